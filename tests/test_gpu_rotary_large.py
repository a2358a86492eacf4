"""Rotary positions of tensors so large that a thread takes two heads, and appends with more
queries than one round of workgroups, against plain implementations in 64 bits."""
import pytest
import torch

import decoder_cases as dc
import token_step_cases as ts
from test_gpu_rotary import check_append, rows_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu(olamd):
    olamd.init(0)
    return olamd


# tokens * heads * D / 16 is 2^20 and more: (batch, tokens, heads, D), odd heads among them
SIZES = [(2, 7301, 9, 128), (1, 18800, 7, 128), (2, 3703, 9, 256), (3, 2740, 8, 256)]


def check(gpu, layout, B, S, H, D, d, interleaved, dtype, in_place=False, offset=0, P=8192):
    assert B * S * H * (D // 16) >= 1 << 20
    g = torch.Generator(device="cuda").manual_seed(B * S + H + d)
    shape = {"tokens": (B * S, H, D), "heads": (B, H, S, D), "joint": (B, S, H * D)}[layout]
    x = (torch.randn(shape, generator=g, device="cuda") * 2).to(dtype)
    c, s = (torch.randn((P, d // 2), generator=g, device="cuda") for _ in range(2))
    pos = torch.randint(0, P, (B * S,) if layout == "tokens" else (B, S), generator=g, device="cuda")
    out = torch.full((x.numel() + offset + 64,), 7.0, dtype=dtype, device="cuda")
    y = out[offset:offset + x.numel()].view(shape)
    if in_place:
        y.copy_(x)
    gpu.rotary_embedding(y if in_place else x, c, s, pos, interleaved, H if layout == "joint" else 0, out=y)
    at = pos.reshape(-1).repeat_interleave(H)
    want, size = ts.rotate(rows_of(x, layout, H), c[at], s[at], interleaved)
    got = rows_of(y, layout, H)
    assert ((got.double() - want).abs() <= ts.rotate_bound(want, size, dtype)).all()
    assert torch.equal(got[:, d:], rows_of(x, layout, H)[:, d:])
    assert (out[:offset] == 7).all() and (out[offset + x.numel():] == 7).all()


@pytest.mark.parametrize("layout", ["tokens", "heads", "joint"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,S,H,D", SIZES)
@pytest.mark.parametrize("typ", ["fp16", "bf16", "fp32"])
def test_embedding(gpu, layout, interleaved, B, S, H, D, typ):
    for d in (D, D // 2, 96):
        check(gpu, layout, B, S, H, D, d, interleaved, dc.TYPE[typ])


@pytest.mark.parametrize("layout", ["tokens", "heads"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("typ", ["bf16", "fp32"])
def test_embedding_in_place_and_off_alignment(gpu, layout, interleaved, typ):
    for d in (128, 64):
        check(gpu, layout, 2, 7301, 9, 128, d, interleaved, dc.TYPE[typ], in_place=True)
        check(gpu, layout, 2, 7301, 9, 128, d, interleaved, dc.TYPE[typ], offset=3)


@pytest.mark.parametrize("new,total,heads,D,d,interleaved", [
    ([1500, 600], [1800, 600], 30, 128, 128, False), ([2000], [2000], 34, 128, 64, True), ([1, 2500, 3], [90, 2500, 70], 26, 80, 32, False),
    ([1] * 400, [1 + 7 * i % 90 for i in range(400)], 32, 128, 128, False), ([1] * 700, [1 + 5 * i % 40 for i in range(700)], 18, 256, 128, True)])
@pytest.mark.parametrize("to,typ", [("fp8", "bf16"), ("int8", "fp16")])
def test_append(gpu, new, total, heads, D, d, interleaved, to, typ):
    b = dc.Batch(sum(total), new, total, 2, D, 16, to, dc.TYPE[typ], slack=1)
    at_once = 64 // (D // 16)
    waves = 1 if sum(new) <= 2 * len(new) else 4
    assert sum(new) * -(-heads // at_once) > 1280 * waves  # past one round
    check_append(gpu, b, heads, d, interleaved, dc.TYPE[typ])


def test_append_with_q_beside_qkv(gpu):
    """One piece of memory: queries to be, rows, queries to be again."""
    b = dc.Batch(3, [1, 40], [9, 70], 2, 64, 16, "fp8", torch.bfloat16)
    rows = dc.randn(dc.gen(4), (41, 6 + 4, 64), torch.bfloat16).cuda()
    c, s = gpu.rotary_tables(70, 64)
    want = gpu.rotary_kv_cache_append(rows, c, s, b.cache(gpu), *b.index())
    n = want.numel()
    for at in (0, n + rows.numel()):
        memory = torch.empty(2 * n + rows.numel(), dtype=torch.bfloat16, device="cuda")
        qkv, q = memory[n:n + rows.numel()].view(rows.shape), memory[at:at + n].view(want.shape)
        qkv.copy_(rows)
        gpu.rotary_kv_cache_append(qkv, c, s, b.cache(gpu), *b.index(), out=q)
        assert torch.equal(q, want) and torch.equal(qkv, rows)
    with pytest.raises(gpu.InvalidArgument, match="overlap"):
        gpu.rotary_kv_cache_append(qkv, c, s, b.cache(gpu), *b.index(), out=memory[n - 8:2 * n - 8].view(want.shape))
