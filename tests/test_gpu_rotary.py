"""Rotary positions: tables, embedding, and the append of a joint projection's rows,
against plain implementations in 64 bits."""
import pytest
import torch

import decoder_cases as dc
import token_step_cases as ts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu(olamd):
    olamd.init(0)
    return olamd


# ---- tables ------------------------------------------------------------------------

def check_tables(gpu, positions, d, base, dtype=torch.float32, **kw):
    cos, sin = gpu.rotary_tables(positions, d, base, dtype=dtype, **kw)
    assert cos.dtype == dtype and cos.shape == sin.shape == (positions, d // 2)
    f, m = ts.frequencies(d, base, kw.get("scaling", "none"), kw.get("factor", 1.0), kw.get("original_positions", 0),
                          kw.get("turns_fast", 32.0), kw.get("turns_slow", 1.0))
    m = kw.get("magnitude", 0.0) or m
    # angles of up to 2^20 in 64 bits are off by less than 2^-28, the functions in fp32 by
    # a few of their ulps at 1, 2^-22, the product with the magnitude by one more
    for got, want in zip((cos, sin), ts.tables(positions, f, m)):
        dc.near(got, want, ts.HALF_STEP[dtype] * want.abs() + 2.0 ** -22 * m)


@pytest.mark.parametrize("positions,d", [(1, 2), (3, 6), (257, 64), (1000, 128), (4097, 80), (5000, 10), (300, 256), (33, 1026)])
@pytest.mark.parametrize("base", [10000.0, 500000.0, 1.5])
def test_tables(gpu, positions, d, base):
    check_tables(gpu, positions, d, base)


@pytest.mark.parametrize("scaling", ["linear", "ntk", "by_parts", "yarn"])
@pytest.mark.parametrize("d,factor,original", [(128, 32.0, 4096), (64, 2.5, 2048), (80, 8.0, 8192), (16, 1.0, 100), (6, 4.0, 7)])
def test_tables_for_long_contexts(gpu, scaling, d, factor, original):
    check_tables(gpu, 700, d, 10000.0, scaling=scaling, factor=factor, original_positions=original)


def test_tables_magnitude_turns_and_types(gpu):
    check_tables(gpu, 100, 64, 10000.0, scaling="yarn", factor=4.0, original_positions=512, turns_fast=8.0, turns_slow=0.5)
    check_tables(gpu, 100, 64, 10000.0, scaling="yarn", factor=4.0, original_positions=512, magnitude=1.0)
    check_tables(gpu, 100, 64, 10000.0, magnitude=2.5)
    for dtype in (torch.float16, torch.bfloat16):
        check_tables(gpu, 100, 48, 10000.0, dtype=dtype)


def test_tables_of_far_positions(gpu):
    """The last of a million positions, whose angles are far past what fp32 has a fraction for."""
    cos, sin = gpu.rotary_tables(1 << 20, 64)
    f, _ = ts.frequencies(64, 10000.0)
    at = torch.tensor([1 << 19, (1 << 20) - 1])
    angle = torch.outer(at.double(), torch.tensor(f, dtype=torch.float64))
    dc.near(cos[at.cuda()], torch.cos(angle), torch.full_like(angle, 2.0 ** -22))
    dc.near(sin[at.cuda()], torch.sin(angle), torch.full_like(angle, 2.0 ** -22))


def test_tables_of_nothing_and_to_the_host(gpu):
    assert gpu.rotary_tables(0, 64)[0].shape == (0, 32)
    out = torch.empty(50, 16), torch.empty(50, 16)
    gpu.rotary_tables(50, 32, out=out)
    assert all(torch.equal(a, b.cpu()) for a, b in zip(out, gpu.rotary_tables(50, 32)))


# ---- embedding -----------------------------------------------------------------------

def rows_of(x, layout, heads):
    """x's rows [n, D], token by token and head by head."""
    if layout == "heads":
        x = x.transpose(1, 2)
    elif layout == "joint":
        x = x.unflatten(-1, (heads, -1))
    return x.reshape(-1, x.shape[-1])


def check_embedding(gpu, layout, B, S, H, D, d, interleaved, dtype, table_dtype=torch.float32, ids=torch.int64, P=97,
                    in_place=False):
    g = dc.gen(B * 1000 + S * 10 + D + d)
    shape = {"tokens": (B * S, H, D), "heads": (B, H, S, D), "joint": (B, S, H * D)}[layout]
    x = dc.randn(g, shape, dtype, 2.0)
    per_token = (B * S,) if layout == "tokens" else (B, S)
    c, s = (dc.randn(g, (P, d // 2) if ids else per_token + (d // 2,), table_dtype) for _ in range(2))
    pos = torch.randint(0, P, per_token, generator=g) if ids else torch.arange(B * S)
    xd = x.cuda()
    got = gpu.rotary_embedding(xd, c.cuda(), s.cuda(), pos.to(ids).cuda() if ids else None, interleaved,
                               H if layout == "joint" else 0, out=xd if in_place else None)
    assert got.dtype == dtype and got.shape == shape
    at = pos.reshape(-1).repeat_interleave(H)
    want, size = ts.rotate(rows_of(x, layout, H), c.reshape(-1, d // 2)[at], s.reshape(-1, d // 2)[at], interleaved)
    got = rows_of(got.cpu(), layout, H)
    dc.near(got, want, ts.rotate_bound(want, size, dtype))
    assert torch.equal(got[:, d:], rows_of(x, layout, H)[:, d:])
    if not in_place:
        assert torch.equal(xd.cpu(), x)


@pytest.mark.parametrize("layout", ["tokens", "heads", "joint"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,S,H,D,d", [(1, 1, 1, 2, 2), (1, 1, 32, 128, 128), (2, 7, 5, 64, 32), (3, 33, 4, 80, 80), (1, 70, 3, 80, 20),
                                       (2, 19, 2, 256, 64), (1, 5, 7, 10, 6), (1, 3, 2, 96, 48), (4, 130, 9, 128, 96), (1, 2, 1, 640, 512)])
@pytest.mark.parametrize("typ", ["fp16", "bf16", "fp32"])
def test_embedding(gpu, layout, interleaved, B, S, H, D, d, typ):
    check_embedding(gpu, layout, B, S, H, D, d, interleaved, dc.TYPE[typ])


@pytest.mark.parametrize("layout", ["tokens", "heads", "joint"])
@pytest.mark.parametrize("typ", ["fp16", "bf16"])
@pytest.mark.parametrize("ids", [None, torch.int32, torch.int64])
@pytest.mark.parametrize("D,d", [(64, 64), (36, 18)])
def test_embedding_by_tables_of_its_type_and_with_and_without_ids(gpu, layout, typ, ids, D, d):
    check_embedding(gpu, layout, 2, 9, 3, D, d, False, dc.TYPE[typ], dc.TYPE[typ], ids)
    check_embedding(gpu, layout, 2, 9, 3, D, d, True, dc.TYPE[typ], torch.float32, ids)


@pytest.mark.parametrize("layout", ["tokens", "heads", "joint"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,d", [(128, 128), (128, 64), (64, 48), (30, 14)])
def test_embedding_in_place(gpu, layout, interleaved, D, d):
    check_embedding(gpu, layout, 3, 41, 6, D, d, interleaved, torch.bfloat16, in_place=True)


def test_embedding_of_memory_off_alignment(gpu):
    """Tensors that begin between 16-byte lines."""
    g = dc.gen(1)
    x, c, s = dc.randn(g, (5, 4, 64), torch.bfloat16), dc.randn(g, (5, 32), torch.float32), dc.randn(g, (5, 32), torch.float32)
    want = gpu.rotary_embedding(x.cuda(), c.cuda(), s.cuda())
    for k in (1, 3):
        odd = [torch.nn.functional.pad(t.reshape(-1), (k, 0)).cuda()[k:].view(t.shape) for t in (x, c, s)]
        out = torch.empty(x.numel() + k, dtype=x.dtype, device="cuda")[k:].view(x.shape)
        assert torch.equal(gpu.rotary_embedding(*odd, out=out), want)


def test_embedding_positions_outside_the_tables(gpu):
    """The rotated dimensions of their tokens are NaN; the others, and other tokens, are as without them."""
    g = dc.gen(2)
    for D, d in ((64, 32), (22, 10)):
        x, c, s = dc.randn(g, (6, 3, D), torch.float16).cuda(), dc.randn(g, (9, d // 2), torch.float32).cuda(), \
            dc.randn(g, (9, d // 2), torch.float32).cuda()
        pos = torch.tensor([0, 8, 9, -1, 3, 2 ** 40], device="cuda")
        got = gpu.rotary_embedding(x, c, s, pos)
        want = gpu.rotary_embedding(x, c, s, pos.clamp(0, 8))
        bad = torch.tensor([2, 3, 5], device="cuda")
        assert torch.isnan(got[bad, :, :d]).all()
        got[bad, :, :d] = want[bad, :, :d]
        assert torch.equal(got, want)


def test_embedding_keeps_infinities_and_nan_to_their_pairs(gpu):
    g = dc.gen(3)
    for interleaved in (False, True):
        for d in (64, 12):
            x, c, s = dc.randn(g, (4, 2, 64), torch.bfloat16), dc.randn(g, (4, d // 2), torch.float32), dc.randn(g, (4, d // 2), torch.float32)
            want = gpu.rotary_embedding(x.cuda(), c.cuda(), s.cuda(), interleaved=interleaved).cpu()
            x[1, 1, 3], x[2, 0, 63] = float("inf"), float("nan")
            got = gpu.rotary_embedding(x.cuda(), c.cuda(), s.cuda(), interleaved=interleaved).cpu()
            pair = (2, 3) if interleaved else (3, 3 + d // 2)
            assert not torch.isfinite(got[1, 1, list(pair)].float()).any()
            hit = torch.zeros(64, dtype=torch.bool)
            hit[list(pair)] = True
            assert torch.equal(got[1, 1, ~hit], want[1, 1, ~hit])
            assert torch.isnan(got[2, 0, 63])
            last = (62, 63) if interleaved else (31, 63)
            hit[:] = False
            hit[list(last) if d == 64 else 63] = True
            assert torch.equal(got[2, 0, ~hit], want[2, 0, ~hit])
            assert torch.equal(got[0], want[0]) and torch.equal(got[3], want[3])


def test_embedding_of_nothing_and_from_the_host(gpu):
    c = torch.zeros(4, 16, device="cuda")
    assert gpu.rotary_embedding(torch.empty((0, 3, 32), device="cuda"), c, c, torch.empty(0, dtype=torch.int64, device="cuda")).shape == (0, 3, 32)
    g = dc.gen(4)
    x, c, s, pos = dc.randn(g, (2, 3, 5, 32), torch.float16), dc.randn(g, (9, 16), torch.float32), dc.randn(g, (9, 16), torch.float32), \
        torch.randint(0, 9, (2, 5), generator=g)
    got = gpu.rotary_embedding(x, c, s, pos)
    assert not got.is_cuda and torch.equal(got, gpu.rotary_embedding(x.cuda(), c.cuda(), s.cuda(), pos.cuda()).cpu())


def test_embedding_of_more_than_4_gb(gpu):
    """Offsets past 32 bits: the last tokens of a tensor of 4.3 GB."""
    T, H, D = 8200, 2048, 128
    x = torch.zeros((T, H, D), dtype=torch.bfloat16, device="cuda")
    tail = dc.randn(dc.gen(5), (2, H, D), torch.bfloat16)
    x[-2:] = tail.cuda()
    c, s = gpu.rotary_tables(T, D)
    want = gpu.rotary_embedding(tail.cuda(), c, s, torch.tensor([T - 2, T - 1], device="cuda"))
    got = gpu.rotary_embedding(x, c, s, out=x)
    assert torch.equal(got[-2:], want) and not got[:-2].any()


# ---- append ----------------------------------------------------------------------------

BATCHES = [([1], [1]), ([1], [200]), ([5], [5]), ([40], [40]), ([33], [100]), ([1, 1, 1, 1], [1, 17, 64, 129]),
           ([0, 3, 0, 1, 0], [7, 3, 0, 33, 100]), ([70, 1, 130, 16], [70, 500, 131, 48]), ([300], [1000]),
           ([2] * 70, [2 + 3 * i for i in range(70)])]


def joint(b, heads, dtype):
    """A batch's rows with queries, keys and values together."""
    return torch.cat([dc.randn(dc.gen(heads), (len(b.k), heads, b.D), dtype), b.k, b.v], 1)


def positions_of(b):
    return torch.tensor([t - n + i for n, t in zip(b.new, b.total) for i in range(n)], dtype=torch.int64)


def check_append(gpu, b, heads, d, interleaved, dtype, table_dtype=torch.float32, ids=None):
    """Queries by the rotation's bound.  The cache against the append's own definition of
    the keys rotated in 64 bits: a key is off by 2^-23 of its products, so a scale is, and a
    code is the nearest to a quotient that is off by as much."""
    g = dc.gen(sum(b.total) + d)
    P = max(b.total + [1])
    c, s = (dc.randn(g, (P, d // 2), table_dtype) for _ in range(2))
    x = joint(b, heads, dtype)
    pos = positions_of(b)
    if ids is not None:
        pos = torch.randint(0, P, pos.shape, generator=g)
    cache = b.cache(gpu)
    q = gpu.rotary_kv_cache_append(x.cuda(), c.cuda(), s.cuda(), cache, *b.index(),
                                   position_ids=None if ids is None else pos.to(ids).cuda(), interleaved=interleaved)
    H = b.H
    y, size = ts.rotate(x[:, :heads + H].reshape(-1, b.D), *(t[pos.repeat_interleave(heads + H)] for t in (c, s)), interleaved)
    y, size = y.reshape(len(x), heads + H, b.D), size.reshape(len(x), heads + H, b.D)
    assert q.dtype == dtype and q.shape == (len(x), heads, b.D)
    dc.near(q, y[:, :heads], ts.rotate_bound(y[:, :heads], size[:, :heads], dtype))
    assert torch.equal(q[..., d:].cpu(), x[:, :heads, d:])
    # values, and everything that keys do not touch, to the bit
    b.k = y[:, heads:].float()
    want = dc.append(b)
    assert torch.equal(cache.v_cache.cpu().view(torch.uint8), want["v_cache"].view(torch.uint8))
    assert torch.equal(cache.v_scale.cpu(), want["v_scale"])
    got, ref = cache.k_cache.cpu().double(), want["k_cache"].double()
    ks, ws = cache.k_scale.cpu().double(), want["k_scale"].double()
    off = float(size.max() if size.numel() else 0) * 2.0 ** -22
    dc.near(ks, ws, off / dc.QMAX[b.to] + 2.0 ** -22 * ws)
    # codes: the same, but where the quotient is that near the middle between two
    differ = got != ref
    assert differ.double().mean() < 1e-3
    step = 2 * dc.half_step(torch.maximum(got.abs(), ref.abs()), b.to)
    assert ((got - ref).abs() <= step)[differ].all()
    return q, cache


@pytest.mark.parametrize("new,total", BATCHES)
@pytest.mark.parametrize("to,typ,bt,D,H,heads,d,interleaved", [
    ("int8", "fp16", 16, 64, 2, 8, 64, False), ("fp8", "bf16", 64, 128, 3, 3, 128, False), ("fp8", "fp16", 32, 80, 1, 5, 32, True),
    ("int8", "bf16", 256, 256, 2, 4, 128, False), ("fp8", "bf16", 16, 16, 8, 32, 16, True), ("fp8", "bf16", 128, 128, 2, 10, 96, False)])
def test_append(gpu, new, total, to, typ, bt, D, H, heads, d, interleaved):
    b = dc.Batch(sum(total) + bt, new, total, H, D, bt, to, dc.TYPE[typ], slack=1)
    check_append(gpu, b, heads, d, interleaved, dc.TYPE[typ])


@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
@pytest.mark.parametrize("new,total", [([1, 1], [9, 70]), ([30, 4], [77, 4])])
def test_append_by_position_ids_and_tables_of_the_rows_type(gpu, ids, new, total):
    b = dc.Batch(5, new, total, 2, 64, 32, "fp8", torch.bfloat16)
    check_append(gpu, b, 4, 32, False, torch.bfloat16, torch.bfloat16, ids)


@pytest.mark.parametrize("new,total", [([1, 2], [70, 9]), ([40, 3], [60, 40])])
def test_append_by_identity_tables_is_the_append(gpu, new, total):
    """cos 1 and sin 0: the bits of kv_cache_append, and q as it was."""
    b = dc.Batch(10, new, total, 2, 64, 16, "fp8", torch.float16)
    x = joint(b, 6, torch.float16).cuda()
    one, zero = torch.ones(100, 32, device="cuda"), torch.zeros(100, 32, device="cuda")
    want = gpu.kv_cache_append(b.k.cuda(), b.v.cuda(), b.cache(gpu), *b.index())
    cache = b.cache(gpu)
    q = gpu.rotary_kv_cache_append(x, one, zero, cache, *b.index())
    assert torch.equal(q, x[:, :6])
    for name in ("k_cache", "v_cache"):
        assert torch.equal(getattr(cache, name).view(torch.uint8), getattr(want, name).view(torch.uint8))
    assert torch.equal(cache.k_scale, want.k_scale) and torch.equal(cache.v_scale, want.v_scale)


@pytest.mark.parametrize("n", [1, 40])
def test_append_leaves_rows_of_no_sequence_and_sequences_that_do_not_fit(gpu, n):
    b = dc.Batch(8, [n] * 4, [100] * 4, 2, 64, 16, "fp8", torch.bfloat16)
    x = torch.nn.functional.pad(joint(b, 4, torch.bfloat16), (0, 0, 0, 0, 3, 5)).cuda()
    c, s = gpu.rotary_tables(100, 64)
    table, start, lengths = b.index()
    good, fresh = b.cache(gpu), b.cache(gpu)
    want = gpu.rotary_kv_cache_append(x, c, s, good, table, start + 3, lengths)
    lengths = lengths.clone()
    lengths[1], lengths[2] = n - 1, 16 * table.shape[1] + 1
    out = torch.full_like(want, 7.0)
    gpu.rotary_kv_cache_append(x, c, s, fresh, table, start + 3, lengths, out=out)
    left = torch.ones(len(out), dtype=torch.bool)
    left[3:3 + n] = left[3 + 3 * n:3 + 4 * n] = False
    assert (out[left.cuda()] == 7).all() and torch.equal(out[~left.cuda()], want[~left.cuda()])
    mine = set(b.table[0].tolist()) | set(b.table[3].tolist())
    for blk in range(len(b.k_scale)):
        for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
            src = getattr(good, name) if blk in mine else getattr(b, name).cuda()
            assert torch.equal(getattr(fresh, name)[blk].view(torch.uint8), src[blk].view(torch.uint8)), (blk, name)


@pytest.mark.parametrize("n", [1, 20])
def test_append_of_positions_outside_the_tables(gpu, n):
    """Their rotated queries are NaN, and their keys make the block's scale one."""
    b = dc.Batch(9, [n, n], [n, 64 + n], 1, 64, 64, "fp8", torch.bfloat16)
    x = joint(b, 2, torch.bfloat16).cuda()
    c, s = gpu.rotary_tables(64, 32)
    cache = b.cache(gpu)
    q = gpu.rotary_kv_cache_append(x, c, s, cache, *b.index())
    assert torch.isfinite(q[:n].float()).all() and torch.isnan(q[n:, :, :32]).all()
    assert torch.equal(q[n:, :, 32:], x[n:, :2, 32:])
    blk = int(b.table[1, 1])
    assert torch.isnan(cache.k_scale[blk]).all() and not cache.k_cache[blk, :, :n].float().any()
    assert torch.isfinite(cache.v_scale[blk]).all() and torch.isfinite(cache.k_scale[int(b.table[0, 0])]).all()


def test_append_of_host_rows(gpu):
    b = dc.Batch(11, [3, 20], [40, 60], 2, 64, 16, "int8", torch.float16)
    x = joint(b, 4, torch.float16)
    c, s = gpu.rotary_tables(60, 64)
    one, two = b.cache(gpu), b.cache(gpu)
    want = gpu.rotary_kv_cache_append(x.cuda(), c, s, one, *b.index())
    got = gpu.rotary_kv_cache_append(x, c.cpu(), s.cpu(), two, *b.index("cpu"))
    assert torch.equal(got, want)
    assert torch.equal(one.k_cache, two.k_cache) and torch.equal(one.v_cache, two.v_cache)


def test_append_of_nothing(gpu):
    b = dc.Batch(2, [0, 0], [5, 0], 2, 64, 16, "int8", torch.float16)
    c, s = gpu.rotary_tables(8, 64)
    cache = b.cache(gpu)
    assert gpu.rotary_kv_cache_append(joint(b, 2, torch.float16).cuda(), c, s, cache, *b.index()).shape == (0, 2, 64)
    assert torch.equal(cache.k_cache.cpu(), b.k_cache)


@pytest.mark.parametrize("new,total", [([1, 1], [300, 70]), ([40, 1], [100, 500])])
def test_captured_and_on_another_stream(gpu, new, total):
    b = dc.Batch(17, new, total, 2, 64, 16, "fp8", torch.bfloat16)
    x, c = joint(b, 8, torch.bfloat16).cuda(), b.cache(gpu)
    idx = b.index()
    pos = positions_of(b).cuda()

    def step():
        cos, sin = gpu.rotary_tables(600, 64)
        q = gpu.rotary_kv_cache_append(x, cos, sin, c, *idx)
        return cos, sin, q, gpu.rotary_embedding(x, cos, sin, pos), gpu.kv_cache_attention(q, c, *idx)

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for _ in range(3):
        for t in got:
            t.zero_()
        step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(got, want))
