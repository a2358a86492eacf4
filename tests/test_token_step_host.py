"""Argument checks of rotary positions, the gated feed-forward and sampling (they run
before any device work, so without a GPU), and known answers of the plain
implementations that the GPU tests compare with."""
import math

import pytest
import torch

import decoder_cases as dc
import token_step_cases as ts
from test_decoder_host import CACHE, cache_args, dev, refused

H16, B16, F32 = torch.float16, torch.bfloat16, torch.float32
U8, I32, I64, E4 = torch.uint8, torch.int32, torch.int64, torch.float8_e4m3fn


def z(*shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype)


# ---- refusals ------------------------------------------------------------------------

@pytest.mark.parametrize("kw,text", [
    (dict(cos=None), "are required"), (dict(sin=None), "are required"), (dict(sin=z(9, 16, dtype=H16)), "both the same"),
    (dict(cos=z(9, 16, dtype=I32), sin=z(9, 16, dtype=I32)), "must be FLOAT"), (dict(cos=z(144)), "cos must be"),
    (dict(sin=z(9, 8)), "sin (cos's)"), (dict(cos=z(9, 0), sin=z(9, 0)), "from 1 to"), (dict(base=1.0), "base"), (dict(base=-2.0), "base"),
    (dict(base=math.inf), "base"), (dict(base=math.nan), "base"), (dict(scaling=5), "scaling"), (dict(scaling=-1), "scaling"),
    (dict(factor=0.5), "factor"), (dict(factor=math.nan), "factor"), (dict(factor=math.inf), "factor"),
    (dict(scaling=2, cos=z(9, 1), sin=z(9, 1)), "ntk"), (dict(scaling=3, original=0), "original_positions"),
    (dict(scaling=4, original=-5), "original_positions"), (dict(scaling=4, original=64, slow=0.0), "slow"),
    (dict(scaling=3, original=64, slow=32.0), "slow"), (dict(scaling=3, original=64, fast=math.inf), "slow"),
    (dict(scaling=3, original=64, fast=math.nan), "slow"), (dict(magnitude=-1.0), "magnitude"), (dict(magnitude=math.nan), "magnitude"),
])
def test_tables_refuse(olamd, kw, text):
    a = dict(base=1e4, scaling=0, factor=1.0, original=0, fast=32.0, slow=1.0, magnitude=0.0, cos=z(9, 16), sin=z(9, 16))
    a.update(kw)
    refused(olamd, "rotary_tables", [*(a[n] for n in ("base", "scaling", "factor", "original", "fast", "slow", "magnitude")),
                                     dev(olamd, a["cos"]), dev(olamd, a["sin"])], text)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "are required"), (dict(y=None), "are required"), (dict(x=z(6, 3, 64, dtype=I32)), "x must be FLOAT"),
    (dict(y=z(6, 3, 64)), "y must have"), (dict(y=z(6, 3, 32, dtype=H16)), "y has"), (dict(x=z(6, 192, dtype=H16)), "x must be ["),
    (dict(x=z(2, 2, 2, 2, 2, dtype=H16)), "x must be ["), (dict(heads=-1), "num_heads"), (dict(heads=5), "must divide"),
    (dict(x=z(2, 3, 5, 64, dtype=H16), heads=4), "not x's"), (dict(x=z(6, 3, 1, dtype=H16)), "head_dim must be"),
    (dict(sin=z(9, 15)), "sin (cos's)"), (dict(cos=z(9, 16, dtype=H16)), "both the same"), (dict(cos=z(9, 16, dtype=B16), sin=z(9, 16, dtype=B16)), "of x's type"),
    (dict(cos=z(9, 33), sin=z(9, 33)), "rotary_dim"), (dict(cos=z(9, 0), sin=z(9, 0)), "rotary_dim"), (dict(cos=z(16), sin=z(16)), "cos must be"),
    (dict(interleaved=2), "interleaved"), (dict(interleaved=-1), "interleaved"), (dict(ids=z(6)), "position_ids must be"),
    (dict(ids=z(5, dtype=I64)), "position_ids ("), (dict(ids=z(1, 6, dtype=I64)), "position_ids ("), (dict(ids=None), "without position_ids"),
    (dict(cos=z(1, 9, 16), sin=z(1, 9, 16)), "with position_ids"), (dict(x=z(2, 3, 64, dtype=H16), heads=2), "position_ids ("),
    (dict(x=z(2, 3, 5, 64, dtype=H16), ids=z(2, 3, dtype=I64)), "position_ids ("),
    (dict(x=z(2, 3, 5, 64, dtype=H16), ids=None, cos=z(10, 16), sin=z(10, 16)), "without position_ids"),
])
def test_embedding_refuses(olamd, kw, text):
    a = dict(x=z(6, 3, 64, dtype=H16), cos=z(9, 16), sin=z(9, 16), ids=z(6, dtype=I64), interleaved=0, heads=0, y=z(6, 3, 64, dtype=H16))
    a.update(kw)
    refused(olamd, "rotary_embedding", [dev(olamd, a["x"]), dev(olamd, a["cos"]), dev(olamd, a["sin"]), dev(olamd, a["ids"]),
                                        a["interleaved"], a["heads"], dev(olamd, a["y"])], text)


@pytest.mark.parametrize("bad", [-1, 9, 2 ** 40])
def test_host_positions_are_checked(olamd, bad):
    ids = z(6, dtype=I64)
    ids[4] = bad
    args = [dev(olamd, z(6, 3, 64, dtype=H16)), dev(olamd, z(9, 16)), dev(olamd, z(9, 16)), olamd.describe(ids), 0, 0,
            dev(olamd, z(6, 3, 64, dtype=H16))]
    refused(olamd, "rotary_embedding", args, "outside the tables")


APPEND = [
    (dict(qkv=None), "are required"), (dict(q=None), "are required"), (dict(cos=None), "are required"),
    (dict(qkv=z(5, 512, dtype=H16)), "qkv must be ["), (dict(qkv=z(5, 8, 64)), "both the same"), (dict(q=z(5, 4, 64, dtype=B16)), "both the same"),
    (dict(q=z(5, 3, 64, dtype=H16)), "heads must be"), (dict(q=z(5, 0, 64, dtype=H16)), "heads must be"), (dict(q=z(4, 4, 64, dtype=H16)), "q ("),
    (dict(q=z(5, 6, 64, dtype=H16)), "qkv ("), (dict(qkv=z(5, 8, 32, dtype=H16)), "qkv ("), (dict(cos=z(9, 20), sin=z(9, 20)), "multiple of 16"),
    (dict(cos=z(9, 40), sin=z(9, 40)), "rotary_dim"), (dict(cos=z(1, 9, 16), sin=z(1, 9, 16)), "cos must be"),
    (dict(sin=z(8, 16)), "sin (cos's)"), (dict(interleaved=3), "interleaved"), (dict(ids=z(4, dtype=I32)), "position_ids ("),
    (dict(ids=z(5)), "position_ids must be"),
]


def append_args(olamd, kw):
    a = dict(qkv=z(5, 8, 64, dtype=H16), cos=z(9, 16), sin=z(9, 16), ids=None, interleaved=0, q=z(5, 4, 64, dtype=H16))
    a.update({k: v for k, v in kw.items() if k in a})
    return [dev(olamd, a["qkv"]), dev(olamd, a["cos"]), dev(olamd, a["sin"]), dev(olamd, a["ids"]), a["interleaved"], dev(olamd, a["q"]),
            *cache_args(olamd, kw)]


@pytest.mark.parametrize("kw,text", CACHE + APPEND)
def test_rotary_append_refuses(olamd, kw, text):
    refused(olamd, "rotary_kv_cache_append", append_args(olamd, kw), text)


def test_rotary_append_refuses_more_blocks_and_heads_than_its_grid_counts(olamd):
    # 65535 sequences and 65536 tokens: up to 65536 blocks of 32768 heads; shapes without memory
    def shaped(dtype, *dims):
        d = dev(olamd, z(*[1] * len(dims), dtype=dtype))
        for i, n in enumerate(dims):
            d.dims[i] = n
        d.size_bytes = math.prod(dims) * dtype.itemsize
        return d

    for kv, text in [(32768, "more than 2^31 blocks and heads"), (32767, "interleaved")]:
        # (the second is refused for another reason: nothing is launched)
        args = [shaped(H16, 65536, 3 * kv, 16), shaped(F32, 9, 8), shaped(F32, 9, 8), olamd.describe(None), 0 if kv == 32768 else 7,
                shaped(H16, 65536, kv, 16), shaped(E4, 9, kv, 16, 16), shaped(E4, 9, kv, 16, 16), shaped(F32, 9, kv), shaped(F32, 9, kv),
                shaped(I32, 65535, 4), shaped(I32, 65536), shaped(I32, 65535)]
        refused(olamd, "rotary_kv_cache_append", args, text)


def test_rotary_append_checks_what_is_on_the_host(olamd):
    args = append_args(olamd, {})
    args[5].location = olamd.HOST
    refused(olamd, "rotary_kv_cache_append", args, "q must be device memory")
    args = append_args(olamd, {})
    args[12] = olamd.describe(torch.tensor([3, 10], dtype=I32))
    refused(olamd, "rotary_kv_cache_append", args, "longer than the tables")
    args = append_args(olamd, {})
    args[3] = olamd.describe(torch.tensor([0, 1, 2, 9, 4], dtype=I32))
    refused(olamd, "rotary_kv_cache_append", args, "outside the tables")


@pytest.mark.parametrize("kw,text", [
    (dict(a=None), "are required"), (dict(gate=None), "are required"), (dict(up_scale=None), "are required"), (dict(y=None), "are required"),
    (dict(gate=z(32, 32, dtype=torch.int8)), "b must be"), (dict(gate=z(32, 24, dtype=U8)), "multiple"), (dict(a=z(4, 96, dtype=H16)), "different lengths"),
    (dict(a=z(4, 64)), "must be FLOAT16 or BFLOAT16"), (dict(a_type=3), "a_type must be"), (dict(gate_scale=z(32, 3, dtype=U8)), "b_scale has"),
    (dict(up=z(31, 32, dtype=U8)), "up (gate's)"), (dict(up=z(32, 16, dtype=U8)), "up (gate's)"), (dict(up=z(32, 32, dtype=torch.int8)), "gate's and"),
    (dict(up_scale=z(32, 1, dtype=U8)), "up_scale (gate_scale's)"), (dict(up_scale=z(32, 2)), "gate's and"), (dict(activation=4), "activation"),
    (dict(activation=-1), "activation"), (dict(y=z(4, 32, dtype=B16)), "a's type"), (dict(y=z(4, 32)), "y without y_scale"),
    (dict(y=z(4, 31, dtype=H16)), "y has"), (dict(y=z(4, 32, dtype=E4)), "y without y_scale"),
    (dict(y_scale=z(4, 1, dtype=U8)), "y with y_scale"), (dict(y=z(4, 32, dtype=E4), y_scale=z(4, 1)), "y with y_scale"),
    (dict(y=z(4, 32, dtype=E4), y_scale=z(4, 2, dtype=U8)), "y_scale has"),
    (dict(gate=z(40, 32, dtype=U8), gate_scale=z(40, 2, dtype=U8), up=z(40, 32, dtype=U8), up_scale=z(40, 2, dtype=U8), y=z(4, 40, dtype=E4),
          y_scale=z(4, 1, dtype=U8)), "N must be a multiple"),
    (dict(a=z(4, 64, dtype=E4), a_scale=z(4, 2, dtype=U8)), "a_type is for"),
])
def test_gated_refuses(olamd, kw, text):
    a = dict(a=z(4, 64, dtype=H16), a_scale=None, a_type=17, gate=z(32, 32, dtype=U8), gate_scale=z(32, 2, dtype=U8), up=z(32, 32, dtype=U8),
             up_scale=z(32, 2, dtype=U8), activation=0, y=z(4, 32, dtype=H16), y_scale=None)
    a.update(kw)
    refused(olamd, "mx_gated_matmul", [v if n in ("a_type", "activation") else dev(olamd, v) for n, v in a.items()], text)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "are required"), (dict(u=None), "are required"), (dict(token=None), "are required"), (dict(x=z(3, 50, dtype=I32)), "logits must be"),
    (dict(x=z(50)), "logits must be ["), (dict(x=z(3, 0)), "vocabulary"), (dict(x=z(1, 1).expand(3, 1 << 21)), "vocabulary"), (dict(u=z(4)), "[rows]"),
    (dict(u=z(3, dtype=H16)), "must be FLOAT"), (dict(T=z(1)), "[rows]"), (dict(T=z(3, dtype=torch.float64)), "must be FLOAT"), (dict(p=z(3, 1)), "[rows]"),
    (dict(m=z(2)), "[rows]"), (dict(k=z(3)), "top_k must be"), (dict(k=z(4, dtype=I32)), "top_k has"), (dict(token=z(3)), "token must be"),
    (dict(token=z(2, dtype=I64)), "token has"), (dict(prob=z(3, dtype=H16)), "probability must be"), (dict(prob=z(4)), "probability ("),
])
def test_sampling_refuses(olamd, kw, text):
    a = dict(x=z(3, 50), u=z(3), T=None, k=None, p=None, m=None, token=z(3, dtype=I64), prob=None)
    a.update(kw)
    args = [dev(olamd, None if v is None else v.contiguous()) for v in a.values()]
    refused(olamd, "sample_tokens", args, text)


def test_python_refuses(olamd):
    x, w, s = z(2, 64, dtype=H16), z(32, 32, dtype=U8), z(32, 2, dtype=U8)
    with pytest.raises(olamd.InvalidArgument, match="activation"):
        olamd.mx_gated_matmul(x, w, s, w, s, "swish")
    with pytest.raises(olamd.InvalidArgument, match="scaling"):
        olamd.rotary_tables(4, 8, scaling="dynamic")


# ---- known answers ---------------------------------------------------------------------

def test_rotation_by_hand():
    x = torch.tensor([[1.0, 2.0, 3.0, 4.0, 5.0, 6.0]])
    c, s = torch.tensor([[0.0, 1.0]]), torch.tensor([[1.0, 0.0]])
    assert ts.rotate(x, c, s, False)[0].tolist() == [[-3.0, 2.0, 1.0, 4.0, 5.0, 6.0]]
    assert ts.rotate(x, c, s, True)[0].tolist() == [[-2.0, 1.0, 3.0, 4.0, 5.0, 6.0]]


def test_scores_of_rotated_rows_go_by_their_distance():
    f, m = ts.frequencies(16, 10000.0)
    assert m == 1.0
    c, s = ts.tables(600, f)
    q, k = torch.randn(2, 1, 16, dtype=torch.float64, generator=dc.gen(1)).unbind(0)
    score = lambda i, j: float((ts.rotate(q, c[i:i + 1], s[i:i + 1], False)[0] * ts.rotate(k, c[j:j + 1], s[j:j + 1], False)[0]).sum())  # noqa: E731
    assert math.isclose(score(7, 3), score(580, 576), abs_tol=1e-9) and math.isclose(score(0, 0), float((q * k).sum()))


def test_scaled_frequencies_by_hand():
    plain, _ = ts.frequencies(8, 10000.0)
    assert [round(v, 12) for v in plain] == [1.0, 0.1, 0.01, 0.001]
    assert ts.frequencies(8, 10000.0, "linear", 4.0)[0] == [v / 4 for v in plain]
    ntk, _ = ts.frequencies(8, 10000.0, "ntk", 4.0)
    assert ntk[0] == 1.0 and math.isclose(ntk[3], plain[3] / 4)  # the slowest pair goes 1 / s as far
    parts, m = ts.frequencies(8, 10000.0, "by_parts", 4.0, original=6283)  # turns: 1000, 100, 10, 1
    assert m == 1.0 and parts[:2] == plain[:2] and math.isclose(parts[3], plain[3] / 4, rel_tol=1e-4)
    assert math.isclose(parts[2], plain[2] * (9 / 31 + 22 / 31 / 4), rel_tol=1e-3)
    yarn, m = ts.frequencies(8, 10000.0, "yarn", 4.0, original=6283)  # at(32) = 1.49, at(1) = 3.00: from 1 to 3
    assert math.isclose(m, 1 + 0.1 * math.log(4)) and yarn[:2] == plain[:2]
    assert math.isclose(yarn[2], plain[2] * (0.5 + 0.5 / 4)) and math.isclose(yarn[3], plain[3] / 4)


def test_activations_by_torch():
    g = torch.linspace(-9, 9, 101, dtype=torch.float64)
    fn = torch.nn.functional
    for kind, want in (("silu", fn.silu(g)), ("gelu", fn.gelu(g)), ("gelu_tanh", fn.gelu(g, approximate="tanh")), ("relu", fn.relu(g))):
        assert torch.allclose(ts.activate(g, kind), want, rtol=1e-9, atol=1e-12)


def test_sampling_by_hand():
    x = [math.log(v) for v in (1, 4, 2, 4, 1)]   # order 1, 3, 2, 0, 4; shares of 12
    pick = lambda u, **kw: ts.sample(x, u, **kw)[0]  # noqa: E731
    assert [pick(u) for u in (0.0, 0.09, 0.4, 0.45, 0.55, 0.9, 0.95)] == [0, 1, 1, 2, 2, 3, 4]
    assert [pick(u, top_k=1) for u in (0.0, 0.99)] == [1, 1] and [pick(u, top_k=2) for u in (0.1, 0.9)] == [1, 3]
    assert [pick(u, top_k=3) for u in (0.1, 0.5, 0.9)] == [1, 2, 3] and [pick(u, top_k=4) for u in (0.0, 0.1)] == [0, 1]
    assert {pick(u / 50, top_p=0.6) for u in range(50)} == {1, 3} and {pick(u / 50, top_p=0.7) for u in range(50)} == {1, 2, 3}
    assert {pick(u / 50, min_p=0.3) for u in range(50)} == {1, 2, 3} and pick(0.99, top_p=0.0) == 1 and pick(0.9, temperature=0.0) == 1
    assert ts.sample(x, 0.2, top_k=2)[1] == pytest.approx(0.5) and ts.sample([-math.inf, math.nan], 0.5) == (-1, 0.0)
    assert [pick(u, temperature=1e-3) for u in (0.1, 0.9)] == [1, 3]
