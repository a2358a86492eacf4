"""Argument checks of the decoder-layer operators (they run before any device
work, so without a GPU) and known answers of the plain implementations that the
GPU tests compare with."""
import ctypes

import numpy as np
import pytest
import torch

import decoder_cases as dc

H16, F32 = torch.float16, torch.float32


def dev(olamd, t, dtype=None, shape=None):
    """Descriptor that names the tensor's memory as device memory: the checks do not look at the payload."""
    if t is None:
        return olamd.describe(None)
    d = olamd.describe(t, dtype, shape)
    d.location = olamd.DEVICE
    return d


def refused(olamd, name, args, text):
    rc = getattr(olamd.lib(), "onnxl_amd_" + name)(*[ctypes.byref(a) if isinstance(a, olamd.Tensor) else a for a in args],
                                                   None)
    assert rc == olamd.INVALID_ARGUMENT, rc
    assert text in olamd.lib().onnxl_amd_last_error().decode()


def norm_args(olamd, **kw):
    a = dict(x=torch.zeros(4, 64, dtype=H16), weight=torch.zeros(64, dtype=H16), residual=None, eps=1e-5, block=0,
             y=torch.zeros(4, 64, dtype=torch.int8), scale=torch.zeros(4, 1), sum=None)
    a.update(kw)
    return [a["x"] if isinstance(a["x"], olamd.Tensor) else dev(olamd, a["x"]), dev(olamd, a["weight"]),
            dev(olamd, a["residual"]), a["eps"], a["block"], dev(olamd, a["y"]), dev(olamd, a["scale"]),
            dev(olamd, a["sum"])]


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "are required"), (dict(y=None), "are required"), (dict(x=torch.zeros(4, 64, dtype=torch.int32)), "x must be"),
    (dict(x=torch.zeros((), dtype=H16)), "last dimension"), (dict(x=torch.zeros(4, 0, dtype=H16)), "empty"),
    (dict(weight=torch.zeros(63, dtype=H16)), "weight has the wrong shape"),
    (dict(weight=torch.zeros(64, dtype=torch.bfloat16)), "weight must have"),
    (dict(residual=torch.zeros(4, 64)), "residual must have"),
    (dict(residual=torch.zeros(3, 64, dtype=H16)), "residual has the wrong shape"),
    (dict(sum=torch.zeros(4, 64, dtype=H16)), "there is no residual"),
    (dict(residual=torch.zeros(4, 64, dtype=H16), sum=torch.zeros(4, 64)), "sum must have"),
    (dict(eps=-1.0), "epsilon"), (dict(eps=float("nan")), "epsilon"), (dict(eps=float("inf")), "epsilon"),
    (dict(y=torch.zeros(4, 64, dtype=torch.uint8)), "y must be"), (dict(y=torch.zeros(4, 32, dtype=torch.int8)), "y has"),
    (dict(block=48), "block_size must be"), (dict(block=-1), "block_size must be"), (dict(block=128), "must divide"),
    (dict(scale=torch.zeros(4, 2)), "y_scale has"), (dict(scale=torch.zeros(4, 1, dtype=H16)), "y_scale must be"),
    (dict(scale=torch.zeros(4, 1, dtype=torch.uint8)), "blocks of 32"),
    (dict(scale=torch.zeros(4, 2, dtype=torch.uint8), block=32), "blocks of 32"),
])
def test_norm_refuses(olamd, kw, text):
    refused(olamd, "rms_norm_quantize", norm_args(olamd, **kw), text)


@pytest.mark.parametrize("x,y,s,text", [
    (torch.zeros(2, 48, dtype=H16), torch.zeros(2, 48, dtype=torch.float8_e4m3fn), torch.zeros(2, 1, dtype=torch.uint8), "multiple"),
    (torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2, 64, dtype=torch.float8_e4m3fn), torch.zeros(2, 2, dtype=torch.uint8),
     "x must be"),
    (torch.zeros(2, 64, dtype=H16), torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2, 2, dtype=torch.uint8), "y must be"),
    (torch.zeros(2, 64, dtype=H16), torch.zeros(2, 32, dtype=torch.float8_e4m3fn), torch.zeros(2, 2, dtype=torch.uint8), "y has"),
    (torch.zeros(2, 64, dtype=H16), torch.zeros(2, 64, dtype=torch.float8_e4m3fn), torch.zeros(2, 2), "y_scale must"),
    (torch.zeros(2, 64, dtype=H16), torch.zeros(2, 64, dtype=torch.float8_e4m3fn), torch.zeros(2, 1, dtype=torch.uint8), "y_scale has"),
])
def test_mx_quantize_refuses(olamd, x, y, s, text):
    refused(olamd, "mx_quantize", [dev(olamd, x), dev(olamd, y), dev(olamd, s)], text)


@pytest.mark.parametrize("kw,text", [
    (dict(b=None), "are required"), (dict(b=torch.zeros(8, 32, dtype=torch.int8)), "b must be"),
    (dict(b=torch.zeros(2, 8, 32, dtype=torch.uint8)), "2-D"), (dict(b=torch.zeros(8, 24, dtype=torch.uint8)), "multiple"),
    (dict(b_scale=torch.zeros(8, 3, dtype=torch.uint8)), "b_scale has"), (dict(b_scale=torch.zeros(8, 2)), "b_scale must"),
    (dict(a=torch.zeros(4, 96, dtype=H16)), "different lengths"), (dict(a=torch.zeros(4, 64)), "must be FLOAT16 or BFLOAT16"),
    (dict(a_type=3), "a_type must be"), (dict(a_type=0), "a_type must be"),
    (dict(a=torch.zeros(4, 64, dtype=torch.float8_e4m3fn)), "a without a_scale"),
    (dict(a=torch.zeros(4, 64, dtype=torch.float8_e4m3fn), a_scale=torch.zeros(4, 2, dtype=torch.uint8)), "a_type is for"),
    (dict(a=torch.zeros(4, 64, dtype=torch.float8_e4m3fn), a_scale=torch.zeros(4, 1, dtype=torch.uint8), a_type=0), "a_scale has"),
    (dict(a=torch.zeros(4, 64, dtype=torch.int8), a_scale=torch.zeros(4, 2, dtype=torch.uint8), a_type=0), "a with a_scale"),
    (dict(y=torch.zeros(4, 8, dtype=torch.bfloat16)), "a's type"), (dict(y=torch.zeros(4, 8)), "y must be"),
    (dict(y=torch.zeros(4, 9, dtype=H16)), "y has"),
])
def test_mx_matmul_refuses(olamd, kw, text):
    a = dict(a=torch.zeros(4, 64, dtype=H16), a_scale=None, a_type=17, b=torch.zeros(8, 32, dtype=torch.uint8),
             b_scale=torch.zeros(8, 2, dtype=torch.uint8), y=torch.zeros(4, 8, dtype=H16))
    a.update(kw)
    refused(olamd, "mx_matmul", [dev(olamd, a["a"]), dev(olamd, a["a_scale"]), a["a_type"], dev(olamd, a["b"]),
                                 dev(olamd, a["b_scale"]), dev(olamd, a["y"])], text)



CACHE = [
    (dict(k_cache=torch.zeros(3, 2, 16, 64)), "the cache must be"), (dict(k_cache=None), "are required"),
    (dict(v_cache=torch.zeros(3, 2, 64, 16, dtype=torch.float8_e4m3fn)), "one type"),
    (dict(v_cache=torch.zeros(3, 2, 16, 64, dtype=torch.int8)), "v_cache"),
    (dict(k_cache=torch.zeros(3, 2, 24, 64, dtype=torch.int8), v_cache=torch.zeros(3, 2, 64, 24, dtype=torch.int8)), "block_tokens"),
    (dict(k_cache=torch.zeros(3, 2, 16, 72, dtype=torch.int8), v_cache=torch.zeros(3, 2, 72, 16, dtype=torch.int8)), "head_dim"),
    (dict(k_cache=torch.zeros(3, 2, 16, 272, dtype=torch.int8), v_cache=torch.zeros(3, 2, 272, 16, dtype=torch.int8)), "head_dim"),
    (dict(k_scale=torch.zeros(3, 1)), "k_scale or v_scale"), (dict(v_scale=torch.zeros(3, 2, dtype=H16)), "must be FLOAT"),
    (dict(table=torch.zeros(2, 3, dtype=torch.int64)), "INT32"), (dict(table=torch.zeros(6, dtype=torch.int32)), "block_table must"),
    (dict(start=torch.zeros(2, dtype=torch.int32)), "query_start"), (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
]


def cache_args(olamd, kw):
    a = dict(k_cache=torch.zeros(3, 2, 16, 64, dtype=torch.int8), v_cache=torch.zeros(3, 2, 64, 16, dtype=torch.int8),
             k_scale=torch.zeros(3, 2), v_scale=torch.zeros(3, 2), table=torch.zeros(2, 3, dtype=torch.int32),
             start=torch.zeros(3, dtype=torch.int32), lengths=torch.zeros(2, dtype=torch.int32))
    a.update({k: v for k, v in kw.items() if k in a})
    return [dev(olamd, a[n]) for n in ("k_cache", "v_cache", "k_scale", "v_scale", "table", "start", "lengths")]


@pytest.mark.parametrize("kw,text", CACHE + [
    (dict(k=torch.zeros(5, 2, 64)), "FLOAT16 or BFLOAT16"), (dict(k=torch.zeros(5, 128, dtype=H16)), "k must be"),
    (dict(k=None), "are required"), (dict(v=torch.zeros(5, 2, 64, dtype=torch.bfloat16)), "both the same"),
    (dict(k=torch.zeros(5, 1, 64, dtype=H16)), "k ([tokens"), (dict(v=torch.zeros(4, 2, 64, dtype=H16)), "v ([tokens"),
])
def test_append_refuses(olamd, kw, text):
    a = dict(k=torch.zeros(5, 2, 64, dtype=H16), v=torch.zeros(5, 2, 64, dtype=H16))
    a.update({k: v for k, v in kw.items() if k in a})
    refused(olamd, "kv_cache_append", [dev(olamd, a["k"]), dev(olamd, a["v"])] + cache_args(olamd, kw), text)


@pytest.mark.parametrize("kw,text", CACHE + [
    (dict(q=torch.zeros(5, 4, 64)), "FLOAT16 or BFLOAT16"), (dict(q=torch.zeros(5, 256, dtype=H16)), "q must be"),
    (dict(q=torch.zeros(5, 3, 64, dtype=H16), out=torch.zeros(5, 3, 64, dtype=H16)), "multiple"),
    (dict(q=torch.zeros(5, 4, 32, dtype=H16)), "different head_dim"), (dict(out=torch.zeros(5, 2, 64, dtype=H16)), "out has"),
    (dict(out=torch.zeros(5, 4, 64, dtype=torch.bfloat16)), "both the same"), (dict(scale=float("nan")), "scale must"),
    (dict(max_query=-1), "max_query"),
])
def test_attention_refuses(olamd, kw, text):
    a = dict(q=torch.zeros(5, 4, 64, dtype=H16), out=torch.zeros(5, 4, 64, dtype=H16), scale=0.1, max_query=0)
    a.update({k: v for k, v in kw.items() if k in a})
    refused(olamd, "kv_cache_attention", [dev(olamd, a["q"])] + cache_args(olamd, kw) +
            [a["scale"], a["max_query"], dev(olamd, a["out"])], text)


@pytest.mark.parametrize("start,lengths,table,text", [
    ([0, 3, 2], [3, 3], 0, "query_start"), ([-1, 3, 5], [9, 9], 0, "query_start"), ([0, 3, 6], [9, 9], 0, "query_start"),
    ([0, 3, 5], [2, 9], 0, "lengths"), ([0, 3, 5], [9, 49], 0, "lengths"), ([0, 3, 5], [9, 9], 3, "block of block_table"),
    ([0, 3, 5], [9, 9], -1, "block of block_table"),
])
def test_host_index_tensors_are_checked(olamd, start, lengths, table, text):
    args = cache_args(olamd, dict(table=torch.full((2, 3), table, dtype=torch.int32),
                                  start=torch.tensor(start, dtype=torch.int32),
                                  lengths=torch.tensor(lengths, dtype=torch.int32)))
    for d in args[4:]:
        d.location = olamd.HOST
    q = torch.zeros(5, 4, 64, dtype=H16)
    refused(olamd, "kv_cache_attention", [dev(olamd, q)] + args + [0.1, 0, dev(olamd, q)], text)


def test_the_cache_stays_on_the_device(olamd):
    args = cache_args(olamd, {})
    args[0].location = olamd.HOST
    q = torch.zeros(5, 4, 64, dtype=H16)
    refused(olamd, "kv_cache_attention", [dev(olamd, q)] + args + [0.1, 0, dev(olamd, q)], "device memory")


def test_strided_tensors_are_refused(olamd):
    x = torch.zeros(4, 128, dtype=H16)[:, ::2]
    with pytest.raises(olamd.InvalidArgument, match="contiguous"):
        olamd.rms_norm_quantize(x, torch.zeros(64, dtype=H16))


# ---- the plain implementations -----------------------------------------------------

def test_mx_quantize_known_answers():
    x = torch.zeros(1, 64)
    x[0, :6] = torch.tensor([6.0, 2.5, -0.25, 0.75, 5.0, -7.0])   # largest 7: exponent 2, scale 2^0
    x[0, 32] = 0.75                                                # exponent -1, scale 2^-3
    v, s = dc.mx_quantize(x, "fp4")
    assert s.tolist() == [[127, 124]]
    assert v[0, :6].tolist() == [6.0, 2.0, -0.0, 1.0, 4.0, -6.0] and v[0, 32] == 6.0
    v, s = dc.mx_quantize(x, "fp8")
    assert s.tolist() == [[127 + 2 - 8, 127 - 1 - 8]]
    assert v[0, :2].tolist() == [384.0, 160.0] and v[0, 5] == -448.0 and v[0, 32] == 384.0
    assert dc.mx_quantize(torch.zeros(1, 32), "fp4")[1].tolist() == [[0]]


def test_mx_fp8_codes_match_a_cast():
    x = dc.randn(dc.gen(0), (50, 64), F32)
    v, s = dc.mx_quantize(x, "fp8")
    scaled = (x.reshape(-1, 32) / torch.exp2(s.reshape(-1, 1).float() - 127)).clamp(-448, 448)
    assert torch.equal(scaled.to(torch.float8_e4m3fn).double().reshape(50, 64), v)


def test_attention_matches_a_dense_softmax():
    b = dc.Batch(1, [3], [37], 2, 16, 16, "fp8", F32, heads=4)
    out, mass, _ = dc.attention(b, 0.25)
    blk = b.table[0, :3].long()
    for h in range(4):
        k = torch.cat([b.k_cache[j, h // 2].double() * b.k_scale[j, h // 2].double() for j in blk])[:37]
        v = torch.cat([b.v_cache[j, h // 2].double().T * b.v_scale[j, h // 2].double() for j in blk])[:37]
        for i in range(3):
            z = torch.exp(b.q[i, h].double() @ k[:35 + i].T * 0.25)
            dc.near(out[i, h], (z[:, None] * v[:35 + i]).sum(0) / z.sum(), torch.full((16,), 1e-12).double())
    assert (mass >= out.abs() - 1e-12).all()


def test_append_grows_a_scale_and_keeps_the_old_tokens():
    b = dc.Batch(1, [1], [3], 1, 16, 16, "int8", F32)
    blk = int(b.table[0, 0])
    b.k_cache[blk], b.k_scale[blk] = 100, 0.01
    b.k[:] = 2.54
    want = dc.append(b)
    assert float(want["k_scale"][blk]) == float(torch.tensor(2.54) / 127)
    assert (want["k_cache"][blk, 0, :2] == 50).all() and (want["k_cache"][blk, 0, 2] == 127).all()
    assert (want["k_cache"][blk, 0, 3:] == 100).all()
