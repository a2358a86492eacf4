"""Edges of the decoder-layer operators that show without a GPU: calls that have
nothing to do end before any device work, and arguments that say something the
operators do not do are refused."""
import ctypes

import pytest
import torch

from test_decoder_host import cache_args, dev

H16 = torch.float16


def status(olamd, name, args):
    """Status and message of a call; NOT_INITIALIZED where it passed its checks and went on to the device."""
    rc = getattr(olamd.lib(), "onnxl_amd_" + name)(*[ctypes.byref(a) if isinstance(a, olamd.Tensor) else a for a in args],
                                                   None)
    return rc, olamd.lib().onnxl_amd_last_error().decode()


@pytest.mark.parametrize("max_query", [0, 1])
@pytest.mark.parametrize("most", [0, 3])
def test_rows_of_an_empty_batch_need_no_device(olamd, max_query, most):
    """Rows of q, k and v, but no sequence: query_start has one entry and lengths none, whose payload is null.  Both
    operators are done before they need the device."""
    cache = cache_args(olamd, dict(table=torch.zeros((0, most), dtype=torch.int32), start=torch.zeros(1, dtype=torch.int32),
                                   lengths=torch.zeros(0, dtype=torch.int32)))
    q, k = torch.zeros(5, 4, 64, dtype=H16), torch.zeros(5, 2, 64, dtype=H16)
    assert status(olamd, "kv_cache_append", [dev(olamd, k), dev(olamd, k)] + cache)[0] == olamd.OK
    assert status(olamd, "kv_cache_attention", [dev(olamd, q)] + cache + [0.1, max_query, dev(olamd, q)])[0] == olamd.OK


@pytest.mark.parametrize("name,values,text", [
    ("start", [0, 3, 2], "query_start"), ("start", [-1, 3, 5], "query_start"), ("start", [0, 3, 6], "query_start"),
    ("start", [4, 2, 5], "query_start"), ("lengths", [-1, 9], "lengths"), ("lengths", [9, 49], "lengths"),
])
@pytest.mark.parametrize("table_on_host", [False, True])
def test_each_host_index_tensor_is_checked(olamd, name, values, text, table_on_host):
    """query_start or lengths in host memory, the other one on the device."""
    cache = cache_args(olamd, {name: torch.tensor(values, dtype=torch.int32)})
    cache[5 if name == "start" else 6].location = olamd.HOST
    if table_on_host:
        cache[4].location = olamd.HOST
    q, k = torch.zeros(5, 4, 64, dtype=H16), torch.zeros(5, 2, 64, dtype=H16)
    for op, args in (("kv_cache_attention", [dev(olamd, q)] + cache + [0.1, 0, dev(olamd, q)]),
                     ("kv_cache_append", [dev(olamd, k), dev(olamd, k)] + cache)):
        rc, message = status(olamd, op, args)
        assert rc == olamd.INVALID_ARGUMENT and text in message, (rc, message)


def test_host_index_tensors_that_fit_pass(olamd):
    """Alone and together; a block table without lengths has entries that nobody reads."""
    for where in ((5,), (6,), (4,), (4, 5), (4, 6), (5, 6)):
        cache = cache_args(olamd, dict(table=torch.full((2, 3), 99 if 6 not in where else 0, dtype=torch.int32),
                                       start=torch.tensor([0, 3, 5], dtype=torch.int32),
                                       lengths=torch.tensor([3, 48], dtype=torch.int32)))
        for i in where:
            cache[i].location = olamd.HOST
        # on to the checks that come after those of the index tensors
        q = torch.zeros(5, 3, 64, dtype=H16)
        rc, message = status(olamd, "kv_cache_attention", [dev(olamd, q)] + cache + [0.1, 0, dev(olamd, q)])
        assert rc == olamd.INVALID_ARGUMENT and "multiple" in message, (where, rc, message)


@pytest.mark.parametrize("kw,text", [
    (dict(output_dtype=10), "output_dtype"), (dict(output_dtype=2), "output_dtype"), (dict(output_dtype=23), "output_dtype"),
    (dict(block_size=64, mx=True), "blocks of 32"), (dict(block_size=-1), "block_size"), (dict(block_size=-1, mx=True), "block_size"),
    (dict(output_dtype=3, mx=True), "FLOAT8E4M3FN"),
])
def test_norm_front_end_refuses_what_it_does_not_do(olamd, kw, text):
    """Types and block sizes that the caller names are taken or refused, never replaced."""
    x = torch.zeros(2, 128, dtype=H16)
    with pytest.raises(olamd.InvalidArgument, match=text):
        olamd.rms_norm_quantize(x, x[0], **kw)


@pytest.mark.parametrize("dtype", [10, 2, 0])
def test_cache_of_another_type_is_refused(olamd, dtype):
    with pytest.raises(olamd.InvalidArgument, match="INT8 or FLOAT8E4M3FN"):
        olamd.KvCache(2, 1, 16, 64, dtype, "cpu")
    assert olamd.KvCache(2, 1, 16, 64, olamd.INT8, "cpu").k_cache.dtype == torch.int8
    assert olamd.KvCache(2, 1, 16, 64, device="cpu").v_cache.dtype == torch.float8_e4m3fn


def test_product_front_end_refuses_another_output_type(olamd):
    """16-bit activations give their own type: another one that the caller names is refused."""
    w, s = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8)
    for dtype in (torch.bfloat16, torch.float32):
        with pytest.raises(olamd.InvalidArgument, match="y must be"):
            olamd.mx_matmul(torch.zeros(2, 64, dtype=H16), w, s, output_dtype=dtype)
