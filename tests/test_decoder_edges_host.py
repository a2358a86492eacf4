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
