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
