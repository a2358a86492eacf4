"""Calls that the operators from the joint projection to the next token refuse, which ran
and gave something else (they are refused before any device work, so without a GPU)."""
import numpy as np
import pytest

from test_decoder_host import refused
from test_token_step_host import append_args


@pytest.mark.parametrize("offset", [0, 256, 5 * 8 * 64 * 2 - 16, 16 - 5 * 4 * 64 * 2])
def test_rotary_append_refuses_q_over_qkv(olamd, offset):
    """q's first row on top of qkv's, inside it, at its end and reaching in from before."""
    args = append_args(olamd, {})
    args[5].data = args[0].data + offset
    refused(olamd, "rotary_kv_cache_append", args, "q may not overlap qkv")


def test_numpy_arrays_reach_the_library(olamd):
    """Each call is refused by the library, for its last dimension; without it outputs of numpy's types were asked of torch."""
    x, w, s = np.zeros((2, 64), np.float16), np.zeros((32, 32), np.uint8), np.zeros((32, 3), np.uint8)
    for call in (lambda: olamd.mx_matmul(x, w, s), lambda: olamd.mx_gated_matmul(x, w, s, w, s),
                 lambda: olamd.rotary_embedding(np.zeros((2, 3, 8), np.float16), np.zeros((2, 5), np.float32), np.zeros((2, 5), np.float32)),
                 lambda: olamd.rms_norm_quantize(x, np.zeros(63, np.float16), x)):
        with pytest.raises(olamd.InvalidArgument):
            call()
