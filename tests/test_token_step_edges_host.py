"""Calls that the operators from the joint projection to the next token refuse, which ran
and gave something else (they are refused before any device work, so without a GPU)."""
import pytest

from test_decoder_host import refused
from test_token_step_host import append_args


@pytest.mark.parametrize("offset", [0, 256, 5 * 8 * 64 * 2 - 16, 16 - 5 * 4 * 64 * 2])
def test_rotary_append_refuses_q_over_qkv(olamd, offset):
    """q's first row on top of qkv's, inside it, at its end and reaching in from before."""
    args = append_args(olamd, {})
    args[5].data = args[0].data + offset
    refused(olamd, "rotary_kv_cache_append", args, "q may not overlap qkv")
