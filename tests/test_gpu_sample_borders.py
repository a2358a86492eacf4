"""Sampling where the way to a border is the long one: rows whose sampled logits say
nothing about top_p's border."""
import numpy as np
import pytest
import torch

import decoder_cases as dc
import token_step_cases as ts
from test_gpu_sample import check

pytestmark = pytest.mark.gpu
VOCAB = 131072


@pytest.fixture(scope="module")
def gpu(olamd):
    olamd.init(0)
    return olamd


def looked_at(vocab, dtype):
    """The places that stand for a long row: a load of each of 1024 threads."""
    n = 4 if dtype == torch.float32 else 8
    first = torch.arange(1024) * (vocab - n) // 1023
    return (first[:, None] + torch.arange(n)).reshape(-1).unique()


def misleading(seed, dtype, top_p):
    """One token has far more weight than any other.  Of the places that stand for the row
    one has a logit 6 octaves lower and the others none; 10000 tokens elsewhere lie 9.5 to
    10.5 octaves lower, and have nine tenths of the weight."""
    g = dc.gen(seed)
    x = torch.full((VOCAB,), float("-inf"))
    at = looked_at(VOCAB, dtype)
    other = torch.ones(VOCAB, dtype=torch.bool)
    other[at] = False
    other = other.nonzero()[:, 0]
    other = other[torch.randperm(len(other), generator=g)]
    octave = float(np.log(2.0))
    x[other[0]] = 3.0
    x[at[torch.randint(0, len(at), (1,), generator=g)]] = 3.0 - 6.0 * octave
    x[other[1:10001]] = 3.0 - octave * (9.5 + torch.rand(10000, generator=g))
    x = x.to(dtype)
    # the tokens from the one place's on do not reach the border
    w = torch.exp(x.double() - 3.0)
    assert w[x >= x[at].max()].sum() < top_p * w.sum()
    return x


@pytest.mark.parametrize("rows", [1, 5, 16, 17])
@pytest.mark.parametrize("typ", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("top_p", [0.5, 0.9, 0.99])
def test_border_below_what_the_rows_sample_says(gpu, rows, typ, top_p):
    x = torch.stack([misleading(100 * rows + r, dc.TYPE[typ], top_p) for r in range(rows)])
    u = torch.rand(rows, generator=dc.gen(rows))
    first = check(gpu, x, u, top_p=top_p)
    for _ in range(3):
        again = check(gpu, x, u, top_p=top_p)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    check(gpu, x, u, top_p=top_p, min_p=2.0 ** -10)


@pytest.mark.parametrize("rows", [4, 20])
def test_rows_with_and_without_a_sample_that_says_something(gpu, rows):
    x, u = ts.randn_logits(21, rows, VOCAB, torch.float32)
    for r in range(0, rows, 2):
        x[r] = misleading(r, torch.float32, 0.9)
    check(gpu, x, u, top_p=0.9)
