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


# ---- shares of sums of more than 53 bits ------------------------------------------------

def near_flat(before, after, n=1 << 20):
    """n equal tokens with tokens of a weight of about 1e-11 before and after them, and all weights in units of 2^-42 of
    the largest.  The sum has 63 bits, and what the small ones add to it is less than 64 bits of a float keep."""
    d = 24.5  # exp(-24.5) 2^42 = 100.7
    unit = float(np.exp(-d) * 2.0 ** 42)
    assert abs(unit - 101) < 0.4
    x = torch.zeros(before + n + after)
    x[:before], x[before + n:] = -d, -d
    return x, [101] * before + [1 << 42] * n + [101] * after


def drawn(weights, u, top_p):
    """The token and how many are kept, by whole numbers: u and top_p are sixteenths."""
    order = sorted(range(len(weights)), key=lambda i: -weights[i])
    total, upto, kept = sum(weights), 0, []
    for i in order:
        if 16 * upto >= round(16 * top_p) * total and kept:
            break
        kept.append(i)
        upto += weights[i]
    kept, upto, total = sorted(kept), 0, sum(weights[i] for i in kept)
    for i in kept:
        upto += weights[i]
        if 16 * upto > round(16 * u) * total:
            return i, len(kept)


@pytest.mark.parametrize("rows", [1, 17])
@pytest.mark.parametrize("typ", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("before,after,u,top_p", [(4, 3, 0.5, 1.0), (0, 4, 0.25, 0.5), (3, 1, 0.5, 0.5), (5, 0, 0.0, 0.25), (1, 6, 0.75, 0.75),
                                                  (0, 4, 0.5, 1.0), (2, 2, 0.9375, 0.9375)])
def test_shares_of_long_sums_are_exact(gpu, rows, typ, before, after, u, top_p):
    x, weights = near_flat(before, after)
    want, kept = drawn(weights, u, top_p)
    x = x.to(dc.TYPE[typ]).cuda().expand(rows, -1).contiguous()
    fill = lambda v: torch.full((rows,), v, device="cuda")  # noqa: E731
    token, prob = gpu.sample_tokens(x, fill(u), None, None, fill(top_p) if top_p < 1 else None)
    assert (token == want).all()
    # a kept token more or less changes the probability by 2^-19 to 2^-20 of itself
    assert ((prob.double().cpu() - 1 / (kept if top_p < 1 else 1 << 20)).abs() < 2.0 ** -22 / kept).all()


def test_tiny_shares(gpu):
    """top_p and u down to fp32's smallest numbers: the first token of the order, and of the index."""
    x, _ = ts.randn_logits(3, 6, 5000, torch.float32)
    tiny = [1e-3, 1e-7, 1e-12, 1e-30, 1e-38, 1e-45]
    p = torch.tensor(tiny)
    check(gpu, x, torch.rand(6, generator=dc.gen(1)), top_p=p)
    check(gpu, x, p)
    token, _ = check(gpu, x, p.flip(0), top_p=p)
    assert torch.equal(token.cpu(), x.argmax(1))
