"""Sampling against the definition in 64 bits: tokens equal, probabilities to fp32."""
import math

import pytest
import torch

import decoder_cases as dc
import token_step_cases as ts

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def gpu(olamd):
    olamd.init(0)
    return olamd


def f32(v):
    return torch.as_tensor(v, dtype=torch.float32)


def check(gpu, x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """Options: a tensor [rows], a number for all rows, or None."""
    rows = len(x)
    spread = lambda v, t: None if v is None else torch.as_tensor(v, dtype=t).expand(rows).contiguous()  # noqa: E731
    u, T, p, m = (spread(v, torch.float32) for v in (u, temperature, top_p, min_p))
    k = spread(top_k, torch.int32)
    dev = [None if t is None else t.cuda() for t in (T, k, p, m)]
    token, prob = gpu.sample_tokens(x.cuda(), u.cuda(), *dev)
    assert token.dtype == torch.int64 and prob.dtype == torch.float32
    at = lambda t, r, off: off if t is None else t[r].item()  # noqa: E731
    for r in range(rows):
        want, wp = ts.sample(x[r].double().numpy(), u[r].item(), at(T, r, 1.0), at(k, r, 0), at(p, r, 1.0), at(m, r, 0.0))
        assert token[r].item() == want, (r, token[r].item(), want)
        # a ratio of two numbers of 42 bits and more, rounded to fp32
        assert abs(prob[r].item() - wp) <= 2.0 ** -22 * wp, (r, prob[r].item(), wp)
    return token, prob


VOCABS = [1, 2, 63, 64, 65, 1000, 1024, 4097, 32000, 50257, 131072, 200003]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("typ", ["fp32", "fp16", "bf16"])
def test_every_option_and_size(gpu, vocab, typ):
    rows = 3 if vocab > 5000 else 9
    x, u = ts.randn_logits(vocab, rows, vocab, dc.TYPE[typ])
    check(gpu, x, u)
    check(gpu, x, u, 0.7)
    check(gpu, x, u, top_k=50)
    check(gpu, x, u, 1.3, top_p=0.9)
    check(gpu, x, u, min_p=0.05)
    check(gpu, x, u, 0.9, 40, 0.95)
    check(gpu, x, u, 1.5, 1000, 0.8, 0.01)
    check(gpu, x, u, 0.0)


@pytest.mark.parametrize("vocab", [777, 40000])
@pytest.mark.parametrize("typ", ["fp32", "bf16"])
def test_rows_that_ask_for_different_things(gpu, vocab, typ):
    rows = 24
    x, u = ts.randn_logits(3, rows, vocab, dc.TYPE[typ], masked=0.5)
    i = torch.arange(rows)
    check(gpu, x, u, f32([0.0, 0.3, 1.0, 2.0])[i % 4], torch.tensor([0, 1, 2, 20, 500, 10 ** 6, -3])[i % 7],
          f32([1.0, 0.5, 0.9, 0.999, 0.0, -1.0, 2.0, NAN])[i % 8], f32([0.0, 0.1, 1.0, 3.0, -1.0, NAN])[i % 6])


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 200, 400, 1100])
def test_row_counts(gpu, rows):
    x, u = ts.randn_logits(rows, rows, 1500, torch.bfloat16)
    check(gpu, x, u, 0.8, 100, 0.9)


@pytest.mark.parametrize("spread", [0.0, 1e-3, 0.3, 1.0, 10.0, 1000.0])
@pytest.mark.parametrize("typ", ["fp32", "fp16"])
@pytest.mark.parametrize("temperature", [0.01, 1.0, 100.0])
def test_flat_and_steep_rows(gpu, spread, typ, temperature):
    """All logits equal, nearly so, and far apart."""
    x, u = ts.randn_logits(7, 3, 9001, dc.TYPE[typ], spread)
    check(gpu, x, u, temperature)
    check(gpu, x, u, temperature, top_k=300)
    check(gpu, x, u, temperature, top_p=0.7)
    check(gpu, x, u, temperature, 5000, 0.5)


@pytest.mark.parametrize("vocab", [5, 300, 20000, 131072])
def test_equal_logits_count_from_the_lowest_index(gpu, vocab):
    """Two values, each many times: borders of top-k and top-p lie among equal logits.  Where shares fall on whole tokens
    all weights are 1, so that every sum is exact and the definition leaves nothing open."""
    x = torch.zeros(4, vocab)
    x[:, ::3] = math.log(4.0)
    for k in (1, 2, vocab // 3, vocab // 3 + 2, vocab - 1, vocab, vocab + 1):
        check(gpu, x, f32([0.0, 0.33, 0.66, 0.99]), top_k=max(k, 1))
    x = torch.ones(4, vocab)
    for p in (0.25, 0.5, 0.75):
        check(gpu, x, f32([0.0, 0.25, 0.5, 0.75]), top_p=p)
        check(gpu, x, f32([0.0, 0.25, 0.5, 0.75]), top_k=(vocab + 1) // 2, top_p=p)


def test_uniform_at_its_ends_and_outside(gpu):
    x, _ = ts.randn_logits(1, 8, 5000, torch.float32)
    x = x[:1].expand(8, -1).contiguous()
    u = f32([0.0, 2.0 ** -30, 1 - 2.0 ** -24, 1.0, 5.0, -1.0, NAN, 0.5])
    for kw in ({}, dict(top_k=7), dict(top_p=0.3), dict(min_p=0.5)):
        check(gpu, x, u, **kw)


def test_every_share_of_a_small_row(gpu):
    """A row of four tokens, and every multiple of a 64th: each takes what its share says."""
    x = f32([[0.0, math.log(2.0), -INF, math.log(3.0)]]).expand(64, -1).contiguous()
    u = torch.arange(64) / 64
    token, prob = check(gpu, x, u)
    assert torch.equal(token.cpu().bincount(minlength=4), torch.tensor([11, 21, 0, 32]))


@pytest.mark.parametrize("vocab", [6, 3000, 70000])
@pytest.mark.parametrize("typ", ["fp32", "fp16", "bf16"])
def test_infinities_nan_and_zeros(gpu, vocab, typ):
    x, u = ts.randn_logits(5, 8, vocab, dc.TYPE[typ])
    x[0] = -INF                       # nothing left
    x[1] = NAN
    x[2, 1:] = -INF                   # one token left
    x[3] = -INF
    x[3, -1] = torch.finfo(x.dtype).min  # the type's lowest number is a logit like others
    x[4, [1, 4]] = INF                # share the weight
    x[5, ::2] = NAN
    x[6] = -0.0
    x[6, vocab // 2:] = 0.0           # the zeros are equal
    x[7] = torch.finfo(x.dtype).min
    for kw in ({}, dict(temperature=0.0), dict(temperature=INF), dict(temperature=NAN), dict(temperature=-1.0), dict(top_k=2),
               dict(top_p=0.5), dict(top_k=3, top_p=0.5, min_p=0.1), dict(temperature=1e-30), dict(temperature=1e30, top_p=0.4)):
        token, prob = check(gpu, x, u, **kw)
        assert token[:2].tolist() == [-1, -1] and not prob[:2].any()
        assert token[2] == 0 and token[3] == vocab - 1 and token[4].item() in (1, 4)


def test_masked_to_the_types_lowest_number(gpu):
    x, u = ts.randn_logits(6, 4, 30000, torch.float32)
    x[:, torch.rand(30000, generator=dc.gen(1)) < 0.9] = torch.finfo(torch.float32).min
    for kw in (dict(top_k=10), dict(top_k=20000), dict(top_p=0.9), dict(temperature=2.0, min_p=0.01), {}):
        check(gpu, x, u, **kw)


def test_types_of_indices_absent_probability_and_host(gpu):
    x, u = ts.randn_logits(2, 5, 4000, torch.float16)
    k = torch.tensor([3, 0, 100, 5000, 1])
    want, prob = gpu.sample_tokens(x.cuda(), u.cuda(), None, k.cuda())
    token = torch.full((5,), -7, dtype=torch.int32, device="cuda")
    gpu.sample_tokens(x.cuda(), u.cuda(), None, k.int().cuda(), out=(token, None))
    assert torch.equal(token.long(), want)
    host = gpu.sample_tokens(x, u, None, k)
    assert not host[0].is_cuda and torch.equal(host[0], want.cpu()) and torch.equal(host[1], prob.cpu())
    assert gpu.sample_tokens(x[:0].cuda(), u[:0].cuda())[0].shape == (0,)


def test_memory_off_alignment(gpu):
    """Rows of odd length, and a tensor that begins between 16-byte lines."""
    for typ in (torch.bfloat16, torch.float32):
        x, u = ts.randn_logits(9, 7, 10007, typ)
        want = gpu.sample_tokens(x.cuda(), u.cuda(), None, None, torch.full((7,), 0.9, device="cuda"))
        for off in (1, 3):
            odd = torch.nn.functional.pad(x.reshape(-1), (off, 0)).cuda()[off:].view(x.shape)
            got = gpu.sample_tokens(odd, u.cuda(), None, None, torch.full((7,), 0.9, device="cuda"))
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_frequencies_follow_the_weights(gpu):
    """4096 evenly spread numbers take every token as often as its weight says, to one."""
    x, _ = ts.randn_logits(4, 1, 37, torch.float32, 1.0)
    u = (torch.arange(4096) + 0.5) / 4096
    token, _ = gpu.sample_tokens(x.expand(4096, -1).contiguous().cuda(), u.cuda())
    want = torch.softmax(x[0].double(), 0) * 4096
    assert ((token.cpu().bincount(minlength=37) - want).abs() <= 1).all()


@pytest.mark.parametrize("rows,vocab", [(1, 131072), (40, 5000), (300, 20000)])
def test_captured_and_on_another_stream(gpu, rows, vocab):
    x, u = (t.cuda() for t in ts.randn_logits(8, rows, vocab, torch.bfloat16))
    T, p = torch.full((rows,), 0.9, device="cuda"), torch.full((rows,), 0.95, device="cuda")
    k = torch.full((rows,), 64, device="cuda")

    def step():
        return (*gpu.sample_tokens(x, u, T, None, p), *gpu.sample_tokens(x, u, T, k, p), *gpu.sample_tokens(x, u))

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
