"""The operators from the joint projection to the next token with numpy arrays, which are
host memory like CPU tensors."""
import pytest
import torch

import decoder_cases as dc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu(olamd):
    olamd.init(0)
    return olamd


def same(got, want):
    pairs = zip(got, want) if isinstance(got, tuple) else [(got, want)]
    return all((g is None and w is None) or (g.dtype == w.dtype and torch.equal(g.cpu().view(torch.uint8), w.cpu().view(torch.uint8)))
               for g, w in pairs)


def test_numpy_arrays(gpu):
    g = dc.gen(1)
    x = dc.randn(g, (5, 64), torch.float16)
    gate, up = dc.mx_weight(g, 32, 64), dc.mx_weight(g, 32, 64)
    c, s = dc.randn(g, (5, 4), torch.float32), dc.randn(g, (5, 4), torch.float32)
    for run, args in ((gpu.mx_matmul, (x, *gate)), (gpu.mx_gated_matmul, (x, *gate, *up)),
                      (gpu.rotary_embedding, (x.view(5, 4, 16), c, s)), (gpu.rms_norm_quantize, (x, x[0].contiguous(), x)),
                      (gpu.sample_tokens, (x, torch.rand(5, generator=g), torch.rand(5, generator=g)))):
        assert same(run(*(a.numpy() for a in args)), run(*(a.cuda() for a in args)))
    b = dc.Batch(2, [2, 3], [5, 9], 1, 64, 16, "int8", torch.float16)
    cache = gpu.kv_cache_append(b.k.cuda(), b.v.cuda(), b.cache(gpu), *b.index())
    assert same(gpu.kv_cache_attention(b.q.numpy(), cache, *b.index()), gpu.kv_cache_attention(b.q.cuda(), cache, *b.index()))
