"""Every kernel of the MX products, plain and gated, over several of its steps, against a
plain implementation in 64 bits (test_mx_plan.py says that these sizes take each)."""
import pytest
import torch

import decoder_cases as dc
import token_step_cases as ts
from mx_kernel_cases import CASES
from test_gpu_gated import KINDS, dense, near_mx

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu(olamd):
    olamd.init(0)
    return olamd


def some(n, most, block=1):
    """Whole blocks of 0 .. n - 1: all of few, else the first, those on both sides of 128 and
    256, the last, and some between."""
    blocks = n // block
    if n <= most:
        at = torch.arange(blocks)
    else:
        edge = [b // block + d for b in (0, 64, 128, 192, 256) for d in (-1, 0, 1)] + [blocks - 1 - d for d in range(3)]
        at = torch.tensor(sorted({b for b in edge if 0 <= b < blocks} | set(range(0, blocks, max(1, blocks * block // most)))))
    return (at[:, None] * block + torch.arange(block)).reshape(-1)


@pytest.mark.parametrize("form,act,M,K,N,x16", CASES)
def test_product(gpu, form, act, M, K, N, x16):
    g = dc.gen(M * 31 + N + K)
    code = gpu.FLOAT8E4M3FN if act == "fp8" else gpu.FLOAT4E2M1
    weights = [dc.mx_weight(g, N, K, 114, 118) for _ in range(1 if form == "plain" else 2)]
    dev = [t.cuda() for w in weights for t in w]
    x = dc.randn(g, (M, K), torch.bfloat16)
    values, scales = dc.mx_quantize(x, act)
    if x16:
        a, kw = x.cuda(), dict(a_type=code)
    else:
        a, s = gpu.mx_quantize(x.cuda(), code)
        kw = dict(a_scale=s)
    rows, cols = some(M, 130), some(N, 600, 32 if form == "gated mx" else 1)
    values, weights = dc.mx_values(values, scales)[rows], [(c[cols], s[cols]) for c, s in weights]
    if form == "plain":
        got = gpu.mx_matmul(a, *dev, **kw)
        want, off = ts.product(values, dense(weights[0]), act)
    else:
        kind = KINDS[(M + N) % 4]
        got = gpu.mx_gated_matmul(a, *dev, kind, mx=form == "gated mx", **kw)
        want, off = ts.gated(values, *(dense(w) for w in weights), act, kind)
    if form == "gated mx":
        assert got[0].shape == (M, N) and got[1].shape == (M, N // 32)
        near_mx(got[0].cpu().float()[rows][:, cols], got[1].cpu()[rows][:, cols[::32] // 32], want, off)
        again = gpu.mx_gated_matmul(a, *dev, kind, mx=True, **kw)
        assert torch.equal(got[0].view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(got[1], again[1])
        return
    assert got.shape == (M, N)
    dc.near(got.cpu()[rows][:, cols], want, dc.ROUND[got.dtype] * want.abs() + off + 2.0 ** -25)
    again = gpu.mx_matmul(a, *dev, **kw) if form == "plain" else gpu.mx_gated_matmul(a, *dev, kind, **kw)
    assert torch.equal(got, again)
