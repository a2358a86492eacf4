"""The gated feed-forward in MX types against a plain implementation in 64 bits."""
import pytest
import torch

import decoder_cases as dc
import token_step_cases as ts

pytestmark = pytest.mark.gpu
KINDS = ["silu", "gelu", "gelu_tanh", "relu"]


@pytest.fixture(scope="module")
def gpu(olamd):
    olamd.init(0)
    return olamd


def dense(w):
    return dc.mx_values(dc.unpack4(w[0]), w[1])


def near_mx(got, scale, h, off):
    """MXFP8 of h: a block's exponent is that of its largest value, which may be off;
    codes are the nearest, half a step of them and the value's own error away."""
    v, b, e = got.cpu().double().reshape(-1, 32), h.reshape(-1, 32), off.reshape(-1, 32)
    lo, hi = ((b.abs() + k * e).clamp(min=0).amax(1, keepdim=True) for k in (-1, 1))
    s = scale.cpu().double().reshape(-1, 1) - 127
    assert (s >= torch.floor(torch.log2(lo.clamp(min=2.0 ** -119))) - 8).all()
    assert (s <= torch.floor(torch.log2(hi.clamp(min=2.0 ** -119))) - 8).all()
    unit = torch.exp2(s)
    want = (b / unit).clamp(-448, 448)
    dc.near(v, want, dc.half_step(torch.maximum(v.abs(), want.abs()), "fp8") + e / unit)


def check(gpu, x, gate, up, act, activation, mx=False, codes=None):
    kw = dict(a_type=gpu.FLOAT8E4M3FN if act == "fp8" else gpu.FLOAT4E2M1) if codes is None else dict(a_scale=codes[1].cuda())
    got = gpu.mx_gated_matmul((x if codes is None else codes[0]).cuda(), gate[0].cuda(), gate[1].cuda(), up[0].cuda(), up[1].cuda(),
                              activation, mx=mx, **kw)
    values, scales = dc.mx_quantize(x, act) if codes is None else (codes[2], codes[1])
    h, off = ts.gated(dc.mx_values(values, scales), dense(gate), dense(up), act, activation)
    if mx:
        assert got[0].dtype == torch.float8_e4m3fn and got[1].dtype == torch.uint8
        near_mx(*got, h, off)
    else:
        assert got.dtype == (x.dtype if codes is None else torch.bfloat16)
        dc.near(got, h, dc.ROUND[got.dtype] * h.abs() + off + 2.0 ** -25)
    return got


def operands(M, N, K, typ, seed=0, lo=114, hi=118):
    """Weights that leave the gate's sums around 1, where the activations bend."""
    g = dc.gen(M * 31 + N + K + seed)
    return dc.randn(g, (M, K), dc.TYPE[typ]), dc.mx_weight(g, N, K, lo, hi), dc.mx_weight(g, N, K, lo, hi)


MNK = [(1, 1, 32), (1, 16, 128), (1, 2048, 4096), (2, 33, 96), (3, 100, 160), (5, 257, 512), (8, 64, 2080), (16, 48, 1056),
       (17, 130, 544), (33, 259, 1024), (64, 512, 1504), (65, 96, 2080), (127, 129, 256), (130, 300, 1120), (256, 256, 512),
       (300, 700, 416), (513, 390, 608), (1, 3, 11008), (31, 1027, 64)]


@pytest.mark.parametrize("M,N,K", MNK)
@pytest.mark.parametrize("act", ["fp8", "fp4"])
@pytest.mark.parametrize("typ", ["bf16", "fp16"])
def test_gated(gpu, M, N, K, act, typ):
    check(gpu, *operands(M, N, K, typ), act, KINDS[(M + N) % 4])


@pytest.mark.parametrize("M,N,K", [(1, 32, 32), (1, 2048, 4096), (2, 96, 160), (9, 32, 2080), (16, 64, 1056), (17, 160, 544), (32, 512, 1024),
                                   (33, 288, 1024), (64, 96, 512), (65, 96, 2080), (130, 320, 1120), (256, 256, 512), (513, 416, 608),
                                   (1, 32, 11008), (31, 1056, 64)])
@pytest.mark.parametrize("act", ["fp8", "fp4"])
def test_gated_to_mxfp8(gpu, M, N, K, act):
    check(gpu, *operands(M, N, K, "bf16", 1), act, KINDS[(M + N // 32) % 4], mx=True)


@pytest.mark.parametrize("M", [1, 20, 40, 100])
@pytest.mark.parametrize("activation", KINDS)
@pytest.mark.parametrize("mx", [False, True])
def test_every_activation(gpu, M, activation, mx):
    """Sums from tiny to far past where an activation is 0 or the identity."""
    x, gate, up = operands(M, 96, 256, "fp16", 2)
    gate[1][:] = torch.randint(104, 122, (96, 1), generator=dc.gen(M)).to(torch.uint8)
    check(gpu, x, gate, up, "fp4", activation, mx)


@pytest.mark.parametrize("M,N,K", MNK[3:])
@pytest.mark.parametrize("act", ["fp8", "fp4"])
def test_gated_of_codes(gpu, M, N, K, act):
    _, gate, up = operands(M, N, K, "bf16", 3, 108, 114)
    g = dc.gen(M + N)
    s = torch.randint(118, 124, (M, K // 32), generator=g).to(torch.uint8)
    if act == "fp8":
        codes = (torch.randn((M, K), generator=g) * 30).clamp(-448, 448).to(torch.float8_e4m3fn)
        values = codes.double()
    else:
        codes = torch.randint(0, 256, (M, K // 2), generator=g).to(torch.uint8)
        values = dc.unpack4(codes)
    check(gpu, None, gate, up, act, "silu", codes=(codes, s, values))


@pytest.mark.parametrize("M,N,K,act", [(1000, 3050, 288, "fp8"), (1000, 3050, 1056, "fp8"), (2000, 4200, 800, "fp4"), (2000, 4200, 1024, "fp4")])
def test_large_tiles_over_several_steps(gpu, M, N, K, act):
    check(gpu, *operands(M, N, K, "bf16"), act, "silu")


@pytest.mark.parametrize("M,N,K,act", [(1000, 6100, 1056, "fp8"), (2000, 8400, 800, "fp4"), (100, 4000, 1312, "fp8"), (100, 4000, 2592, "fp4"),
                                       (1000, 6100, 8480, "fp8")])
def test_plain_products_by_tiles_over_several_steps(gpu, M, N, K, act):
    """(the last on four waves; its rows and columns are looked at by a sample)"""
    x, w, _ = operands(M, N, K, "bf16")
    got = gpu.mx_matmul(x.cuda(), w[0].cuda(), w[1].cuda(), a_type=gpu.FLOAT8E4M3FN if act == "fp8" else gpu.FLOAT4E2M1)
    rows, cols = torch.arange(0, M, 1 if K < 3000 else 17), torch.arange(0, N, 1 if K < 3000 else 23)
    want, off = ts.product(dc.mx_values(*dc.mx_quantize(x, act))[rows], dense(w)[cols], act)
    dc.near(got.cpu()[rows][:, cols], want, dc.ROUND[got.dtype] * want.abs() + off + 2.0 ** -25)


@pytest.mark.parametrize("M,N,K,act", [(1000, 3050, 96, "fp8"), (1900, 4000, 64, "fp8"), (2000, 4200, 64, "fp4"), (40, 5700, 96, "fp8"),
                                       (61, 3600, 288, "fp8"), (50, 6301, 96, "fp4")])
def test_wide(gpu, M, N, K, act):
    """Sizes that take each of the tiles, and wide weights of few rows."""
    check(gpu, *operands(M, N, K, "bf16", 4), act, "silu")
    if N % 32 == 0:
        check(gpu, *operands(M, N, K, "bf16", 4), act, "silu", mx=True)


@pytest.mark.parametrize("M", [1, 20, 300])
def test_places_gate_and_up(gpu, M):
    """ReLU of distinct positive gates times distinct ups, one nonzero activation a row: products exact to the bit, so that
    a column of either weight in another's place shows."""
    K, N = 416, 160
    g = dc.gen(9)
    gate, up = dc.mx_weight(g, N, K, 124, 130), dc.mx_weight(g, N, K, 120, 134)
    gate = (gate[0] & 0x77, gate[1])
    x = torch.zeros((M, K))
    k = (torch.arange(M) * 37) % K
    x[torch.arange(M), k] = 1.0
    want = (dense(gate)[:, k] * dense(up)[:, k]).T
    for act in (gpu.FLOAT8E4M3FN, gpu.FLOAT4E2M1):
        args = (x.to(torch.bfloat16).cuda(), gate[0].cuda(), gate[1].cuda(), up[0].cuda(), up[1].cuda(), "relu")
        got = gpu.mx_gated_matmul(*args, a_type=act)
        assert torch.equal(got.cpu().double(), want.to(torch.bfloat16).double())
        codes, scale = gpu.mx_gated_matmul(*args, a_type=act, mx=True)
        q, s = gpu.mx_quantize(want.float().contiguous().cuda())
        # (a sum with the weight -0 in it is +0, where the product by itself is -0: zeros are equal here)
        assert torch.equal(scale, s) and torch.equal(codes.float(), q.float())


@pytest.mark.parametrize("M", [1, 20, 40, 300])
@pytest.mark.parametrize("mx", [False, True])
def test_keeps_nan_to_its_row_and_column(gpu, M, mx):
    x, gate, up = operands(M, 96, 256, "fp16", 5)
    for activation in KINDS:
        run = lambda: gpu.mx_gated_matmul(x.cuda(), gate[0].cuda(), gate[1].cuda(), up[0].cuda(), up[1].cuda(), activation, mx=mx)  # noqa: E731
        want = run()
        x0, g0, u0 = x.clone(), gate[1].clone(), up[1].clone()
        x[M // 2, 77] = float("inf")
        gate[1][33, 2], up[1][70, 3] = 255, 255
        got = run()
        x, gate, up = x0, (gate[0], g0), (up[0], u0)
        if mx:
            # a column's NaN is its whole block's
            nan = got[1] == 255
            assert nan[M // 2].all() and nan[:, 1:].all() and not got[0][M // 2].float().any()
            keep = torch.arange(M) != M // 2
            assert torch.equal(got[1][keep, 0], want[1][keep, 0])
            assert torch.equal(got[0][keep, :32].view(torch.uint8), want[0][keep, :32].view(torch.uint8))
        else:
            assert torch.isnan(got[M // 2]).all() and torch.isnan(got[:, [33, 70]]).all()
            got[M // 2], got[:, [33, 70]] = want[M // 2], want[:, [33, 70]]
            assert torch.equal(got, want)


def test_of_nothing_of_rank_3_and_from_the_host(gpu):
    x, gate, up = operands(6, 64, 64, "bf16", 6)
    w = (*gate, *up)
    d = tuple(t.cuda() for t in w)
    assert gpu.mx_gated_matmul(x[:0].cuda(), *d).shape == (0, 64)
    got = gpu.mx_gated_matmul(x.view(2, 3, 64).cuda(), *d)
    assert got.shape == (2, 3, 64) and torch.equal(got.view(6, 64), gpu.mx_gated_matmul(x.cuda(), *d))
    assert torch.equal(gpu.mx_gated_matmul(x, *w), gpu.mx_gated_matmul(x.cuda(), *d).cpu())
    y, s = gpu.mx_gated_matmul(x, *w, mx=True)
    yd, sd = gpu.mx_gated_matmul(x.cuda(), *d, mx=True)
    assert torch.equal(y.view(torch.uint8), yd.cpu().view(torch.uint8)) and torch.equal(s, sd.cpu())
    none = torch.empty((32, 0), dtype=torch.uint8, device="cuda")
    for M in (3, 200):
        empty = torch.empty((M, 0), dtype=torch.float16, device="cuda")
        assert not gpu.mx_gated_matmul(empty, none, none, none, none).any()
        y, s = gpu.mx_gated_matmul(empty, none, none, none, none, mx=True)
        assert not y.float().any() and not s.any()


@pytest.mark.parametrize("M", [1, 40, 200])
def test_whole_block_captured_and_on_another_stream(gpu, M):
    """Gated product to MXFP8 and the product that takes it back, and the 16-bit form."""
    x, gate, up = operands(M, 512, 256, "bf16", 7)
    down = tuple(t.cuda() for t in dc.mx_weight(dc.gen(8), 256, 512))
    x, w = x.cuda(), tuple(t.cuda() for t in (*gate, *up))

    def block():
        h, s = gpu.mx_gated_matmul(x, *w, mx=True)
        return h.view(torch.uint8), s, gpu.mx_matmul(h, *down, s), gpu.mx_matmul(gpu.mx_gated_matmul(x, *w, "gelu"), *down)

    want = block()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = block()
    side.synchronize()
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = block()
    for _ in range(3):
        for t in got:
            t.zero_()
        block()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(got, want))
