"""RMS norm with 8-bit output, MX quantization and product, paged 8-bit cache
and its attention, against plain implementations in 64 bits."""
import pytest
import torch

import decoder_cases as dc

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def gpu(olamd):
    olamd.init(0)
    return olamd


# ---- RMS norm ------------------------------------------------------------------

def check_norm(gpu, x, w, r, to, block, mx=False, eps=1e-5, out=None):
    got, scale, total = gpu.rms_norm_quantize(x.cuda(), w.cuda(), None if r is None else r.cuda(), eps, block,
                                              gpu.INT8 if to == "int8" else gpu.FLOAT8E4M3FN, mx, out)
    v, h = dc.norm(x, w, r, eps)
    if r is None:
        assert total is None
    else:
        assert torch.equal(total.cpu(), h)
    D = x.shape[-1]
    block = 32 if mx else block or D
    vb = v.reshape(-1, block)
    top = vb.abs().amax(1, keepdim=True)
    code, s = got.cpu().double().reshape(-1, block), scale.cpu().double().reshape(-1, 1)
    if mx:
        s = torch.exp2(s - 127)
        # the power of two is top's, up to the fp32 error of a top beside a power of two
        lo, hi = (torch.floor(torch.log2(top * f)) - 8 for f in (1 - 2.0 ** -20, 1 + 2.0 ** -20))
        assert ((s == torch.exp2(lo)) | (s == torch.exp2(hi)) | (top == 0)).all()
    else:
        dc.near(s, top / dc.QMAX[to], top / dc.QMAX[to] * 2.0 ** -20)
    want = (vb / s.clamp(min=1e-300)).clamp(-dc.QMAX[to], dc.QMAX[to])
    # half a step of the code, and the fp32 steps before the rounding
    dc.near(code, want, dc.half_step(torch.maximum(code.abs(), want.abs()), to) + want.abs() * 2.0 ** -19)


@pytest.mark.parametrize("rows,D", [(1, 1), (1, 4096), (3, 7), (2, 255), (5, 1000), (7, 2049), (33, 5001), (2, 16384),
                                    (2, 20011), (700, 64)])
@pytest.mark.parametrize("typ", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("to", ["int8", "fp8"])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_per_row(gpu, rows, D, typ, to, residual):
    g = dc.gen(rows * 7 + D)
    x, r = dc.randn(g, (rows, D), dc.TYPE[typ], 3.0), dc.randn(g, (rows, D), dc.TYPE[typ], 2.0)
    check_norm(gpu, x, dc.randn(g, (D,), dc.TYPE[typ]), r if residual else None, to, 0)


@pytest.mark.parametrize("block", [32, 64, 128, 256])
@pytest.mark.parametrize("rows,D", [(1, 256), (3, 768), (9, 4096), (130, 1280), (2, 33024)])
@pytest.mark.parametrize("typ,to", [("bf16", "fp8"), ("fp16", "int8"), ("fp32", "fp8")])
def test_norm_per_block(gpu, block, rows, D, typ, to):
    g = dc.gen(block + D)
    check_norm(gpu, dc.randn(g, (rows, D), dc.TYPE[typ]), dc.randn(g, (D,), torch.float32),
               dc.randn(g, (rows, D), dc.TYPE[typ]), to, block)


@pytest.mark.parametrize("rows,D", [(1, 32), (3, 96), (17, 4096), (200, 2080), (3, 16416)])
@pytest.mark.parametrize("typ", ["fp16", "bf16"])
def test_norm_mxfp8(gpu, rows, D, typ):
    g = dc.gen(D)
    check_norm(gpu, dc.randn(g, (rows, D), dc.TYPE[typ]), dc.randn(g, (D,), dc.TYPE[typ]),
               dc.randn(g, (rows, D), dc.TYPE[typ]), "fp8", 32, mx=True)


def test_norm_shape_of_rank_3_and_zero_rows(gpu):
    g = dc.gen(3)
    check_norm(gpu, dc.randn(g, (2, 3, 96), torch.float16), dc.randn(g, (96,), torch.float16), None, "int8", 32)
    y, s, _ = gpu.rms_norm_quantize(torch.empty((0, 64), dtype=torch.float16, device="cuda"),
                                    torch.ones(64, dtype=torch.float16, device="cuda"))
    assert y.shape == (0, 64) and s.shape == (0, 1)


@pytest.mark.parametrize("alias", ["x", "residual"])
@pytest.mark.parametrize("D", [512, 4099, 40000])
def test_norm_sum_in_place(gpu, alias, D):
    g = dc.gen(D)
    x, r, w = (dc.randn(g, s, torch.bfloat16) for s in ((5, D), (5, D), (D,)))
    xd, rd = x.cuda(), r.cuda()
    y = torch.empty((5, D), dtype=torch.int8, device="cuda")
    s = torch.empty((5, 1), dtype=torch.float32, device="cuda")
    want = gpu.rms_norm_quantize(xd.clone(), w.cuda(), rd.clone(), output_dtype=gpu.INT8)
    gpu.rms_norm_quantize(xd, w.cuda(), rd, output_dtype=gpu.INT8, out=(y, s, xd if alias == "x" else rd))
    assert torch.equal(y, want[0]) and torch.equal(s, want[1])
    assert torch.equal(xd if alias == "x" else rd, want[2])


@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("to,block", [("int8", 0), ("fp8", 0), ("fp8", 64)])
def test_norm_of_what_is_not_finite(gpu, bad, to, block):
    """The row's scales are NaN and its codes zero; the other rows are as without it."""
    g = dc.gen(5)
    x, w = dc.randn(g, (4, 320), torch.float16), dc.randn(g, (320,), torch.float16)
    code = gpu.INT8 if to == "int8" else gpu.FLOAT8E4M3FN
    want = gpu.rms_norm_quantize(x.cuda(), w.cuda(), None, 1e-5, block, code)
    x[2, 100] = bad
    y, s, _ = gpu.rms_norm_quantize(x.cuda(), w.cuda(), None, 1e-5, block, code)
    # an infinite value makes the others 0: only its own block has a NaN
    if bad != bad:
        assert torch.isnan(s[2]).all() and not y[2].float().any()
    else:
        assert torch.isnan(s[2, 100 // block if block else 0]) and not y[2].float().any()
    keep = [0, 1, 3]
    assert torch.equal(y[keep].view(torch.uint8), want[0][keep].view(torch.uint8)) and torch.equal(s[keep], want[1][keep])


@pytest.mark.parametrize("to", ["int8", "fp8"])
def test_norm_of_zeros_and_tiny_values(gpu, to):
    """Zero rows: zero scale and codes (no division by zero, eps 0 among them: NaN scale); values whose scale is
    below the smallest normal number count as zero."""
    x = torch.zeros((2, 64), dtype=torch.float32, device="cuda")
    x[1] = 1e-38
    w = torch.ones(64, dtype=torch.float32, device="cuda")
    code = gpu.INT8 if to == "int8" else gpu.FLOAT8E4M3FN
    y, s, _ = gpu.rms_norm_quantize(x, w, None, 1e-5, 0, code)
    assert not y[0].float().any() and s[0] == 0
    assert bool(y[1].float().any()) == (float(s[1]) > 0) and (s[1] == 0 or float(s[1]) >= 2.0 ** -126)
    y, s, _ = gpu.rms_norm_quantize(x, w, None, 0.0, 0, code)
    assert torch.isnan(s[0]) and not y[0].float().any()


# ---- MX quantization -------------------------------------------------------------

def check_mx_quantize(gpu, x, to):
    codes, scale = gpu.mx_quantize(x.cuda(), gpu.FLOAT8E4M3FN if to == "fp8" else gpu.FLOAT4E2M1)
    want, ws = dc.mx_quantize(x, to)
    assert torch.equal(scale.cpu(), ws)
    got = codes.cpu().double() if to == "fp8" else dc.unpack4(codes.cpu())
    assert torch.equal(got, want) and torch.equal(torch.signbit(got), torch.signbit(want))


@pytest.mark.parametrize("to", ["fp8", "fp4"])
@pytest.mark.parametrize("typ", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (5, 4096), (2, 3, 160), (700, 64), (1, 11008)])
def test_mx_quantize(gpu, to, typ, shape):
    g = dc.gen(shape[-1])
    x = dc.randn(g, shape, torch.float32) * torch.exp2(torch.randint(-12, 9, (*shape[:-1], 1), generator=g).float())
    check_mx_quantize(gpu, x.to(dc.TYPE[typ]), to)


@pytest.mark.parametrize("to", ["fp8", "fp4"])
def test_mx_quantize_ties_saturation_and_range(gpu, to):
    """Every midpoint of the grid and its neighbours, blocks whose largest value saturates, zero blocks, negative
    zeros and values near both ends of fp32."""
    grid = dc.e4m3_grid() if to == "fp8" else dc.E2M1[:8]
    v = torch.cat((grid, (grid[1:] + grid[:-1]) / 2)).float()
    v = torch.cat((v, torch.nextafter(v, torch.tensor(INF)), -v))
    top = 480.0 if to == "fp8" else 7.5  # rounds above the largest code
    v = torch.nn.functional.pad(v, (0, -len(v) % 31)).reshape(-1, 31)
    x = torch.cat((torch.cat((v, torch.full((len(v), 1), float(grid[-1]))), 1),
                   torch.cat((v[:1], torch.full((1, 1), top)), 1), torch.zeros(1, 32), -torch.zeros(1, 32)))
    x = torch.cat((x, x * 2.0 ** -100, x * 2.0 ** 110 if to == "fp8" else x * 2.0 ** 120, x * 2.0 ** -126))
    check_mx_quantize(gpu, x, to)


@pytest.mark.parametrize("to", ["fp8", "fp4"])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_mx_quantize_of_what_is_not_finite(gpu, to, bad):
    x = dc.randn(dc.gen(2), (2, 96), torch.bfloat16)
    x[1, 40] = bad
    code = gpu.FLOAT8E4M3FN if to == "fp8" else gpu.FLOAT4E2M1
    codes, scale = gpu.mx_quantize(x.cuda(), code)
    bits = codes.view(torch.uint8).cpu()
    assert scale[1, 1] == 255 and (scale.cpu() == 255).sum() == 1
    n = bits.shape[1] // 3
    assert not bits[1, n:2 * n].any()
    x[1, 32:64] = 0
    want, _ = gpu.mx_quantize(x.cuda(), code)
    assert torch.equal(want.view(torch.uint8).cpu(), bits)


# ---- MX product --------------------------------------------------------------------

def check_mx_product(a, a_scale_values, b, bs, got, act):
    """a in 64 bits (codes times scales).  fp32 sums of exact products: K / 128
    roundings and the alignment inside an instruction, bounded by 2^-20 of the
    sum of magnitudes; one rounding of the result.  For E4M3 activations the
    instruction adds the products of 16 consecutive k aligned to the largest of
    them, what is below 2^-13 of it cut off (measured: 2^-13 is kept and 2^-14
    is not; E2M1 products span less than that and lose nothing), so each such
    group may be off by 16 * 2^-13 of its largest product."""
    w = dc.mx_values(dc.unpack4(b), bs)
    a = dc.mx_values(a, a_scale_values)
    want, mass = a @ w.T, a.abs() @ w.abs().T
    bound = dc.ROUND[got.dtype] * want.abs() + 2.0 ** -20 * mass + 2.0 ** -25
    if act == "fp8":
        for k in range(0, a.shape[1], 16):
            top = (a[:, None, k].abs() * w[None, :, k].abs())
            for j in range(k + 1, k + 16):
                torch.maximum(top, a[:, None, j].abs() * w[None, :, j].abs(), out=top)
            bound += 2.0 ** -9 * top
    dc.near(got, want, bound)


MNK = [(1, 1, 32), (1, 16, 128), (1, 4096, 4096), (2, 33, 96), (3, 100, 160), (5, 257, 512), (8, 64, 2080), (16, 48, 1056),
       (17, 130, 544), (33, 259, 1024), (64, 512, 3040), (65, 96, 4128), (127, 129, 256), (130, 300, 1120), (256, 256, 512),
       (300, 1000, 416), (513, 770, 1184), (1, 3, 11008), (31, 2049, 64)]


@pytest.mark.parametrize("M,N,K", MNK)
@pytest.mark.parametrize("act", ["fp8", "fp4"])
@pytest.mark.parametrize("typ", ["bf16", "fp16"])
def test_mx_matmul_quantizes_its_activations(gpu, M, N, K, act, typ):
    g = dc.gen(M * 31 + N + K)
    x = dc.randn(g, (M, K), dc.TYPE[typ])
    b, bs = dc.mx_weight(g, N, K)
    got = gpu.mx_matmul(x.cuda(), b.cuda(), bs.cuda(), a_type=gpu.FLOAT8E4M3FN if act == "fp8" else gpu.FLOAT4E2M1)
    assert got.dtype == x.dtype and got.shape == (M, N)
    check_mx_product(*dc.mx_quantize(x, act), b, bs, got, act)


@pytest.mark.parametrize("M,N,K,act", [(1000, 6100, 96, "fp8"), (1900, 4000, 64, "fp8"), (2000, 4200, 64, "fp4"),
                                       (40, 11300, 96, "fp8"), (61, 7200, 288, "fp8"), (50, 12301, 96, "fp4")])
def test_mx_matmul_of_wide_products(gpu, M, N, K, act):
    """Sizes that take each of the tiles, and wide weights of few rows."""
    g = dc.gen(M + N + K)
    x = dc.randn(g, (M, K), torch.bfloat16)
    b, bs = dc.mx_weight(g, N, K)
    got = gpu.mx_matmul(x.cuda(), b.cuda(), bs.cuda(), a_type=gpu.FLOAT8E4M3FN if act == "fp8" else gpu.FLOAT4E2M1)
    check_mx_product(*dc.mx_quantize(x, act), b, bs, got, act)


@pytest.mark.parametrize("M,N,K", MNK[3:])
@pytest.mark.parametrize("act", ["fp8", "fp4"])
def test_mx_matmul_of_codes(gpu, M, N, K, act):
    """Scales that differ widely from block to block of a row, on both sides."""
    g = dc.gen(M + N * 17 + K)
    b, bs = dc.mx_weight(g, N, K, 110, 140)
    s = torch.randint(110, 140, (M, K // 32), generator=g).to(torch.uint8)
    if act == "fp8":
        codes = (torch.randn((M, K), generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        a = codes.double()
    else:
        codes = torch.randint(0, 256, (M, K // 2), generator=g).to(torch.uint8)
        a = dc.unpack4(codes)
    got = gpu.mx_matmul(codes.cuda(), b.cuda(), bs.cuda(), s.cuda())
    assert got.dtype == torch.bfloat16
    check_mx_product(a, s, b, bs, got, act)


def test_mx_matmul_places_every_value(gpu):
    """One nonzero activation and distinct weights: the k of both operands and the block of both scales."""
    K, N = 416, 48
    g = dc.gen(9)
    b, bs = dc.mx_weight(g, N, K, 100, 150)
    x = torch.diag(torch.ones(K)).to(torch.bfloat16)
    for act in (gpu.FLOAT8E4M3FN, gpu.FLOAT4E2M1):
        for rows in (slice(0, K), slice(100, 108), slice(415, 416)):
            got = gpu.mx_matmul(x[rows].cuda().contiguous(), b.cuda(), bs.cuda(), a_type=act)
            assert torch.equal(got.cpu().double(), dc.mx_values(dc.unpack4(b), bs).T[rows].to(torch.bfloat16).double())


@pytest.mark.parametrize("M", [1, 40, 300])
@pytest.mark.parametrize("act", ["fp8", "fp4"])
def test_mx_matmul_keeps_nan_to_its_row_and_column(gpu, M, act):
    g = dc.gen(M)
    x = dc.randn(g, (M, 256), torch.float16)
    b, bs = dc.mx_weight(g, 70, 256)
    code = gpu.FLOAT8E4M3FN if act == "fp8" else gpu.FLOAT4E2M1
    want = gpu.mx_matmul(x.cuda(), b.cuda(), bs.cuda(), a_type=code)
    x[M // 2, 77] = INF
    bs[33, 2] = 255
    got = gpu.mx_matmul(x.cuda(), b.cuda(), bs.cuda(), a_type=code)
    assert torch.isnan(got[M // 2]).all() and torch.isnan(got[:, 33]).all()
    got[M // 2], got[:, 33] = want[M // 2], want[:, 33]
    assert torch.equal(got, want)


def test_mx_matmul_of_nothing_and_of_rank_3(gpu):
    g = dc.gen(1)
    b, bs = dc.mx_weight(g, 20, 64)
    assert gpu.mx_matmul(torch.empty((0, 64), dtype=torch.float16, device="cuda"), b.cuda(), bs.cuda()).shape == (0, 20)
    x = dc.randn(g, (2, 3, 64), torch.bfloat16)
    got = gpu.mx_matmul(x.cuda(), b.cuda(), bs.cuda())
    assert got.shape == (2, 3, 20)
    check_mx_product(*(t.reshape(6, -1) for t in dc.mx_quantize(x, "fp8")), b, bs, got.reshape(6, 20), "fp8")
    zero = torch.empty((3, 0), dtype=torch.float16, device="cuda")
    got = gpu.mx_matmul(zero, torch.empty((5, 0), dtype=torch.uint8, device="cuda"),
                        torch.empty((5, 0), dtype=torch.uint8, device="cuda"))
    assert got.shape == (3, 5) and not got.any()


# ---- cache: append -------------------------------------------------------------------

BATCHES = [([1], [1]), ([1], [200]), ([5], [5]), ([40], [40]), ([33], [100]), ([1, 1, 1, 1], [1, 17, 64, 129]),
           ([0, 3, 0, 1, 0], [7, 3, 0, 33, 100]), ([70, 1, 130, 16], [70, 500, 131, 48]), ([300], [1000]),
           ([2] * 70, [2 + 3 * i for i in range(70)])]


def same(got, want):
    return torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("new,total", BATCHES)
@pytest.mark.parametrize("to,typ,bt,D,H", [("int8", "fp16", 16, 64, 2), ("fp8", "bf16", 64, 128, 3), ("fp8", "fp16", 32, 80, 1),
                                           ("int8", "bf16", 256, 256, 2), ("fp8", "bf16", 16, 16, 8)])
def test_append(gpu, new, total, to, typ, bt, D, H):
    b = dc.Batch(sum(total) + bt, new, total, H, D, bt, to, dc.TYPE[typ], slack=1)
    want = dc.append(b)
    c = gpu.kv_cache_append(b.k.cuda(), b.v.cuda(), b.cache(gpu), *b.index())
    for name in ("k_cache", "v_cache"):
        assert same(getattr(c, name), want[name]), name
    for name in ("k_scale", "v_scale"):
        assert torch.equal(getattr(c, name).cpu(), want[name]), name


@pytest.mark.parametrize("to", ["int8", "fp8"])
def test_append_token_by_token(gpu, to):
    """A block filled by single tokens of growing size: its scale grows and the kept codes follow."""
    D, bt, H = 64, 16, 2
    g = dc.gen(4)
    xs = dc.randn(g, (40, H, D), torch.float32) * torch.exp2(torch.arange(40) / 4.0)[:, None, None]
    b = dc.Batch(1, [1], [40], H, D, bt, to, torch.bfloat16)
    c = b.cache(gpu)
    table, start, _ = b.index()
    for t in range(40):
        b.k, b.v = xs[t:t + 1].to(torch.bfloat16), -xs[t:t + 1].to(torch.bfloat16)
        b.total, b.new = [t + 1], [1]
        want = dc.append(b)
        for n, v in want.items():
            setattr(b, n, v)
        gpu.kv_cache_append(b.k.cuda(), b.v.cuda(), c, table, start,
                            torch.tensor([t + 1], dtype=torch.int32, device="cuda"))
        assert same(c.k_cache, want["k_cache"]) and same(c.v_cache, want["v_cache"]), t
        assert torch.equal(c.k_scale.cpu(), want["k_scale"]) and torch.equal(c.v_scale.cpu(), want["v_scale"]), t


@pytest.mark.parametrize("to", ["int8", "fp8"])
def test_append_of_zeros_and_of_what_is_not_finite(gpu, to):
    b = dc.Batch(3, [2, 2], [2, 20], 2, 64, 16, to, torch.float16)
    b.k[:2] = 0           # a fresh block of zeros: scale 0
    b.v[3, 1, 5] = NAN    # the second sequence, head 1
    want = dc.append(b)
    c = gpu.kv_cache_append(b.k.cuda(), b.v.cuda(), b.cache(gpu), *b.index())
    blk0, blk1 = int(b.table[0, 0]), int(b.table[1, 1])
    assert not c.k_scale[blk0].any() and not c.k_cache[blk0, :, :2].float().any()
    assert torch.isnan(c.v_scale[blk1, 1]) and not c.v_cache[blk1, 1, :, :4].float().any()
    assert same(c.v_cache[blk1, 0], want["v_cache"][blk1, 0]) and same(c.k_cache[blk1], want["k_cache"][blk1])


def test_append_leaves_what_does_not_fit(gpu):
    """Device-resident numbers that do not fit leave their sequence out; the others are appended."""
    b = dc.Batch(8, [2, 2, 2, 2], [20, 20, 20, 20], 2, 64, 16, "fp8", torch.bfloat16)
    good = dc.append(b)
    c = b.cache(gpu)
    table, start, lengths = b.index()
    table[0, 1] = 10 ** 6                                   # outside the cache
    lengths[1] = 1                                          # fewer than the new tokens
    lengths[2] = 16 * table.shape[1] + 1                    # past the table
    gpu.kv_cache_append(b.k.cuda(), b.v.cuda(), c, table, start, lengths)
    used = b.table[3, :2].tolist()
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        got, was = getattr(c, name).cpu(), getattr(b, name)
        for blk in range(len(was)):
            assert same(got[blk], good[name][blk] if blk in used else was[blk]), (name, blk)


# ---- cache: attention ------------------------------------------------------------------

def check_attention(gpu, b, scale=None, max_query=0, cache=None):
    scale_ = b.D ** -0.5 if scale is None else scale
    got = gpu.kv_cache_attention(b.q.cuda(), cache or b.cache(gpu), *b.index(), scale, max_query)
    out, mass, mag = dc.attention(b, scale_)
    dc.near(got, out, dc.attention_bound(out, mass, mag, b.q.dtype))
    return got


@pytest.mark.parametrize("new,total", BATCHES)
@pytest.mark.parametrize("to,typ,bt,D,H,group", [("int8", "fp16", 16, 64, 2, 4), ("fp8", "bf16", 64, 128, 1, 8),
                                                 ("fp8", "fp16", 32, 80, 2, 5), ("int8", "bf16", 128, 256, 1, 1),
                                                 ("fp8", "bf16", 16, 16, 3, 3), ("int8", "fp16", 256, 128, 1, 20)])
@pytest.mark.parametrize("hint", [False, True])
def test_attention(gpu, new, total, to, typ, bt, D, H, group, hint):
    b = dc.Batch(sum(total) + D, new, total, H, D, bt, to, dc.TYPE[typ], heads=H * group, slack=2)
    check_attention(gpu, b, max_query=max(new) if hint else 0)


@pytest.mark.parametrize("D", list(range(16, 257, 16)))
@pytest.mark.parametrize("new,total", [([1, 2], [70, 300]), ([150], [210])])
def test_attention_head_dims(gpu, D, new, total):
    check_attention(gpu, dc.Batch(D, new, total, 2, D, 32, "fp8", torch.bfloat16, heads=4))


@pytest.mark.parametrize("total", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000, 5000])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_attention_lengths(gpu, total, new):
    if new <= total:
        check_attention(gpu, dc.Batch(total, [new], [total], 2, 128, 16, "int8", torch.float16, heads=8), max_query=new)


@pytest.mark.parametrize("new", [1, 60])
def test_attention_long(gpu, new):
    """Long enough that the work on one sequence is split many ways."""
    check_attention(gpu, dc.Batch(1, [new], [40000], 1, 64, 64, "fp8", torch.bfloat16, heads=2))


@pytest.mark.parametrize("new,total", [([1, 2, 1], [5, 90, 257]), ([50, 20], [50, 300])])
def test_attention_ignores_what_is_past_the_length(gpu, new, total):
    """NaN codes past a sequence's last token, NaN scales of blocks it does not use, table entries past its end."""
    b = dc.Batch(6, new, total, 2, 128, 64, "fp8", torch.bfloat16, heads=4, slack=3)
    want = check_attention(gpu, b)
    used = set()
    for i, t in enumerate(total):
        for j in range(-(-t // 64)):
            blk = int(b.table[i, j])
            used.add(blk)
            n = min(t - j * 64, 64)
            b.k_cache.view(torch.uint8)[blk, :, n:] = 0x7f
            b.v_cache.view(torch.uint8)[blk, :, :, n:] = 0xff
        b.table[i, -(-t // 64):] = 10 ** 9 - i
    for blk in set(range(len(b.k_scale))) - used:
        b.k_cache.view(torch.uint8)[blk] = 0x7f
        b.v_cache.view(torch.uint8)[blk] = 0x7f
        b.k_scale[blk] = NAN
        b.v_scale[blk] = INF
    got = gpu.kv_cache_attention(b.q.cuda(), b.cache(gpu), *b.index())
    assert torch.equal(got, want)


@pytest.mark.parametrize("new,total", [([1], [300]), ([40], [300])])
@pytest.mark.parametrize("to", ["int8", "fp8"])
def test_attention_scales_of_any_size(gpu, new, total, to):
    """Block scales from 2^-100 to 2^100 of v, zero scales, and scores so far apart that one token has all the weight."""
    b = dc.Batch(7, new, total, 1, 64, 16, to, torch.bfloat16, heads=2)
    for big in (-100, 100):
        b.v_scale = torch.full_like(b.v_scale, 2.0 ** big)
        got = gpu.kv_cache_attention(b.q.cuda(), b.cache(gpu), *b.index())
        out, mass, mag = dc.attention(b, 0.125)
        dc.near(got, out, dc.attention_bound(out, mass, mag, b.q.dtype))
    b.v_scale = torch.exp2((torch.arange(b.v_scale.numel()) % 7 * 6 - 18).float()).reshape(b.v_scale.shape)
    b.v_scale[int(b.table[0, 2])] = 0
    b.k_scale[int(b.table[0, 3])] = 0
    check_attention(gpu, b)
    check_attention(gpu, b, scale=40.0)
    check_attention(gpu, b, scale=0.0)
    check_attention(gpu, b, scale=-0.3)


@pytest.mark.parametrize("typ", ["fp16", "bf16"])
@pytest.mark.parametrize("new,total", [([1], [100]), ([30], [100])])
def test_attention_queries_of_any_size(gpu, typ, new, total):
    b = dc.Batch(12, new, total, 1, 64, 16, "int8", dc.TYPE[typ], heads=4)
    b.q[:, 0] *= 2.0 ** (14 if typ == "fp16" else 30)
    b.q[:, 1] *= 2.0 ** (-14 if typ == "fp16" else -40)
    b.q[:, 2] = 0
    check_attention(gpu, b)


@pytest.mark.parametrize("new,total", [([2], [100]), ([40], [100])])
def test_attention_keeps_nan_to_its_row(gpu, new, total):
    b = dc.Batch(13, new, total, 2, 128, 16, "fp8", torch.float16, heads=4)
    want = check_attention(gpu, b)
    b.q[1, 2, 7] = NAN
    got = gpu.kv_cache_attention(b.q.cuda(), b.cache(gpu), *b.index())
    assert torch.isnan(got[1, 2]).all()
    got[1, 2] = want[1, 2]
    assert torch.equal(got, want)
    # a block whose values were not finite gives NaN to the rows that see it
    b = dc.Batch(13, new, total, 2, 128, 16, "fp8", torch.float16, heads=4)
    b.v_scale[int(b.table[0, 0]), 1] = NAN
    got = gpu.kv_cache_attention(b.q.cuda(), b.cache(gpu), *b.index())
    assert torch.isnan(got[:, 2:]).all() and torch.equal(got[:, :2], want[:, :2])


@pytest.mark.parametrize("n", [2, 40])
def test_attention_of_what_does_not_fit_is_nan(gpu, n):
    b = dc.Batch(8, [n] * 4, [100] * 4, 2, 64, 16, "fp8", torch.bfloat16, heads=4)
    want = check_attention(gpu, b)
    table, start, lengths = b.index()
    table[0, 3] = -7
    lengths[1] = n - 1
    lengths[2] = 16 * table.shape[1] + 1
    got = gpu.kv_cache_attention(b.q.cuda(), b.cache(gpu), table, start, lengths)
    assert torch.isnan(got[:3 * n]).all() and torch.equal(got[3 * n:], want[3 * n:])


@pytest.mark.parametrize("hint", [1, 20, 50, 10 ** 6])
def test_attention_with_a_wrong_hint(gpu, hint):
    b = dc.Batch(3, [1, 50, 3, 20], [100, 90, 30, 300], 2, 64, 16, "fp8", torch.bfloat16, heads=4)
    check_attention(gpu, b, max_query=hint)


@pytest.mark.parametrize("to", ["int8", "fp8"])
def test_prompt_attention_scales_of_any_size(gpu, to):
    """As above, with enough rows for the kernel of prompts."""
    test_attention_scales_of_any_size(gpu, [100], [300], to)


@pytest.mark.parametrize("typ", ["fp16", "bf16"])
def test_prompt_attention_queries_of_any_size(gpu, typ):
    test_attention_queries_of_any_size(gpu, typ, [60], [160])


def test_prompt_attention_keeps_nan_to_its_row(gpu):
    test_attention_keeps_nan_to_its_row(gpu, [90], [150])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [127, 128, 129, 255, 256, 257, 600])
def test_attention_row_counts(gpu, D, rows):
    """Rows beside the kernels' own counts, one sequence over many pieces."""
    check_attention(gpu, dc.Batch(rows + D, [rows], [rows + 2300], 1, D, 64, "fp8", torch.bfloat16))


@pytest.mark.parametrize("batch", [64, 65, 70, 300])
def test_attention_of_many_sequences(gpu, batch):
    """Single tokens of many sequences, among them prompts, empty sequences and ones without new tokens."""
    new = [(1, 1, 0, 1, 2, 45, 1)[i % 7] for i in range(batch)]
    total = [n + (37 * i) % 210 if n or i % 2 else 0 for i, n in enumerate(new)]
    check_attention(gpu, dc.Batch(batch, new, total, 2, 64, 16, "int8", torch.float16, heads=4))


def test_attention_of_many_sequences_of_which_some_do_not_fit(gpu):
    b = dc.Batch(9, [2] * 70, [50] * 70, 2, 64, 16, "fp8", torch.bfloat16, heads=4)
    want = check_attention(gpu, b)
    table, start, lengths = b.index()
    lengths[3] = 1
    lengths[69] = 16 * table.shape[1] + 1
    got = gpu.kv_cache_attention(b.q.cuda(), b.cache(gpu), table, start, lengths)
    bad = torch.zeros(140, dtype=torch.bool)
    bad[6:8] = bad[138:] = True
    assert torch.isnan(got[bad.cuda()]).all() and torch.equal(got[~bad.cuda()], want[~bad.cuda()])


@pytest.mark.parametrize("new,total", [([1, 2], [70, 9]), ([200, 3], [260, 40])])
def test_attention_leaves_rows_of_no_sequence_alone(gpu, new, total):
    b = dc.Batch(10, new, total, 2, 64, 16, "int8", torch.bfloat16, heads=4)
    want = check_attention(gpu, b)
    table, start, lengths = b.index()
    q = torch.nn.functional.pad(b.q, (0, 0, 0, 0, 3, 5)).cuda()
    out = torch.full_like(q, 7.0)
    gpu.kv_cache_attention(q, b.cache(gpu), table, start + 3, lengths, out=out)
    assert torch.equal(out[3:-5], want) and (out[:3] == 7).all() and (out[-5:] == 7).all()


def test_nothing_to_do(gpu):
    b = dc.Batch(2, [0, 0], [5, 0], 2, 64, 16, "int8", torch.float16, heads=2)
    assert gpu.kv_cache_attention(b.q.cuda(), b.cache(gpu), *b.index()).shape == (0, 2, 64)
    c = gpu.kv_cache_append(b.k.cuda(), b.v.cuda(), b.cache(gpu), *b.index())
    assert same(c.k_cache, b.k_cache)


# ---- together ----------------------------------------------------------------------------

def test_host_tensors_are_staged(gpu):
    b = dc.Batch(21, [3, 20], [40, 60], 2, 64, 16, "int8", torch.float16, heads=4)
    want = gpu.kv_cache_attention(b.q.cuda(), b.cache(gpu), *b.index())
    got = gpu.kv_cache_attention(b.q, b.cache(gpu), *b.index("cpu"))
    assert not got.is_cuda and torch.equal(got, want.cpu())
    x, w = dc.randn(dc.gen(1), (3, 64), torch.float16), torch.ones(64, dtype=torch.float16)
    assert torch.equal(gpu.rms_norm_quantize(x, w)[0].view(torch.uint8),
                       gpu.rms_norm_quantize(x.cuda(), w.cuda())[0].view(torch.uint8).cpu())
    m, ms = dc.mx_weight(dc.gen(2), 30, 64)
    assert torch.equal(gpu.mx_matmul(x, m, ms), gpu.mx_matmul(x.cuda(), m.cuda(), ms.cuda()).cpu())


@pytest.mark.parametrize("new,total", [([1, 1], [300, 70]), ([40, 1], [100, 2000])])
def test_captured_and_on_another_stream(gpu, new, total):
    """Every operator on a stream of its own, captured into a graph and replayed with other work between: the same
    bits as eager calls."""
    b = dc.Batch(17, new, total, 2, 64, 16, "fp8", torch.bfloat16, heads=8)
    g = dc.gen(3)
    T, D = sum(new), 256
    x, w = dc.randn(g, (T, D), torch.bfloat16).cuda(), dc.randn(g, (D,), torch.bfloat16).cuda()
    m, ms = (t.cuda() for t in dc.mx_weight(g, 512, D))
    c, idx, k, v, q = b.cache(gpu), b.index(), b.k.cuda(), b.v.cuda(), b.q.cuda()

    def layer():
        y, s, total_ = gpu.rms_norm_quantize(x, w, x, mx=True)
        p = gpu.mx_matmul(y, m, ms, s)
        gpu.kv_cache_append(k, v, c, *idx)
        return p, total_, gpu.kv_cache_attention(q, c, *idx), gpu.mx_matmul(x, m, ms, a_type=gpu.FLOAT4E2M1)

    want = layer()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = layer()
    side.synchronize()
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = layer()
    for _ in range(3):
        for t in got:
            t.zero_()
        layer()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(got, want))


def test_same_call_same_bits(gpu):
    b = dc.Batch(30, [1] * 5, [900, 10, 3000, 77, 1500], 2, 128, 64, "int8", torch.float16, heads=16)
    c, idx, q = b.cache(gpu), b.index(), b.q.cuda()
    first = gpu.kv_cache_attention(q, c, *idx)
    assert all(torch.equal(gpu.kv_cache_attention(q, c, *idx), first) for _ in range(5))
