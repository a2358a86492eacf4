"""Edges of the decoder-layer operators on the GPU, against plain implementations in 64 bits: rows beside blocks that
are not in the cache, values at the ends of fp32, sizes past one launch, a query_start that falls."""
import pytest
import torch

import decoder_cases as dc
from test_gpu_decoder import check_norm, same

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def gpu(olamd):
    olamd.init(0)
    return olamd


# ---- attention beside a block outside the cache ---------------------------------

@pytest.mark.parametrize("new,blocks", [(5, 2), (5, 70), (150, 0), (700, 3)])
@pytest.mark.parametrize("to,typ,D,bt", [("fp8", "bf16", 64, 16), ("fp8", "fp16", 128, 64), ("fp8", "bf16", 80, 32),
                                         ("fp8", "bf16", 256, 128), ("int8", "fp16", 128, 16)])
@pytest.mark.parametrize("bad", [-7, 10 ** 9])
def test_rows_before_a_bad_block_are_as_without_it(gpu, new, blocks, to, typ, D, bt, bad):
    """The last block of a sequence is outside the cache.  Rows that see a token of it are NaN, and those before are
    right, whatever block 0 of the cache holds (NaN codes and scales here, as memory that nobody wrote may)."""
    total = (-(-new // bt) + blocks) * bt + 3
    b = dc.Batch(new + D, [new], [total], 2, D, bt, to, dc.TYPE[typ], heads=4)
    spare = next(i for i in range(1, len(b.k_scale)) if i not in b.table)
    b.table[b.table == 0] = spare
    out, mass, mag = dc.attention(b, D ** -0.5)
    for t in (b.k_cache, b.v_cache):
        t.view(torch.uint8)[0] = 0x7f
    b.k_scale[0], b.v_scale[0] = NAN, INF
    table, start, lengths = b.index()
    table[0, -1] = bad
    got = gpu.kv_cache_attention(b.q.cuda(), b.cache(gpu), table, start, lengths)
    before = new - 3  # the three tokens of the last block come last
    dc.near(got[:before], out[:before], dc.attention_bound(out, mass, mag, b.q.dtype)[:before])
    assert torch.isnan(got[before:]).all()


# ---- sizes past one launch (2^32 threads) ------------------------------------------

def test_norm_of_more_rows_than_a_launch_takes(gpu):
    rows = 2 ** 26 + 3
    x = torch.randn((rows, 1), dtype=torch.float16, device="cuda")
    w = torch.ones(1, dtype=torch.float16, device="cuda")
    y, s, _ = gpu.rms_norm_quantize(x, w, output_dtype=gpu.INT8)
    for part in range(0, rows, 2 ** 24):
        rows_of = slice(part, min(rows, part + 2 ** 24))
        want = gpu.rms_norm_quantize(x[rows_of], w, output_dtype=gpu.INT8)
        assert torch.equal(y[rows_of], want[0]) and torch.equal(s[rows_of], want[1])


def test_mx_product_with_more_columns_than_a_launch_takes(gpu):
    N = 2 ** 27 + 40
    x = dc.randn(dc.gen(1), (1, 32), torch.bfloat16).cuda()
    b = torch.randint(0, 256, (N, 16), dtype=torch.uint8, device="cuda")
    s = torch.randint(118, 124, (N, 1), dtype=torch.uint8, device="cuda")
    y = gpu.mx_matmul(x, b, s)
    for part in range(0, N, 2 ** 25):
        cols = slice(part, min(N, part + 2 ** 25))
        assert torch.equal(y[:, cols], gpu.mx_matmul(x, b[cols], s[cols]))


# ---- a query_start that falls -----------------------------------------------------------

@pytest.mark.parametrize("start", [[0, 9, 2, 4, 6], [0, 2, 100, 4, 8], [0, 8, 0, 8, 8], [8, 6, 4, 2, 0], [-3, 2, 4, 1, 8]])
@pytest.mark.parametrize("n", [2, 40])
def test_a_falling_query_start_stays_inside(gpu, start, n):
    """Which results such a batch gives is not said, but it reads and writes nothing beyond its rows and blocks: blocks
    of the cache that its table does not name and rows past `tokens` stay as they are."""
    b = dc.Batch(8, [2 * n] * 4, [3 * n + 20] * 4, 2, 64, 16, "fp8", torch.bfloat16, heads=4)
    start = torch.tensor(start, dtype=torch.int32) * n
    tokens = 8 * n
    c = b.cache(gpu)
    table, _, lengths = b.index()
    k, v, q = b.k[:tokens].cuda(), b.v[:tokens].cuda(), b.q[:tokens].cuda()
    out = torch.full((tokens + 64, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    gpu.kv_cache_attention(q, c, table, start.cuda(), lengths, out=out[:tokens])
    gpu.kv_cache_append(k, v, c, table, start.cuda(), lengths)
    assert (out[tokens:] == 7).all()
    free = [i for i in range(len(b.k_scale)) if i not in b.table]
    assert len(free) == 3
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        assert same(getattr(c, name)[free], getattr(b, name)[free]), name


# ---- values at the ends of fp32 ------------------------------------------------------------

@pytest.mark.parametrize("D", [64, 1000, 4096, 16384, 20011])
@pytest.mark.parametrize("typ", ["bf16", "fp32"])
@pytest.mark.parametrize("size,eps", [(1e20, 1e-5), (1e25, 1e-5), (3e36, 0.0), (1e-25, 0.0), (1e-33, 0.0), (1e-20, 1e-30)])
def test_norm_of_rows_whose_squares_leave_fp32(gpu, D, typ, size, eps):
    """Sums of squares above fp32's largest number and below its smallest, in rows beside ordinary ones."""
    g = dc.gen(D)
    x, r = dc.randn(g, (5, D), dc.TYPE[typ]), dc.randn(g, (5, D), dc.TYPE[typ])
    x[1::2] *= size
    r[1::2] *= size
    w = dc.randn(g, (D,), torch.float32)
    check_norm(gpu, x, w, r, "fp8", 0, eps=eps)
    check_norm(gpu, x, w, None, "int8", 0, eps=eps)
    if D % 32 == 0:
        check_norm(gpu, x, w, r, "int8", 32, eps=eps)
        check_norm(gpu, x, w, r, "fp8", 32, mx=True, eps=eps)


@pytest.mark.parametrize("new,total", [([1], [1]), ([1], [100]), ([2, 1], [700, 9]), ([150], [150]), ([150], [700])])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_attention_of_scores_near_the_ends_of_fp32(gpu, new, total, sign):
    """Every token of the cache has one key, so every weight is the same, at scores of 2^104 to 2^110 in size."""
    b = dc.Batch(3, new, total, 1, 64, 16, "int8", torch.bfloat16, heads=2)
    b.k_cache[:], b.k_scale[:], b.v_scale[:] = 64, 1.0, 2.0 ** -7
    b.q[:] = sign * 2.0 ** 95
    b.q[:, 1] *= 2.0 ** 6
    got = gpu.kv_cache_attention(b.q.cuda(), b.cache(gpu), *b.index(), 0.125)
    at = 0
    for i, (n, t) in enumerate(zip(new, total)):
        blk = b.table[i, :-(-t // 16)].long()
        v = (b.v_cache[blk].double() * 2.0 ** -7).permute(1, 0, 3, 2).reshape(-1, 64)[:t]
        for j in range(n):
            seen = v[:t - n + j + 1]
            want, mass = seen.mean(0), seen.abs().mean(0)
            for h in range(2):
                dc.near(got[at + j, h], want, dc.ROUND[torch.bfloat16] * want.abs() + 2.0 ** -10 * mass + 2.0 ** -24)
        at += n


# ---- a cache past 4 GB ------------------------------------------------------------------------

@pytest.mark.parametrize("new", [3, 200])
@pytest.mark.parametrize("H,bt,D", [(8, 64, 128), (4, 256, 64)])
def test_cache_whose_offsets_pass_32_bits(gpu, new, H, bt, D):
    """Blocks on both sides of 2^32 bytes, appended to and attended over: as in a small cache."""
    total = new + 5 * bt + 7
    b = dc.Batch(new, [new], [total], H, D, bt, "fp8", torch.bfloat16, heads=2 * H)
    line = 2 ** 32 // (H * bt * D)
    blocks = line + len(b.k_scale)
    order = torch.arange(b.table.shape[1], dtype=torch.int32) * (1 - 2 * (torch.arange(b.table.shape[1]) % 2)) + line
    big = gpu.KvCache(blocks, H, bt, D)
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        small, large = getattr(b, name).cuda(), getattr(big, name)
        large.view(torch.uint8).fill_(0x7f)
        for i in range(b.table.shape[1]):
            large[int(order[i])] = small[int(b.table[0, i])]
    c, (table, start, lengths) = b.cache(gpu), b.index()
    far = order.to(torch.int32)[None].cuda()
    k, v, q = b.k.cuda(), b.v.cuda(), b.q.cuda()
    gpu.kv_cache_append(k, v, c, table, start, lengths)
    gpu.kv_cache_append(k, v, big, far, start, lengths)
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        for i in range(b.table.shape[1]):
            assert same(getattr(big, name)[int(order[i])], getattr(c, name)[int(b.table[0, i])].cpu()), (name, i)
    assert torch.equal(gpu.kv_cache_attention(q, big, far, start, lengths),
                       gpu.kv_cache_attention(q, c, table, start, lengths))
