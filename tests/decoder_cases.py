"""Plain implementations, in 64 bits on the CPU, of the decoder-layer operators
(RMS norm with 8-bit output, MX quantization and product, paged 8-bit cache and
its attention), and builders of their inputs."""
import numpy as np
import torch

QMAX = {"int8": 127.0, "fp8": 448.0}
CODE = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
# half a unit in the last place, relative, of a result rounded once
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                    dtype=torch.float64)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


# ---- RMS norm ----------------------------------------------------------------

def norm(x, weight, residual, eps):
    """(v, h): h = x + residual rounded to x's type, v its norm in 64 bits."""
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    f = h.double()
    return f / torch.sqrt((f * f).mean(-1, keepdim=True) + eps) * weight.double(), h


def half_step(code, to):
    """Half the distance from |code| to the next larger code (fp8: 3 bits of
    fraction, subnormal steps of 2^-9)."""
    if to == "int8":
        return torch.full_like(code, 0.5)
    a = code.abs().clamp(min=2.0 ** -6)
    return torch.exp2(torch.floor(torch.log2(a)) - 4)


# ---- MX ------------------------------------------------------------------------

def mx_quantize(x, to):
    """(codes as values in 64 bits, E8M0 bytes) of finite x [.., K]: the nearest
    code found by searching the type's grid."""
    emax, top_code = (8, 448.0) if to == "fp8" else (2, 6.0)
    b = x.double().reshape(-1, 32)
    top = b.abs().max(1, keepdim=True).values
    e = torch.where(top > 0, torch.floor(torch.log2(top)), torch.tensor(-1000.0, dtype=torch.float64)) - emax
    # log2 may round up to the next whole number: compare with the power itself
    e = torch.where((top > 0) & (torch.exp2(e + emax) > top), e - 1, e).clamp(min=-127)
    v = b / torch.exp2(e)
    grid = e4m3_grid() if to == "fp8" else E2M1[:8]
    mid = (grid[1:] + grid[:-1]) / 2
    a = v.abs().clamp(max=top_code)
    lo, hi = torch.bucketize(a, mid), torch.bucketize(a, mid, right=True)
    q = grid[torch.where(lo % 2 == 0, lo, hi)]  # even code on a midpoint
    return torch.copysign(q, v).reshape(x.shape), (e + 127).to(torch.uint8).reshape(*x.shape[:-1], -1)


def e4m3_grid():
    c = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn)
    return c.double()


def unpack4(codes):
    """Values of packed E2M1 codes [.., K / 2]."""
    c = codes.to(torch.int64)
    return E2M1[torch.stack((c & 15, c >> 4), -1).flatten(-2)]


def mx_values(values, scale):
    return (values.reshape(-1, 32) * torch.exp2(scale.double().reshape(-1, 1) - 127)).reshape(values.shape)


def mx_weight(g, N, K, lo=118, hi=124):
    return (torch.randint(0, 256, (N, K // 2), generator=g).to(torch.uint8),
            torch.randint(lo, hi, (N, K // 32), generator=g).to(torch.uint8))


# ---- cache -----------------------------------------------------------------------

class Batch:
    """A cache with random contents and a batch of sequences over it: counts of
    new tokens and lengths with them."""

    def __init__(self, seed, new, total, kv_heads, D, bt, to, dtype, heads=None, slack=0, spare=3):
        g = gen(seed)
        self.new, self.total, self.H, self.D, self.bt, self.to = list(new), list(total), kv_heads, D, bt, to
        need = [-(-t // bt) for t in total]
        blocks = sum(need) + spare
        order = torch.randperm(blocks, generator=g).to(torch.int32)
        self.table = torch.full((len(need), max(need + [0]) + slack), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.start = torch.tensor([sum(self.new[:i]) for i in range(len(self.new) + 1)], dtype=torch.int32)
        self.lengths = torch.tensor(total, dtype=torch.int32)
        T = sum(self.new)
        if to == "int8":
            code = lambda s: torch.randint(-127, 128, s, generator=g).to(torch.int8)  # noqa: E731
        else:
            code = lambda s: (torch.randn(s, generator=g) * 120).clamp(-448, 448).to(torch.float8_e4m3fn)  # noqa: E731
        self.k_cache, self.v_cache = code((blocks, kv_heads, bt, D)), code((blocks, kv_heads, D, bt))
        self.k_scale = (torch.rand((blocks, kv_heads), generator=g) + 0.5) * (2.0 / QMAX[to])
        self.v_scale = (torch.rand((blocks, kv_heads), generator=g) + 0.5) * (2.0 / QMAX[to])
        self.k, self.v = randn(g, (T, kv_heads, D), dtype), randn(g, (T, kv_heads, D), dtype)
        self.q = randn(g, (T, heads or kv_heads, D), dtype)

    def cache(self, olamd):
        c = olamd.KvCache.__new__(olamd.KvCache)
        c.k_cache, c.v_cache = self.k_cache.cuda(), self.v_cache.cuda()
        c.k_scale, c.v_scale = self.k_scale.cuda(), self.v_scale.cuda()
        return c

    def index(self, where="cuda"):
        return tuple(t.to(where) for t in (self.table, self.start, self.lengths))


def code8(v, to):
    """Codes of fp32 values, as the definition rounds them (ties to even)."""
    v = v.clamp(-QMAX[to], QMAX[to])
    return v.round().to(torch.int8) if to == "int8" else v.to(torch.float8_e4m3fn)


def append(b):
    """k_cache, v_cache, k_scale, v_scale after the append, in the definition's
    own fp32 steps (one division for the scale, one for its inverse, one
    product a value): every implementation of them has the same bits."""
    out = {n: getattr(b, n).clone() for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    for i, (n, t) in enumerate(zip(b.new, b.total)):
        first, at = t - n, int(b.start[i])
        for j in range(first // b.bt, -(-t // b.bt)) if n else ():
            blk = int(b.table[i, j])
            lo, hi = max(first - j * b.bt, 0), min(t - j * b.bt, b.bt)
            for name in "kv":
                x = getattr(b, name)[at + j * b.bt + lo - first:at + j * b.bt + hi - first].float().transpose(0, 1)
                c = out[name + "_cache"][blk]
                c = c if name == "k" else c.transpose(1, 2)
                s = out[name + "_scale"][blk]
                top = x.abs().amax((1, 2)) / torch.tensor(QMAX[b.to])
                top = torch.where(top < 2.0 ** -126, torch.zeros_like(top), top)
                now = torch.maximum(s, top) if lo else top
                inv = torch.where(now > 0, 1.0 / now, torch.zeros_like(now))[:, None, None]
                if lo:
                    again = code8(c[:, :lo].float() * (s[:, None, None] * inv), b.to)
                    c[:, :lo] = torch.where((now != s)[:, None, None], again.float(), c[:, :lo].float()).to(CODE[b.to])
                c[:, lo:hi] = code8(x * inv, b.to)
                s.copy_(now)
    return out


def attention(b, scale, q=None):
    """(out, bound) in 64 bits: bound[t, h, d] is the sum of p |v|, and the
    largest of sum |q||k| * scale, what errors are measured by."""
    q = (b.q if q is None else q).double()
    out, mass = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros(q.shape[:2], dtype=torch.float64)
    group = q.shape[1] // b.H
    for i, (n, t) in enumerate(zip(b.new, b.total)):
        if not n:
            continue
        rows = slice(int(b.start[i]), int(b.start[i]) + n)
        blk = b.table[i, :-(-t // b.bt)].long()
        k = (b.k_cache[blk].double() * b.k_scale[blk].double()[..., None, None]).transpose(0, 1).reshape(b.H, -1, b.D)
        v = (b.v_cache[blk].double() * b.v_scale[blk].double()[..., None, None]).permute(1, 0, 3, 2)
        k, v = k[:, :t], v.reshape(b.H, -1, b.D)[:, :t]
        late = torch.arange(t) > torch.arange(t - n, t)[:, None]
        for h in range(q.shape[1]):
            z = (q[rows, h] @ k[h // group].T * scale).masked_fill(late, float("-inf"))
            p = torch.softmax(z, -1)
            out[rows, h], mass[rows, h] = p @ v[h // group], p @ v[h // group].abs()
            mag[rows, h] = (q[rows, h].abs() @ k[h // group].abs().T * abs(scale)).masked_fill(late, 0).amax(-1)
    return out, mass, mag


def attention_bound(out, mass, mag, dtype):
    """What a kernel may be off by.  Its weights are rounded to 11 bits (2^-11)
    and the exponential, its argument's rounding and the division add no more
    than that again; the fp32 score of D <= 256 products of exact factors is
    off by at most 2^-20 of sum |q||k|, which the exponential turns into the
    same relative error of a weight; the result is rounded once."""
    return ROUND[dtype] * out.abs() + (2.0 ** -10 + 2.0 ** -20 * mag[..., None]) * mass + 2.0 ** -24


def near(got, want, bound):
    """Asserts |got - want| <= bound everywhere (64 bits)."""
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} values off; worst {float((off / bound).max()):.3g} of "
                           f"the bound at {np.unravel_index(int((off / bound).argmax()), tuple(off.shape))}")
