"""Plain implementations, in 64 bits on the CPU, of the operators from a layer's
joint projection to the next token (rotary positions, gated feed-forward,
sampling), and how far a kernel may be from them."""
import math

import numpy as np
import torch

import decoder_cases as dc

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


# ---- rotary positions ------------------------------------------------------------

def frequencies(d, base, scaling="none", s=1.0, original=0, fast=32.0, slow=1.0):
    """(angle per position of every pair, the tables' magnitude) by the header's
    formulas, one pair after the other."""
    f = []
    for i in range(d // 2):
        plain = base ** (-2 * i / d)
        if scaling == "none":
            f.append(plain)
        elif scaling == "linear":
            f.append(plain / s)
        elif scaling == "ntk":
            f.append((base * s ** (d / (d - 2))) ** (-2 * i / d))
        else:
            if scaling == "by_parts":
                k = (original * plain / (2 * math.pi) - slow) / (fast - slow)
            else:
                lo, hi = (d * math.log(original / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (fast, slow))
                lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), d - 1)
                k = 1 - (i - lo) / (hi - lo if hi - lo > 0.001 else 0.001)
            k = min(max(k, 0.0), 1.0)
            f.append(plain * k + plain / s * (1 - k))
    return f, 0.1 * math.log(s) + 1 if scaling == "yarn" else 1.0


def tables(positions, f, m=1.0):
    angle = torch.outer(torch.arange(positions, dtype=torch.float64), torch.tensor(f, dtype=torch.float64))
    return m * torch.cos(angle), m * torch.sin(angle)


def rotate(x, c, s, interleaved):
    """(y, size) in 64 bits: x [n, D], tables [n, d / 2]; size = |a c| + |b s| of every
    value, what an fp32 sum of the two products may be off by 2^-23 of."""
    x, c, s = x.double(), c.double(), s.double()
    d = 2 * c.shape[-1]
    i = torch.arange(d // 2)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, d // 2 + i)
    y, size = x.clone(), torch.zeros_like(x)
    a, b = x[:, ia], x[:, ib]
    y[:, ia], y[:, ib] = a * c - b * s, a * s + b * c
    size[:, ia], size[:, ib] = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
    return y, size


def rotate_bound(y, size, dtype):
    """Two products and a sum in fp32, rounded once to the type (a subnormal half by
    2^-25)."""
    return HALF_STEP[dtype] * y.abs() + 2.0 ** -23 * size + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -140)


# ---- gated feed-forward ------------------------------------------------------------

def activate(g, kind):
    if kind == "silu":
        return g / (1 + torch.exp(-g))
    if kind == "gelu":
        return 0.5 * g * torch.erfc(-g * math.sqrt(0.5))
    if kind == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
    return g.clamp(min=0)


def product(a, w, act):
    """(a w^T, what a kernel's fp32 sum may be off by): as check_mx_product of the plain
    product has it, without the rounding of the result."""
    off = 2.0 ** -20 * (a.abs() @ w.abs().T)
    if act == "fp8":
        for k in range(0, a.shape[1], 16):
            top = torch.zeros_like(off)
            for j in range(k, k + 16):
                torch.maximum(top, a[:, None, j].abs() * w[None, :, j].abs(), out=top)
            off += 2.0 ** -9 * top
    return a @ w.T, off


def gated(a, gate, up, act, activation):
    """(h, bound before the result's rounding).  No activation's slope is above 1.13;
    its own fp32 steps are a few ulps, and those of an exponent of size up to g^2."""
    (g, eg), (u, eu) = product(a, gate, act), product(a, up, act)
    f = activate(g, activation)
    ef = 1.13 * eg + 2.0 ** -19 * (1 + g * g) * f.abs()
    return f * u, ef * (u.abs() + eu) + f.abs() * eu


# ---- sampling ------------------------------------------------------------------------

def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability) of one row of logits (a sequence of floats), by the
    definition, in 64 bits."""
    x = np.asarray(x, dtype=np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    if not (x > -np.inf).any():
        return -1, 0.0
    order = np.lexsort((np.arange(len(x)), -x))
    if not temperature > 0:
        return int(order[0]), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        d = np.where(x == x.max(), 0.0, (x.max() - x) / temperature)
    d = np.where(np.isnan(d), np.inf, d)  # beside an infinite logit, at an infinite temperature
    w = np.where(x > -np.inf, np.exp(-d), 0.0)
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        upto = np.cumsum(w[order])
        before = np.concatenate(([0.0], upto[:-1]))
        keep = before < max(top_p, 0.0) * upto[-1]
        keep[0] = True
        order = order[keep]
    if min_p > 0:
        order = order[w[order] >= min(min_p, 1.0)]
    order = np.sort(order)
    upto = np.cumsum(w[order])
    u = min(u, 1 - 2.0 ** -24) if u > 0 else 0.0
    at = int(np.searchsorted(upto, u * upto[-1], side="right"))
    return int(order[at]), float(w[order[at]] / upto[-1])


def randn_logits(seed, rows, vocab, dtype, spread=3.0, masked=0.0):
    g = dc.gen(seed)
    x = torch.randn((rows, vocab), generator=g) * spread
    if masked:
        x.masked_fill_(torch.rand((rows, vocab), generator=g) < masked, float("-inf"))
        x[:, vocab // 2] = 0.0
    return x.to(dtype), torch.rand(rows, generator=g)
