"""Timed cases of the 8-bit and 4-bit decoder layer: the operators around the
quantized products when a language model is served on one MI355X.

A case is a dict of plain values whose "kind" names the operator:

  norm    RMS norm with the residual's addition, output in 8 bits with scales
  mx      microscaled 4-bit product: 16-bit activations quantised to blocks of
          32 (MXFP8 or MXFP4) times MXFP4 weights
  normmx  the norm with MXFP8 output, then the product: a layer's input
          projection as it is called
  append  new keys and values into a paged 8-bit cache with one scale for each
          block of tokens and head
  attend  causal attention of the newest tokens over that cache

``listed()`` names the cases, ``draw(rng)`` draws one more of the same ranges,
``prepare`` / ``run`` make and run one, ``work`` gives the bytes and operations
it cannot do without and ``exact`` the result in 64 bits.  Where ``own`` is
false, ``run`` computes the operator from elementary torch operations in 32
bits; where it is true it makes the library's calls, through the handles that
a session keeps per node.
"""
import importlib.util
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

own = False

FP8, FP4 = 17, 23  # ONNX codes of FLOAT8E4M3FN and FLOAT4E2M1
QMAX = {"int8": 127.0, "fp8": 448.0}
TORCH8 = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TORCH16 = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
TINY = 2.0 ** -126  # a scale below the smallest normal number counts as zero


def _package():
    if "onnx_light_amd" not in sys.modules:
        path = os.path.join(ROOT, "onnx-light_amd", "__init__.py")
        spec = importlib.util.spec_from_file_location("onnx_light_amd", path,
                                                      submodule_search_locations=[os.path.dirname(path)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["onnx_light_amd"] = mod
        spec.loader.exec_module(mod)
        mod.init(0)
    return sys.modules["onnx_light_amd"]


# ---- cases ------------------------------------------------------------------

def listed():
    return [
        # one sequence decoding: a single row, where the launch is the cost
        {"name": "norm_token", "kind": "norm", "rows": 1, "D": 4096, "type": "bf16", "residual": True, "to": "fp8",
         "block": 0},
        # a decoding batch with a width that divides by nothing, for the int8 products
        {"name": "norm_batch", "kind": "norm", "rows": 61, "D": 5001, "type": "fp16", "residual": False, "to": "int8",
         "block": 0},
        # a long prompt of a wide model: the memory rate
        {"name": "norm_prompt", "kind": "norm", "rows": 8192, "D": 8192, "type": "bf16", "residual": True, "to": "fp8",
         "block": 128},
        # one sequence decoding through an up projection
        {"name": "mx_token", "kind": "mx", "M": 1, "K": 4096, "N": 14336, "type": "bf16", "act": "fp8"},
        # a decoding batch through a down projection, ragged in M and N
        {"name": "mx_batch", "kind": "mx", "M": 33, "K": 11008, "N": 4099, "type": "fp16", "act": "fp4"},
        # a long prompt through a square projection: the matrix cores' rate
        {"name": "mx_prompt", "kind": "mx", "M": 4096, "K": 8192, "N": 8192, "type": "bf16", "act": "fp4"},
        # a prompt of ordinary length entering a layer: norm, MXFP8 activations, joint projection
        {"name": "layer_input", "kind": "normmx", "M": 1000, "K": 4096, "N": 6144, "type": "bf16"},
        # 64 sequences decoding: one token each into its block
        {"name": "append_token", "kind": "append", "batch": 64, "new": 1, "new_least": 1, "longest": 8192,
         "shortest": 200, "kv_heads": 8, "D": 128, "block": 16, "type": "bf16", "to": "fp8"},
        # four prompts entering the cache
        {"name": "append_prompt", "kind": "append", "batch": 4, "new": 4096, "new_least": 1500, "longest": 4096,
         "shortest": 1500, "kv_heads": 8, "D": 128, "block": 64, "type": "bf16", "to": "fp8"},
        # one sequence decoding over a cache of ordinary length
        {"name": "attend_token", "kind": "attend", "batch": 1, "new": 1, "new_least": 1, "longest": 8191,
         "shortest": 8191, "heads": 32, "kv_heads": 8, "D": 128, "block": 64, "type": "fp16", "to": "int8"},
        # 64 sequences of very different lengths decoding: the memory rate
        {"name": "attend_batch", "kind": "attend", "batch": 64, "new": 1, "new_least": 1, "longest": 16384,
         "shortest": 500, "heads": 64, "kv_heads": 8, "D": 128, "block": 16, "type": "bf16", "to": "fp8"},
        # two chunks of long prompts over what is in the cache already: the matrix cores' rate
        {"name": "attend_prompt", "kind": "attend", "batch": 2, "new": 4096, "new_least": 2048, "longest": 8192,
         "shortest": 5000, "heads": 32, "kv_heads": 8, "D": 128, "block": 64, "type": "bf16", "to": "int8"},
    ]


def _log(rng, lo, hi, step=1):
    """A size from lo to hi, spread over its logarithm, a multiple of step."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step
    return min(max(v, -(-lo // step) * step), hi // step * step)


def draw(rng):
    kind = rng.choice(["norm", "mx", "normmx", "append", "attend", "attend"])
    typ, to = rng.choice(["bf16", "fp16"]), rng.choice(["fp8", "int8"])
    if kind == "norm":
        block = rng.choice([0, 0, 64, 128]) if to == "fp8" else 0
        return {"kind": kind, "rows": _log(rng, 1, 8192), "D": _log(rng, 256, 8192, block or 1), "type": typ,
                "residual": rng.random() < 0.6, "to": to, "block": block}
    if kind in ("mx", "normmx"):
        d = {"kind": kind, "M": _log(rng, 1, 4096), "K": _log(rng, 512, 8192, rng.choice([32, 128])),
             "N": _log(rng, 256, 8192, rng.choice([1, 64])), "type": typ}
        return dict(d, act=rng.choice(["fp8", "fp4"])) if kind == "mx" else d
    d = {"kind": kind, "kv_heads": rng.choice([1, 2, 4, 8]), "D": rng.choice([64, 80, 128, 128, 256]),
         "block": rng.choice([16, 32, 64, 128]), "type": typ, "to": to if kind == "attend" else "fp8"}
    prompt = rng.random() < 0.4
    if prompt:
        d["batch"] = rng.randint(1, 3)
        d["new"] = _log(rng, 20, 2048)
        d["new_least"] = rng.randint(1, d["new"])
        d["longest"] = d["new"] + _log(rng, 1, 4096)
        d["shortest"] = rng.randint(d["new"], d["longest"])
    else:
        d["batch"] = _log(rng, 1, 64)
        d["new"] = rng.choice([1, 1, 1, 2, 4, 7])
        d["new_least"] = rng.randint(1, d["new"])
        d["longest"] = _log(rng, 16, 8192)
        d["shortest"] = rng.randint(min(d["longest"], 8), d["longest"])
    if kind == "attend":
        d["heads"] = d["kv_heads"] * rng.choice([1, 2, 4, 5, 8])
    while _cost(d) > 1e10:  # the largest listed cases'
        d["batch"], d["longest"] = max(1, d["batch"] // 2), max(1, d["longest"] // 2)
        d["new"] = min(d["new"], d["longest"])
        d["new_least"], d["shortest"] = min(d["new_least"], d["new"]), min(d["shortest"], d["longest"])
    return d


def _cost(case):
    """Bytes, or operations where those take longer."""
    w = work(case)
    return max(w["bytes"] * 8, w["flops"] / 50)


def _spread(hi, lo, n, turn):
    """n whole numbers from lo to hi in mixed order, both ends among them."""
    if n == 1:
        return [hi]
    return [hi - (hi - lo) * ((i * turn) % n) // (n - 1) for i in range(n)]


def _turn(n):
    """A step that is coprime to n, so that i * step runs through all of range(n)."""
    return next(t for t in range(max(1, n * 5 // 8), 2 * n + 2) if math.gcd(t, n) == 1)


def _lens(case):
    """(new tokens, tokens in the cache after them) of every sequence."""
    n = case["batch"]
    new = _spread(case["new"], case["new_least"], n, 1)
    total = _spread(case["longest"], case["shortest"], n, _turn(n))
    return new, [max(t, a) for t, a in zip(total, new)]


# ---- inputs -----------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _hidden(g, rows, D, dtype):
    """Hidden states: a few channels far larger than the rest."""
    loud = 1.0 + 20.0 * (torch.rand((D,), generator=g, device="cuda") < 0.01)
    return (torch.randn((rows, D), generator=g, device="cuda") * loud).to(dtype)


def _mx_weight(g, N, K):
    """Codes, two in a byte, and block exponents of weights of moderate size."""
    w = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
    s = torch.randint(118, 124, (N, K // 32), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
    return w, s


def _codes(g, to, shape):
    if to == "int8":
        return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float16) * 120).clamp_(-448, 448).to(TORCH8[to])


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g, kind, dt = _gen(seed), case["kind"], TORCH16[case["type"]]
    if kind == "norm":
        d = {"x": _hidden(g, case["rows"], case["D"], dt), "w": _randn(g, (case["D"],), dt, 0.2) + 1}
        if case["residual"]:
            d["r"] = _hidden(g, case["rows"], case["D"], dt)
        return d
    if kind in ("mx", "normmx"):
        w, s = _mx_weight(g, case["N"], case["K"])
        d = {"x": _hidden(g, case["M"], case["K"], dt), "b": w, "b_scale": s}
        if kind == "normmx":
            d["r"], d["w"] = _hidden(g, case["M"], case["K"], dt), _randn(g, (case["K"],), dt, 0.2) + 1
        return d
    new, total = _lens(case)
    bt, H, D, to = case["block"], case["kv_heads"], case["D"], case["to"]
    need = [-(-t // bt) for t in total]
    blocks = sum(need) + 2
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(need), max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    start = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    k_scale = (torch.rand((blocks, H), generator=g, device="cuda") * 0.5 + 0.75) * (3.0 / QMAX[to])
    v_scale = (torch.rand((blocks, H), generator=g, device="cuda") * 0.5 + 0.75) * (3.0 / QMAX[to])
    d = {"k_cache": _codes(g, to, (blocks, H, bt, D)), "v_cache": _codes(g, to, (blocks, H, D, bt)),
         "k_scale": k_scale, "v_scale": v_scale, "table": table, "start": start,
         "lengths": torch.tensor(total, dtype=torch.int32, device="cuda")}
    if kind == "append":
        d["k"], d["v"] = _randn(g, (sum(new), H, D), dt), _randn(g, (sum(new), H, D), dt)
    else:
        d["q"] = _randn(g, (sum(new), case["heads"], D), dt)
    return d


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if own:
        _handles(case, s)
    return s


def _handles(case, s):
    """The outputs' buffers and the prepared calls that a session keeps per node."""
    pkg, kind, x = _package(), case["kind"], s.get("x")
    call = s["calls"] = []

    def new(shape, dtype):
        return torch.empty(shape, dtype=dtype, device="cuda")

    if kind in ("norm", "normmx"):
        mx = kind == "normmx"
        rows, D = x.shape
        s["y"] = new((rows, D), TORCH8["fp8" if mx else case["to"]])
        s["y_scale"] = new((rows, D // 32), torch.uint8) if mx else new((rows, D // (case["block"] or D)), torch.float32)
        s["sum"] = new((rows, D), x.dtype) if "r" in s else None
        call.append(pkg.prepare("rms_norm_quantize", x, s["w"], s.get("r"), EPS, 32 if mx else case["block"], s["y"],
                                s["y_scale"], s["sum"]))
        if mx:
            s["out"] = new((rows, case["N"]), x.dtype)
            call.append(pkg.prepare("mx_matmul", s["y"], s["y_scale"], 0, s["b"], s["b_scale"], s["out"]))
    elif kind == "mx":
        s["out"] = new((case["M"], case["N"]), x.dtype)
        call.append(pkg.prepare("mx_matmul", x, None, FP8 if case["act"] == "fp8" else FP4, s["b"], s["b_scale"],
                                s["out"]))
    elif kind == "append":
        call.append(pkg.prepare("kv_cache_append", s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"],
                                s["v_scale"], s["table"], s["start"], s["lengths"]))
    else:
        s["out"] = torch.empty_like(s["q"])
        call.append(pkg.prepare("kv_cache_attention", s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                                s["table"], s["start"], s["lengths"], 1.0 / math.sqrt(case["D"]), case["new"],
                                s["out"]))


# ---- one pass ---------------------------------------------------------------

def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        for c in state["calls"]:
            c()
        if kind == "norm":
            q = state["y"]
            if case["to"] == "int8":  # the values that the codes stand for
                q = (q.to(torch.float32) * state["y_scale"]).to(torch.bfloat16)
            return {"y": q, "scale": state["y_scale"], "sum": state["sum"]}
        if kind == "normmx":
            return {"out": state["out"], "sum": state["sum"]}
        if kind == "append":
            return {n: state[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
        return {"out": state["out"]}
    if kind == "norm":
        y, total = _norm(state)
        q, scale = _quantize8(y, case["to"], case["block"] or case["D"])
        if case["to"] == "int8":
            q = (q.to(torch.float32) * scale).to(torch.bfloat16)
        return {"y": q, "scale": scale, "sum": total}
    if kind == "mx":
        return {"out": _mx_product(_mx_values(state["x"].float(), case["act"]), state).to(state["x"].dtype)}
    if kind == "normmx":
        y, total = _norm(state)
        return {"out": _mx_product(_mx_values(y, "fp8"), state).to(state["x"].dtype), "sum": total}
    if kind == "append":
        return _append(state)
    return {"out": _attend(state)}


def _norm(s):
    """x + r rounded to the type, and its RMS norm in 32 bits."""
    h = s["x"] if "r" not in s else (s["x"].float() + s["r"].float()).to(s["x"].dtype)
    f = h.float()
    return f * (1.0 / torch.sqrt(f.square().mean(-1, keepdim=True) + EPS)) * s["w"].float(), h if "r" in s else None


def _inverse(scale):
    return torch.where(scale > 0, 1.0 / scale, 0.0)


def _scales(amax, to):
    s = amax / QMAX[to]
    return torch.where(s < TINY, 0.0, s)


def _round8(v, to):
    v = v.clamp(-QMAX[to], QMAX[to])
    return (v.round() if to == "int8" else v).to(TORCH8[to])


def _quantize8(y, to, block):
    b = y.unflatten(-1, (-1, block))
    scale = _scales(b.abs().amax(-1), to)
    return _round8(b * _inverse(scale).unsqueeze(-1), to).flatten(-2), scale


def _mx_values(x, act):
    """What the codes and block exponents of x stand for: 2^e times the nearest
    E4M3 or E2M1 value, e = floor(log2 of the block's largest) - that type's."""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top)[1] - 1 - (8 if act == "fp8" else 2)).clamp(-127, 127)
    e = torch.where(top > 0, e, -127).float()
    v = b * torch.exp2(-e)
    if act == "fp8":
        v = v.clamp(-448, 448).to(torch.float8_e4m3fn).float()
    else:
        a = v.abs().clamp(max=6.0)
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        v = torch.copysign(torch.round(a / step) * step, v)
    return (v * torch.exp2(e)).flatten(-2)


E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _mx_product(a, s):
    lut = torch.tensor(E2M1, device="cuda")
    w = torch.stack((lut[(s["b"] & 15).int()], lut[(s["b"] >> 4).int()]), -1).flatten(-2)
    w = (w.unflatten(-1, (-1, 32)) * torch.exp2(s["b_scale"].float() - 127).unsqueeze(-1)).flatten(-2)
    return a @ w.t()


def _append(s):
    case = s["case"]
    to, bt, B = case["to"], case["block"], case["batch"]
    start, length, table = s["start"].long(), s["lengths"].long(), s["table"].long()
    count = start[1:] - start[:-1]
    rows = torch.arange(s["k"].shape[0], device="cuda")
    seq = torch.bucketize(rows, start[1:], right=True)
    pos = length[seq] - count[seq] + rows - start[seq]
    block, off = table[seq, pos // bt], pos % bt
    first = length - count
    head = table[torch.arange(B, device="cuda"), (first // bt).clamp(max=table.shape[1] - 1)]  # the block a sequence goes on in
    keep = (first % bt > 0) & (count > 0)
    old_tokens = torch.arange(bt, device="cuda") < (first % bt).unsqueeze(-1)
    for name, vals in (("k", s["k"].float()), ("v", s["v"].float())):
        cache, scale = s[name + "_cache"], s[name + "_scale"]
        amax = torch.zeros_like(scale).index_reduce_(0, block, vals.abs().amax(-1), "amax")
        carried = torch.zeros_like(scale).index_add_(0, head, scale[head] * keep.unsqueeze(-1))
        fresh = torch.maximum(carried, _scales(amax, to))
        touched = torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, block, True)
        ratio = (carried[head] * _inverse(fresh[head]))[:, :, None, None]
        old = cache[head]
        again = _round8(old.float() * ratio, to)
        kept = (old_tokens & keep.unsqueeze(-1))[:, None, :, None] if name == "k" else \
            (old_tokens & keep.unsqueeze(-1))[:, None, None, :]
        # sequences with no block to go on in put back what they took
        byte = cache.view(torch.uint8)
        byte[head] = torch.where(kept, again.view(torch.uint8), old.view(torch.uint8))
        new = _round8(vals * _inverse(fresh[block]).unsqueeze(-1), to).view(torch.uint8)
        if name == "k":
            byte[block, :, off] = new
        else:
            byte[block, :, :, off] = new
        scale.copy_(torch.where(touched.unsqueeze(-1), fresh, scale))
    return {n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}


def _attend(s):
    case = s["case"]
    bt, H, D, B = case["block"], case["kv_heads"], case["D"], case["batch"]
    group = case["heads"] // H
    start, length, table = s["start"].long(), s["lengths"].long(), s["table"].long()
    count = start[1:] - start[:-1]
    most, wide = case["new"], table.shape[1] * bt
    # queries padded to [B, H, group * most, D]
    i = torch.arange(most, device="cuda")
    there = i < count.unsqueeze(-1)
    row = (start[:-1].unsqueeze(-1) + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().unflatten(2, (H, group)).permute(0, 2, 3, 1, 4).reshape(B, H, group * most, D)
    k = s["k_cache"][table].float() * s["k_scale"][table][..., None, None]        # [B, blocks, H, bt, D]
    k = k.permute(0, 2, 4, 1, 3).reshape(B, H, D, wide)
    p = torch.matmul(q, k).mul_(1.0 / math.sqrt(D)).unflatten(2, (group, most))
    del k
    pos = length.unsqueeze(-1) - count.unsqueeze(-1) + i
    seen = (torch.arange(wide, device="cuda") <= pos.unsqueeze(-1)) & there.unsqueeze(-1)  # [B, most, wide]
    p.masked_fill_(~seen[:, None, None], float("-inf"))
    p.sub_(p.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    v = s["v_cache"][table].float() * s["v_scale"][table][..., None, None]        # [B, blocks, H, D, bt]
    v = v.permute(0, 2, 1, 4, 3).reshape(B, H, wide, D)
    v.masked_fill_((torch.arange(wide, device="cuda") >= length.unsqueeze(-1))[:, None, :, None], 0.0)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (group, most)) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, most, H * group, D)
    return o[there].to(s["q"].dtype)


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "norm":
        n = case["rows"] * case["D"]
        scales = case["rows"] * (case["D"] // case["block"] if case["block"] else 1)
        # x, and with a residual that and the sum; one byte out; the weight and the scales
        return {"bytes": n * (7 if case["residual"] else 3) + 2 * case["D"] + 4 * scales, "flops": 6 * n}
    if kind in ("mx", "normmx"):
        M, K, N = case["M"], case["K"], case["N"]
        b = N * K // 2 + N * K // 32 + 2 * M * N + 2 * M * K
        return {"bytes": b + (4 * M * K + 2 * K if kind == "normmx" else 0), "flops": 2 * M * N * K}
    new, total = _lens(case)
    H, D, bt = case["kv_heads"], case["D"], case["block"]
    if kind == "append":
        # the new tokens in 16 bits and out in 8, the tokens before them in a block gone on in, the scales
        old = sum((t - n) % bt for n, t in zip(new, total))
        touched = sum(-(-t // bt) - (t - n) // bt for n, t in zip(new, total))
        return {"bytes": 2 * H * (sum(new) * D * 3 + old * D * 2 + touched * 8), "flops": 2 * sum(new) * H * D * 4}
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))
    blocks = sum(-(-t // bt) for t in total)
    return {"bytes": 2 * sum(total) * H * D + 2 * blocks * H * 4 + 4 * sum(new) * case["heads"] * D,
            "flops": 4 * pairs * case["heads"] * D}


# ---- the same in 64 bits ----------------------------------------------------

def _exact8(y, to):
    """The nearest values of the 8-bit type, ties to even, of finite y in its range."""
    if to == "int8":
        return torch.round(y).clamp(-127, 127)
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return (torch.round(y / step) * step).clamp(-448, 448)


def _exact_scaled(y, to, block):
    shape = y.shape
    y = y.reshape(-1, block)
    scale = y.abs().max(1, keepdim=True).values / QMAX[to]
    code = _exact8(torch.where(scale > 0, y / scale, torch.zeros_like(y)), to)
    return code.reshape(shape), scale.reshape(*shape[:-1], -1), (code * scale).reshape(shape)


def _exact_norm(d):
    x = d["x"].double()
    if "r" in d:
        x = (x + d["r"].double()).to(d["x"].dtype).double()
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * d["w"].double(), x


def _exact_mx(x, act):
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    b = x.reshape(-1, 32)
    top = b.abs().max(1, keepdim=True).values
    unit = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -140))) - (8 if act == "fp8" else 2))
    v = b / unit
    if act == "fp8":
        return (_exact8(v.clamp(-448, 448), "fp8") * unit).reshape(x.shape)
    g = torch.tensor(grid, dtype=torch.float64, device=x.device)
    mid = (g[1:] + g[:-1]) / 2
    a = v.abs()
    lo, hi = torch.bucketize(a, mid), torch.bucketize(a, mid, right=True)
    pick = torch.where(lo % 2 == 0, lo, hi)  # on a midpoint lo != hi, and the even code is taken
    return (torch.sign(v) * g[pick] * unit).reshape(x.shape)


def _exact_weight(d):
    c = torch.stack((d["b"] % 16, d["b"] // 16), -1).reshape(d["b"].shape[0], -1).int()
    e, m = (c % 8) // 2, (c % 2).double()
    mag = torch.where(e > 0, torch.exp2(e.double() - 1) * (1 + m / 2), m / 2)
    mag = torch.where(c >= 8, -mag, mag)
    return mag * torch.exp2(d["b_scale"].double() - 127).repeat_interleave(32, 1)


def exact(case, seed):
    d, kind = _inputs(case, seed), case["kind"]
    if kind == "norm":
        y, h = _exact_norm(d)
        code, scale, value = _exact_scaled(y, case["to"], case["block"] or case["D"])
        return {"y": value if case["to"] == "int8" else code, "scale": scale, "sum": h if "r" in d else None}
    if kind == "mx":
        return {"out": _exact_mx(d["x"].double(), case["act"]) @ _exact_weight(d).T}
    if kind == "normmx":
        y, h = _exact_norm(d)
        return {"out": _exact_mx(y, "fp8") @ _exact_weight(d).T, "sum": h}
    if kind == "append":
        return _exact_append(case, d)
    return {"out": _exact_attend(case, d)}


def _exact_append(case, d):
    new, total = _lens(case)
    bt, to = case["block"], case["to"]
    out = {n: d[n].double() for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    table, at = d["table"].tolist(), 0
    for i, (n, t) in enumerate(zip(new, total)):
        first = t - n
        for j in range(first // bt, -(-t // bt)):
            blk, lo, hi = table[i][j], max(first - j * bt, 0), min(t - j * bt, bt)
            rows = slice(at + j * bt + lo - first, at + j * bt + hi - first)
            for name in "kv":
                x = d[name][rows].double().transpose(0, 1)                          # [H, tokens, D]
                cache = out[name + "_cache"][blk]
                cache = cache if name == "k" else cache.transpose(1, 2)             # a view, [H, bt, D]
                s = out[name + "_scale"][blk]
                was = s.clone() if lo else torch.zeros_like(s)
                now = torch.maximum(was, x.abs().amax((1, 2)) / QMAX[to])
                if lo:
                    cache[:, :lo] = _exact8(cache[:, :lo] * (was / now)[:, None, None], to)
                cache[:, lo:hi] = _exact8(x / now[:, None, None], to)
                s.copy_(now)
        at += n
    return out


def _exact_attend(case, d):
    new, total = _lens(case)
    H, D = case["kv_heads"], case["D"]
    group = case["heads"] // H
    out = torch.empty(d["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, t) in enumerate(zip(new, total)):
        blk = d["table"][i, :-(-t // case["block"])].long()
        late = torch.arange(t, device="cuda") > torch.arange(t - n, t, device="cuda").unsqueeze(1)
        for h in range(H):
            k = (d["k_cache"][blk, h].double() * d["k_scale"][blk, h].double()[:, None, None]).reshape(-1, D)[:t]
            v = (d["v_cache"][blk, h].double() * d["v_scale"][blk, h].double()[:, None, None]).transpose(1, 2)
            v = v.reshape(-1, D)[:t]
            for j in range(h * group, (h + 1) * group):
                w = d["q"][at:at + n, j].double() @ k.T / math.sqrt(D)
                out[at:at + n, j] = torch.softmax(w.masked_fill(late, float("-inf")), -1) @ v
        at += n
    return out
