"""Timed cases of the operators that carry a quantized decoder layer from its
joint projection to the next token: positions, the gated feed-forward and the
choice of the token, when a language model is served on one MI355X.

A case is a dict of plain values whose "kind" names the operator:

  tables  cosine and sine tables of rotary positions, plain or scaled for
          contexts longer than a model was trained on
  rope    rotary positions of queries or keys: half and interleaved pairs, all
          or part of a head, the layouts of the ONNX operator and [tokens,
          heads, head_dim]
  append  the joint projection's rows into the paged 8-bit cache: queries
          rotated, keys rotated and quantised, values quantised
  gated   gated feed-forward with MXFP4 weights: both projections, the
          activation and the product
  ffn     the same with MXFP8 output, and the product that takes it back
  sample  a token from logits and given random numbers: temperature, top-k,
          top-p, min-p

``listed()`` names the cases, ``draw(rng)`` draws one more of the same ranges,
``prepare`` / ``run`` make and run one, ``work`` gives the bytes and operations
it cannot do without and ``exact`` the result in 64 bits.  Where ``own`` is
false, ``run`` computes the operator from elementary torch operations in 32
bits (64 for angles and for a token's cumulated weights); where it is true it
makes the library's calls, through the handles that a session keeps per node.
"""
import importlib.util
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

own = False

FP8, FP4 = 17, 23  # ONNX codes of FLOAT8E4M3FN and FLOAT4E2M1
TORCH = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SCALINGS = ["none", "linear", "ntk", "by_parts", "yarn"]  # the library's numbers for them
ACTIVATIONS = ["silu", "gelu", "gelu_tanh", "relu"]       # the same
BASE = 10000.0
TINY = 2.0 ** -126  # a cache scale below the smallest normal number counts as zero


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
        # a session's tables for a short window: the launch is the cost
        {"name": "tables_window", "kind": "tables", "positions": 8192, "rot": 128, "scaling": "none", "factor": 1.0,
         "original": 0},
        # tables of a window 32 times as long as the model was trained on: the memory rate
        {"name": "tables_long", "kind": "tables", "positions": 1000003, "rot": 128, "scaling": "yarn", "factor": 32.0,
         "original": 32768},
        # the queries of 64 sequences decoding
        {"name": "rope_token", "kind": "rope", "layout": "tokens", "batch": 64, "seq": 1, "heads": 32, "D": 128,
         "rot": 128, "interleaved": False, "type": "bf16", "positions": 16384},
        # the ONNX operator on two long prompts, half of each head rotated: the memory rate
        {"name": "rope_prompt", "kind": "rope", "layout": "heads", "batch": 2, "seq": 8191, "heads": 40, "D": 128,
         "rot": 64, "interleaved": True, "type": "fp16", "positions": 16384},
        # 64 sequences decoding: one token each, from the joint projection to the cache
        {"name": "append_token", "kind": "append", "batch": 64, "new": 1, "new_least": 1, "longest": 8192,
         "shortest": 200, "heads": 32, "kv_heads": 8, "D": 128, "rot": 128, "interleaved": False, "block": 16,
         "type": "bf16"},
        # four prompts entering the cache
        {"name": "append_prompt", "kind": "append", "batch": 4, "new": 4096, "new_least": 1500, "longest": 4096,
         "shortest": 1500, "heads": 32, "kv_heads": 8, "D": 128, "rot": 128, "interleaved": False, "block": 64,
         "type": "bf16"},
        # one sequence decoding through the two projections
        {"name": "gated_token", "kind": "gated", "M": 1, "K": 4096, "N": 14336, "type": "bf16", "act": "fp8",
         "activation": "silu"},
        # a decoding batch, ragged in M and N
        {"name": "gated_batch", "kind": "gated", "M": 33, "K": 5120, "N": 13001, "type": "fp16", "act": "fp4",
         "activation": "gelu_tanh"},
        # a prompt of ordinary length through the whole feed-forward block
        {"name": "ffn_prompt", "kind": "ffn", "M": 1000, "K": 4096, "N": 14336, "type": "bf16", "act": "fp8",
         "activation": "silu"},
        # a long prompt through a wide layer: the matrix cores' rate
        {"name": "gated_prompt", "kind": "gated", "M": 4096, "K": 8192, "N": 14336, "type": "bf16", "act": "fp4",
         "activation": "silu"},
        # the next token of one sequence
        {"name": "sample_token", "kind": "sample", "rows": 1, "vocab": 128000, "type": "fp32", "temperature": 0.8,
         "top_k": 50, "top_p": 0.95, "min_p": 0.0, "spread": 3.0, "masked": 0.0},
        # the next tokens of a large batch, no top-k to cut the vocabulary short
        {"name": "sample_batch", "kind": "sample", "rows": 256, "vocab": 131072, "type": "bf16", "temperature": 1.0,
         "top_k": 0, "top_p": 0.9, "min_p": 0.02, "spread": 2.5, "masked": 0.0},
    ]


def _log(rng, lo, hi, step=1):
    """A size from lo to hi, spread over its logarithm, a multiple of step."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step
    return min(max(v, -(-lo // step) * step), hi // step * step)


def draw(rng):
    kind = rng.choice(["tables", "rope", "append", "append", "gated", "gated", "ffn", "sample", "sample", "sample"])
    typ = rng.choice(["bf16", "fp16"])
    if kind == "tables":
        scaling = rng.choice(SCALINGS)
        factor = 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 32.0])
        return {"kind": kind, "positions": _log(rng, 1000, 500000), "rot": rng.choice([32, 64, 80, 128, 256]),
                "scaling": scaling, "factor": factor, "original": rng.choice([4096, 8192, 32768])}
    if kind in ("rope", "append"):
        D = rng.choice([64, 80, 128, 128, 256])
        d = {"kind": kind, "D": D, "rot": rng.choice([D, D, D // 2 // 16 * 16, 32]),
             "interleaved": rng.random() < 0.4, "type": typ}
        if kind == "rope":
            d.update(layout=rng.choice(["tokens", "heads", "joint"]), batch=_log(rng, 1, 16), seq=_log(rng, 1, 4096),
                     heads=rng.choice([1, 4, 8, 24, 32, 40]), positions=8192, type=rng.choice(["bf16", "fp16", "fp32"]))
            while _cost(d) > 5e9:
                d["seq"] = max(1, d["seq"] // 2)
            return d
        d.update(kv_heads=rng.choice([1, 2, 4, 8]), block=rng.choice([16, 32, 64, 128]))
        d["heads"] = d["kv_heads"] * rng.choice([1, 2, 4, 5, 8])
        if rng.random() < 0.5:
            d["batch"], d["new"] = rng.randint(1, 4), _log(rng, 20, 4096)
            d["new_least"] = rng.randint(1, d["new"])
            d["longest"] = d["new"] + _log(rng, 1, 4096)
            d["shortest"] = rng.randint(d["new"], d["longest"])
        else:
            d["batch"], d["new"] = _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 4, 7])
            d["new_least"] = rng.randint(1, d["new"])
            d["longest"] = _log(rng, 16, 8192)
            d["shortest"] = rng.randint(min(d["longest"], 8), d["longest"])
        return d
    if kind in ("gated", "ffn"):
        return {"kind": kind, "M": _log(rng, 1, 4096), "K": _log(rng, 512, 8192, rng.choice([32, 128])),
                "N": _log(rng, 256, 8192, 32 if kind == "ffn" else rng.choice([1, 64])), "type": typ,
                "act": "fp8" if kind == "ffn" else rng.choice(["fp8", "fp4"]), "activation": rng.choice(ACTIVATIONS)}
    return {"kind": kind, "rows": _log(rng, 1, 128), "vocab": _log(rng, 1000, 200000),
            "type": rng.choice(["bf16", "fp16", "fp32"]), "temperature": rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]),
            "top_k": rng.choice([0, 0, 1, 20, 50, 200, 2000]), "top_p": rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]),
            "min_p": rng.choice([0.0, 0.0, 0.02, 0.1]), "spread": rng.choice([1.0, 2.0, 4.0]),
            "masked": rng.choice([0.0, 0.0, 0.5, 0.99])}


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


def _rand(g, shape):
    return torch.rand(shape, generator=g, device="cuda")


def _hidden(g, rows, D, dtype):
    """Hidden states: a few channels far larger than the rest."""
    loud = 1.0 + 20.0 * (_rand(g, (D,)) < 0.01)
    return (torch.randn((rows, D), generator=g, device="cuda") * loud).to(dtype)


def _mx_weight(g, N, K):
    """Codes, two in a byte, and block exponents of weights that keep a product near its input's size."""
    w = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
    s = torch.randint(118, 122, (N, K // 32), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
    return w, s


def _table_inputs(g, positions, rot):
    """Tables as a session holds them, of a base that is each seed's own."""
    base = BASE * (1.0 + float(_rand(g, (1,))))
    f = base ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    a = torch.arange(positions, device="cuda", dtype=torch.float64).unsqueeze(1) * f
    return torch.cos(a).float(), torch.sin(a).float()


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g, kind = _gen(seed), case["kind"]
    dt = TORCH[case["type"]] if "type" in case else None
    if kind == "tables":
        return {"base": BASE * (1.0 + float(_rand(g, (1,))))}
    if kind == "rope":
        B, S, H, D = case["batch"], case["seq"], case["heads"], case["D"]
        shape = {"tokens": (B * S, H, D), "heads": (B, H, S, D), "joint": (B, S, H * D)}[case["layout"]]
        c, s = _table_inputs(g, case["positions"], case["rot"])
        # every sequence from a place of its own on
        first = torch.randint(0, case["positions"] - S + 1, (B, 1), generator=g, device="cuda")
        pos = first + torch.arange(S, device="cuda")
        return {"x": _randn(g, shape, dt), "cos": c, "sin": s,
                "positions": pos.reshape(-1) if case["layout"] == "tokens" else pos}
    if kind == "append":
        return _append_inputs(g, case, dt)
    if kind in ("gated", "ffn"):
        d = {"x": _hidden(g, case["M"], case["K"], dt)}
        d["gate"], d["gate_scale"] = _mx_weight(g, case["N"], case["K"])
        d["up"], d["up_scale"] = _mx_weight(g, case["N"], case["K"])
        if kind == "ffn":
            d["down"], d["down_scale"] = _mx_weight(g, case["K"], case["N"])
        return d
    B, V = case["rows"], case["vocab"]
    x = torch.randn((B, V), generator=g, device="cuda") * case["spread"]
    # a few tokens that the model is for, above the rest
    likely = torch.randint(0, V, (B, 8), generator=g, device="cuda")
    x.scatter_add_(1, likely, (2 + 2 * _rand(g, (B, 8))) * case["spread"])
    if case["masked"]:
        # what a grammar does not allow next; something it always does
        allowed = torch.randint(0, V, (B, 1), generator=g, device="cuda")
        x.masked_fill_((_rand(g, (B, V)) < case["masked"]).scatter_(1, allowed, False), float("-inf"))
    k = case["top_k"]
    # the requests of a batch differ in what they ask for
    return {"x": x.to(dt), "u": _rand(g, (B,)), "temperature": case["temperature"] * (0.5 + _rand(g, (B,))),
            "top_k": (torch.randint(1, k + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if k else None),
            "top_p": 1 - (1 - case["top_p"]) * (0.2 + 0.8 * _rand(g, (B,))) if case["top_p"] < 1 else None,
            "min_p": case["min_p"] * (0.5 + _rand(g, (B,))) if case["min_p"] else None}


def _append_inputs(g, case, dt):
    new, total = _lens(case)
    bt, H, D = case["block"], case["kv_heads"], case["D"]
    need = [-(-t // bt) for t in total]
    blocks = sum(need) + 2
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(need), max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    start = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    scale = [(_rand(g, (blocks, H)) * 0.5 + 0.75) * (3.0 / 448.0) for _ in range(2)]
    codes = [(torch.randn((blocks, H, bt, D), generator=g, device="cuda", dtype=torch.float16) * 120)
             .clamp_(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
    c, s = _table_inputs(g, max(total), case["rot"])
    return {"qkv": _randn(g, (sum(new), case["heads"] + 2 * H, D), dt), "cos": c, "sin": s, "k_cache": codes[0],
            "v_cache": codes[1].view(blocks, H, D, bt), "k_scale": scale[0], "v_scale": scale[1], "table": table,
            "start": start, "lengths": torch.tensor(total, dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if own:
        _handles(case, s)
    return s


def _handles(case, s):
    """The outputs' buffers and the prepared calls that a session keeps per node."""
    pkg, kind = _package(), case["kind"]
    call = s["calls"] = []

    def new(shape, dtype):
        return torch.empty(shape, dtype=dtype, device="cuda")

    if kind == "tables":
        s["out"] = {n: new((case["positions"], case["rot"] // 2), torch.float32) for n in ("cos", "sin")}
        call.append(pkg.prepare("rotary_tables", s["base"], SCALINGS.index(case["scaling"]), case["factor"],
                                case["original"], 32.0, 1.0, 0.0, s["out"]["cos"], s["out"]["sin"]))
    elif kind == "rope":
        s["out"] = {"y": torch.empty_like(s["x"])}
        call.append(pkg.prepare("rotary_embedding", s["x"], s["cos"], s["sin"], s["positions"],
                                int(case["interleaved"]), case["heads"] if case["layout"] == "joint" else 0,
                                s["out"]["y"]))
    elif kind == "append":
        s["q"] = new((s["qkv"].shape[0], case["heads"], case["D"]), s["qkv"].dtype)
        s["out"] = {n: s[n] for n in ("q", "k_cache", "v_cache", "k_scale", "v_scale")}
        call.append(pkg.prepare("rotary_kv_cache_append", s["qkv"], s["cos"], s["sin"], None, int(case["interleaved"]),
                                s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["start"],
                                s["lengths"]))
    elif kind in ("gated", "ffn"):
        M, N, x = case["M"], case["N"], s["x"]
        act = FP8 if case["act"] == "fp8" else FP4
        ffn = kind == "ffn"
        h = new((M, N), torch.float8_e4m3fn if ffn else x.dtype)
        hs = new((M, N // 32), torch.uint8) if ffn else None
        call.append(pkg.prepare("mx_gated_matmul", x, None, act, s["gate"], s["gate_scale"], s["up"], s["up_scale"],
                                ACTIVATIONS.index(case["activation"]), h, hs))
        if ffn:
            y = new((M, case["K"]), x.dtype)
            call.append(pkg.prepare("mx_matmul", h, hs, 0, s["down"], s["down_scale"], y))
        s["out"] = {"y": y if ffn else h}
    else:
        s["out"] = {"token": new((case["rows"],), torch.int64), "probability": new((case["rows"],), torch.float32)}
        call.append(pkg.prepare("sample_tokens", s["x"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"],
                                s["out"]["token"], s["out"]["probability"]))


# ---- one pass ---------------------------------------------------------------

def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        for c in state["calls"]:
            c()
        return state["out"]
    if kind == "tables":
        c, s = _tables(case, state["base"])
        return {"cos": c, "sin": s}
    if kind == "rope":
        return {"y": _rope(state)}
    if kind == "append":
        return _append(state)
    if kind == "sample":
        token, p = _sample(state)
        return {"token": token, "probability": p}
    h = _gated(_mx_values(state["x"].float(), case["act"]), state)
    if kind == "ffn":
        h = _mx_values(h, "fp8") @ _weight(state, "down").t()
    return {"y": h.to(state["x"].dtype)}


def _frequencies(case, base):
    """Angle per position of every pair of dimensions, and what cosine and sine are multiplied by."""
    d, how, s, L = case["rot"], case["scaling"], case["factor"], case["original"]
    i = torch.arange(d // 2, device="cuda", dtype=torch.float64)
    if how == "ntk":  # the base grows, so that the slowest pair turns 1 / s as far
        base = base * s ** (d / (d - 2))
    f = base ** (-2 * i / d)
    if how == "linear":
        return f / s, 1.0
    if how == "by_parts":  # what turns often in L positions stays, what hardly turns is slowed down
        keep = ((L * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return f * keep + f / s * (1 - keep), 1.0
    if how == "yarn":  # the same along the dimensions, and sharper scores
        def at(turns):
            return d * math.log(L / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), d - 1)
        slow = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / s * slow + f * (1 - slow), 0.1 * math.log(s) + 1.0 if s > 1 else 1.0
    return f, 1.0


def _tables(case, base):
    f, m = _frequencies(case, base)
    a = torch.arange(case["positions"], device="cuda", dtype=torch.float64).unsqueeze(1) * f
    return (torch.cos(a) * m).float(), (torch.sin(a) * m).float()


def _rotate(x, c, s, rot, interleaved):
    """x [.., D] in 32 bits, its first rot dimensions turned by tables [.., rot / 2]."""
    r, rest = x[..., :rot], x[..., rot:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rot // 2], r[..., rot // 2:])
    a, b = a * c - b * s, a * s + b * c
    r = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((r, rest), -1)


def _rope(st):
    case, x = st["case"], st["x"]
    c, s = st["cos"][st["positions"]], st["sin"][st["positions"]]
    f = x.float()
    if case["layout"] == "heads":
        c, s = c.unsqueeze(1), s.unsqueeze(1)
    else:
        f = f.unflatten(-1, (case["heads"], case["D"])) if case["layout"] == "joint" else f
        c, s = c.unsqueeze(-2), s.unsqueeze(-2)
    return _rotate(f, c, s, case["rot"], case["interleaved"]).reshape(x.shape).to(x.dtype)


def _inverse(scale):
    return torch.where(scale > 0, 1.0 / scale, 0.0)


def _round8(v):
    return v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _append(st):
    case = st["case"]
    bt, B, H, Hk = case["block"], case["batch"], case["heads"], case["kv_heads"]
    start, length, table = st["start"].long(), st["lengths"].long(), st["table"].long()
    count = start[1:] - start[:-1]
    rows = torch.arange(st["qkv"].shape[0], device="cuda")
    seq = torch.bucketize(rows, start[1:], right=True)
    pos = length[seq] - count[seq] + rows - start[seq]
    f = st["qkv"].float()
    c, s = st["cos"][pos].unsqueeze(1), st["sin"][pos].unsqueeze(1)
    q = _rotate(f[:, :H], c, s, case["rot"], case["interleaved"]).to(st["qkv"].dtype)
    k = _rotate(f[:, H:H + Hk], c, s, case["rot"], case["interleaved"])
    block, off = table[seq, pos // bt], pos % bt
    first = length - count
    head = table[torch.arange(B, device="cuda"), (first // bt).clamp(max=table.shape[1] - 1)]  # the block a sequence goes on in
    keep = (first % bt > 0) & (count > 0)
    old_tokens = torch.arange(bt, device="cuda") < (first % bt).unsqueeze(-1)
    for name, vals in (("k", k), ("v", f[:, H + Hk:])):
        cache, scale = st[name + "_cache"], st[name + "_scale"]
        amax = torch.zeros_like(scale).index_reduce_(0, block, vals.abs().amax(-1), "amax") / 448.0
        carried = torch.zeros_like(scale).index_add_(0, head, scale[head] * keep.unsqueeze(-1))
        fresh = torch.maximum(carried, torch.where(amax < TINY, 0.0, amax))
        touched = torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, block, True)
        ratio = (carried[head] * _inverse(fresh[head]))[:, :, None, None]
        old = cache[head]
        again = _round8(old.float() * ratio)
        kept = (old_tokens & keep.unsqueeze(-1))[:, None, :, None] if name == "k" else \
            (old_tokens & keep.unsqueeze(-1))[:, None, None, :]
        # sequences with no block to go on in put back what they took
        byte = cache.view(torch.uint8)
        byte[head] = torch.where(kept, again.view(torch.uint8), old.view(torch.uint8))
        codes = _round8(vals * _inverse(fresh[block]).unsqueeze(-1)).view(torch.uint8)
        if name == "k":
            byte[block, :, off] = codes
        else:
            byte[block, :, :, off] = codes
        scale.copy_(torch.where(touched.unsqueeze(-1), fresh, scale))
    return dict({n: st[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}, q=q)


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


def _weight(st, name):
    lut = torch.tensor(E2M1, device="cuda")
    w, s = st[name], st[name + "_scale"]
    w = torch.stack((lut[(w & 15).int()], lut[(w >> 4).int()]), -1).flatten(-2)
    return (w.unflatten(-1, (-1, 32)) * torch.exp2(s.float() - 127).unsqueeze(-1)).flatten(-2)


def _gated(a, st):
    g, how = a @ _weight(st, "gate").t(), st["case"]["activation"]
    if how == "silu":
        g = g / (1 + torch.exp(-g))
    elif how == "gelu":
        g = 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    elif how == "gelu_tanh":
        g = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))
    else:
        g = g.clamp(min=0)
    return g * (a @ _weight(st, "up").t())


def _sample(st):
    # in 64 bits: a token's place among cumulated weights, and the border of top-p
    x = st["x"].double()
    # larger logits first, the lower index first among equals
    x, index = torch.sort(x, dim=-1, descending=True, stable=True)
    T = st["temperature"].double().unsqueeze(-1)
    greedy = ~(T > 0)
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, 1.0, T))
    rank = torch.arange(x.shape[1], device="cuda")
    keep = ~greedy | (rank == 0)
    if st["top_k"] is not None:
        keep &= rank < st["top_k"].unsqueeze(-1)
    w = w * keep
    if st["top_p"] is not None:
        upto = torch.cumsum(w, -1)
        before = torch.cat((torch.zeros_like(upto[:, :1]), upto[:, :-1]), -1)
        keep &= before < st["top_p"].double().unsqueeze(-1) * upto[:, -1:]
    if st["min_p"] is not None:
        keep &= w >= st["min_p"].double().unsqueeze(-1)
    w = torch.zeros_like(w).scatter_(1, index, w * keep)
    upto = torch.cumsum(w, -1)
    token = torch.searchsorted(upto, st["u"].double().unsqueeze(-1) * upto[:, -1:], right=True)
    return token.squeeze(-1), (w.gather(1, token) / upto[:, -1:]).float().squeeze(-1)


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "tables":
        n = case["positions"] * case["rot"] // 2
        return {"bytes": 8 * n, "flops": 20 * n}
    if kind == "rope":
        n, size = case["batch"] * case["seq"] * case["heads"] * case["D"], 4 if case["type"] == "fp32" else 2
        # the tables' rows once for each position
        rows = min(case["batch"] * case["seq"], case["positions"])
        return {"bytes": 2 * n * size + rows * case["rot"] * 4 + 8 * case["batch"] * case["seq"],
                "flops": 3 * n * case["rot"] // case["D"]}
    if kind in ("gated", "ffn"):
        M, K, N = case["M"], case["K"], case["N"]
        weights = 3 if kind == "ffn" else 2
        return {"bytes": weights * (N * K // 2 + N * K // 32) + 2 * M * K + 2 * M * (K if kind == "ffn" else N),
                "flops": 2 * weights * M * N * K}
    if kind == "sample":
        n, size = case["rows"] * case["vocab"], 4 if case["type"] == "fp32" else 2
        return {"bytes": n * size + 32 * case["rows"], "flops": 4 * n}
    new, total = _lens(case)
    H, Hk, D, bt = case["heads"], case["kv_heads"], case["D"], case["block"]
    # the joint rows in, queries out in 16 bits, keys and values in 8; the tokens before them in a block gone on
    # in; scales, tables
    old = sum((t - n) % bt for n, t in zip(new, total))
    touched = sum(-(-t // bt) - (t - n) // bt for n, t in zip(new, total))
    rows = min(sum(new), max(total))
    return {"bytes": sum(new) * D * (4 * H + 6 * Hk) + 2 * Hk * (old * D * 2 + touched * 8) + rows * case["rot"] * 4,
            "flops": sum(new) * (3 * (H + Hk) * case["rot"] + 8 * Hk * D)}


# ---- the same in 64 bits ----------------------------------------------------

def _exact8(y):
    """The nearest E4M3 values, ties to even, of finite y."""
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return (torch.round(y / step) * step).clamp(-448, 448)


def _exact_mx(x, act):
    b = x.reshape(-1, 32)
    top = b.abs().max(1, keepdim=True).values
    unit = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -118))) - (8 if act == "fp8" else 2))
    v = b / unit
    if act == "fp8":
        return (_exact8(v.clamp(-448, 448)) * unit).reshape(x.shape)
    g = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    mid = (g[1:] + g[:-1]) / 2
    a = v.abs()
    lo, hi = torch.bucketize(a, mid), torch.bucketize(a, mid, right=True)
    pick = torch.where(lo % 2 == 0, lo, hi)  # on a midpoint lo != hi, and the even code is taken
    return (torch.sign(v) * g[pick] * unit).reshape(x.shape)


def _exact_weight(d, name):
    b, s = d[name], d[name + "_scale"]
    c = torch.stack((b % 16, b // 16), -1).reshape(b.shape[0], -1)
    e, m = (c % 8) // 2, (c % 2).double()
    mag = torch.where(e > 0, torch.exp2(e.double() - 1) * (1 + m / 2), m / 2)
    mag = torch.where(c >= 8, -mag, mag)
    return mag.mul_(torch.exp2(s.double() - 127).repeat_interleave(32, 1))


def _exact_gated(d, case):
    a = _exact_mx(d["x"].double(), case["act"])
    g = a @ _exact_weight(d, "gate").T
    fn = torch.nn.functional
    act = {"silu": fn.silu, "gelu": fn.gelu, "gelu_tanh": lambda v: fn.gelu(v, approximate="tanh"), "relu": fn.relu}
    return act[case["activation"]](g).mul_(a @ _exact_weight(d, "up").T)


def _exact_turn(x, angle_cos, angle_sin, rot, interleaved):
    """x [n, D] in 64 bits as complex numbers times (cos + i sin) [n, rot / 2]."""
    n = x.shape[0]
    y = x.clone()
    pairs = x[:, :rot].reshape(n, rot // 2, 2) if interleaved else x[:, :rot].reshape(n, 2, rot // 2).transpose(1, 2)
    z = torch.view_as_complex(pairs.contiguous()) * torch.complex(angle_cos, angle_sin)
    z = torch.view_as_real(z)
    y[:, :rot] = (z if interleaved else z.transpose(1, 2)).reshape(n, rot)
    return y


def exact(case, seed):
    d, kind = _inputs(case, seed), case["kind"]
    if kind == "tables":
        return _exact_tables(case, d["base"])
    if kind == "rope":
        H, D = case["heads"], case["D"]
        x = d["x"].double()
        x = x.transpose(1, 2) if case["layout"] == "heads" else x
        at = d["positions"].reshape(-1).repeat_interleave(H)
        y = _exact_turn(x.reshape(-1, D), d["cos"][at].double(), d["sin"][at].double(), case["rot"], case["interleaved"])
        if case["layout"] == "heads":
            return {"y": y.reshape(case["batch"], case["seq"], H, D).transpose(1, 2).contiguous()}
        return {"y": y.reshape(d["x"].shape)}
    if kind == "append":
        return _exact_append(case, d)
    if kind == "sample":
        return _exact_sample(case, d)
    h = _exact_gated(d, case)
    return {"y": _exact_mx(h, "fp8") @ _exact_weight(d, "down").T if kind == "ffn" else h}


def _exact_tables(case, base):
    d, s, L, how = case["rot"], case["factor"], case["original"], case["scaling"]
    f, m = [], 1.0
    if how == "yarn":
        m = 1.0 + 0.1 * math.log(s)
        first, last = (d / 2 * math.log(L / (2 * math.pi * turns)) / math.log(base) for turns in (32.0, 1.0))
        first, last = max(0, math.floor(first)), min(d - 1, math.ceil(last))
    for i in range(d // 2):
        plain = math.exp(-2 * i / d * math.log(base))
        if how == "none":
            f.append(plain)
        elif how == "linear":
            f.append(plain / s)
        elif how == "ntk":
            f.append(math.exp(-2 * i / d * (math.log(base) + d / (d - 2) * math.log(s))))
        else:
            if how == "by_parts":
                share = (L / (2 * math.pi / plain) - 1.0) / 31.0
            else:
                share = 1 - (i - first) / (last - first if last > first else 0.001)
            share = min(1.0, max(0.0, share))
            f.append(plain * (share + (1 - share) / s))
    angle = torch.outer(torch.arange(case["positions"], device="cuda").double(),
                        torch.tensor(f, dtype=torch.float64, device="cuda"))
    return {"cos": m * torch.cos(angle), "sin": m * torch.sin(angle)}


def _exact_append(case, d):
    new, total = _lens(case)
    bt, H, Hk, D, rot = case["block"], case["heads"], case["kv_heads"], case["D"], case["rot"]
    out = {n: d[n].double() for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    x = d["qkv"].double()
    out["q"] = torch.empty((x.shape[0], H, D), dtype=torch.float64, device="cuda")
    table, at = d["table"].tolist(), 0
    for i, (n, t) in enumerate(zip(new, total)):
        first = t - n
        turn = [d[name][first:t].double().repeat_interleave(H + Hk, 0) for name in ("cos", "sin")]
        qk = _exact_turn(x[at:at + n, :H + Hk].reshape(-1, D), *turn, rot, case["interleaved"]).reshape(n, H + Hk, D)
        out["q"][at:at + n] = qk[:, :H]
        both = {"k": qk[:, H:], "v": x[at:at + n, H + Hk:]}
        for j in range(first // bt, -(-t // bt)):
            blk, lo, hi = table[i][j], max(first - j * bt, 0), min(t - j * bt, bt)
            for name in "kv":
                y = both[name][j * bt + lo - first:j * bt + hi - first].transpose(0, 1)   # [H, tokens, D]
                cache = out[name + "_cache"][blk]
                cache = cache if name == "k" else cache.transpose(1, 2)                   # a view, [H, bt, D]
                s = out[name + "_scale"][blk]
                was = s.clone() if lo else torch.zeros_like(s)
                now = torch.maximum(was, y.abs().amax((1, 2)) / 448.0)
                if lo:
                    cache[:, :lo] = _exact8(cache[:, :lo] * (was / now)[:, None, None])
                cache[:, lo:hi] = _exact8(y / now[:, None, None])
                s.copy_(now)
        at += n
    return out


def _exact_sample(case, d):
    B, V = case["rows"], case["vocab"]
    token = torch.empty(B, dtype=torch.int64, device="cuda")
    prob = torch.empty(B, dtype=torch.float64, device="cuda")
    T, u = d["temperature"].tolist(), d["u"].tolist()
    k, p, m = ([None] * B if d[n] is None else d[n].tolist() for n in ("top_k", "top_p", "min_p"))
    for b in range(B):
        x = d["x"][b].double()
        if not T[b] > 0:
            token[b], prob[b] = x.argmax(), 1.0
            continue
        w = torch.softmax(x / T[b], 0)
        order = torch.argsort(x, descending=True, stable=True)
        if k[b] is not None:
            order = order[:k[b]]
        if p[b] is not None:
            share = w[order] / w[order].sum()
            order = order[torch.cumsum(share, 0) - share < p[b]]
        if m[b] is not None:
            order = order[w[order] >= m[b] * w.max()]
        order = torch.sort(order).values
        upto = torch.cumsum(w[order], 0)
        at = order[int((upto <= u[b] * upto[-1]).sum())]
        token[b], prob[b] = at, w[at] / upto[-1]
    return {"token": token, "probability": prob}
