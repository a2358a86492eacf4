"""A decoder layer with MXFP4 weights, MXFP8 activations and an 8-bit paged
cache: two prompts of different lengths enter it, then both sequences go on one
token at a time, each token drawn from the logits of the one before.

    python examples/decoder_layer.py [--hidden 2048] [--prompt 700] [--tokens 8]

The quantized products, plain and gated, the norms, the rotation by position, the
cache and its attention, and the choice of a token are the framework's; the sum
behind the layer and the embeddings' lookup are torch's.
Prints how far the outputs are from the same layer in 64 bits on the CPU, and on
a GPU the time of a step.
"""
from __future__ import annotations

import argparse
import importlib.util
import math
import os
import sys
import time

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load():
    """The framework's package (its folder's name is no Python name)."""
    if "onnx_light_amd" not in sys.modules:
        path = os.path.join(ROOT, "onnx-light_amd", "__init__.py")
        spec = importlib.util.spec_from_file_location("onnx_light_amd", path)
        sys.modules["onnx_light_amd"] = module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
    return sys.modules["onnx_light_amd"]


class Shape:
    def __init__(self, hidden=2048, heads=16, kv_heads=4, head_dim=128, inner=5632):
        self.hidden, self.heads, self.kv_heads, self.head_dim, self.inner = hidden, heads, kv_heads, head_dim, inner

    def matrices(self) -> dict:
        """Rows and columns of the weights: every product is x @ w^T."""
        rows = (self.heads + 2 * self.kv_heads) * self.head_dim
        return {"qkv": (rows, self.hidden), "o": (self.hidden, self.heads * self.head_dim),
                "gate_up": (2 * self.inner, self.hidden), "down": (self.hidden, self.inner)}


def random_weights(shape: Shape, seed=0) -> dict:
    """bfloat16 weights on the CPU, scaled so that a product keeps its input's size."""
    g = torch.Generator().manual_seed(seed)
    w = {n: (torch.randn(s, generator=g) / math.sqrt(s[1])).bfloat16() for n, s in shape.matrices().items()}
    for n in ("norm1", "norm2"):
        w[n] = (1 + 0.1 * torch.randn(shape.hidden, generator=g)).bfloat16()
    return w


def rotate(x, positions):
    """Rotates pairs of dimensions (i, i + D / 2) of x [tokens, heads, D] by
    position * 10000^(-2 i / D): the plain layer's form of the rotary tables."""
    half = x.shape[-1] // 2
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    turn = positions.to(wide)[:, None] * 10000.0 ** (-torch.arange(half, device=x.device, dtype=wide) / half)
    c, s = torch.cos(turn)[:, None], torch.sin(turn)[:, None]
    a, b = x[..., :half].to(wide), x[..., half:].to(wide)
    return torch.cat([a * c - b * s, a * s + b * c], -1).to(x.dtype)


class Sequences:
    """The paged cache of a batch: blocks are handed out as sequences grow."""

    def __init__(self, ola, shape: Shape, batch: int, longest: int, block_tokens=64, dtype=None):
        self.ola, self.block_tokens = ola, block_tokens
        self.most = -(-longest // block_tokens)
        self.cache = ola.KvCache(batch * self.most, shape.kv_heads, block_tokens, shape.head_dim,
                                 ola.FLOAT8E4M3FN if dtype is None else dtype)
        self.free = list(range(batch * self.most))
        self.table = torch.zeros((batch, self.most), dtype=torch.int32)
        self.held = [0] * batch     # blocks of each sequence
        self.length = [0] * batch   # tokens of each sequence

    def grow(self, new):
        """Room for new[b] tokens of every sequence: (block_table, query_start,
        lengths) on the GPU."""
        for b, n in enumerate(new):
            self.length[b] += n
            while self.held[b] * self.block_tokens < self.length[b]:
                self.table[b, self.held[b]] = self.free.pop()
                self.held[b] += 1
        start = [sum(new[:b]) for b in range(len(new) + 1)]
        return (self.table.cuda(), torch.tensor(start, dtype=torch.int32, device="cuda"),
                torch.tensor(self.length, dtype=torch.int32, device="cuda"))


class DecoderLayer:
    """Weights, and tables of positions for sequences of up to `longest` tokens."""

    def __init__(self, ola, shape: Shape, weights: dict, longest=8192):
        self.ola, self.shape = ola, shape
        self.tables = ola.rotary_tables(longest, shape.head_dim)  # cos, sin
        self.norm1, self.norm2 = weights["norm1"].cuda(), weights["norm2"].cuda()
        self.w = {n: ola.mx_quantize(weights[n].cuda(), ola.FLOAT4E2M1) for n in shape.matrices()}
        # codes and scales of the gate's rows, then of those it is multiplied by
        self.gate, self.up = zip(*(t.split(shape.inner) for t in self.w["gate_up"]))

    def dense(self) -> dict:
        """The weights that the quantized ones stand for, in 64 bits on the CPU."""
        values = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
        out = {"norm1": self.norm1.cpu().double(), "norm2": self.norm2.cpu().double()}
        for n, (codes, scales) in self.w.items():
            c = codes.cpu()
            c = torch.stack([c & 15, c >> 4], -1).flatten(-2).long()
            v = values[c & 7] * (1 - 2 * (c >> 3).double())
            out[n] = v * torch.exp2(scales.cpu().double() - 127).repeat_interleave(32, -1)
        return out

    def norm(self, x, weight, residual=None):
        y, scale, total = self.ola.rms_norm_quantize(x, weight, residual, mx=True)
        return y, scale, x if residual is None else total

    def product(self, name, a, a_scale=None):
        return self.ola.mx_matmul(a, *self.w[name], a_scale, output_dtype=torch.bfloat16)

    def __call__(self, x, sequences: Sequences, new):
        """x bfloat16 [tokens, hidden], the new[b] new tokens of sequence b one
        sequence after the other."""
        return self.step(x, sequences.cache, *self.grow(sequences, new), max(new))

    def grow(self, sequences: Sequences, new):
        """Sequences.grow inside the tables of positions: lengths on the GPU are not checked
        against them by the library, and a position outside makes NaN."""
        if max(held + n for held, n in zip(sequences.length, new)) > len(self.tables[0]):
            raise ValueError(f"a sequence has more tokens than the layer's {len(self.tables[0])} positions")
        return sequences.grow(new)

    def step(self, x, cache, table, start, lengths, most):
        """The same on the GPU alone; no sequence has more than `most` new tokens."""
        s, ola = self.shape, self.ola
        y, scale, x = self.norm(x, self.norm1)
        qkv = self.product("qkv", y, scale).view(len(x), -1, s.head_dim)
        q = ola.rotary_kv_cache_append(qkv, *self.tables, cache, table, start, lengths)
        o = ola.kv_cache_attention(q, cache, table, start, lengths, max_query=most)
        o = self.product("o", o.view(len(x), -1))  # 16-bit rows, quantized by the product
        y, scale, x = self.norm(o, self.norm2, x)  # x + o, and its norm
        h, h_scale = ola.mx_gated_matmul(y, *self.gate, *self.up, a_scale=scale, mx=True)
        return x + self.product("down", h, h_scale)


class Vocabulary:
    """Embeddings of tokens, and from the layer's outputs the next ones."""

    def __init__(self, ola, hidden: int, size=32000, seed=2):
        g = torch.Generator().manual_seed(seed)
        self.ola = ola
        self.rows = torch.randn((size, hidden), generator=g).bfloat16().cuda()
        head = torch.randn((size, hidden), generator=g).mul_(2 * hidden ** -0.5).bfloat16()
        self.w = ola.mx_quantize(head.cuda(), ola.FLOAT4E2M1)

    def next(self, y, start, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
        """(token, probability) after each sequence's last row of y."""
        logits = self.ola.mx_matmul(y[start[1:].long() - 1], *self.w)
        return self.ola.sample_tokens(logits, uniform, temperature, top_k, top_p, min_p)


def plain_layer(shape: Shape, w: dict, x, length: int):
    """The layer in 64 bits for one sequence: x [length, hidden] from position 0."""
    def norm(h, weight):
        return h * weight / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-5)

    x = x.double()
    qkv = (norm(x, w["norm1"]) @ w["qkv"].T).view(length, -1, shape.head_dim)
    q, k, v = qkv.split([shape.heads, shape.kv_heads, shape.kv_heads], 1)
    at = torch.arange(length)
    group = shape.heads // shape.kv_heads
    q, k, v = rotate(q, at), rotate(k, at).repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    p = torch.stack([q[:, h] @ k[:, h].T for h in range(shape.heads)]) * shape.head_dim ** -0.5
    p = p.masked_fill(at[None, :] > at[:, None], -math.inf).softmax(-1)
    o = torch.stack([p[h] @ v[:, h] for h in range(shape.heads)], 1).reshape(length, -1)
    x = x + o @ w["o"].T
    gate, up = (norm(x, w["norm2"]) @ w["gate_up"].T).chunk(2, -1)
    return x + (torch.nn.functional.silu(gate) * up) @ w["down"].T


def run(ola, shape: Shape, prompts, tokens: int, dtype=None, seed=0):
    """Runs prompts and then `tokens` single tokens of every sequence; returns the
    layer, the inputs and the outputs of each sequence in order of position."""
    layer = DecoderLayer(ola, shape, random_weights(shape, seed), max(prompts) + tokens)
    g = torch.Generator().manual_seed(seed + 1)
    inputs = [torch.randn(n + tokens, shape.hidden, generator=g).bfloat16() for n in prompts]
    sequences = Sequences(ola, shape, len(prompts), max(prompts) + tokens, dtype=dtype)
    outputs = [[] for _ in prompts]
    y = layer(torch.cat([x[:n] for x, n in zip(inputs, prompts)]).cuda(), sequences, list(prompts))
    for b, part in enumerate(y.split(list(prompts))):
        outputs[b].append(part.cpu())
    for t in range(tokens):
        y = layer(torch.stack([x[n + t] for x, n in zip(inputs, prompts)]).cuda(), sequences, [1] * len(prompts))
        for b in range(len(prompts)):
            outputs[b].append(y[b:b + 1].cpu())
    return layer, inputs, [torch.cat(o) for o in outputs]


def generate(layer: DecoderLayer, words: Vocabulary, prompts, tokens: int, seed=0):
    """Lets prompts (lists of tokens) go on by `tokens` drawn ones each, at temperature
    0.8 of the 50 likeliest and 95 % of their weight; returns the drawn tokens."""
    batch = len(prompts)
    g = torch.Generator(device="cuda").manual_seed(seed)
    rules = (torch.full((batch,), 0.8, device="cuda"), torch.full((batch,), 50, dtype=torch.int32, device="cuda"),
             torch.full((batch,), 0.95, device="cuda"))
    sequences = Sequences(layer.ola, layer.shape, batch, max(map(len, prompts)) + tokens)
    ids, new, drawn = torch.tensor(sum(prompts, []), device="cuda"), [len(p) for p in prompts], []
    for _ in range(tokens):
        table, start, lengths = layer.grow(sequences, new)
        y = layer.step(words.rows[ids], sequences.cache, table, start, lengths, max(new))
        ids, _ = words.next(y, start, torch.rand(batch, generator=g, device="cuda"), *rules)
        drawn.append(ids)
        new = [1] * batch
    return torch.stack(drawn, 1).tolist() if drawn else [[] for _ in prompts]


def error(layer: DecoderLayer, x, y) -> float:
    """How far y is from the layer in 64 bits, of what the layer adds to x (root
    mean squares)."""
    want = plain_layer(layer.shape, layer.dense(), x, len(x))
    return float((y.double() - want).square().mean().sqrt() / (want - x.double()).square().mean().sqrt())


def main():
    a = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    a.add_argument("--hidden", type=int, default=2048)
    a.add_argument("--prompt", type=int, default=700)
    a.add_argument("--tokens", type=int, default=8)
    a = a.parse_args()
    ola = load()
    ola.init(0)
    shape = Shape(hidden=a.hidden)
    prompts = [a.prompt, max(1, a.prompt // 3)]
    layer, inputs, outputs = run(ola, shape, prompts, a.tokens)
    for b, (x, y) in enumerate(zip(inputs, outputs)):
        print(f"sequence {b}: {prompts[b]} tokens of prompt and {a.tokens} single ones, "
              f"error {error(layer, x, y):.3f} of what the layer adds")
    words = Vocabulary(ola, shape.hidden)
    for b, drawn in enumerate(generate(layer, words, [[i % len(words.rows) for i in range(n)] for n in prompts], a.tokens)):
        print(f"sequence {b} goes on with tokens {drawn}")
    for name, new in (("prompt", prompts), ("token", [1] * len(prompts))):
        x = torch.randn(sum(new), shape.hidden, device="cuda").bfloat16()
        times = []
        for _ in range(6):
            sequences = Sequences(ola, shape, len(new), max(new))
            torch.cuda.synchronize()
            t = time.perf_counter()
            layer(x, sequences, new)
            torch.cuda.synchronize()
            times.append(time.perf_counter() - t)
        print(f"{name} step of {sum(new)} tokens: {sorted(times)[2] * 1e6:.0f} us")


if __name__ == "__main__":
    main()
