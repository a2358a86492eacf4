"""A decoding step's operators together, from a token's row to the next token, and calls of
them at the ends of what they take."""
import importlib.util
import os

import pytest
import torch

import token_step_cases as ts
from test_gpu_sample import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu(olamd):
    olamd.init(0)
    return olamd


@pytest.fixture(scope="module")
def ex():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decoder_layer.py")
    spec = importlib.util.spec_from_file_location("decoder_layer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


class Step:
    """A step of a layer and a vocabulary on tensors that stay where they are."""

    def __init__(self, gpu, ex, layer, words, held, new, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.layer, self.words, self.most = layer, words, max(new)
        s = layer.shape
        self.sequences = ex.Sequences(gpu, s, len(new), 256)
        self.cache = self.sequences.cache
        for t in self.cache.tensors():
            t.view(torch.uint8).zero_()
        self.table, start, lengths = self.sequences.grow(held)
        filled = torch.randn((sum(held), s.hidden), generator=g, device="cuda").bfloat16()
        layer.step(filled, self.cache, self.table, start, lengths, max(held))
        self.start = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
        # room for the steps to come, whose blocks are in the table from the start
        self.table, _, _ = self.sequences.grow([120 - h for h in held])
        self.lengths = torch.tensor([h + n for h, n in zip(held, new)], dtype=torch.int32, device="cuda")
        self.ids = torch.randint(0, len(words.rows), (sum(new),), generator=g, device="cuda")
        self.uniform = torch.rand(len(new), generator=g, device="cuda")
        self.rules = [torch.full((len(new),), v, dtype=t, device="cuda")
                      for v, t in ((0.9, torch.float32), (40, torch.int32), (0.9, torch.float32), (0.01, torch.float32))]

    def __call__(self):
        y = self.layer.step(self.words.rows[self.ids], self.cache, self.table, self.start, self.lengths, self.most)
        return (y, *self.words.next(y, self.start, self.uniform, *self.rules))

    def on(self, token, seed):
        """To the next step."""
        self.lengths += (self.start[1:] - self.start[:-1])
        self.ids.copy_(token.repeat_interleave((self.start[1:] - self.start[:-1]).long()))
        self.uniform.copy_(torch.rand(len(self.uniform), generator=torch.Generator().manual_seed(seed)))

    def state(self):
        return [t.view(torch.uint8).clone() for t in self.cache.tensors()]

    def back(self, state):
        for t, s in zip(self.cache.tensors(), state):
            t.view(torch.uint8).copy_(s)


def captured(step, side):
    with torch.cuda.stream(side):
        step()
        step()  # (again, which is the same: its tokens are in the cache, at their scales)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    return graph, out


def test_captured_steps_go_on_as_eager_ones(gpu, ex):
    """Two graphs, one of single tokens, one of a few a sequence, share a workspace; each
    replay is the eager step's, with eager work and the other graph's between."""
    shape = ex.Shape(hidden=512, heads=8, kv_heads=2, head_dim=64, inner=736)
    layer = ex.DecoderLayer(gpu, shape, ex.random_weights(shape), 256)
    words = ex.Vocabulary(gpu, 512, 70000)  # rows of it are shared by workgroups
    steps = [Step(gpu, ex, layer, words, [5, 64, 33], [1, 1, 1], 1), Step(gpu, ex, layer, words, [40, 1], [7, 2], 2)]
    side = torch.cuda.Stream()
    before = [s.state() for s in steps]
    graphs = [captured(s, side) for s in steps]
    for s, b in zip(steps, before):
        s.back(b)
    for i in range(4):
        eager = []
        for s in steps:
            was = s.state()
            eager.append((*(t.clone() for t in s()), s.state()))
            s.back(was)
        for (graph, out), s, (y, token, prob, after) in zip(graphs, steps, eager):
            for t in out:
                t.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.isfinite(y.float()).all() and (token >= 0).all() and (token < 70000).all()
            for got, want in zip((*out, *s.state()), (y, token, prob, *after)):
                assert torch.equal(got, want), i
            s.on(token, i)
    assert not torch.equal(steps[0].state()[0], before[0][0])


def test_drawn_tokens_are_the_definitions(gpu, ex):
    """The logits of the layer's outputs, and the token of the definition in 64 bits."""
    shape = ex.Shape(hidden=256, heads=4, kv_heads=4, head_dim=64, inner=512)
    layer = ex.DecoderLayer(gpu, shape, ex.random_weights(shape), 256)
    words = ex.Vocabulary(gpu, 256, 5001)
    s = Step(gpu, ex, layer, words, [9, 100], [3, 1], 3)
    y, token, prob = s()
    logits = gpu.mx_matmul(y[[2, 3]].contiguous(), *words.w).cpu().double()
    for b in range(2):
        want, p = ts.sample(logits[b].numpy(), s.uniform[b].item(), *(r[b].item() for r in s.rules))
        assert token[b].item() == want and abs(prob[b].item() - p) <= 2.0 ** -22 * p


def test_generate_runs_and_repeats(gpu, ex):
    shape = ex.Shape(hidden=256, heads=4, kv_heads=2, head_dim=64, inner=512)
    layer = ex.DecoderLayer(gpu, shape, ex.random_weights(shape))
    words = ex.Vocabulary(gpu, 256, 1000)
    a, b = (ex.generate(layer, words, [[1, 2, 3], [999], list(range(70))], 5, seed=4) for _ in range(2))
    assert a == b and [len(t) for t in a] == [5, 5, 5] and all(0 <= t < 1000 for row in a for t in row)


# ---- rows shared by workgroups, and the largest vocabulary --------------------------------

@pytest.mark.parametrize("rows", [1, 15, 16, 17])
@pytest.mark.parametrize("typ", [torch.float32, torch.bfloat16])
def test_shared_rows_with_long_lists(gpu, rows, typ):
    """A spread of nearly nothing puts all tokens into a few bins: no list has room, and the
    border goes by the logits' bits; a top_k above what the threads' largest logits say."""
    x, u = ts.randn_logits(5, rows, 66001, typ, spread=1e-3)
    check(gpu, x, u, top_k=600)
    check(gpu, x, u, top_p=0.5)
    check(gpu, x, u, 1.0, 20000, 0.7, 0.999)
    x, u = ts.randn_logits(6, rows, 66001, typ, spread=4.0)
    check(gpu, x, u, top_k=513)
    check(gpu, x, u, 1.0, 5000, 0.99)


@pytest.mark.parametrize("rows", [2, 17])
def test_shared_rows_that_ask_for_different_things(gpu, rows):
    x, u = ts.randn_logits(7, rows, 80000, torch.bfloat16)
    x[0] = float("-inf")
    x[1, 100:] = torch.finfo(torch.bfloat16).min
    r = torch.arange(rows)
    T = torch.where(r % 5 == 2, torch.zeros(rows), 0.5 + r / rows)
    k, p = torch.tensor([0, 7, 512, 513, 1, 90000, -3] * 3)[:rows], torch.tensor([0.9, 1.0, 0.3, 0.0, 2.0] * 4)[:rows]
    check(gpu, x, u, T, k, p, torch.tensor([0.0, 0.2, -1.0] * 6)[:rows])


@pytest.mark.parametrize("rows", [1, 17])
@pytest.mark.parametrize("typ", [torch.float32, torch.bfloat16])
def test_largest_vocabulary(gpu, rows, typ):
    x, u = ts.randn_logits(8, rows, 2 ** 21 - 1, typ)
    check(gpu, x, u)
    check(gpu, x, u, 0.8, 50, 0.95)
    check(gpu, x, u, top_p=0.9)


def test_no_rows(gpu):
    empty = torch.empty(0, device="cuda")
    token, prob = gpu.sample_tokens(torch.empty(0, 1000, device="cuda"), empty, empty)
    assert token.shape == (0,) and prob.shape == (0,)
