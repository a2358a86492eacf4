"""The example of a decoder layer: its operators together, prompts first, then
single tokens, against the layer in 64 bits."""
import importlib.util
import math
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("decoder_layer", os.path.join(ROOT, "examples", "decoder_layer.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_rotation_keeps_lengths_and_depends_on_distance():
    ex = example()
    x, y = torch.randn(2, 3, 1, 16, dtype=torch.float64).unbind(0)
    at = torch.tensor([0, 5, 900])
    a = ex.rotate(x, at)
    assert torch.allclose(a.norm(dim=-1), x.norm(dim=-1))
    assert torch.equal(a[0], x[0])
    far = (ex.rotate(x, at + 7) * ex.rotate(y, at + 7)).sum(-1)
    assert torch.allclose((a * ex.rotate(y, at)).sum(-1), far)


def test_plain_layer_is_causal():
    ex = example()
    shape = ex.Shape(hidden=64, heads=4, kv_heads=2, head_dim=16, inner=96)
    w = {n: t.double() for n, t in ex.random_weights(shape).items()}
    x = torch.randn(9, 64, dtype=torch.float64)
    assert torch.allclose(ex.plain_layer(shape, w, x, 9)[:5], ex.plain_layer(shape, w, x[:5], 5))


@pytest.mark.gpu
@pytest.mark.parametrize("prompts,tokens", [([150, 37], 3), ([1, 64, 65], 2), ([300], 1)])
@pytest.mark.parametrize("int8", [False, True])
def test_layer(olamd, prompts, tokens, int8):
    """Eight things are rounded to 8 bits on the way from x to the layer's output:
    both norms' outputs, the two other products' inputs, k, v, and through the
    scores q's and k's errors once more.  Each has a relative error of at most
    2^-4 (E4M3; INT8 codes of a block are nearer), a root mean square of 2^-4 /
    sqrt(3); their sum bounds what they make together."""
    olamd.init(0)
    ex = example()
    shape = ex.Shape(hidden=512, heads=8, kv_heads=2, head_dim=64, inner=704)
    layer, inputs, outputs = ex.run(olamd, shape, prompts, tokens, dtype=olamd.INT8 if int8 else olamd.FLOAT8E4M3FN)
    for x, y in zip(inputs, outputs):
        assert y.shape == x.shape and torch.isfinite(y.float()).all()
        assert ex.error(layer, x, y) < 8 * 2.0 ** -4 / math.sqrt(3)


@pytest.mark.gpu
def test_prompt_at_once_or_in_parts(olamd):
    """A prompt in one step and the same tokens one by one give the layer's output
    within the same bound of each other, twice."""
    olamd.init(0)
    ex = example()
    shape = ex.Shape(hidden=256, heads=4, kv_heads=4, head_dim=64, inner=512)
    _, _, whole = ex.run(olamd, shape, [70], 0)
    layer, inputs, parts = ex.run(olamd, shape, [1], 69)
    x = torch.randn(70, 256, generator=torch.Generator().manual_seed(1)).bfloat16()
    assert torch.equal(inputs[0], x)
    added = (whole[0].double() - x.double()).square().mean().sqrt()
    off = (whole[0].double() - parts[0].double()).square().mean().sqrt()
    assert off < 2 * 8 * 2.0 ** -4 / math.sqrt(3) * added
