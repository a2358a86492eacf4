"""The example of a decoder layer at lengths that its defaults do not have."""
import pytest
import torch

from test_decoder_layer import example


class NoLibrary:
    """What a cache's bookkeeping needs of the library."""
    FLOAT8E4M3FN = 17

    @staticmethod
    def KvCache(*args):
        return None


def test_layer_refuses_sequences_that_its_tables_do_not_reach():
    ex = example()
    shape = ex.Shape(hidden=64, heads=4, kv_heads=2, head_dim=16, inner=96)
    layer = object.__new__(ex.DecoderLayer)
    layer.tables = torch.empty(100, 8), torch.empty(100, 8)
    sequences = ex.Sequences(NoLibrary, shape, 2, 200)
    sequences.length = [99, 7]
    with pytest.raises(ValueError, match="100 positions"):
        layer.grow(sequences, [2, 1])
    with pytest.raises(ValueError, match="100 positions"):
        layer.grow(sequences, [0, 94])
    assert sequences.length == [99, 7] and sequences.held == [0, 0]  # nothing has grown


@pytest.mark.gpu
def test_prompt_past_eight_thousand_tokens(olamd):
    olamd.init(0)
    ex = example()
    shape = ex.Shape(hidden=128, heads=2, kv_heads=1, head_dim=64, inner=192)
    layer, _, outputs = ex.run(olamd, shape, [8190, 5], 4)
    assert all(torch.isfinite(y.float()).all() for y in outputs) and [len(y) for y in outputs] == [8194, 9]
    words = ex.Vocabulary(olamd, 128, 500)
    drawn = ex.generate(layer, words, [[i % 500 for i in range(8190)], [1, 2]], 4)
    assert [len(d) for d in drawn] == [4, 4] and all(0 <= t < 500 for d in drawn for t in d)
    with pytest.raises(ValueError, match="8194 positions"):
        ex.generate(layer, words, [[i % 500 for i in range(8190)]], 6)


@pytest.mark.gpu
def test_nothing_to_draw(olamd):
    olamd.init(0)
    ex = example()
    shape = ex.Shape(hidden=128, heads=2, kv_heads=1, head_dim=64, inner=192)
    layer = ex.DecoderLayer(olamd, shape, ex.random_weights(shape), 64)
    assert ex.generate(layer, ex.Vocabulary(olamd, 128, 500), [[1, 2], [3]], 0) == [[], []]
