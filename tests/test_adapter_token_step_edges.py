"""The rotary embedding's graph node and the attribute that says how many dimensions turn,
which ONNX's operator has beside the tables that say it too."""
import pytest

from test_adapter_token_step import program  # noqa: F401

NODE = "RotaryEmbedding;x:10:2,3,5,32 c:1:9,8 s:1:9,8 p:6:2,5;y;rotary_embedding_dim="


@pytest.mark.parametrize("dim", [0, 16])
def test_dimensions_of_the_tables(program, dim):  # noqa: F811
    assert program(f"{NODE}{dim}") == ["rotary 10H[2,3,5,32]1920 1H[9,8]288 1H[9,8]288 6H[2,5]40 0 0 10H[2,3,5,32]1920", "out y 10 [2,3,5,32] 0"]


@pytest.mark.parametrize("dim", [8, 32, -16])
def test_other_dimensions_are_refused(program, dim):  # noqa: F811
    """Before the library is called, which would turn the tables' 16."""
    lines = program(f"{NODE}{dim}")
    assert len(lines) == 1 and lines[0].startswith("invalid "), lines
