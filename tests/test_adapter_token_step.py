"""The adapter's graph nodes from a layer's joint projection to the next token, as
test_adapter_decoder.py has those of the layer: registered, and what they make of a
node's inputs and attributes, against a stand-in runtime."""
import os
import re
import shutil
import subprocess

import pytest

from test_adapter_decoder import ADAPTER, MAIN, ROOT, _part

OPERATORS = ["MxGatedMatMul", "RotaryTables", "RotaryEmbedding", "RotaryKvCacheAppend", "SampleTokens"]


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    text = open(ADAPTER).read()
    base = _part(text, "// ONNX TensorProto data types used below.", "// MatMul output shape as the reference")
    sizes = re.search(r"size_t ByteSize\(.*\n", text).group(0)
    helpers = _part(text, "// The value of an optional FLOAT scalar input.", "// ai.rt.amd:RmsNormQuantize(x, weight")
    cache = _part(text, "// The four tensors of a cache that the graph holds", "// ai.rt.amd:KvCacheAppend(k, v")
    nodes = _part(text, "// Operators from a decoder layer's joint projection", "std::once_flag g_registered;")
    makes = "".join(f'    if (n.type == "{op}") k = std::make_unique<Mi355x{op}>(kc, nullptr);\n' for op in OPERATORS)
    main = re.sub(r'(    if \(n\.type == .*\n)+', makes.replace("\\", r"\\"), MAIN)
    source = tmp_path_factory.mktemp("adapter") / "nodes.cc"
    source.write_text('#include "adapter_token_step_runtime.hpp"\nnamespace mi355x {\n' + base + sizes + helpers + cache + nodes +
                      "}  // namespace mi355x\n" + main)
    exe = source.with_suffix("")
    subprocess.run(["g++", "-std=c++17", "-O0", "-Wall", "-Werror", "-Wno-unused-function", "-I", os.path.join(ROOT, "include"), "-I",
                    os.path.join(ROOT, "tests"), str(source), "-o", str(exe)], check=True)

    def run(case, refuse=None):
        out = subprocess.run([str(exe)] + ([refuse] if refuse else []), input=case + "\n", capture_output=True, text=True,
                             check=True, timeout=60).stdout
        return out.splitlines()

    return run


@pytest.mark.parametrize("op", OPERATORS)
def test_node_is_registered(op):
    text = open(ADAPTER).read()
    assert re.search(rf"class Mi355x{op} : public Mi355xKernel\b", text)
    assert f'static constexpr const char *name = "onnxl_amd:CPU:ai.rt.amd:{op}";' in text
    assert f'Register<Mi355x{op}>(kFusedDomain, "{op}");' in text


CACHE = "kc:17:3,2,16,64 vc:17:3,2,64,16 ks:1:3,2 vs:1:3,2 t:6:2,3 s:6:3 l:6:2"
CACHE_CALL = "17D[3,2,16,64]6144 17D[3,2,64,16]6144 1D[3,2]24 1D[3,2]24 6H[2,3]24 6H[3]12 6H[2]8"
CACHE_OUT = ["out a 17 [3,2,16,64] 1", "out b 17 [3,2,64,16] 1", "out c 1 [3,2] 1", "out d 1 [3,2] 1"]


@pytest.mark.parametrize("case,lines", [
    ("MxGatedMatMul;a:10:5,64 g:2:64,32 gs:2:64,2 u:2:64,32 us:2:64,2;y;activation=2 a_type=23",
     ["gated 10H[5,64]640 - 23 2H[64,32]2048 2H[64,2]128 2H[64,32]2048 2H[64,2]128 2 10H[5,64]640 -", "out y 10 [5,64] 0"]),
    ("MxGatedMatMul;a:17:5,64 g:2:64,32 gs:2:64,2 u:2:64,32 us:2:64,2 as:2:5,2;y s;mx=1",
     ["gated 17H[5,64]320 2H[5,2]10 0 2H[64,32]2048 2H[64,2]128 2H[64,32]2048 2H[64,2]128 0 17H[5,64]320 2H[5,2]10",
      "out y 17 [5,64] 0", "out s 2 [5,2] 0"]),
    ("MxGatedMatMul;a:2:5,32 g:2:64,32 gs:2:64,2 u:2:64,32 us:2:64,2 as:2:5,2;y",
     ["gated 2H[5,32]160 2H[5,2]10 0 2H[64,32]2048 2H[64,2]128 2H[64,32]2048 2H[64,2]128 0 16H[5,64]640 -", "out y 16 [5,64] 0"]),
    ("RotaryTables;;c s;positions=7 rotary_dim=32", ["tables 10000 0 1 0 32 1 0 1H[7,16]448 1H[7,16]448", "out c 1 [7,16] 0", "out s 1 [7,16] 0"]),
    ("RotaryTables;- - - b:1 m:1;c s;positions=7 rotary_dim=32 scaling=4 original_positions=64",
     ["tables 10000 4 1 64 32 0.5 0.5 1H[7,16]448 1H[7,16]448", "out c 1 [7,16] 0", "out s 1 [7,16] 0"]),
    ("RotaryEmbedding;x:10:2,3,5,32 c:1:9,8 s:1:9,8 p:6:2,5;y", ["rotary 10H[2,3,5,32]1920 1H[9,8]288 1H[9,8]288 6H[2,5]40 0 0 10H[2,3,5,32]1920",
                                                                "out y 10 [2,3,5,32] 0"]),
    ("RotaryEmbedding;x:1:2,5,96 c:1:2,5,8 s:1:2,5,8;y;interleaved=1 num_heads=3",
     ["rotary 1H[2,5,96]3840 1H[2,5,8]320 1H[2,5,8]320 - 1 3 1H[2,5,96]3840", "out y 1 [2,5,96] 0"]),
    (f"RotaryKvCacheAppend;x:10:5,8,64 c:1:9,16 n:1:9,16 - {CACHE};q a b c d",
     [f"rotary append 10H[5,8,64]5120 1H[9,16]576 1H[9,16]576 - 0 10D[5,4,64]2560 {CACHE_CALL}", "out q 10 [5,4,64] 1", *CACHE_OUT]),
    (f"RotaryKvCacheAppend;x:16:5,8,64 c:16:9,16 n:16:9,16 p:6:5 {CACHE};q a b c d;interleaved=1",
     [f"rotary append 16H[5,8,64]5120 16H[9,16]288 16H[9,16]288 6H[5]20 1 16D[5,4,64]2560 {CACHE_CALL}", "out q 16 [5,4,64] 1", *CACHE_OUT]),
    ("SampleTokens;x:10:3,50 u:1:3;t", ["sample 10H[3,50]300 1H[3]12 - - - - 7H[3]3 -", "out t 7 [3] 0"]),
    ("SampleTokens;x:1:3,50 u:1:3 T:1:3 k:6:3 p:1:3 m:1:3;t p",
     ["sample 1H[3,50]600 1H[3]12 1H[3]12 6H[3]12 1H[3]12 1H[3]12 7H[3]3 1H[3]12", "out t 7 [3] 0", "out p 1 [3] 0"]),
])
def test_node_calls_the_library(program, case, lines):
    """Type, place, shape and bytes of every argument, and of the node's outputs (the stand-in has INT64 values of a byte);
    no buffer is left."""
    assert program(case) == lines


@pytest.mark.parametrize("case", [
    "MxGatedMatMul;a:10:5,64 g:2:64,32 gs:2:64,2 u:2:64,32;y", "MxGatedMatMul;a:10:5,64 g:2:2,64,32 gs:2:64,2 u:2:64,32 us:2:64,2;y",
    "MxGatedMatMul;a:10:5,64 g:2:64,32 gs:2:64,2 u:2:64,32 us:2:64,2;y s", "MxGatedMatMul;a:10:5,64 g:2:64,32 gs:2:64,2 u:2:64,32 us:2:64,2;y;mx=1",
    "RotaryTables;;c s;positions=7", "RotaryTables;;c s;rotary_dim=32", "RotaryTables;;c s;positions=7 rotary_dim=31",
    "RotaryTables;b:10;c s;positions=7 rotary_dim=32", "RotaryEmbedding;x:10 c:1:9,8 s:1:9,8;y", "RotaryEmbedding;x:10:2,3,32 c:1:9,8;y",
    f"RotaryKvCacheAppend;x:10:5,4,64 c:1:9,16 n:1:9,16 - {CACHE};q a b c d", f"RotaryKvCacheAppend;x:10:5,8,64 c:1:9,16 n:1:9,16 - {CACHE};q a b c",
    "SampleTokens;x:10:50 u:1:3;t", "SampleTokens;x:10:3,50;t",
])
def test_node_refuses(program, case):
    """Before the library is called."""
    lines = program(case)
    assert len(lines) == 1 and lines[0].startswith("invalid "), lines


def test_node_passes_on_what_the_library_refuses(program):
    assert program("SampleTokens;x:10:3,50 u:1:4;t", refuse="no") == ["sample 10H[3,50]300 1H[4]16 - - - - 7H[3]3 -", "invalid no"]
