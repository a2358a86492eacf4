"""The adapter's graph nodes of a decoder layer: registered, and what they make
of a node's inputs and attributes.  Their section of the adapter is compiled
against a stand-in runtime (adapter_runtime.hpp) whose library writes down every
call, since the adapter as a whole compiles inside the onnx-light tree only."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ADAPTER = os.path.join(ROOT, "adapter", "register_mi355x.cc")
OPERATORS = ["RmsNormQuantize", "MxQuantize", "MxMatMul", "KvCacheAppend", "KvCacheAttention"]

MAIN = r"""
// stdin: one case a line: op;inputs;outputs;attributes.  An input is name:type:dims or empty, an attribute name=value
#include <iostream>
#include <sstream>
using namespace mi355x;
static std::vector<std::string> Split(const std::string &s, char c) {
  std::vector<std::string> v;
  std::string t;
  std::istringstream in(s);
  while (std::getline(in, t, c)) v.push_back(t);
  if (!s.empty() && s.back() == c) v.push_back("");
  return v;
}
int main(int argc, char **argv) {
  if (argc > 1) refuse = argv[1];
  std::string line;
  while (std::getline(std::cin, line)) {
    const auto f = Split(line, ';');
    NodeProto n;
    rt::RuntimeContext ctx;
    n.type = f[0];
    for (const auto &i : Split(f[1], ' ')) {
      const auto p = Split(i, ':');
      n.in.push_back(p.empty() || p[0] == "-" ? "" : p[0]);
      if (n.in.back().empty()) continue;
      rt::Tensor t;
      t.data_type = std::stoi(p[1]);
      int64_t count = 1;
      if (p.size() > 2)
        for (const auto &d : Split(p[2], ',')) t.shape.d.push_back(std::stoll(d)), count *= t.shape.d.back();
      t.data.assign(rt::PackedByteSize(t.data_type, count), 0);
      if (t.data_type == 1 && p.size() == 2) {
        const float half = 0.5f;
        std::memcpy(t.data.data(), &half, 4);
      }
      ctx.values[n.in.back()] = t;
    }
    for (const auto &o : Split(f[2], ' ')) n.out.push_back(o == "-" ? "" : o);
    if (f.size() > 3)
      for (const auto &a : Split(f[3], ' ')) n.attributes[Split(a, '=')[0]] = std::stoll(Split(a, '=')[1]);
    const rt::KernelContext kc{&n};
    std::unique_ptr<rt::KernelBase> k;
    if (n.type == "RmsNormQuantize") k = std::make_unique<Mi355xRmsNormQuantize>(kc, nullptr);
    if (n.type == "MxQuantize") k = std::make_unique<Mi355xMxQuantize>(kc, nullptr);
    if (n.type == "MxMatMul") k = std::make_unique<Mi355xMxMatMul>(kc, nullptr);
    if (n.type == "KvCacheAppend") k = std::make_unique<Mi355xKvCacheAppend>(kc, nullptr);
    if (n.type == "KvCacheAttention") k = std::make_unique<Mi355xKvCacheAttention>(kc, nullptr);
    try {
      k->Run(ctx);
      for (const auto &o : n.out) {
        if (o.empty()) continue;
        if (!ctx.values.count(o)) {
          std::printf("missing %s\n", o.c_str());
          continue;
        }
        const rt::Tensor &t = ctx.values.at(o);
        std::printf("out %s %d [", o.c_str(), t.data_type);
        for (size_t i = 0; i < t.shape.size(); ++i) std::printf(i ? ",%lld" : "%lld", (long long)t.shape[i]);
        std::printf("] %d\n", t.data.empty() ? -1 : t.data[0]);
      }
    } catch (const std::invalid_argument &e) {
      std::printf("invalid %s\n", e.what());
    }
    k.reset();
    if (live_buffers) std::printf("%d buffers left\n", live_buffers);
  }
}
"""


def _part(text, first, last):
    return text[text.index(first):text.index(last)]


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    text = open(ADAPTER).read()
    base = _part(text, "// ONNX TensorProto data types used below.", "// MatMul output shape as the reference")
    sizes = re.search(r"size_t ByteSize\(.*\n", text).group(0)
    nodes = _part(text, "// The value of an optional FLOAT scalar input.",
                  "// ---------------------------------------------------------------------------\n// Registration.")
    tmp = tmp_path_factory.mktemp("adapter")
    source = tmp / "nodes.cc"
    source.write_text('#include "adapter_runtime.hpp"\nnamespace mi355x {\n' + base + sizes + nodes +
                      "}  // namespace mi355x\n" + MAIN)
    exe = tmp / "nodes"
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


@pytest.mark.parametrize("case,lines", [
    ("RmsNormQuantize;x:10:3,64 w:10:64;y s",
     ["norm 10H[3,64]384 10H[64]128 - 1e-05 0 17H[3,64]192 1H[3,1]12 -", "out y 17 [3,64] 0", "out s 1 [3,1] 0"]),
    ("RmsNormQuantize;x:16:3,64 w:1:64 r:16:3,64 e:1;y s t;block_size=32 output_dtype=3",
     ["norm 16H[3,64]384 1H[64]256 16H[3,64]384 0.5 32 3H[3,64]192 1H[3,2]24 16H[3,64]384", "out y 3 [3,64] 0",
      "out s 1 [3,2] 0", "out t 16 [3,64] 0"]),
    ("RmsNormQuantize;x:16:3,64 w:16:64 r:16:3,64;y s;mx=1",
     ["norm 16H[3,64]384 16H[64]128 16H[3,64]384 1e-05 32 17H[3,64]192 2H[3,2]6 -", "out y 17 [3,64] 0", "out s 2 [3,2] 0"]),
    ("MxQuantize;x:10:2,64;y s", ["quantize 10H[2,64]256 17H[2,64]128 2H[2,2]4", "out y 17 [2,64] 0", "out s 2 [2,2] 0"]),
    ("MxQuantize;x:10:2,64;y s;output_dtype=23",
     ["quantize 10H[2,64]256 23H[2,64]64 2H[2,2]4", "out y 2 [2,32] 0", "out s 2 [2,2] 0"]),
    ("MxMatMul;a:10:5,64 b:2:8,32 bs:2:8,2;y;a_type=23",
     ["matmul 10H[5,64]640 - 23 2H[8,32]256 2H[8,2]16 10H[5,8]80", "out y 10 [5,8] 0"]),
    ("MxMatMul;a:17:5,64 b:2:8,32 bs:2:8,2 as:2:5,2;y;output_dtype=10",
     ["matmul 17H[5,64]320 2H[5,2]10 0 2H[8,32]256 2H[8,2]16 10H[5,8]80", "out y 10 [5,8] 0"]),
    ("MxMatMul;a:2:5,32 b:2:8,32 bs:2:8,2 as:2:5,2;y",
     ["matmul 2H[5,32]160 2H[5,2]10 0 2H[8,32]256 2H[8,2]16 16H[5,8]80", "out y 16 [5,8] 0"]),
    ("KvCacheAppend;k:10:5,2,64 v:10:5,2,64 kc:17:3,2,16,64 vc:17:3,2,64,16 ks:1:3,2 vs:1:3,2 t:6:2,3 s:6:3 l:6:2;a b c d",
     ["append 10H[5,2,64]1280 10H[5,2,64]1280 17D[3,2,16,64]6144 17D[3,2,64,16]6144 1D[3,2]24 1D[3,2]24 6H[2,3]24 6H[3]12 6H[2]8",
      "out a 17 [3,2,16,64] 1", "out b 17 [3,2,64,16] 1", "out c 1 [3,2] 1", "out d 1 [3,2] 1"]),
    ("KvCacheAttention;q:16:5,4,64 kc:3:3,2,16,64 vc:3:3,2,64,16 ks:1:3,2 vs:1:3,2 t:6:2,3 s:6:3 l:6:2;y",
     ["attention 16H[5,4,64]2560 3D[3,2,16,64]6144 3D[3,2,64,16]6144 1D[3,2]24 1D[3,2]24 6H[2,3]24 6H[3]12 6H[2]8 0.125 0 "
      "16H[5,4,64]2560", "out y 16 [5,4,64] 0"]),
    ("KvCacheAttention;q:16:5,4,64 kc:3:3,2,16,64 vc:3:3,2,64,16 ks:1:3,2 vs:1:3,2 t:6:2,3 s:6:3 l:6:2 f:1;y;max_query=3",
     ["attention 16H[5,4,64]2560 3D[3,2,16,64]6144 3D[3,2,64,16]6144 1D[3,2]24 1D[3,2]24 6H[2,3]24 6H[3]12 6H[2]8 0.5 3 "
      "16H[5,4,64]2560", "out y 16 [5,4,64] 0"]),
])
def test_node_calls_the_library(program, case, lines):
    """Type, place (host or device), shape and bytes of every argument, and of the node's outputs; no buffer is left."""
    assert program(case) == lines


@pytest.mark.parametrize("case", [
    "MxQuantize;x:10:2,64;y s;output_dtype=3", "MxQuantize;x:10:2,64;y s;output_dtype=10",
    "MxQuantize;x:10;y s", "RmsNormQuantize;x:10 w:10:64;y s", "RmsNormQuantize;x:10:3,64 w:10:64;y s;block_size=-1",
    "MxMatMul;a:10:5,64 b:2:2,8,32 bs:2:8,2;y", "KvCacheAttention;q:16:5,256 kc:3:3,2,16,64 vc:3:3,2,64,16 ks:1:3,2 vs:1:3,2 t:6:2,3 s:6:3 l:6:2;y",
    "KvCacheAppend;k:10:5,2,64 v:10:5,2,64 kc:17:3,2,16,64 vc:17:3,2,64,16 ks:1:3,2 - t:6:2,3 s:6:3 l:6:2;a b c d",
])
def test_node_refuses(program, case):
    """Before the library is called."""
    lines = program(case)
    assert len(lines) == 1 and lines[0].startswith("invalid "), lines


@pytest.mark.parametrize("case,call", [
    # a sum that nothing is added for, and blocks that MXFP8 does not have: the library sees them and refuses
    ("RmsNormQuantize;x:10:3,64 w:10:64;y s t", "norm 10H[3,64]384 10H[64]128 - 1e-05 0 17H[3,64]192 1H[3,1]12 10H[3,64]384"),
    ("RmsNormQuantize;x:10:3,64 w:10:64;y s;mx=1 block_size=64",
     "norm 10H[3,64]384 10H[64]128 - 1e-05 64 17H[3,64]192 2H[3,1]3 -"),
])
def test_node_passes_on_what_the_library_refuses(program, case, call):
    assert program(case, refuse="no") == [call, "invalid no"]
