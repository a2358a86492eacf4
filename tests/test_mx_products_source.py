"""What the compiler cannot see in the MX products' kernels: assembly statements that read
a matrix instruction's result get no wait states before them."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onnx-light_amd", "csrc")


@pytest.mark.parametrize("name", ["mx_gemm.hpp", "mx_stream.hpp", "mx_gate.hpp", "mx.hip"])
def test_assembly_is_of_loads_and_waits_alone(name):
    text = open(os.path.join(CSRC, name)).read()
    for statement in re.findall(r'\basm\s*(?:volatile\s*)?\(\s*"([^"]*)"', text):
        for instruction in filter(None, statement.split(r"\n\t")):
            assert instruction.startswith(("s_", "buffer_load")), instruction


def test_launches_are_cut_into_pieces():
    """A launch of 2^32 threads or more along x runs in part without an error: with 512 threads a tile 2^30 rows by a narrow
    weight are that many, so every grid is a piece's count."""
    grids = re.findall(r"<<<([^,]+),", open(os.path.join(CSRC, "mx.hip")).read())
    assert len(grids) >= 6
    for grid in grids:
        assert grid in ("count", "dim3(count"), grid


def test_pieces_cover_every_workgroup(tmp_path):
    """LaunchInPieces, compiled for the host, for as many tiles as 2^31 rows have."""
    text = open(os.path.join(CSRC, "decoder.hpp")).read()
    body = text[text.index("template <typename F> void LaunchInPieces"):]
    (tmp_path / "p.cpp").write_text("#include <cstdint>\n#include <cstdio>\n#include <initializer_list>\n" + body[:body.index("\n}\n") + 3] + """
int main() {
  for (int64_t groups : {int64_t(1), int64_t(1) << 22, (int64_t(1) << 23) + 5, int64_t(1) << 24})
    LaunchInPieces(groups, 512, [&](int64_t first, unsigned count) { std::printf("%lld %lld %u\\n", (long long)groups, (long long)first, count); });
}
""")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", str(tmp_path / "p.cpp"), "-o", str(tmp_path / "p")], check=True)
    at = {}
    for line in subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout.splitlines():
        groups, first, count = map(int, line.split())
        assert first == at.get(groups, 0) and 0 < count * 512 < 2 ** 32
        at[groups] = first + count
    assert len(at) == 4 and all(k == v for k, v in at.items())
