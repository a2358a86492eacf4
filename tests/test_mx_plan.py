"""Which kernel an MX product takes (csrc/mx_plan.hpp, compiled for the host)."""
import ctypes
import os
import subprocess

import pytest

from mx_kernel_cases import BOTH, CASES

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onnx-light_amd", "csrc")
OUTPUT = {"plain": 0, "gated": 1, "gated mx": 2}
CUS = 256

SHIM = """#include "mx_plan.hpp"
#include <cstdio>
using namespace onnxl_amd;
extern "C" void plan(int64_t M, int64_t N, int64_t K, int x, int a_fp4, int output, char *out) {
  const mx::Sizes p{M, N, K, x != 0, a_fp4 != 0, output, 256};
  if (mx::Streams(p)) {
    const mx::StreamPlan s = mx::PlanStream(p);
    std::sprintf(out, "stream %d %d %d %d", s.nt, s.mt, (int)mx::OwnQuant(p), s.split > 1);
  } else {
    const mx::GemmPlan t = mx::PlanGemm(p);
    std::sprintf(out, "tiles %d %d %d %d %d", t.mb, t.nb, t.stages, t.wm, t.wn);
  }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """(form, act, M, K, N, activations of 16 bits) -> the kernel, as a text."""
    d = tmp_path_factory.mktemp("mx_plan")
    (d / "p.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, str(d / "p.cpp"), "-o", str(d / "p.so")],
                   check=True)
    f = ctypes.CDLL(str(d / "p.so")).plan
    f.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int] * 3 + [ctypes.c_char_p]
    text = ctypes.create_string_buffer(64)

    def of(form, act, M, K, N, x=True):
        f(M, N, K, int(x), int(act == "fp4"), OUTPUT[form], text)
        return text.value.decode()

    return of


# (form, act, rows, K, N, us streaming, us by tiles), measured on an MI355X
MEASURED = [
    ("plain", "fp8", 17, 4096, 14336, 15.5, 17.1), ("plain", "fp8", 17, 14336, 14336, 41.7, 47.8), ("plain", "fp8", 32, 4096, 20480, 23.3, 17.9),
    ("plain", "fp8", 33, 28672, 4096, 42.9, 68.3), ("plain", "fp8", 48, 28672, 4096, 51.5, 68.7), ("plain", "fp8", 64, 28672, 4096, 60.8, 69.4),
    ("plain", "fp8", 33, 28672, 8192, 71.4, 80.3), ("plain", "fp8", 64, 512, 20480, 17.3, 8.0), ("plain", "fp8", 64, 512, 14336, 14.3, 7.9),
    ("plain", "fp8", 48, 512, 14336, 10.7, 7.7), ("plain", "fp8", 64, 1024, 8192, 11.3, 8.9), ("plain", "fp8", 48, 14336, 8192, 46.4, 39.8),
    ("plain", "fp4", 33, 28672, 8192, 54.4, 63.0), ("plain", "fp4", 64, 28672, 4096, 43.4, 49.6), ("plain", "fp4", 64, 512, 28672, 15.6, 7.7),
    ("plain", "fp4", 64, 1024, 14336, 13.0, 8.1), ("plain", "fp4", 33, 8192, 12288, 27.1, 21.1), ("plain", "fp4", 48, 14336, 4096, 18.6, 28.3),
    ("gated", "fp8", 17, 2048, 8192, 9.5, 12.8), ("gated", "fp8", 17, 14336, 8192, 38.3, 44.3), ("gated", "fp8", 32, 8192, 8192, 33.8, 28.3),
    ("gated", "fp8", 64, 1024, 5632, 13.5, 9.8), ("gated", "fp4", 48, 1024, 11008, 12.2, 9.0), ("gated", "fp4", 24, 4096, 11008, 21.0, 17.7),
    ("gated mx", "fp8", 32, 4096, 14336, 27.1, 19.4), ("gated mx", "fp8", 24, 8192, 28672, 90.9, 77.8), ("gated mx", "fp8", 32, 2048, 8192, 8.7, 12.1),
    ("gated mx", "fp4", 20, 4096, 28672, 43.1, 31.0), ("gated mx", "fp4", 32, 8192, 14336, 42.4, 29.1), ("gated mx", "fp4", 17, 2048, 14336, 10.9, 12.4),
]


@pytest.mark.parametrize("form,act,M,K,N,stream,tiles", MEASURED)
def test_few_rows_take_the_faster_kernel(plan, form, act, M, K, N, stream, tiles):
    """Sizes on both sides of the rule's lines, each more than a tenth apart (a few less)."""
    assert plan(form, act, M, K, N).startswith("stream" if stream < tiles else "tiles")


def test_every_kernel_that_a_size_takes_is_tested(plan):
    """Of a sweep of sizes, each kernel (and for the streaming one, K shared by workgroups or not) is a size's of the GPU
    tests too; sizes that take a kernel in fewer than three of its steps do not count there."""
    rows = [1, 2, 3, 4, 8, 16, 17, 24, 31, 32, 33, 40, 48, 49, 56, 64, 65, 100, 128, 129, 200, 256, 300, 513, 700, 1000, 2000, 4096, 10000]
    widths = [1, 16, 33, 64, 100, 257, 512, 1000, 1056, 2048, 2600, 3050, 4096, 5700, 6100, 8192, 9000, 11008, 14336, 20000, 28672, 60000]
    lengths = [32, 96, 256, 288, 512, 544, 800, 1056, 1312, 2048, 2080, 2592, 4096, 6016, 8192, 8480, 14336, 28672]
    met = {(form, act, plan(form, act, M, K, N, x)) for form in OUTPUT for act in BOTH for M in rows for N in widths for K in lengths
           for x in (True, False) if form != "gated mx" or N % 32 == 0}
    tested = {(form, act, plan(form, act, M, K, N, x)) for form, act, M, K, N, x in CASES
              if K >= 768 or plan(form, act, M, K, N, x).startswith("stream")}
    assert len(met) > 80 and not met - tested, met - tested
