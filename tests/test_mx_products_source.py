"""What the compiler cannot see in the MX products' kernels: assembly statements that read
a matrix instruction's result get no wait states before them."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onnx-light_amd", "csrc")


@pytest.mark.parametrize("name", ["mx_gemm.hpp", "mx_stream.hpp", "mx_gate.hpp", "mx.hip"])
def test_assembly_is_of_loads_and_waits_alone(name):
    text = open(os.path.join(CSRC, name)).read()
    for statement in re.findall(r'\basm\s*(?:volatile\s*)?\(\s*"([^"]*)"', text):
        for instruction in filter(None, statement.split(r"\n\t")):
            assert instruction.startswith(("s_", "buffer_load")), instruction
