"""No kernel with MFMAs has instructions in inline assembly: the compiler puts the waits that an MFMA in flight needs between
instructions that it knows, and does not know what assembly does to the registers.  (An empty assembly statement, which hides a
value from the optimiser, has no instructions.)"""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "blog_amd", "csrc")
# asm("...") or asm volatile("..."), and its first string
STATEMENT = re.compile(r'\basm\b\s*(?:volatile\s*)?\(\s*"([^"]*)"')


def _sources():
    return {os.path.basename(p): open(p).read() for p in sorted(glob.glob(os.path.join(CSRC, "*.h*")))}


def test_instructions_in_assembly_stand_where_no_mfma_is():
    found = {(name, text) for name, code in _sources().items() for text in STATEMENT.findall(code) if text}
    assert found == {("qlin_device.hpp", "v_cvt_f16_f32 %0, %1"), ("qlin_q4k_stream.hip", "v_and_b32 %0, %1, %2")}
    sources = _sources()
    assert "mfma" not in sources["qlin_q4k_stream.hip"]
    # the conversion's users: dequantization, and the quantizers of Q8_1 rows
    users = {name for name, code in sources.items() if "f32_to_f16_bits(" in code}
    assert users == {"qlin_device.hpp", "qlin_dequant.hip", "qlin_q8_1.hpp"}
    assert "mfma" not in sources["qlin_dequant.hip"]
    for name, code in sources.items():
        if '#include "qlin_q8_1.hpp"' in code:
            for kernel in re.split(r"__global__", code)[1:]:
                body = kernel[:kernel.find("\n}\n")]
                assert not (re.search(r"\bquantize_\w+\s*\(", body) and "mfma" in body), name
