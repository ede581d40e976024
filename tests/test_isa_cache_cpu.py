"""The same hazards of inline asm in the cache library's kernels, compiled with the flags that each of them ships with
(no GPU)."""
import re
import subprocess

import pytest

from fastdecisions_amd import _build
from test_isa_cpu import (test_a_wait_state_between_m0_and_the_copy_that_reads_it,  # noqa: F401  (run on `kernels` below)
                          test_no_asm_leaves_a_global_load_into_registers_in_flight,
                          test_registers_of_asm_lds_reads_are_untouched_until_their_wait)

COPIES = re.compile(r"load_lds|gqa_tile\.h")  # copies to LDS of its own, or the shared one
SOURCES = [s for s in _build.CACHE_SOURCES if s.endswith(".hip") and COPIES.search((_build.CSRC / s).read_text())]


def test_the_attention_is_among_them():
    assert "paged_gqa.hip" in SOURCES


@pytest.fixture(scope="module", params=SOURCES)
def kernels(request):
    """{function: [(opcode, register operands, inside an asm block, text)]} in program order."""
    flags = [*_build.COMMON_FLAGS, "-x", "hip", *_build.DEVICE_FLAGS, *_build.EXTRA_FLAGS.get(request.param, [])]
    out = subprocess.run([_build.hipcc(), *flags, "--cuda-device-only", "-S", str(_build.CSRC / request.param), "-o", "-"],
                         check=True, capture_output=True, text=True)
    found, current, in_asm = {}, None, False
    for line in out.stdout.splitlines():
        name = re.match(r"(_Z\w+):", line)
        if name:
            current = found.setdefault(name[1], [])
        elif "#ASMSTART" in line or "#ASMEND" in line:
            in_asm = "#ASMSTART" in line
        else:
            text = line.split(";")[0].strip()
            if current is not None and text and not text.startswith(".") and not text.endswith(":"):
                op, _, rest = text.partition(" ")
                current.append((op, re.findall(r"[vsa]\[\d+:\d+\]|\b[vsa]\d+\b|\bm0\b", rest), in_asm, text))
    found = {name: ins for name, ins in found.items() if ins}
    assert len(found) > 1
    return found
