"""CPU: inline assembly that writes a named register says so to the compiler."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "starneig_amd", "csrc")


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip"))), ids=os.path.basename)
def test_registers_that_inline_assembly_writes_are_clobbers(path):
    for statement in re.findall(r"\basm\b\s*(?:volatile\s*)?\(.*?\);", open(path).read(), re.S):
        strings = re.findall(r'"((?:[^"\\]|\\.)*)"', statement)
        for line in re.split(r"\\n(?:\\t)?", strings[0]):
            written = re.match(r"\s*[sv]_\w+\s+(m0|vcc|exec|scc|[sv]\d+)\b", line)
            assert written is None or written.group(1) in strings[1:], (written.group(1), statement)
