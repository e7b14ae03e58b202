"""Shared arrays that a kernel reads or writes 16 bytes at a time say so in their declaration: without it their place is the linker's choice."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "torch_ggml_ops_b200" / "csrc"
WIDE = r"(?:u?int4|float4|longlong2|ulonglong2|double2)"


@pytest.mark.parametrize("source", sorted(p.name for p in CSRC.glob("*.cu*")))
def test_arrays_used_in_wide_words_are_aligned(source):
    text = (CSRC / source).read_text()
    used = set(re.findall(rf"reinterpret_cast<(?:const )?{WIDE}\s*\*>\(&?(\w+)", text))
    for declaration in re.findall(r"^[^/\n]*__shared__[^;]*;", text, re.M):
        if re.search(rf"\b{WIDE}\b|align", declaration):
            continue
        names = set(re.findall(r"(\w+)\s*(?:\[|,|;)", declaration))
        assert not names & used, f"{source}: {declaration.strip()}"
