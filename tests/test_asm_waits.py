"""Wait states in the kernels' inline asm, which the compiler does not look into (sources alone; no GPU)."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "nebulasd_amd" / "csrc"


def lds_loads():
    """(file, instructions) of every asm string that loads to LDS."""
    found = []
    for path in sorted(CSRC.iterdir()):
        for text in re.findall(r'asm volatile\(\s*"((?:[^"\\]|\\.)*)"', path.read_text()):
            parts = [x.strip() for x in text.replace("\\t", "").split("\\n") if x.strip()]
            if any(x.startswith("global_load_lds") for x in parts):
                found.append(pytest.param(parts, id=f"{path.name}-{len(found)}"))
    return found


@pytest.mark.parametrize("parts", lds_loads())
def test_loads_to_lds_wait_behind_m0(parts):
    """A load to LDS comes one wait state at least behind the write of m0 that says where to (s_nop n: n + 1 states), and
    five behind a base in scalar registers, which a VALU may have written just before the asm."""
    load = next(i for i, x in enumerate(parts) if x.startswith("global_load_lds"))
    write = max(i for i, x in enumerate(parts[:load]) if x.startswith("s_mov_b32 m0"))
    states = sum(int(x.split()[1]) + 1 for x in parts[write + 1:load] if x.startswith("s_nop"))
    base = parts[load].split(",")[1].split()[0]
    assert states >= (1 if base == "off" else 5)


def test_there_are_loads_to_lds():
    assert len(lds_loads()) >= 9
