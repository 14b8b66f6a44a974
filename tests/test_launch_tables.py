"""The tables that go with the attention's launches, as host code builds them (no GPU)."""

from __future__ import annotations

import ctypes
import subprocess

import numpy as np
import pytest

from nebulasd_amd.build import CSRC, ROOT

_SOURCE = """
#include "nsd_common.h"
extern "C" void make(const uint64_t* from, int n, uint64_t* out, int whole) {
  uint64_t t[96];
  std::fill(t, t + 96, 0xabababababababab);  // what lies on the stack
  if (whole) {
    std::copy(from, from + n, t);
    nsd::end_table(t, n);
  } else {
    nsd::short_table(t, from, n);
  }
  std::copy(t, t + 96, out);
}
"""


@pytest.fixture(scope="module")
def make(tmp_path_factory):
    at = tmp_path_factory.mktemp("tables")
    (at / "tables.cpp").write_text(_SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", f"-I{ROOT / 'include'}",
                    str(at / "tables.cpp"), "-o", str(at / "tables.so")], check=True)
    return ctypes.CDLL(str(at / "tables.so")).make


@pytest.mark.parametrize("whole", [0, 1])
@pytest.mark.parametrize("n", [0, 1, 50, 95, 96])
def test_tables_end_in_zeros(make, n, whole):
    """The filled entries and nothing else of a longer table, whose rest nobody wrote."""
    from_, out = np.full(448, 0xcd, np.uint64), np.zeros(96, np.uint64)
    from_[:n] = np.arange(1, n + 1)
    make(from_.ctypes.data_as(ctypes.c_void_p), n, out.ctypes.data_as(ctypes.c_void_p), whole)
    assert (out[:n] == np.arange(1, n + 1)).all() and not out[n:].any()
