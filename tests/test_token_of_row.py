"""The token that a packed row is: the kernels' own arithmetic, compiled for the
host, at numbers whose sums pass 64 bits."""

import ctypes
import itertools
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "torchlib-xpu_amd" / "csrc"
LO, HI = -2 ** 63, 2 ** 63 - 1

# The branch behind it as the kernels have it: table entries below `width` are read.
SOURCE = r"""
#include "token_of_row.h"
extern "C" int64_t token(int64_t start, int64_t row, int64_t offset) {
  return mx::attn::token_of_row(start, row, offset);
}
extern "C" int64_t entry(int64_t start, int64_t row, int64_t offset, int64_t width) {
  const int64_t t = mx::attn::token_of_row(start, row, offset);
  const int64_t e = t >= 0 ? t >> 4 : width;
  return e < width ? e : -1;
}
"""


def compilers():
    found = [c for c in ("/opt/rocm/llvm/bin/clang++", "g++") if shutil.which(c)]
    return found or [pytest.param(None, marks=pytest.mark.skip(reason="no host compiler"))]


@pytest.fixture(scope="module", params=compilers())
def lib(request, tmp_path_factory):
    where = tmp_path_factory.mktemp("token_of_row")
    (where / "t.cpp").write_text(SOURCE)
    subprocess.run([request.param, "-O3", "-std=c++17", "-shared", "-fPIC", f"-I{CSRC}", str(where / "t.cpp"), "-o",
                    str(where / "t.so")], check=True, timeout=120)
    lib = ctypes.CDLL(str(where / "t.so"))
    lib.token.argtypes, lib.token.restype = [ctypes.c_int64] * 3, ctypes.c_int64
    lib.entry.argtypes, lib.entry.restype = [ctypes.c_int64] * 4, ctypes.c_int64
    return lib


STARTS = [LO, LO + 1, -2 ** 33, -1, 0, 1, 5, 2 ** 31, 2 ** 40, HI - 6, HI - 1, HI]
ROWS = [0, 1, 5, 2 ** 26 - 1, 2 ** 40]
OFFSETS = [LO, LO + 5, -2 ** 33, -1, 0, 1, 4, 2 ** 26, 2 ** 40, HI]


def test_against_whole_numbers(lib):
    for start, row, offset in itertools.product(STARTS, ROWS, OFFSETS):
        t = start + row - offset
        want = t if start >= 0 and offset <= row and row - offset <= HI and t <= HI else -1
        assert lib.token(start, row, offset) == want, (start, row, offset)


def test_no_entry_before_the_table_or_past_it(lib):
    for width in (0, 1, 100):
        for start, row, offset in itertools.product(STARTS, ROWS, OFFSETS):
            assert -1 <= lib.entry(start, row, offset, width) < max(width, 0) or width == 0
            t = start + row - offset
            inside = start >= 0 and offset <= row and 0 <= t < 16 * width
            assert lib.entry(start, row, offset, width) == (t // 16 if inside else -1), (start, row, offset)
