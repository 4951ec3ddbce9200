"""The arithmetic of row numbers (ops/csrc/ska_rows.h) near 2^31, on the host:
the kernels' own functions, over sequences that need no memory."""

import ctypes
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(
    os.path.abspath(__file__))), "spark_sklearn_amd", "ops", "csrc")
MOST = 2 ** 31 - 65537          # entries or rows, the operators' limit

SOURCE = """
#include <cstdint>
#include "ska_rows.h"

// sorted keys without memory: key i is i / each
struct Keys {
  int64_t n, each;
  int64_t operator[](int64_t i) const {
    if (i < 0 || i >= n) throw i;
    return i / each;
  }
};

// -1: a position outside the keys was read
extern "C" int64_t find(int64_t n, int64_t each, int64_t g) {
  try {
    return ska::lower_bound(Keys{n, each}, (int)n, g);
  } catch (int64_t) {
    return -1;
  }
}

extern "C" int64_t count(int64_t first, int64_t last, int64_t shift) {
  return ska::part_count((int)first, (int)last, (int)shift);
}

extern "C" int64_t end(int64_t at, int64_t last, int64_t shift) {
  return ska::part_end((int)at, (int)last, (int)shift);
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    folder = tmp_path_factory.mktemp("rows")
    source, built = folder / "rows.cpp", folder / "rows.so"
    source.write_text(SOURCE)
    # sums that pass 32 bits wrap round, as they do in the kernels
    subprocess.run(
        [compiler, "-std=c++17", "-O1", "-fwrapv", "-shared", "-fPIC",
         "-I", CSRC, str(source), "-o", str(built)], check=True)
    lib = ctypes.CDLL(str(built))
    for name in ("find", "count", "end"):
        getattr(lib, name).restype = ctypes.c_int64
    return lib


@pytest.mark.parametrize("n", [0, 1, 2, 1000, 2 ** 30 - 1, 2 ** 30 + 1,
                               1_500_000_000, MOST])
@pytest.mark.parametrize("groups", [1, 3, 8192, 10007, 2 ** 24 - 1])
def test_lower_bound(host, n, groups):
    each = max(1, n // groups)
    for g in sorted({0, 1, 2, groups // 3, groups // 2, groups - 1, groups,
                     n // each}):
        at = host.find(*(ctypes.c_int64(v) for v in (n, each, g)))
        assert at == min(n, g * each)


@pytest.mark.parametrize("shift", [6, 8, 9, 16, 20, 22, 30])
@pytest.mark.parametrize("first,last", [
    (0, 0), (0, 1), (5, 5), (3, 1000), (0, 2 ** 30), (1, 2 ** 30 + 2),
    (0, MOST), (1, MOST), (12345, MOST), (MOST - 70000, MOST),
    (MOST - 1, MOST), (MOST, MOST)])
def test_parts(host, first, last, shift):
    size = 1 << shift
    count = host.count(*(ctypes.c_int64(v) for v in (first, last, shift)))
    assert count == -(-(last - first) // size)
    for part in (0, 1, count // 2, count - 2, count - 1):
        if not 0 <= part < count:
            continue
        at = first + part * size
        end = host.end(*(ctypes.c_int64(v) for v in (at, last, shift)))
        assert end == min(last, at + size)


def test_a_group_that_ends_before_it_begins_has_no_parts(host):
    """As offsets that decrease would have it."""
    assert host.count(*(ctypes.c_int64(v) for v in (900, 100, 8))) == 0
