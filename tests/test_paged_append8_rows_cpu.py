"""The rows of `paged_append8`'s tasks, in the kernel's own arithmetic compiled for the host, against
Python's whole numbers: lengths are read on the device and may be any 32-bit number."""
from __future__ import annotations

import ctypes
import random
import shutil
import subprocess

import pytest

from conftest import PKG

SOURCE = """
#include "paged8_rows.cuh"
extern "C" void rows(int n, int c, int top, int L, int span, int k, int* out) {
  const simsd::PagedRows8 r = simsd::paged_rows8(n, c, top, L, span, k);
  out[0] = r.at, out[1] = r.lo, out[2] = r.hi;
}
"""


@pytest.fixture(scope="module")
def rows(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("rows")
    (d / "rows.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-O1", "-fwrapv", "-std=c++17", "-fPIC", "-shared", "-I", str(PKG / "csrc"), "-o", str(d / "rows.so"),
                    str(d / "rows.cpp")], check=True)
    fn = ctypes.CDLL(str(d / "rows.so")).rows

    def call(*args):
        out = (ctypes.c_int * 3)()
        fn(*args, out)
        return tuple(out)

    return call


def expected(n, c, top, L, span, k):
    """None, or (first position of the span, rows lo .. hi - 1)."""
    at = ((n - c) // span + k) * span
    first, last = max(n - c, at), min(top, at + span)
    if c == 0 or first >= last:
        return None
    return at, first - (n - L), last - (n - L)


def check(rows, n, count, cap, L, span):
    c = min(n, max(0, min(count, L)))
    top = min(n, cap)
    seen = []
    for k in range((L + span - 2) // span + 1):          # as many spans as L neighbouring tokens can touch
        at, lo, hi = rows(n, c, top, L, span, k)
        want = expected(n, c, top, L, span, k)
        if want is None:
            assert lo >= hi, (n, count, cap, L, span, k)
            continue
        assert (at, lo, hi) == want, (n, count, cap, L, span, k)
        assert 0 <= L - c <= lo < hi <= L and 0 <= at < top
        seen += range(lo, hi)
    assert seen == list(range(L - c, L - (n - max(top, n - c)))), (n, count, cap, L, span)   # every place's row, once


MAX = 0x7FFFFFFF
LENGTHS = [0, 1, 15, 16, 17, 50, 1000, 0x3FFFFFFF, 0x40000000, 0x7FFEFFFF, 0x7FFF0000, 0x7FFF0001, 0x7FFFF800, 0x7FFFF810,
           0x7FFFFFEF, 0x7FFFFFF0, 0x7FFFFFFE, MAX]


@pytest.mark.parametrize("span", [1, 7, 16, 24, 64, 128, 4096])
def test_rows_of_lengths_up_to_the_largest(rows, span):
    for n in LENGTHS:
        for L, count in ((1, 1), (2, 2), (4, 4), (4, 1), (4, 0), (300, 300), (300, 7), (2048, 10), (2048, 2048)):
            for cap in (0, 48, 1008, n, n - 1, 0x7FFF0000):
                check(rows, n, count, max(0, min(cap, 0x7FFF0000)), L, span)


def test_rows_of_any_length(rows):
    rng = random.Random(0)
    for _ in range(3000):
        n = rng.choice([rng.randrange(MAX + 1), MAX - rng.randrange(5000), rng.randrange(5000)])
        L = rng.randrange(1, 600)
        cap = min(0x7FFF0000, max(0, rng.choice([n - rng.randrange(700), n + 1, rng.randrange(5000)])))
        check(rows, n, rng.randrange(-2, L + 3), cap, L, rng.choice([1, 3, 8, 16, 40, 128]))
