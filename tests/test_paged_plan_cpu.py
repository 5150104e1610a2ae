"""How many CTAs paged attention starts where a device has more SMs than a B200: no more than its join of a cut
sequence has shared memory for, and counters."""
from __future__ import annotations

import shutil
import subprocess
import sys

import pytest

from kernels import _lib

# What the smallest tcgen05 form has behind its CTA's barriers: 64 dims, 128 rows, the 8-bit cache (four fp16 tiles and
# eight 8-bit ones of 128 keys, 16 KB of O, a KB of maxima and sums, eight units of scales).
ROOM = 4 * 16384 + 8 * 8192 + 16384 + 1024 + 8 * 1536

SIZES = """
import ctypes, sys
ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
for name in ("simsd_paged_attention_workspace_size", "simsd_paged_attention8_workspace_size"):
    fn = getattr(lib, name)
    fn.restype, fn.argtypes = ctypes.c_size_t, [ctypes.c_int] * 4
    for L in (1, 8, 16, 32, 64, 128, 500):
        for D in (64, 128):
            print(name, L, D, fn(L, 1, 1, D))
"""


def sizes(tmp_path, sms):
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    (tmp_path / "sms.c").write_text(f"int simsd_device_sm_count(void) {{ return {sms}; }}\n")
    subprocess.run([cc, "-shared", "-fPIC", "-o", str(tmp_path / "sms.so"), str(tmp_path / "sms.c")], check=True)
    out = subprocess.run([sys.executable, "-c", SIZES, str(tmp_path / "sms.so"), str(_lib.LIB_PATH)], check=True,
                         capture_output=True, text=True).stdout.split("\n")
    return [(w[0], int(w[1]), int(w[2]), int(w[3])) for w in map(str.split, out) if len(w) == 4]


def grid_of(size, D, nr):
    up = lambda v: -(-v // 256) * 256  # noqa: E731
    for grid in range(1, 1025):
        if _lib.PAGED_COUNTER_BYTES + up(2 * grid * D * nr * 4) + up(2 * grid * nr * 8) == size:
            return grid
    raise AssertionError((size, D, nr))


@pytest.mark.parametrize("sms", [1, 148, 160, 200, 700])
def test_the_join_has_room_for_the_parts_of_every_cta(tmp_path, sms):
    for name, rows, D, size in sizes(tmp_path, sms):
        bits8 = "attention8" in name
        nr = next(n for n in (8, 16, 32, 64, 128, 10 ** 6) if rows <= n)
        if bits8 and nr == 16:
            continue                         # either form may take these rows
        nr = min(nr, 128)
        grid = grid_of(size, D, nr)
        assert grid <= _lib.PAGED_COUNTER_BYTES // 4
        if nr == 8:                          # what this device's SMs hold at once: the library has asked for `sms`
            assert grid == min((3 if bits8 else 2) * sms, 1024)
        if nr >= 32:
            assert grid * nr * 8 <= ROOM and grid <= sms, (name, rows, D, grid)
            if sms <= 148:
                assert grid == sms
