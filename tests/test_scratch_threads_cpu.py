"""Calls that share a stream's scratch are made with the GIL held, so that no other thread's
launch comes between the two of a verification."""
from __future__ import annotations

import ctypes
import threading
import time

import pytest

from kernels import _lib

FUNCFLAG_PYTHONAPI = 4                 # ctypes: the GIL is kept over the call


@pytest.mark.parametrize("name", ["simsd_paged_attention", "simsd_speculative_verify"])
def test_the_gil_is_held(name):
    fn = getattr(_lib.lib(), name)
    assert type(fn)._flags_ & FUNCFLAG_PYTHONAPI
    assert (fn.restype, list(fn.argtypes)) == (_lib.SIGNATURES[name][0], _lib.SIGNATURES[name][1])


def test_the_ctypes_way_goes_through_them():
    """The same function objects are what paged_attention and speculative_verify call and what the binding is bound to."""
    plain = ctypes.CDLL(str(_lib.LIB_PATH))
    for name in ("simsd_paged_attention", "simsd_speculative_verify"):
        assert getattr(_lib.lib(), name) is getattr(_lib.lib(), name)
        at = lambda f: ctypes.cast(f, ctypes.c_void_p).value  # noqa: E731
        assert at(getattr(_lib.lib(), name)) == at(getattr(plain, name))


def test_a_held_call_keeps_other_threads_out():
    """What the flag does: during such a call no other thread runs Python."""
    libc = ctypes.PyDLL(None)
    ticks, stop = [], threading.Event()

    def tick():
        while not stop.is_set():
            ticks.append(time.perf_counter())

    t = threading.Thread(target=tick)
    t.start()
    time.sleep(0.05)
    a = time.perf_counter()
    libc.usleep(200000)
    b = time.perf_counter()
    stop.set()
    t.join()
    assert not [x for x in ticks if a + 0.02 < x < b - 0.02]
