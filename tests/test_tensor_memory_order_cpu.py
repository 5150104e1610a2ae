"""Order of tensor-memory accesses in the tcgen05 attention kernels, read from their source: after a wait on a
barrier that says that the tensor cores, or other threads, are done with a piece of tensor memory, the waiting
thread's next access of it comes after a `tc_fence_after()` that it cannot have jumped over."""
from __future__ import annotations

import re

import pytest

from conftest import PKG

FILES = sorted(p.name for p in (PKG / "csrc").glob("paged_attn*_tc.cuh"))
# barriers that products or tensor-memory stores complete
WAIT = r"wait(?:_all)?\s*\(\s*(?:smem_u32\s*\(\s*)?(?:s_full|p_full|q_full|pv_done|drained)\b"
TOKEN = re.compile(rf"(?P<open>{{)|(?P<close>}})|(?P<fence>\btc_fence_after\(\))|(?P<wait>\b(?:mbar_)?{WAIT})"
                   r"|(?P<access>\b(?:tmem_ld16|ptc_st16|ptc_mma)\s*\()")


def unordered(text: str) -> list[int]:
    """Lines of accesses that some wait before them reaches without a fence in between.  A block starts with what
    holds before it, and what is fenced inside it (it may not run) does not count behind it."""
    text = re.sub(r"//[^\n]*", "", text)
    state, bad = [True], []
    for t in TOKEN.finditer(text):
        if t["open"]:
            state.append(state[-1])
        elif t["close"]:
            state.pop()
        elif t["fence"]:
            before = text[:t.start()].rstrip()
            state[-1] = state[-1] or before[-1] in ";{}"          # not the statement of an if
        elif t["wait"]:
            state[-1] = False
        elif not state[-1]:
            bad.append(text.count("\n", 0, t.start()) + 1)
    assert state == [True], "braces do not match"
    return bad


def test_the_reading_finds_a_fence_that_may_be_jumped_over():
    wait, store = "if (!wait_all(pv_done, 1)) break;", "ptc_st16(at, x);"
    assert unordered(f"{{ {wait} tc_fence_after(); {store} }}") == []
    assert unordered(f"{{ if (n > 0) {{ {wait} tc_fence_after(); }} {store} }}") == []
    assert unordered(f"{{ {wait} {store} }}") == [1]
    assert unordered(f"{{ {wait} if (up) {{ tc_fence_after(); {store} }} \n {store} }}") == [2]
    assert unordered(f"{{ {wait} if (up) tc_fence_after(); {store} }}") == [1]


@pytest.mark.parametrize("name", FILES)
def test_tensor_memory_is_accessed_after_a_fence(name):
    text = (PKG / "csrc" / name).read_text()
    assert len(re.findall(WAIT, text)) >= 5 and unordered(text) == []


def test_both_kernels_are_read():
    assert FILES == ["paged_attn8_tc.cuh", "paged_attn_tc.cuh"]
