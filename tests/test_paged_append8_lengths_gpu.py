"""`paged_append8` of sequences whose lengths are past every table, up to the largest 32-bit number: flagged, and
nothing of the cache is written."""
from __future__ import annotations

import pytest
import torch

from kernels import _lib
from kernels.paged_cache import rope_table
from kernels.paged_cache8 import cache8, paged_append8

pytestmark = pytest.mark.gpu
DEV = "cuda"
MAX = 0x7FFFFFFF


@pytest.mark.parametrize("D,ps,block", [(128, 16, 16), (64, 16, 4), (128, 7, 1), (64, 48, 24), (128, 128, 128)])
@pytest.mark.parametrize("L,count", [(1, None), (2, None), (4, 1), (300, 7), (2048, 10), (33, 0)])
def test_lengths_past_the_tables_are_flagged_and_write_nothing(D, ps, block, L, count):
    Hq, Hk, lens = 2, 1, [MAX, MAX - 1, MAX - 15, 0x7FFFF810, 0x7FFFF7FF, 0x7FFF0001, 0x40000000, 20]
    B = len(lens)
    g = torch.Generator(device=DEV).manual_seed(L + ps)
    pages = -(-2100 // ps) + 1
    cache = cache8(pages * B, Hk, ps, D, block, DEV)
    for t in cache[:2]:
        t.view(torch.uint8).random_(0, 120, generator=g)
    for t in cache[2:]:
        t.fill_(0.5)
    before = [t.clone() for t in cache]
    table = torch.arange(pages * B, dtype=torch.int32, device=DEV).view(B, pages)
    cos, sin = rope_table(4096, D, 1e6, DEV)
    qkv = torch.randn(B, L, (Hq + 2 * Hk) * D, generator=g, device=DEV).to(torch.bfloat16)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    with torch.inference_mode():
        q = paged_append8(qkv, Hq, Hk, *cache, table, ints(lens), cos, sin, count=None if count is None else ints([count] * B))
    flagged = bool(_lib.device_error() & _lib.DEV_ERR_BAD_INDEX)
    _lib.clear_device_error()
    new = L if count is None else count
    assert flagged == (new > 0)
    assert bool((q[:-1] == 0).all())
    # the last one is as it would be alone: its new tokens in its own pages, the others' pages as they were
    kept = min(new, 20)
    assert bool((q[-1, L - kept:].float().abs().amax((-1, -2)) > 0).all()) and bool((q[-1, : L - kept] == 0).all())
    for a, b in zip(before, cache):
        assert torch.equal(a[: pages * (B - 1)].view(torch.uint8), b[: pages * (B - 1)].view(torch.uint8))
