"""Appends to blocks whose scale is no power of two (a cache that was quantised elsewhere).

A new number is multiplied by the scale's fp32 reciprocal (2^-24 off, and the product 2^-24) and rounded to e4m3: half a
step, 2^-4 of it or 2^-10 s, and 2^-22 of it for the rest.  Where the scale grows it becomes a power of two, and an older
number is multiplied by the ratio (exact but for one rounding) and rounded once: the same bound."""
from __future__ import annotations

import pytest
import torch

from kernels import _lib
from kernels.paged_cache import rope_table
from kernels.paged_cache8 import F8, paged_append8
from test_paged_cache8_gpu import BF, DEV, cache_of, gen, ints, power, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ps,block,n,c", [(16, 16, 11, 3), (16, 4, 31, 1), (24, 24, 40, 7), (64, 64, 60, 40), (7, 7, 20, 4)])
@pytest.mark.parametrize("size", [0.01, 1.0, 50.0])
def test_append_to_other_scales(ps, block, n, c, size):
    g = gen(n + ps)
    Hq, Hk, D = 2, 3, 64
    table, pages = tables(g, [n], ps)
    k, ks = cache_of(g, pages, Hk, ps, D, block, pow2=False)
    v, vs = cache_of(g, pages, Hk, ps, D, block, pow2=False)
    before = [t.clone() for t in (k, v, ks, vs)]
    cos, sin = rope_table(64, 0, 1e6, DEV)                        # no rotation, no norm: keys and values are the rows' own
    qkv = (torch.randn(1, c, (Hq + 2 * Hk) * D, generator=g, device=DEV) * size).to(BF)
    with torch.inference_mode():
        paged_append8(qkv, Hq, Hk, k, v, ks, vs, table, ints([n]), cos, sin)
    assert _lib.device_error() == 0
    old = n - c
    for i, (cache, scale) in enumerate(((k, ks), (v, vs))):
        x = qkv[0, :, (Hq + i * Hk) * D: (Hq + (i + 1) * Hk) * D].double().view(c, Hk, D)
        for lo in range(old // block * block, n, block):
            page, at = int(table[0, lo // ps]), lo % ps
            first, last = max(lo, old), min(lo + block, n)
            new = x[first - old: last - old].transpose(0, 1)
            s, s0 = scale[page, :, at // block].double(), before[2 + i][page, :, at // block].double()
            want = power(new.abs().amax((1, 2)))
            assert torch.equal(s, torch.maximum(s0, want) if lo < old else want)
            s = s[:, None, None]
            got = cache.view(torch.uint8)[page, :, at: at + last - lo].view(F8).double() * s
            held = before[i].view(torch.uint8)[page, :, at: at + first - lo].view(F8).double() * s0[:, None, None]
            for a, b in ((got[:, : first - lo], held), (got[:, first - lo:], new)):
                bound = torch.maximum(2.0 ** -4 * b.abs(), 2.0 ** -10 * s) + 2.0 ** -22 * b.abs()
                assert bool(((a - b).abs() <= bound).all()), (i, lo)
            same = (s[:, 0, 0] == s0) & (lo < old)                # a scale that has not grown leaves older numbers alone
            assert torch.equal(got[same, : first - lo], held[same])
