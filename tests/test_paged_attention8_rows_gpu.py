"""Attention over the 8-bit cache at every number of rows a KV head (query heads of a group times tokens) around those
where it takes its rows another way, against 64 bits (bounds: test_paged_cache8_gpu.py)."""
from __future__ import annotations

import pytest
import torch

from kernels import _lib
from kernels.paged_cache8 import paged_attention8
from test_paged_cache8_gpu import BF, DEV, FP, cache_of, check_attention, gen, ints, poison, randn, spread_scales, stale, tables, values

pytestmark = pytest.mark.gpu


# query heads of a group, tokens
@pytest.mark.parametrize("G,L", [(8, 1), (9, 1), (3, 3), (2, 5), (11, 1), (4, 3), (13, 1), (7, 2), (5, 3), (4, 4), (16, 1), (1, 16),
                                 (17, 1), (1, 17), (3, 6), (8, 4), (33, 1)])
@pytest.mark.parametrize("D,ps,block,dtype,window,mask", [(128, 16, 16, BF, None, False), (64, 24, 8, FP, 90, False),
                                                          (128, 7, 1, FP, None, True), (64, 64, 64, BF, 200, True)])
def test_rows_match_64_bits(G, L, D, ps, block, dtype, window, mask):
    g = gen(100 * G + L + D)
    Hk, lens = 2, [700, 0, 129, 5, 2048]
    B = len(lens)
    table, pages = tables(g, lens, ps)
    k, ks = cache_of(g, pages, Hk, ps, D, block)
    v, vs = cache_of(g, pages, Hk, ps, D, block)
    free = stale(table, lens, pages, ps)
    poison(k, ks, free)
    poison(v, vs, free)
    q = randn(g, B, L, G * Hk, D, dtype=dtype, scale=2.0)
    tail = None
    if mask:
        tail = torch.rand(B, L, L, generator=g, device=DEV) < 0.5
        tail[:, 0] = False
    sinks = 3 if window else 0
    with torch.inference_mode():
        o, lse = paged_attention8(q, k, v, ks, vs, table, ints(lens), tail_mask=tail, return_lse=True, window=window, sinks=sinks)
        again = paged_attention8(q, k, v, ks, vs, table, ints(lens), tail_mask=tail, window=window, sinks=sinks)
    check_attention(q, values(k, ks), values(v, vs), spread_scales(vs, ps), table, lens, D ** -0.5, tail, o, lse, window, sinks)
    assert torch.equal(o, again) and _lib.device_error() == 0
