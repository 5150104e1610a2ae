"""`paged_reserve` and `paged_append8` together: sequences that ask for less than L tokens, or that the pool cannot serve,
keep what they hold, number for number and scale for scale."""
from __future__ import annotations

import pytest
import torch

from kernels import _lib
from kernels.paged_cache import rope_table
from kernels.paged_cache8 import cache8, paged_append8
from kernels.paged_tables import page_pool, paged_reserve

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("ps,block", [(16, 16), (16, 4), (24, 24)])
def test_what_was_not_served_leaves_older_tokens_alone(ps, block):
    Hq, Hk, D, L = 4, 2, 64, 6
    g = torch.Generator(device=DEV).manual_seed(ps)
    lens = [ps - 2, 2 * ps, 5, 3 * ps - 1, 0, ps]
    held_pages = [-(-n // ps) for n in lens]
    B, pool = len(lens), sum(held_pages) + 2                      # two more pages than the sequences hold
    cos, sin = rope_table(512, D, 1e6, DEV)
    table, held, free, left = page_pool(B, 8, pool, DEV)
    cache = cache8(pool, Hk, ps, D, block, DEV)
    new = lambda n, scale: (torch.randn(B, n, (Hq + 2 * Hk) * D, generator=g, device=DEV) * scale).to(torch.bfloat16)  # noqa: E731
    with torch.inference_mode():
        start = torch.zeros_like(held)
        _, _, total = paged_reserve(table, start, held, free, left, max(lens), ps, ints(lens))
        paged_append8(new(max(lens), 1.0), Hq, Hk, *cache, table, total, cos, sin, count=total - start)
        assert total.tolist() == lens and left.tolist() == [2] and _lib.device_error() == 0
        rows = table.clone()
        before = [t.clone() for t in cache]
        asked = [6, 3, 0, 4, 2, 6]                                # 1 + 1 + 0 + 1 + 1 + 1 pages: the first two are served
        n = total.clone()
        _, _, total = paged_reserve(table, n, held, free, left, L, ps, ints(asked))
        served = (total - n).tolist()
        assert served == [6, 3, 0, 0, 0, 0] and _lib.device_error() & _lib.DEV_ERR_CAPACITY
        _lib.clear_device_error()
        # tokens a thousand times as large: a block that one of them reaches gets another scale
        q = paged_append8(new(L, 1000.0), Hq, Hk, *cache, table, total, cos, sin, count=total - n)
    assert _lib.device_error() == 0
    for b in range(B):
        assert bool((q[b, : L - served[b]] == 0).all()) and bool((q[b, L - served[b]:] != 0).any((-1, -2)).all())
        for j in range(0, lens[b], block):
            page, at = int(rows[b, j // ps]), j % ps
            if j + block > lens[b] and served[b]:                 # the open block of a sequence that went on
                continue
            for i in range(2):
                keep = slice(at, at + min(block, lens[b] - j))
                assert torch.equal(cache[i].view(torch.uint8)[page, :, keep], before[i].view(torch.uint8)[page, :, keep]), (b, j)
                assert torch.equal(cache[2 + i][page, :, at // block], before[2 + i][page, :, at // block]), (b, j)
