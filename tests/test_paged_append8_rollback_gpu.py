"""Tokens that are taken back from the 8-bit cache: the block that they ended in may keep a scale that only they needed,
and its kept tokens are as far off as that scale's smallest numbers are apart, no further."""
from __future__ import annotations

import pytest
import torch

from kernels import _lib
from kernels.paged_cache import rope_table
from kernels.paged_cache8 import F8, cache8, paged_append8

pytestmark = pytest.mark.gpu
DEV = "cuda"


def values(cache, i, page, block):
    return cache[i].view(torch.uint8)[page].view(F8).double() * cache[2 + i][page].double().repeat_interleave(block, -1)[..., None]


@pytest.mark.parametrize("ps,block", [(16, 16), (32, 8), (64, 64)])
@pytest.mark.parametrize("size", [1.0, 30.0, 3000.0])
def test_rejected_drafts_bound_the_error_of_kept_tokens(ps, block, size):
    Hq, Hk, D, kept, drafted = 2, 2, 64, block - 5, 4
    g = torch.Generator(device=DEV).manual_seed(int(size) + ps)
    ints = lambda v: torch.tensor([v], dtype=torch.int32, device=DEV)  # noqa: E731
    cos, sin = rope_table(256, 0, 1e6, DEV)                       # no rotation, no norm: keys and values are the rows' own
    cache, table = cache8(3, Hk, ps, D, block, DEV), torch.tensor([[1, 2]], dtype=torch.int32, device=DEV)
    rows = lambda n, f: (torch.randn(1, n, (Hq + 2 * Hk) * D, generator=g, device=DEV) * f).to(torch.bfloat16)  # noqa: E731
    old, outliers, new = rows(kept, 1.0), rows(drafted, size), rows(2, 1.0)
    with torch.inference_mode():
        paged_append8(old, Hq, Hk, *cache, table, ints(kept), cos, sin)
        own = [s[1].clone() for s in cache[2:]]
        paged_append8(outliers, Hq, Hk, *cache, table, ints(kept + drafted), cos, sin)
        raised = [s[1].clone() for s in cache[2:]]
        paged_append8(new, Hq, Hk, *cache, table, ints(kept + 2), cos, sin)
        for i in range(2):
            at = slice((Hq + i * Hk) * D, (Hq + (i + 1) * Hk) * D)
            for part, j in ((old, 0), (new, kept)):
                x = part[0, :, at].double().view(-1, Hk, D).transpose(0, 1)
                got = values(cache, i, 1, block)[:, j: j + x.shape[1]]
                # a token is rounded once at the scale it was written with and once at the one that was raised
                first = own[i] if j == 0 else raised[i]
                s0, s1 = (s.double()[:, :1, None] for s in (first, raised[i]))
                bound = torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -10 * s0) + torch.where(s1 > s0, 2.0 ** -10 * s1, 0.0)
                assert bool(((got - x).abs() <= bound).all()), (i, j, float(((got - x).abs() / bound).max()))
            top = outliers[0, :, at].double().abs().amax()
            assert float(raised[i][:, 0].max()) >= float(top) / 448 and float(raised[i][:, 0].max()) <= float(top) / 224 + 1
            assert torch.equal(cache[2 + i][1, :, 0], raised[i][:, 0])        # it does not come down ..
        paged_append8(rows(3, 1.0), Hq, Hk, *cache, table, ints(3), cos, sin)
        if size == 3000.0:
            assert bool((cache[2][1, :, 0] < raised[0][:, 0]).all())          # .. until the block's first token is written anew
    assert _lib.device_error() == 0
