"""A window that no key of the table lies behind is no window, bit for bit and for every number of rows: the call takes the
form that it takes without one."""
from __future__ import annotations

import pytest
import torch

from kernels.paged_cache import paged_attention
from kernels.paged_cache8 import cache8, paged_attention8

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("L,Hq,Hk,D,mask", [(1, 8, 2, 128, False), (4, 8, 2, 128, False), (8, 8, 2, 128, True), (32, 8, 2, 128, False),
                                            (40, 8, 2, 64, True), (9, 4, 2, 64, False), (17, 32, 8, 128, True)])
def test_a_window_as_long_as_the_table_is_none(bits, L, Hq, Hk, D, mask):
    g = torch.Generator(device=DEV).manual_seed(L)
    lens, ps, B = [1500, 64, 3, 2048], 16, 4
    places = 2048
    table = torch.randperm(B * places // ps, generator=g, device=DEV).to(torch.int32).view(B, -1)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = torch.randn(B, L, Hq, D, generator=g, device=DEV).to(torch.bfloat16)
    tail = torch.rand(L, L, generator=g, device=DEV) < 0.6 if mask else None
    k, v = (torch.randn(B * places // ps, Hk, ps, D, generator=g, device=DEV) for _ in range(2))
    if bits == 16:
        attend = lambda **kw: paged_attention(q, k.bfloat16(), v.bfloat16(), table, n, tail_mask=tail, return_lse=True, **kw)  # noqa: E731
    else:
        cache = cache8(B * places // ps, Hk, ps, D, 16, DEV)
        for to, x in zip(cache, (k, v)):
            to.copy_((x * 64).clamp(-448, 448))
        for s in cache[2:]:
            s.fill_(2.0 ** -6)
        attend = lambda **kw: paged_attention8(q, *cache, table, n, tail_mask=tail, return_lse=True, **kw)  # noqa: E731
    with torch.inference_mode():
        want = attend()
        for window, sinks in ((places, 0), (places + 1, 7), (1 << 30, 3), (1 << 45, 1 << 45)):
            for a, b in zip(want, attend(window=window, sinks=sinks)):
                assert torch.equal(a, b), (window, sinks)
        # one token less: the form that counts it.  Nothing of the first three is hidden, so that both are the same sums of
        # p_j v_j, each with weights and output rounded once to bf16 at most: 2 (2^-8 + 2^-8) max |v|
        o, lse = attend(window=places - 1)
        assert float((o.float() - want[0].float())[:3].abs().max()) <= 2.0 ** -6 * float(v.abs().max())
