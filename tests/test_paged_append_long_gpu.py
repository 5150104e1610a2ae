"""Appends of more tokens than the GPU holds CTAs, so that a CTA takes several: its ring of
loads goes round, slots, positions and rotary rows are fetched ahead.  Tolerances are those
of test_paged_cache_gpu.py's append."""
from __future__ import annotations

import pytest
import torch

from kernels import _lib
from kernels.paged_cache import paged_append, rope_table
from test_paged_cache_gpu import BF, DEV, FP, append_reference, cache, gen, near, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [593, 1777, 4001])
@pytest.mark.parametrize("Hq,Hk,D,R,ps,layout,dtype,norm,skip", [
    (8, 2, 128, 128, 16, "hnd", BF, True, 0.1), (14, 2, 64, 32, 24, "nhd", FP, False, 0.0),
    (3, 1, 64, 64, 7, "both", BF, True, 0.5), (32, 8, 128, 64, 1, "nhd", FP, True, 0.02)])
def test_many_tokens_match_64_bits(T, Hq, Hk, D, R, ps, layout, dtype, norm, skip):
    g = gen(T + Hq)
    pages = -(-T // ps) + 2
    kc, vc = cache(g, pages, Hk, ps, D, dtype, layout), cache(g, pages, Hk, ps, D, dtype, layout)
    k0, v0 = kc.clone(), vc.clone()
    qkv = randn(g, T, (Hq + 2 * Hk) * D, dtype=dtype)
    slots = torch.randperm(pages * ps, generator=g, device=DEV)[:T]
    slots[torch.rand(T, generator=g, device=DEV) < skip] = -1
    positions = torch.randint(0, 5000, (T,), generator=g, device=DEV)
    cos, sin = rope_table(5000, R, 1e6, DEV)
    qw = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(dtype) if norm else None
    kw = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(dtype) if norm else None
    qkv[slots < 0] = float("nan")
    with torch.inference_mode():
        q = paged_append(qkv, Hq, Hk, kc, vc, slots, positions, cos, sin, qw, kw, 1e-6)
    kept = slots >= 0
    rq, rk, rv, (mq, mk) = append_reference(qkv[kept], Hq, Hk, D, slots[kept], positions[kept], cos, sin, qw, kw, 1e-6)
    near(q[kept], rq, mq, dtype)
    assert bool((q[~kept] == 0).all())
    at = slots[kept]
    near(kc[at // ps, :, at % ps], rk, mk, dtype)
    assert torch.equal(vc[at // ps, :, at % ps].double(), rv)
    k0[at // ps, :, at % ps] = kc[at // ps, :, at % ps]
    v0[at // ps, :, at % ps] = vc[at // ps, :, at % ps]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)
    assert _lib.device_error() == 0
