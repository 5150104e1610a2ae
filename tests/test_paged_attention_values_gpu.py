"""Values that are not finite, in keys that rows see and in keys that they do not, at every
number of rows per KV head; loads of long strides and of heads that share their keys.

Finite outputs: the bounds of test_paged_cache_gpu.py.  Others: +inf, -inf or NaN as in the
64-bit form (every weight there is well above the smallest 16-bit number).
"""
from __future__ import annotations

import math

import pytest
import torch

from kernels import _lib
from kernels.paged_cache import paged_attention
from test_paged_cache_gpu import BF, DEV, FP, U, cache, check_attention, gen, randn, tables

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


def check_values(q, kc, vc, table, lens, scale, tail, o):
    """As check_attention, for outputs that may be infinite or NaN."""
    B, L, Hq, D = q.shape
    Hk, ps = kc.shape[1], kc.shape[2]
    u = U[q.dtype]
    for b, n in enumerate(lens):
        pages = table[b, : -(-n // ps)].long()
        k = kc[pages].transpose(1, 2).reshape(-1, Hk, D)[:n].double()
        v = vc[pages].transpose(1, 2).reshape(-1, Hk, D)[:n].double()
        for t in range(L):
            see = torch.arange(n, device=DEV) < n - L
            for i in range(max(0, L - n), L):
                see[n - L + i] = i <= t if tail is None else bool(tail[t, i])
            got = o[b, t].double()
            if not bool(see.any()):
                assert bool((got == 0).all())
                continue
            z = torch.einsum("hgd,nhd->hgn", q[b, t].double().view(Hk, Hq // Hk, D), k[see]) * scale
            p = torch.softmax(z, -1)[..., None]                                  # [Hk, G, n, 1]
            terms = p * v[see].transpose(0, 1)[:, None]
            ref, spread = terms.sum(2).reshape(Hq, D), terms.abs().sum(2).reshape(Hq, D)
            fine = ref.isfinite()
            assert torch.equal(got.isnan(), ref.isnan()), (b, t)
            assert torch.equal(got.isposinf(), ref.isposinf()) and torch.equal(got.isneginf(), ref.isneginf()), (b, t)
            bound = (u + 2.0 ** -12) * spread + u * ref.abs() + 2.0 ** -24
            assert bool(((got - ref).abs() <= bound)[fine].all()), (b, t)


ROWS = [(2, 8, 2), (4, 8, 2), (5, 8, 2), (8, 8, 2), (16, 8, 2), (32, 8, 2), (40, 8, 2)]     # 8 .. 160 rows a KV head


@pytest.mark.parametrize("L,Hq,Hk", ROWS)
@pytest.mark.parametrize("D,ps,dtype,where", [(128, 16, BF, "one"), (64, 24, FP, "one"), (128, 7, FP, "many"),
                                              (64, 16, BF, "many"), (128, 16, BF, "both signs")])
def test_infinite_values_of_old_keys_stay_infinite(L, Hq, Hk, D, ps, dtype, where):
    g = gen(L + D)
    lens = [700, 333, 150]
    table, pages = tables(g, lens, ps)
    kc, vc = cache(g, pages, Hk, ps, D, dtype, "hnd"), cache(g, pages, Hk, ps, D, dtype, "hnd")
    q = randn(g, len(lens), L, Hq, D, dtype=dtype)
    for b, n in enumerate(lens):
        for i, j in enumerate({"one": [n // 2], "many": [0, 3, 40, 41, 70, 100, n - L - 1],
                               "both signs": [2, 60, n - L - 2]}[where]):
            vc[table[b, j // ps].long(), 0, j % ps, 5] = -INF if where == "both signs" and i == 1 else INF
            vc[table[b, j // ps].long(), Hk - 1, j % ps, (9 * i + 1) % D] = -INF
    with torch.inference_mode():
        o, lse = paged_attention(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=DEV), return_lse=True)
    check_values(q, kc, vc, table, lens, D ** -0.5, None, o)
    assert bool(lse.isfinite().all()) and _lib.device_error() == 0


@pytest.mark.parametrize("L,Hq,Hk", [(2, 8, 2), (4, 8, 2), (8, 2, 2), (3, 5, 1), (16, 1, 1), (8, 8, 2), (16, 8, 2), (32, 8, 2)])
@pytest.mark.parametrize("D,ps,dtype,masked", [(128, 16, BF, False), (64, 24, FP, True), (128, 5, FP, False),
                                               (64, 16, BF, True)])
@pytest.mark.parametrize("bad,keys", [(INF, False), (NAN, False), (NAN, True)])
def test_values_of_drafted_tokens_reach_the_rows_that_see_them(L, Hq, Hk, D, ps, dtype, masked, bad, keys):
    g = gen(L * Hq + D)
    lens = [300, L, 21 + L]
    table, pages = tables(g, lens, ps)
    kc, vc = cache(g, pages, Hk, ps, D, dtype, "nhd"), cache(g, pages, Hk, ps, D, dtype, "nhd")
    for b, n in enumerate(lens):
        for j in {n - 1, n - 1 - L // 3}:
            at = table[b, j // ps].long(), j % ps
            vc[at[0], :, at[1], 3] = bad
            vc[at[0], Hk - 1, at[1], D - 1] = bad
            if keys:
                kc[at[0], 0, at[1], 7] = bad
    q = randn(g, len(lens), L, Hq, D, dtype=dtype)
    mask = None
    if masked:
        mask = torch.rand(L, L, generator=g, device=DEV) < 0.5
        mask[0] = False
    with torch.inference_mode():
        o = paged_attention(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=DEV), tail_mask=mask)
    check_values(q, kc, vc, table, lens, D ** -0.5, mask, o)


@pytest.mark.parametrize("L,D,ps,dtype,lens", [(8, 128, 16, BF, [300, 5, 129]), (5, 64, 48, FP, [1000, 0, 64]),
                                               (32, 128, 32, BF, [257, 40]), (4, 64, 16, BF, [4000]), (16, 128, 64, FP, [700, 90]),
                                               (2, 128, 16, BF, [300, 5, 129])])
def test_heads_that_share_one_cache(L, D, ps, dtype, lens):
    """A head stride of 0 (one cache expanded over the KV heads), for which there is no TMA map."""
    g = gen(L + ps)
    Hk, Hq = 4, 16
    table, pages = tables(g, lens, ps)
    kc, vc = (cache(g, pages, 1, ps, D, dtype, "hnd").expand(pages, Hk, ps, D) for _ in range(2))
    q = randn(g, len(lens), L, Hq, D, dtype=dtype, scale=2.0)
    with torch.inference_mode():
        o, lse = paged_attention(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=DEV), return_lse=True)
    check_attention(q, kc, vc, table, lens, D ** -0.5, None, o, lse)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("L", [8, 16, 32])
def test_offsets_past_32_bits_with_many_rows(L):
    """Pages 2^30 elements apart: page 3 starts past the 32-bit range, in elements and in bytes."""
    g = gen(L)
    ps, Hk, D, step = 16, 2, 128, 1 << 30
    raw = [torch.empty(3 * step + Hk * ps * D, dtype=BF, device=DEV) for _ in range(2)]
    kc, vc = (r.as_strided((4, Hk, ps, D), (step, ps * D, D, 1)) for r in raw)
    kc.copy_(randn(g, 4, Hk, ps, D))
    vc.copy_(randn(g, 4, Hk, ps, D))
    table = torch.tensor([[3, 1, 2, 0]], dtype=torch.int32, device=DEV)
    q = randn(g, 1, L, 8, D)
    with torch.inference_mode():
        o, lse = paged_attention(q, kc, vc, table, torch.tensor([61], dtype=torch.int32, device=DEV), return_lse=True)
    check_attention(q, kc, vc, table, [61], D ** -0.5, None, o, lse)
