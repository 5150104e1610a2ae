"""Paged key-value cache (kernels/paged_cache.py) against a plain 64-bit
implementation.

Tolerances.  u is half a step of the 16-bit type relative to the value (2^-8
bf16, 2^-11 fp16).  Append: one rounding, u |ref|, plus the 32-bit arithmetic
before it, 2^-20 of |a c| + |b s| (a dot of <= 13 dependent additions, rsqrt and
three products), plus half the smallest fp16 step.  Attention: with spread =
sum_j p_j |v_j| and d = 2^-20 scale max_j sum_i |q_i k_ji| the error of a score,
the weights may be rounded to 16 bits for the second product (u spread), every
weight moves by 2 d + 2^-16 (score, exponential, and up to 256 dependent
additions), and o is rounded once (u |ref|).  lse: d + 2^-16 + 2^-22 |lse|.
"""
from __future__ import annotations

import math

import pytest
import torch

from kernels import _lib
from kernels.paged_cache import paged_append, paged_attention, rope_table

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16
U = {BF: 2.0 ** -8, FP: 2.0 ** -11}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def cache(g, pages, Hk, ps, D, dtype, layout):
    if layout == "nhd":
        return randn(g, pages, ps, Hk, D, dtype=dtype).transpose(1, 2)
    if layout == "both":     # k or v of a [pages, 2, Hk, ps, D] allocation
        return randn(g, pages, 2, Hk, ps, D, dtype=dtype)[:, 1]
    return randn(g, pages, Hk, ps, D, dtype=dtype)


# ------------------------------------------------------------------ append
def append_reference(qkv, Hq, Hk, D, slots, positions, cos, sin, qw, kw, eps):
    """(q, k, v, magnitude) in 64 bits, [T, heads, D]."""
    x = qkv.double().view(qkv.shape[0], Hq + 2 * Hk, D)
    R = 2 * cos.shape[1]
    c, s = cos.double()[positions][:, None], sin.double()[positions][:, None]
    out, mag = [], []
    for part, w in ((x[:, :Hq], qw), (x[:, Hq:Hq + Hk], kw)):
        if w is not None:
            part = part / (part.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
        a, b, rest = part[..., : R // 2], part[..., R // 2: R], part[..., R:]
        out.append(torch.cat([a * c - b * s, b * c + a * s, rest], -1))
        mag.append(torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), rest.abs()], -1))
    return out[0], out[1], x[:, Hq + Hk:], mag


def near(got, ref, mag, dtype):
    bound = U[dtype] * ref.abs() + 2.0 ** -20 * mag * (1 + U[dtype]) + (2.0 ** -25 if dtype == FP else 2.0 ** -130)
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("T,Hq,Hk,D,R,ps,layout,dtype,norm,skip", [
    (1, 32, 8, 128, 128, 16, "hnd", BF, True, 0.0), (5, 32, 8, 128, 64, 1, "nhd", BF, True, 0.3),
    (77, 14, 2, 64, 32, 24, "both", FP, False, 0.2), (33, 3, 1, 64, 64, 7, "hnd", FP, True, 0.0),
    (300, 4, 4, 128, 0, 64, "nhd", BF, False, 0.0), (2, 64, 8, 128, 112, 16, "both", BF, True, 0.5),
    (130, 7, 1, 64, 16, 5, "nhd", BF, True, 0.9)])
def test_append_matches_64_bits(T, Hq, Hk, D, R, ps, layout, dtype, norm, skip):
    g = gen(T + Hq)
    pages = -(-T // ps) + 2
    kc, vc = cache(g, pages, Hk, ps, D, dtype, layout), cache(g, pages, Hk, ps, D, dtype, layout)
    k0, v0 = kc.clone(), vc.clone()
    qkv = randn(g, T, (Hq + 2 * Hk) * D + 8, dtype=dtype)[:, : (Hq + 2 * Hk) * D]      # rows apart
    slots = torch.randperm(pages * ps, generator=g, device=DEV)[:T]
    slots[torch.rand(T, generator=g, device=DEV) < skip] = -1
    positions = torch.randint(0, 5000, (T,), generator=g, device=DEV)
    cos, sin = rope_table(5000, R, 1e6, DEV)
    qw = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(dtype) if norm else None
    kw = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(dtype) if norm else None
    qkv[slots < 0] = float("nan")                          # padding rows hold anything
    positions[slots < 0] = -7
    with torch.inference_mode():
        q = paged_append(qkv, Hq, Hk, kc, vc, slots, positions, cos, sin, qw, kw, 1e-6)
    kept = slots >= 0
    rq, rk, rv, (mq, mk) = append_reference(qkv[kept], Hq, Hk, D, slots[kept], positions[kept], cos, sin, qw, kw, 1e-6)
    assert q.shape == (T, Hq, D)
    near(q[kept], rq, mq, dtype)
    assert bool((q[~kept] == 0).all())
    at = slots[kept]
    near(kc[at // ps, :, at % ps], rk, mk, dtype)
    assert torch.equal(vc[at // ps, :, at % ps].double(), rv)
    k0[at // ps, :, at % ps] = kc[at // ps, :, at % ps]
    v0[at // ps, :, at % ps] = vc[at // ps, :, at % ps]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)     # no other slot moved
    assert _lib.device_error() == 0


def test_append_bad_indices_are_flagged_and_skipped():
    g = gen(1)
    kc, vc = cache(g, 4, 2, 16, 64, BF, "hnd"), cache(g, 4, 2, 16, 64, BF, "hnd")
    k0, v0 = kc.clone(), vc.clone()
    qkv = randn(g, 3, 8 * 64)
    cos, sin = rope_table(10, 64, 1e6, DEV)
    slots = torch.tensor([64, 3, 1 << 40], device=DEV)
    positions = torch.tensor([0, 10, 0], device=DEV)       # slot 3's position lies past the table
    with torch.inference_mode():
        q = paged_append(qkv, 4, 2, kc, vc, slots, positions, cos, sin)
    assert _lib.device_error() & _lib.DEV_ERR_BAD_INDEX
    _lib.clear_device_error()
    assert torch.equal(kc, k0) and torch.equal(vc, v0) and bool((q == 0).all())


def test_append_of_no_tokens():
    g = gen(2)
    kc, vc = cache(g, 4, 2, 16, 64, BF, "hnd"), cache(g, 4, 2, 16, 64, BF, "hnd")
    cos, sin = rope_table(10, 64, 1e6, DEV)
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    with torch.inference_mode():
        assert paged_append(randn(g, 0, 8 * 64), 4, 2, kc, vc, none, none, cos, sin).shape == (0, 4, 64)


# ------------------------------------------------------------------ attention
def tables(g, lens, ps, spare=2, junk=-1):
    """(page_table, pages): every sequence's pages in any order, `junk` after its last."""
    need = [-(-n // ps) for n in lens]
    pages, width = sum(need) + spare, max(max(need), 1)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    t = torch.full((len(lens), width), junk, dtype=torch.int32, device=DEV)
    at = 0
    for b, k in enumerate(need):
        t[b, :k] = order[at:at + k]
        at += k
    return t, pages


def check_attention(q, kc, vc, table, lens, scale, tail, o, lse):
    B, L, Hq, D = q.shape
    Hk, ps = kc.shape[1], kc.shape[2]
    G, u = Hq // Hk, U[q.dtype]
    for b, n in enumerate(lens):
        pages = table[b, : -(-n // ps)].long()
        k = kc[pages].transpose(1, 2).reshape(-1, Hk, D)[:n].double()        # [n, Hk, D]
        v = vc[pages].transpose(1, 2).reshape(-1, Hk, D)[:n].double()
        for t in range(L):
            see = torch.arange(n, device=DEV) < n - L
            for i in range(max(0, L - n), L):
                see[n - L + i] = i <= t if tail is None else bool((tail if tail.ndim == 2 else tail[b])[t, i])
            got, gl = o[b, t].double(), lse[b, t].double()
            if not bool(see.any()):
                assert bool((got == 0).all()) and bool((gl == -math.inf).all()), (b, t)
                continue
            qq = q[b, t].double().view(Hk, G, D)
            z = torch.einsum("hgd,nhd->hgn", qq, k[see]) * scale
            p = torch.softmax(z, -1)
            d = torch.einsum("hgd,nhd->hgn", qq.abs(), k[see].abs()).amax(-1).view(Hq) * abs(scale) * 2.0 ** -20
            ref = torch.einsum("hgn,nhd->hgd", p, v[see]).reshape(Hq, D)
            spread = torch.einsum("hgn,nhd->hgd", p, v[see].abs()).reshape(Hq, D)
            bound = (u + 2 * d[:, None] + 2.0 ** -16) * spread + u * ref.abs() + (2.0 ** -25 if u == U[FP] else 0) + 1e-30
            err = (got - ref).abs()
            assert bool((err <= bound).all()), (b, t, n, float((err / bound).max()))
            rl = torch.logsumexp(z, -1).view(Hq)
            el = (gl - rl).abs()
            assert bool((el <= d + 2.0 ** -16 + 2.0 ** -22 * rl.abs()).all()), (b, t, n, float(el.max()))


# lengths around tile, page and split edges; groups of 1 to 16 query heads; 1 to 40 rows a head;
# pages of one token, odd pages, pages larger than any sequence
ATT = [
    ([1], 1, 32, 8, 128, 16, "hnd", BF, None), ([0, 1, 2, 0], 1, 8, 8, 128, 16, "nhd", BF, None),
    ([15, 16, 17, 63, 64, 65, 127, 128, 129], 1, 32, 8, 128, 16, "hnd", BF, None),
    ([1000, 3, 0, 517], 1, 16, 1, 128, 1, "nhd", BF, None), ([700, 701], 1, 14, 2, 64, 24, "both", FP, None),
    ([333, 40, 1], 1, 5, 5, 64, 7, "hnd", FP, None), ([5000], 1, 32, 8, 128, 16, "hnd", BF, None),
    ([20000, 100], 1, 8, 2, 128, 64, "nhd", FP, None), ([2048] * 3, 1, 8, 8, 64, 4096, "hnd", BF, None),
    ([4, 5, 100, 0, 2, 1], 4, 32, 8, 128, 16, "hnd", BF, None),            # shorter than its queries: rows see nothing
    ([64, 200, 1500], 8, 32, 8, 128, 16, "nhd", BF, "each"), ([90, 130], 5, 40, 8, 128, 32, "hnd", FP, "one"),
    ([300, 37, 16], 16, 16, 2, 64, 24, "both", BF, "each"), ([777, 12], 3, 12, 1, 64, 8, "nhd", FP, "each"),
    ([513, 40], 40, 8, 8, 128, 16, "hnd", BF, "one"), ([257, 31], 33, 6, 2, 64, 16, "hnd", BF, None),
    # 17 to 128 rows and more, pages of other than 8 tokens among them
    ([200, 65, 5, 0], 8, 16, 2, 128, 7, "hnd", BF, "each"), ([130, 300], 6, 32, 8, 64, 1, "nhd", FP, None),
    ([1000, 129, 128, 127], 32, 32, 8, 128, 16, "hnd", BF, "each"), ([2500, 12], 20, 20, 4, 128, 40, "both", FP, "one"),
    ([260, 3], 70, 2, 1, 128, 64, "nhd", BF, "one"), ([6000], 4, 32, 4, 128, 128, "hnd", BF, None),
    ([9000, 8000], 17, 8, 2, 64, 8, "nhd", BF, None), ([640] * 9, 1, 24, 1, 128, 16, "hnd", BF, None),
    ([10] * 200, 1, 8, 4, 64, 16, "hnd", BF, None), ([0] * 5, 2, 4, 2, 128, 16, "hnd", BF, None),
]


@pytest.mark.parametrize("lens,L,Hq,Hk,D,ps,layout,dtype,tail", ATT)
def test_attention_matches_64_bits(lens, L, Hq, Hk, D, ps, layout, dtype, tail):
    g = gen(sum(lens) + Hq)
    B = len(lens)
    table, pages = tables(g, lens, ps)
    kc, vc = cache(g, pages, Hk, ps, D, dtype, layout), cache(g, pages, Hk, ps, D, dtype, layout)
    used = torch.zeros(pages * ps, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        j = torch.arange(n, device=DEV)
        used[table[b, j // ps].long() * ps + j % ps] = True
    free = ~used.view(pages, 1, ps, 1)
    kc.masked_fill_(free, float("nan"))                    # stale memory holds anything
    vc.masked_fill_(free, float("inf"))
    q = randn(g, B, L, Hq, D, dtype=dtype, scale=2.0)
    mask = None
    if tail is not None:
        mask = torch.rand(*((B,) if tail == "each" else ()), L, L, generator=g, device=DEV) < 0.5
        mask[..., 0, :] = False
    with torch.inference_mode():
        o, lse = paged_attention(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=DEV), tail_mask=mask,
                                 return_lse=True)
    assert o.shape == q.shape and lse.shape == (B, L, Hq)
    check_attention(q, kc, vc, table, lens, D ** -0.5, mask, o, lse)
    assert _lib.device_error() == 0


def test_attention_single_token_form_scale_and_large_scores():
    g = gen(7)
    lens = [400, 31]
    table, pages = tables(g, lens, 16)
    kc, vc = cache(g, pages, 2, 16, 128, BF, "hnd"), cache(g, pages, 2, 16, 128, BF, "hnd")
    q = randn(g, 2, 8, 128, scale=30.0)                    # scores of some hundreds: one key takes all the weight
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    with torch.inference_mode():
        o, lse = paged_attention(q, kc, vc, table, n, scale=0.125, return_lse=True)
        assert torch.equal(o, paged_attention(q, kc, vc, table, n, scale=0.125))
    check_attention(q[:, None], kc, vc, table, lens, 0.125, None, o[:, None], lse[:, None])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attention_masked_drafts_do_not_reach_other_rows(bad):
    """A drafted token whose key and value overflowed harms only the rows that see it."""
    g = gen(8)
    lens, L, ps = [300, 8, 21], 8, 16
    table, pages = tables(g, lens, ps)
    kc, vc = cache(g, pages, 2, ps, 128, BF, "hnd"), cache(g, pages, 2, ps, 128, BF, "hnd")
    for b, n in enumerate(lens):
        for j in (n - 3, n - 2):                           # drafted tokens 5 and 6
            kc[table[b, j // ps].long(), :, j % ps] = bad
            vc[table[b, j // ps].long(), :, j % ps] = bad
    q = randn(g, 3, L, 8, 128)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    with torch.inference_mode():
        o, lse = paged_attention(q, kc, vc, table, n, return_lse=True)
    for b, k in enumerate(lens):
        pages_b = table[b, : -(-k // ps)].long()
        kk = kc[pages_b].transpose(1, 2).reshape(-1, 2, 128)[:k].double()
        vv = vc[pages_b].transpose(1, 2).reshape(-1, 2, 128)[:k].double()
        for t in range(5):
            m = k - L + t + 1
            z = torch.einsum("hgd,nhd->hgn", q[b, t].double().view(2, 4, 128), kk[:m]) * 128 ** -0.5
            ref = torch.einsum("hgn,nhd->hgd", torch.softmax(z, -1), vv[:m]).reshape(8, 128)
            spread = torch.einsum("hgn,nhd->hgd", torch.softmax(z, -1), vv[:m].abs()).reshape(8, 128)
            assert bool(((o[b, t].double() - ref).abs() <= 2.0 ** -7 * spread + 1e-30).all()), (b, t)
            assert bool(torch.isfinite(lse[b, t]).all())
        assert not bool(torch.isfinite(o[b, 5:].float()).all())


def test_attention_offsets_past_32_bits():
    """Pages 2^30 elements apart: page 3 starts past the 32-bit range."""
    g = gen(9)
    ps, Hk, D, step = 16, 2, 128, 1 << 30
    raw = [torch.empty(3 * step + Hk * ps * D, dtype=BF, device=DEV) for _ in range(2)]
    kc, vc = (r.as_strided((4, Hk, ps, D), (step, ps * D, D, 1)) for r in raw)
    kc.copy_(randn(g, 4, Hk, ps, D))
    vc.copy_(randn(g, 4, Hk, ps, D))
    table = torch.tensor([[3, 1, 2, 0]], dtype=torch.int32, device=DEV)
    q = randn(g, 1, 1, 8, D)
    qkv = randn(g, 1, 12 * D)
    cos, sin = rope_table(8, D, 1e6, DEV)
    slot = torch.tensor([3 * ps + 5], device=DEV)
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    with torch.inference_mode():
        paged_append(qkv, 8, Hk, kc, vc, slot, zero, cos, sin)
        assert torch.equal(vc[3, :, 5], qkv.view(12, D)[10:]) and torch.equal(kc[3, :, 5], qkv.view(12, D)[8:10])
        o, lse = paged_attention(q, kc, vc, table, torch.tensor([61], dtype=torch.int32, device=DEV), return_lse=True)
    check_attention(q, kc, vc, table, [61], D ** -0.5, None, o, lse)


def test_attention_bad_pages_and_lengths_are_flagged():
    g = gen(10)
    kc, vc = cache(g, 4, 2, 16, 64, BF, "hnd"), cache(g, 4, 2, 16, 64, BF, "hnd")
    q = randn(g, 3, 1, 4, 64)
    table = torch.tensor([[0, 4], [1, -1], [2, 3]], dtype=torch.int32, device=DEV)   # two bad pages
    with torch.inference_mode():
        o = paged_attention(q, kc, vc, table, torch.tensor([32, 32, 10], dtype=torch.int32, device=DEV))
        assert _lib.device_error() & _lib.DEV_ERR_BAD_INDEX
        _lib.clear_device_error()
        ref = paged_attention(q[2:], kc, vc, table[2:], torch.tensor([10], dtype=torch.int32, device=DEV))
        assert torch.equal(o[2:], ref) and _lib.device_error() == 0
        # a length past the table counts up to its end; a negative one counts as none
        o = paged_attention(q, kc, vc, table[2:].expand(3, 2), torch.tensor([33, 32, -5], dtype=torch.int32, device=DEV))
        assert _lib.device_error() & _lib.DEV_ERR_BAD_INDEX
        _lib.clear_device_error()
        ref = paged_attention(q[:2], kc, vc, table[2:].expand(2, 2), torch.tensor([32, 32], dtype=torch.int32, device=DEV))
        assert torch.equal(o[:2], ref) and bool((o[2] == 0).all())


def test_attention_is_repeatable_on_streams_and_in_graphs():
    """Equal bits on every call, on another stream, and from a graph replayed as the sequences grow."""
    g = gen(11)
    lens = [3000, 17, 900, 0]
    table, pages = tables(g, [4000] * 4, 16)
    kc, vc = cache(g, pages, 8, 16, 128, BF, "hnd"), cache(g, pages, 8, 16, 128, BF, "hnd")
    q = randn(g, 4, 1, 32, 128)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    with torch.inference_mode():
        first = [t.clone() for t in paged_attention(q, kc, vc, table, n, return_lse=True)]
        for _ in range(3):
            again = paged_attention(q, kc, vc, table, n, return_lse=True)
            assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
        streams = [torch.cuda.Stream() for _ in range(3)]
        outs = []
        for s in streams * 3:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(paged_attention(q, kc, vc, table, n, return_lse=True))
        torch.cuda.synchronize()
        for a in outs:
            assert torch.equal(a[0], first[0]) and torch.equal(a[1], first[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = paged_attention(q, kc, vc, table, n, return_lse=True)
        for k in (1, 400, 1000):
            n.copy_(torch.tensor(lens, dtype=torch.int32, device=DEV) + k)
            graph.replay()
            now = paged_attention(q, kc, vc, table, n, return_lse=True)
            assert torch.equal(now[0], held[0]) and torch.equal(now[1], held[1])


def test_attention_of_nothing():
    g = gen(12)
    kc, vc = cache(g, 4, 2, 16, 64, BF, "hnd"), cache(g, 4, 2, 16, 64, BF, "hnd")
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    with torch.inference_mode():
        o = paged_attention(randn(g, 0, 1, 4, 64), kc, vc, none.view(0, 3), none)
        assert o.shape == (0, 1, 4, 64)
        # sequences without a page yet
        o = paged_attention(randn(g, 2, 1, 4, 64), kc, vc, none.view(2, 0), torch.zeros(2, dtype=torch.int32, device=DEV))
        assert bool((o == 0).all())


def test_append_then_attend_is_plain_attention():
    """Tokens appended one call at a time, then read back: causal attention over them."""
    g = gen(13)
    T, Hq, Hk, D, ps = 50, 8, 2, 128, 16
    kc, vc = torch.zeros(6, Hk, ps, D, dtype=BF, device=DEV), torch.zeros(6, Hk, ps, D, dtype=BF, device=DEV)
    table = torch.tensor([[5, 0, 3, 1]], dtype=torch.int32, device=DEV)
    cos, sin = rope_table(64, D, 1e4, DEV)
    qkv = randn(g, T, (Hq + 2 * Hk) * D)
    pos = torch.arange(T, device=DEV)
    slots = table[0, pos // ps].long() * ps + pos % ps
    w = torch.ones(D, dtype=BF, device=DEV)
    with torch.inference_mode():
        whole = paged_append(qkv, Hq, Hk, kc.clone(), vc.clone(), slots, pos, cos, sin, w, w)
        outs = []
        for t in range(T):
            q = paged_append(qkv[t:t + 1], Hq, Hk, kc, vc, slots[t:t + 1], pos[t:t + 1], cos, sin, w, w)
            assert torch.equal(q, whole[t:t + 1])
            outs.append(paged_attention(q, kc, vc, table, torch.tensor([t + 1], dtype=torch.int32, device=DEV)))
    o = torch.cat(outs).double()
    k = kc[table[0].long()].transpose(1, 2).reshape(-1, Hk, D)[:T].double().repeat_interleave(Hq // Hk, 1)
    v = vc[table[0].long()].transpose(1, 2).reshape(-1, Hk, D)[:T].double().repeat_interleave(Hq // Hk, 1)
    z = torch.einsum("thd,nhd->htn", whole.double(), k) * D ** -0.5
    z = z.masked_fill(~torch.ones(T, T, device=DEV).tril().bool(), -math.inf)
    p = torch.softmax(z, -1)
    ref, spread = torch.einsum("htn,nhd->thd", p, v), torch.einsum("htn,nhd->thd", p, v.abs())
    assert bool(((o - ref).abs() <= 2.0 ** -7 * spread + 2.0 ** -8 * ref.abs()).all())
