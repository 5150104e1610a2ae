"""The paged cache held in 8 bits (kernels/paged_cache8.py) against a plain 64-bit
implementation.

Tolerances.  u is half a step of the 16-bit type relative to the value (2^-8 bf16, 2^-11
fp16), 2^-4 of e4m3's, whose smallest numbers are 2^-9 apart (half: 2^-10 s).  Append: the
32-bit arithmetic before a rounding errs by 2^-20 of |a c| + |b s| (a dot of <= 13 dependent
additions, rsqrt and three products).  Attention: with spread = sum_j p_j |v_j| and d =
2^-20 scale max_j sum_i |q_i k_ji| the error of a score, plus 2^-38 of the row's largest |q|
times sum_i |k_ji| for what its fp16 form drops, the weights p_j vs_j are rounded to fp16
(2^-11 spread; those under 2^-14 by 2^-25 at most where the largest is over 2^7: n 2^-32 448
max_j p_j vs_j), every weight moves by 2 d + 2^-16 (score, exponential, and up to 256
dependent additions), and o is rounded once (u |ref|).  lse: d + 2^-16 + 2^-22 |lse|.
"""
from __future__ import annotations

import math

import pytest
import torch

from kernels import _lib
from kernels.paged_cache import paged_attention, rope_table
from kernels.paged_cache8 import F8, cache8, paged_append8, paged_attention8

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16
U = {BF: 2.0 ** -8, FP: 2.0 ** -11}
NAN8 = 0x7F


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def power(top):
    """The smallest power of two s, 2^-64 to 2^64, with top <= 448 s (64 bits)."""
    m, e = torch.frexp(top.double())
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.ldexp(torch.ones_like(m), torch.where(top > 0, e, -64).clamp(-64, 64))


def cache_of(g, pages, Hk, ps, D, block, layout="hnd", pow2=True):
    """A quantised cache whose blocks have different magnitudes."""
    x = torch.randn(pages, Hk, ps // block, block, D, generator=g, device=DEV)
    x *= torch.exp(torch.randn(pages, Hk, ps // block, 1, 1, generator=g, device=DEV))
    top = x.abs().amax((-1, -2))
    scale = power(top).float() if pow2 else top / 448 * 1.01
    x = (x / scale[..., None, None]).clamp(-448, 448).to(F8).view(pages, Hk, ps, D)
    if layout == "nhd":
        x = x.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(F8)
    if layout == "both":         # k or v of a [pages, 2, ..] allocation
        whole = torch.zeros(pages, 2, Hk, ps, D, dtype=torch.uint8, device=DEV)
        whole[:, 1] = x.view(torch.uint8)
        x = whole.view(F8)[:, 1]
    return x, scale.contiguous()


def values(cache, scale):
    """[pages, Hk, ps, D] in 64 bits."""
    n = cache.shape[2] // scale.shape[2]
    x = cache.view(torch.uint8).contiguous().view(F8).double()
    return x * scale.double().repeat_interleave(n, 2)[..., None]


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


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ append
def turned(part, weight, pos, cos, sin, eps):
    """(value, magnitude of its rotation's terms) in 64 bits of [n, heads, D] at positions [n]."""
    R = 2 * cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    if weight is not None:
        part = part / (part.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    a, b, rest = part[..., : R // 2], part[..., R // 2: R], part[..., R:]
    return (torch.cat([a * c - b * s, b * c + a * s, rest], -1),
            torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), rest.abs()], -1))


def check_append(before, after, q, qkv, Hq, Hk, table, lens, count, cos, sin, qw, kw, eps=1e-6):
    """before, after: (k_cache, v_cache, k_scale, v_scale)."""
    B, L = qkv.shape[:2]
    D, ps = after[0].shape[3], after[0].shape[2]
    bs = ps // after[2].shape[2]
    x = qkv.double().view(B, L, Hq + 2 * Hk, D)
    dtype = qkv.dtype
    want = [[c.view(torch.uint8).clone() for c in before[:2]], [s.clone() for s in before[2:]]]
    for b, (n, c) in enumerate(zip(lens, count)):
        c = min(n, max(0, min(c, L)))
        old = n - c
        assert bool((q[b, : L - c] == 0).all())
        if c == 0:
            continue
        pos = torch.arange(old, n, device=DEV)
        ref, mag = turned(x[b, L - c:, :Hq], qw, pos, cos, sin, eps)
        err = (q[b, L - c:].double() - ref).abs()
        bound = U[dtype] * ref.abs() + 2.0 ** -20 * mag * (1 + U[dtype]) + (2.0 ** -25 if dtype == FP else 2.0 ** -130)
        assert bool((err <= bound).all()), (b, float((err / bound).max()))
        k, km = turned(x[b, L - c:, Hq:Hq + Hk], kw, pos, cos, sin, eps)
        v = x[b, L - c:, Hq + Hk:]
        for i, (y, e) in enumerate(((k, km * 2.0 ** -20), (v, torch.zeros_like(v)))):
            for lo in range(old // bs * bs, n, bs):
                page, at = int(table[b, lo // ps]), lo % ps
                first, last = max(lo, old), min(lo + bs, n)
                part, pe = y[first - old: last - old].transpose(0, 1), e[first - old: last - old].transpose(0, 1)
                fine = part.isfinite()
                top = part.abs().where(fine, torch.zeros((), dtype=torch.float64, device=DEV)).amax((1, 2))
                slack = pe.where(fine, torch.zeros((), dtype=torch.float64, device=DEV)).amax((1, 2))
                s, s0 = after[2 + i][page, :, at // bs].double(), before[2 + i][page, :, at // bs].double()
                lows, highs = power((top - slack).clamp(min=0)), power(top + slack)
                if lo < old:
                    lows, highs = torch.maximum(lows, s0), torch.maximum(highs, s0)
                assert bool(((s == lows) | (s == highs)).all()), (b, i, lo)
                codes = after[i].view(torch.uint8)[page, :, at: at + bs]
                got = codes.view(F8).double() * s[:, None, None]
                new = got[:, first - lo: last - lo]
                assert torch.equal(new.isnan(), ~fine)
                edge = torch.maximum(2.0 ** -4 * part.abs(), 2.0 ** -10 * s[:, None, None].expand_as(part)) + pe * 1.0625
                over = part.abs() > 448 * s[:, None, None]          # past the largest scale
                assert bool(((new - part).abs() <= edge)[fine & ~over].all()), (b, i, lo)
                assert bool((new.abs() == 448 * s[:, None, None])[fine & over].all())
                if first > lo:       # the older tokens: exact but near the smallest numbers
                    held = before[i].view(torch.uint8)[page, :, at: at + first - lo].view(F8).double() * s0[:, None, None]
                    now = got[:, : first - lo]
                    big = held.abs() >= 2.0 ** -6 * s[:, None, None]
                    assert torch.equal(now[big], held[big]) and torch.equal(now.isnan(), held.isnan())
                    near = (now - held).abs() <= 2.0 ** -10 * s[:, None, None]
                    assert bool((near | held.isnan()).all())
                want[0][i][page, :, at: at + last - lo] = codes[:, : last - lo]
                want[1][i][page, :, at // bs] = after[2 + i][page, :, at // bs]
    # nothing else moved
    for i in range(2):
        assert torch.equal(after[i].view(torch.uint8), want[0][i])
        assert torch.equal(after[2 + i], want[1][i]) or torch.equal(after[2 + i].nan_to_num(7.0), want[1][i].nan_to_num(7.0))


APPEND = [
    # new tokens, length with them, heads, dims, rotated, pages, block, layout, type, norm, count
    ([1], [1], 32, 8, 128, 128, 16, 16, "hnd", BF, True, None), ([1] * 3, [16, 17, 33], 32, 8, 128, 128, 16, 16, "nhd", BF, True, None),
    ([5] * 4, [3, 5, 21, 700], 14, 2, 64, 32, 24, 8, "both", FP, False, [5, 4, 0, 2]),
    ([40] * 2, [100, 40], 7, 1, 64, 64, 64, 64, "nhd", BF, True, [33, 40]), ([130], [333], 8, 8, 128, 0, 128, 128, "hnd", BF, True, None),
    ([17] * 3, [1000, 18, 17], 4, 2, 128, 112, 16, 1, "hnd", FP, True, [17, 1, -3]), ([9], [9], 3, 1, 64, 16, 7, 7, "hnd", BF, False, [50]),
    ([3] * 2, [4, 50], 16, 4, 128, 64, 1, 1, "nhd", BF, True, None), ([300], [300], 2, 1, 128, 128, 48, 24, "both", BF, True, None),
    ([16] * 2, [32, 31], 8, 2, 64, 64, 32, 2, "hnd", BF, True, None),
    # blocks of less than 16 tokens that start, end and were begun before the call, over pages of less than 16 too
    ([21] * 4, [21, 22, 530, 100], 6, 2, 128, 128, 8, 8, "hnd", BF, True, [21, 9, 20, 1]), ([50] * 2, [77, 51], 4, 4, 64, 32, 4, 4, "nhd", FP, False, None),
    ([100], [131], 2, 2, 128, 64, 24, 8, "both", BF, True, None), ([70], [75], 3, 3, 64, 64, 12, 3, "hnd", BF, True, None),
]


@pytest.mark.parametrize("new,lens,Hq,Hk,D,R,ps,block,layout,dtype,norm,count", APPEND)
def test_append_matches_64_bits(new, lens, Hq, Hk, D, R, ps, block, layout, dtype, norm, count):
    g = gen(sum(lens) + Hq)
    B, L = len(lens), new[0]
    table, pages = tables(g, lens, ps)
    k, ks = cache_of(g, pages, Hk, ps, D, block, layout)
    v, vs = cache_of(g, pages, Hk, ps, D, block, layout)
    before = [t.clone() for t in (k, v, ks, vs)]
    W = (Hq + 2 * Hk) * D
    qkv = (torch.randn(B, L, W + 8, generator=g, device=DEV) * torch.exp(torch.randn(B, L, 1, generator=g, device=DEV))).to(dtype)
    qkv = qkv[..., :W]                                             # rows apart
    for b, c in enumerate(count or [L] * B):
        qkv[b, : L - min(max(c, 0), lens[b], L)] = float("nan")    # padding rows hold anything
    cos, sin = rope_table(1024, R, 1e6, DEV)
    qw = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(dtype) if norm else None
    kw = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(dtype) if norm else None
    with torch.inference_mode():
        q = paged_append8(qkv, Hq, Hk, k, v, ks, vs, table, ints(lens), cos, sin, qw, kw,
                          count=None if count is None else ints(count))
    assert q.shape == (B, L, Hq, D)
    check_append(before, (k, v, ks, vs), q, qkv, Hq, Hk, table, lens, count or [L] * B, cos, sin, qw, kw)
    assert _lib.device_error() == 0


def test_append_token_by_token_is_one_append_up_to_the_scales_growth():
    """Blocks filled a token at a time end with the same scales, and with numbers that are a
    rounding or two further off only where the scale grew."""
    g = gen(3)
    Hq, Hk, D, ps, T = 4, 2, 128, 16, 40
    table, pages = tables(g, [48], ps)
    cos, sin = rope_table(64, D, 1e4, DEV)
    qkv = randn(g, 1, T, (Hq + 2 * Hk) * D, scale=0.2) * torch.exp(torch.linspace(0, 3, T, device=DEV))[None, :, None].to(BF)
    a, b = cache8(pages, Hk, ps, D, 16, DEV), cache8(pages, Hk, ps, D, 16, DEV)
    with torch.inference_mode():
        whole = paged_append8(qkv, Hq, Hk, *a, table, ints([T]), cos, sin)
        for t in range(T):
            q = paged_append8(qkv[:, t], Hq, Hk, *b, table, ints([t + 1]), cos, sin)
            assert torch.equal(q, whole[:, t])
    assert torch.equal(a[2], b[2]) and torch.equal(a[3], b[3])
    for i in range(2):
        x, y = values(a[i], a[2 + i]), values(b[i], b[2 + i])
        s = a[2 + i].double().repeat_interleave(16, 2)[..., None]
        assert bool(((x - y).abs() <= 5 * 2.0 ** -10 * s).all())   # up to five growths of a block's scale
        big = x.abs() >= 2.0 ** -6 * s
        assert torch.equal(x[big], y[big])


def test_append_numbers_that_are_not_finite_and_zeros():
    g = gen(4)
    Hq, Hk, D, ps = 2, 1, 64, 16
    table, pages = tables(g, [16], ps)
    cos, sin = rope_table(32, 0, 1e4, DEV)
    for kind, dtype in (("zero", BF), ("tiny", BF), ("huge", BF), ("bad", FP)):
        qkv = randn(g, 1, 10, (Hq + 2 * Hk) * D, dtype=dtype)
        if kind == "zero":
            qkv.zero_()
        if kind == "tiny":
            qkv.mul_(2.0 ** -100)
        if kind == "huge":
            qkv.mul_(2.0 ** 100)
        if kind == "bad":
            qkv[0, 3, 130] = float("nan")
            qkv[0, 4, 200] = float("inf")
            qkv[0, 5, 140] = float("-inf")
        c = cache8(pages, Hk, ps, D, 16, DEV)
        before = [t.clone() for t in c]
        with torch.inference_mode():
            q = paged_append8(qkv, Hq, Hk, *c, table, ints([10]), cos, sin)
        check_append(before, c, q, qkv, Hq, Hk, table, [10], [10], cos, sin, None, None)
        page = int(table[0, 0])
        for s in c[2:]:
            s = float(s[page, 0, 0])
            assert {"zero": s == 2.0 ** -64, "tiny": s == 2.0 ** -64, "huge": s == 2.0 ** 64, "bad": s < 1.0}[kind], (kind, s)


def test_append_bad_indices_are_flagged_and_skipped():
    g = gen(5)
    Hq, Hk, D, ps = 4, 2, 64, 16
    k, ks = cache_of(g, 4, Hk, ps, D, 16)
    v, vs = cache_of(g, 4, Hk, ps, D, 16)
    before = [t.clone() for t in (k, v, ks, vs)]
    cos, sin = rope_table(40, D, 1e4, DEV)
    qkv = randn(g, 1, 3, (Hq + 2 * Hk) * D)

    def call(row, n, **kw):
        with torch.inference_mode():
            q = paged_append8(qkv, Hq, Hk, k, v, ks, vs, ints([row]), ints([n]), cos, sin, **kw)
        bad = _lib.device_error()
        _lib.clear_device_error()
        return q, bad

    for row, n in (([0, 4, 1], 20), ([0, -1, 1], 20), ([4, 1, 1], 3)):           # pages that are none
        q, bad = call(row, n)
        assert bad & _lib.DEV_ERR_BAD_INDEX and bool(q.isfinite().all()) and bool((q != 0).any())
        for a, b in zip(before, (k, v, ks, vs)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    q, bad = call([0, 1, 2], 50)                                                  # past the page table
    assert bad & _lib.DEV_ERR_BAD_INDEX and bool((q[0, 1:] == 0).all())
    q, bad = call([0, 1, 2], 42)                                                  # past cos / sin
    assert bad & _lib.DEV_ERR_BAD_INDEX and bool((q[0, 1:] == 0).all()) and bool((q[0, 0] != 0).any())
    mid = [t.clone() for t in (k, v, ks, vs)]
    q, bad = call([0, 1, 2], -5)                                                  # no tokens at all
    assert bad == 0 and bool((q == 0).all())
    q, bad = call([3, 3, 3], 9, count=ints([0]))
    assert bad == 0 and bool((q == 0).all())
    for a, b in zip(mid, (k, v, ks, vs)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_append_of_nothing():
    c = cache8(2, 2, 16, 64, 16, DEV)
    cos, sin = rope_table(10, 64, 1e6, DEV)
    with torch.inference_mode():
        assert paged_append8(torch.empty(0, 3, 8 * 64, dtype=BF, device=DEV), 4, 2, *c, ints([]).view(0, 2), ints([]), cos,
                             sin).shape == (0, 3, 4, 64)
        assert paged_append8(torch.empty(2, 0, 8 * 64, dtype=BF, device=DEV), 4, 2, *c, ints([[0], [1]]), ints([0, 3]), cos,
                             sin).shape == (2, 0, 4, 64)
        # sequences without a page: a new token has no place
        q = paged_append8(torch.ones(2, 1, 8 * 64, dtype=BF, device=DEV), 4, 2, *c, ints([]).view(2, 0), ints([0, 1]), cos, sin)
        assert bool((q == 0).all()) and _lib.device_error() & _lib.DEV_ERR_BAD_INDEX
        _lib.clear_device_error()


# ------------------------------------------------------------------ attention
def check_attention(q, K, V, vscale, table, lens, scale, tail, o, lse, window=None, sinks=0, weight=2.0 ** -11):
    """K, V: the caches' values [pages, Hk, ps, D] in 64 bits; vscale [pages, Hk, ps] the scales of the values."""
    B, L, Hq, D = q.shape
    Hk, ps = K.shape[1], K.shape[2]
    G, u = Hq // Hk, U[q.dtype]
    for b, n in enumerate(lens):
        pages = table[b, : -(-n // ps)].long().clamp(0, K.shape[0] - 1)
        k = K[pages].transpose(1, 2).reshape(-1, Hk, D)[:n]                       # [n, Hk, D]
        v = V[pages].transpose(1, 2).reshape(-1, Hk, D)[:n]
        s = vscale[pages].transpose(1, 2).reshape(-1, Hk)[:n]
        j = torch.arange(n, device=DEV)
        for t in range(L):
            see = j < n - L
            for i in range(max(0, L - n), L):
                see[n - L + i] = i <= t if tail is None else bool((tail if tail.ndim == 2 else tail[b])[t, i])
            if window is not None:
                see &= (j > n - L + t - window) | (j < sinks)
            got, gl = o[b, t].double(), lse[b, t].double()
            if not bool(see.any()):
                assert bool((got == 0).all()) and bool((gl == -math.inf).all()), (b, t)
                continue
            qq = q[b, t].double().view(Hk, G, D)
            z = torch.einsum("hgd,nhd->hgn", qq, k[see]) * scale
            p = torch.softmax(z, -1)
            d = torch.einsum("hgd,nhd->hgn", qq.abs(), k[see].abs()).amax(-1) * 2.0 ** -20
            d = d + qq.abs().amax(-1) * k[see].abs().sum(-1).amax(0)[:, None] * 2.0 ** -38
            d = (d * abs(scale)).view(Hq)
            ref = torch.einsum("hgn,nhd->hgd", p, v[see]).reshape(Hq, D)
            spread = torch.einsum("hgn,nhd->hgd", p, v[see].abs()).reshape(Hq, D)
            small = n * 2.0 ** -32 * 448 * (p * s[see].T[:, None]).amax(-1).view(Hq)
            bound = (weight + 2 * d[:, None] + 2.0 ** -16) * spread + small[:, None] + u * ref.abs() + 1e-30
            bound = bound + (2.0 ** -25 if u == U[FP] else 0)
            err = (got - ref).abs()
            assert bool((err <= bound).all()), (b, t, n, float((err / bound).max()))
            rl = torch.logsumexp(z, -1).view(Hq)
            el = (gl - rl).abs()
            assert bool((el <= d + 2.0 ** -16 + 2.0 ** -22 * rl.abs()).all()), (b, t, n, float(el.max()))


def spread_scales(scale, ps):
    return scale.double().repeat_interleave(ps // scale.shape[2], 2)


def stale(table, lens, pages, ps):
    """Which slots of the cache no sequence uses, [pages, ps]."""
    used = torch.zeros(pages * ps, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        j = torch.arange(n, device=DEV)
        used[table[b, j // ps].long() * ps + j % ps] = True
    return ~used.view(pages, ps)


def poison(cache, scale, free):
    """NaN in unused slots, and in the scales of blocks without a used one."""
    cache.view(torch.uint8).masked_fill_(free[:, None, :, None], NAN8)
    n = cache.shape[2] // scale.shape[2]
    scale.masked_fill_(free.view(free.shape[0], -1, n).all(-1)[:, None], float("nan"))


# lengths around tile, page and split edges; groups of 1 to 16 query heads; 1 to 40 rows a head;
# pages of one token, odd pages, pages larger than any sequence; blocks of one token to whole pages
ATT = [
    ([1], 1, 32, 8, 128, 16, 16, "hnd", BF, None), ([0, 1, 2, 0], 1, 8, 8, 128, 16, 4, "nhd", BF, None),
    ([31, 32, 33, 127, 128, 129, 255, 256, 257], 1, 32, 8, 128, 16, 16, "hnd", BF, None),
    ([1000, 3, 0, 517], 1, 16, 1, 128, 1, 1, "nhd", BF, None), ([700, 701], 1, 14, 2, 64, 24, 8, "both", FP, None),
    ([333, 40, 1], 1, 5, 5, 64, 7, 7, "hnd", FP, None), ([5000], 1, 32, 8, 128, 16, 1, "hnd", BF, None),
    ([20000, 100], 1, 8, 2, 128, 64, 64, "nhd", FP, None), ([2048] * 3, 1, 8, 8, 64, 4096, 128, "hnd", BF, None),
    ([4, 5, 100, 0, 2, 1], 4, 32, 8, 128, 16, 16, "hnd", BF, None),        # shorter than its queries: rows see nothing
    ([64, 200, 1500], 8, 32, 8, 128, 16, 8, "nhd", BF, "each"), ([90, 130], 5, 40, 8, 128, 32, 32, "hnd", FP, "one"),
    ([300, 37, 16], 16, 16, 2, 64, 24, 12, "both", BF, "each"), ([777, 12], 3, 12, 1, 64, 8, 2, "nhd", FP, "each"),
    ([513, 40], 40, 8, 8, 128, 16, 16, "hnd", BF, "one"), ([257, 31], 33, 6, 2, 64, 16, 16, "hnd", BF, None),
    ([200, 65, 5, 0], 8, 16, 2, 128, 7, 1, "hnd", BF, "each"), ([130, 300], 6, 32, 8, 64, 1, 1, "nhd", FP, None),
    ([1000, 129, 128, 127], 32, 32, 8, 128, 16, 16, "hnd", BF, "each"), ([260, 3], 70, 2, 1, 128, 64, 16, "nhd", BF, "one"),
    ([6000], 4, 32, 4, 128, 128, 128, "hnd", BF, None), ([10] * 200, 1, 8, 4, 64, 16, 8, "hnd", BF, None),
    ([0] * 5, 2, 4, 2, 128, 16, 16, "hnd", BF, None), ([640] * 9, 1, 24, 1, 128, 16, 16, "hnd", BF, None),
    # many units a CTA: every ring goes round, with and without TMA
    ([2500 + 97 * i for i in range(12)], 4, 32, 8, 128, 16, 16, "hnd", BF, None), ([3000, 1, 5000, 900] * 4, 3, 28, 4, 64, 4, 2, "nhd", FP, "each"),
    ([4000] * 6, 20, 32, 8, 128, 64, 64, "hnd", BF, "one"), ([40000, 30000], 2, 64, 8, 128, 1, 1, "hnd", BF, None),
]


@pytest.mark.parametrize("lens,L,Hq,Hk,D,ps,block,layout,dtype,tail", ATT)
def test_attention_matches_64_bits(lens, L, Hq, Hk, D, ps, block, layout, dtype, tail):
    g = gen(sum(lens) + Hq)
    B = len(lens)
    table, pages = tables(g, lens, ps)
    k, ks = cache_of(g, pages, Hk, ps, D, block, layout, pow2=dtype == BF)
    v, vs = cache_of(g, pages, Hk, ps, D, block, layout, pow2=dtype == BF)
    free = stale(table, lens, pages, ps)
    poison(k, ks, free)
    poison(v, vs, free)
    q = randn(g, B, L, Hq, D, dtype=dtype, scale=2.0)
    mask = None
    if tail is not None:
        mask = torch.rand(*((B,) if tail == "each" else ()), L, L, generator=g, device=DEV) < 0.5
        mask[..., 0, :] = False
    with torch.inference_mode():
        o, lse = paged_attention8(q, k, v, ks, vs, table, ints(lens), tail_mask=mask, return_lse=True)
    assert o.shape == q.shape and lse.shape == (B, L, Hq)
    check_attention(q, values(k, ks), values(v, vs), spread_scales(vs, ps), table, lens, D ** -0.5, mask, o, lse)
    assert _lib.device_error() == 0


# (window, sinks) through the 8-bit and the 16-bit cache: windows of one key, inside a unit, over its
# edges, longer than any sequence; no sinks, some, more than the window leaves out
WINDOW = [
    ([1, 2, 50, 200, 1000], 1, 32, 8, 128, 16, "hnd", BF, None, 1, 0), ([5, 64, 65, 300, 4000], 1, 8, 2, 128, 16, "nhd", BF, None, 64, 4),
    ([700, 129, 900], 1, 14, 2, 64, 24, "both", FP, None, 100, 70), ([333, 40, 1], 1, 5, 5, 64, 7, "hnd", FP, None, 31, 1),
    ([20000, 9000], 1, 8, 2, 128, 64, "nhd", BF, None, 500, 130), ([3000, 10], 1, 16, 1, 128, 1, "hnd", BF, None, 257, 2),
    ([64, 200, 1500], 8, 32, 8, 128, 16, "nhd", BF, "each", 20, 5), ([90, 130, 4], 5, 40, 8, 128, 32, "hnd", FP, "one", 3, 40),
    ([300, 37, 16, 0], 16, 16, 2, 64, 24, "both", BF, None, 10, 0), ([513, 40], 40, 8, 8, 128, 16, "hnd", BF, "one", 17, 1),
    ([1000, 128], 32, 32, 8, 128, 16, "hnd", BF, None, 300, 64), ([777, 12], 3, 12, 1, 64, 8, "nhd", FP, "each", 1 << 30, 3),
    ([500, 1200], 2, 8, 2, 128, 16, "hnd", BF, None, 100, 10000), ([400, 90], 1, 8, 8, 64, 16, "hnd", FP, None, 60, 15),
]


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("lens,L,Hq,Hk,D,ps,layout,dtype,tail,window,sinks", WINDOW)
def test_window_matches_64_bits(lens, L, Hq, Hk, D, ps, layout, dtype, tail, window, sinks, bits):
    """Pages of which no key is visible have been given back: their entries are no pages."""
    g = gen(sum(lens) + Hq)
    B = len(lens)
    table, pages = tables(g, lens, ps)
    k, ks = cache_of(g, pages, Hk, ps, D, 1 if ps % 2 else 2, layout)
    v, vs = cache_of(g, pages, Hk, ps, D, 1 if ps % 2 else 2, layout)
    free = stale(table, lens, pages, ps)
    gone = table.clone()
    for b, n in enumerate(lens):
        first = max(0, n - L + 1 - window)
        hidden = [j for j in range(n) if sinks <= j < first]
        for j in hidden:
            free[table[b, j // ps].long(), j % ps] = True
        for page in range(-(-n // ps)):
            keys = range(page * ps, min(n, (page + 1) * ps))
            if all(sinks <= j < first for j in keys):
                gone[b, page] = -1 if page % 2 else 1 << 30
    poison(k, ks, free)
    poison(v, vs, free)
    q = randn(g, B, L, Hq, D, dtype=dtype, scale=2.0)
    mask = None
    if tail is not None:
        mask = torch.rand(*((B,) if tail == "each" else ()), L, L, generator=g, device=DEV) < 0.5
        mask[..., 0, :] = False
    K, V, S, weight = values(k, ks), values(v, vs), spread_scales(vs, ps), 2.0 ** -11
    with torch.inference_mode():
        if bits == 8:
            o, lse = paged_attention8(q, k, v, ks, vs, gone, ints(lens), tail_mask=mask, return_lse=True, window=window, sinks=sinks)
        else:
            k16, v16 = K.to(dtype), V.to(dtype)
            K, V, S, weight = k16.double(), v16.double(), torch.zeros_like(S), U[dtype]
            o, lse = paged_attention(q, k16, v16, gone, ints(lens), tail_mask=mask, return_lse=True, window=window, sinks=sinks)
    check_attention(q, K, V, S, table, lens, D ** -0.5, mask, o, lse, window, sinks, weight)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("bits", [8, 16])
def test_a_window_over_everything_is_no_window(bits):
    g = gen(21)
    lens, ps = [300, 37, 1], 16
    table, pages = tables(g, lens, ps)
    k, ks = cache_of(g, pages, 2, ps, 128, 16)
    v, vs = cache_of(g, pages, 2, ps, 128, 16)
    k16, v16 = values(k, ks).to(BF), values(v, vs).to(BF)
    f = (lambda q, **kw: paged_attention8(q, k, v, ks, vs, table, ints(lens), **kw)) if bits == 8 else \
        (lambda q, **kw: paged_attention(q, k16, v16, table, ints(lens), **kw))
    with torch.inference_mode():
        for L in (1, 2, 4):
            q = randn(g, 3, L, 8, 128)
            assert torch.equal(f(q), f(q, window=300)) and torch.equal(f(q), f(q, window=1 << 40, sinks=1 << 40))
            assert torch.equal(f(q), f(q, sinks=5))


def test_attention_single_token_form_scale_and_large_scores():
    g = gen(7)
    lens = [400, 31]
    table, pages = tables(g, lens, 16)
    k, ks = cache_of(g, pages, 2, 16, 128, 16)
    v, vs = cache_of(g, pages, 2, 16, 128, 16)
    q = randn(g, 2, 8, 128, scale=30.0)                    # scores of some hundreds: one key takes all the weight
    K, V, S = values(k, ks), values(v, vs), spread_scales(vs, 16)
    with torch.inference_mode():
        for scale in (0.125, -0.125):
            o, lse = paged_attention8(q, k, v, ks, vs, table, ints(lens), scale=scale, return_lse=True)
            assert torch.equal(o, paged_attention8(q, k, v, ks, vs, table, ints(lens), scale=scale))
            check_attention(q[:, None], K, V, S, table, lens, scale, None, o[:, None], lse[:, None])


@pytest.mark.parametrize("kind", ["queries", "scales", "values", "zero"])
def test_attention_magnitudes(kind):
    """Queries from 2^-60 to 2^60, scales 2^-60 to 2^60 in one sequence, zero scales of zero blocks."""
    g = gen(17)
    lens, ps, D = [700, 33], 16, 128
    table, pages = tables(g, lens, ps)
    k, ks = cache_of(g, pages, 2, ps, D, 16)
    v, vs = cache_of(g, pages, 2, ps, D, 16)
    q = randn(g, 2, 2, 8, D)
    scale = D ** -0.5
    if kind == "queries":          # rows of very different sizes, the scores small again by the keys
        size = torch.tensor([2.0 ** -60, 1.0, 2.0 ** 60, 2.0 ** 20], device=DEV).repeat(2)
        q = (q.float() * size[:, None]).to(BF)
        ks *= 2.0 ** -60
    if kind in ("scales", "values"):
        vs *= torch.exp2(torch.randint(-60, 60, vs.shape, generator=g, device=DEV).float())
    if kind == "values":
        ks *= torch.exp2(torch.randint(-20, 2, ks.shape, generator=g, device=DEV).float())
    if kind == "zero":
        for c, s in ((k, ks), (v, vs)):
            hit = torch.rand(s.shape, generator=g, device=DEV) < 0.3
            s.masked_fill_(hit, 0.0)
            c.view(torch.uint8).masked_fill_(hit.repeat_interleave(16, 2)[..., None], 0)
    with torch.inference_mode():
        o, lse = paged_attention8(q, k, v, ks, vs, table, ints(lens), scale=scale, return_lse=True)
    check_attention(q, values(k, ks), values(v, vs), spread_scales(vs, ps), table, lens, scale, None, o, lse)


@pytest.mark.parametrize("where", ["key", "value", "key scale", "value scale"])
def test_attention_masked_drafts_do_not_reach_other_rows(where):
    """A drafted token whose stored numbers or scale are NaN harms only the rows that see it."""
    g = gen(8)
    lens, L, ps = [300, 8, 21], 8, 16
    table, pages = tables(g, lens, ps)
    k, ks = cache_of(g, pages, 2, ps, 128, 1)
    v, vs = cache_of(g, pages, 2, ps, 128, 1)
    clean = values(k, ks), values(v, vs), spread_scales(vs, ps)
    for b, n in enumerate(lens):
        for j in (n - 3, n - 2):                           # drafted tokens 5 and 6
            page, at = table[b, j // ps].long(), j % ps
            if where in ("key", "value"):
                (k if where == "key" else v).view(torch.uint8)[page, :, at, 7] = NAN8
            else:
                (ks if where == "key scale" else vs)[page, :, at] = float("nan")
    q = randn(g, 3, L, 8, 128)
    with torch.inference_mode():
        o, lse = paged_attention8(q, k, v, ks, vs, table, ints(lens), return_lse=True)
    tail = torch.ones(L, L, dtype=torch.bool, device=DEV).tril()
    for b, n in enumerate(lens):
        for t in range(5):
            one = tail.clone()
            check_attention(q[b:b + 1, : t + 1], *clean, table[b:b + 1], [n - L + t + 1], 128 ** -0.5, one[: t + 1, : t + 1],
                            o[b:b + 1, : t + 1], lse[b:b + 1, : t + 1])
        assert bool(o[b, 5:].float().isnan().any(-1).all())


def test_attention_offsets_past_32_bits():
    """Pages 2^31 bytes apart: page 2 starts past the 32-bit range."""
    g = gen(9)
    ps, Hk, D, step = 16, 2, 128, 1 << 31
    raw = [torch.empty(2 * step + Hk * ps * D, dtype=torch.uint8, device=DEV) for _ in range(2)]
    k, v = (r.view(F8).as_strided((3, Hk, ps, D), (step, ps * D, D, 1)) for r in raw)
    small = [cache_of(g, 3, Hk, ps, D, 16) for _ in range(2)]
    (ks, vs) = (s for _, s in small)
    k.view(torch.uint8).copy_(small[0][0].view(torch.uint8))
    v.view(torch.uint8).copy_(small[1][0].view(torch.uint8))
    table = ints([[2, 1, 0]])
    before = [t.clone() for t in (k, v, ks, vs)]
    qkv = randn(g, 1, 2, 12 * D)
    cos, sin = rope_table(64, D, 1e6, DEV)
    with torch.inference_mode():
        q = paged_append8(qkv, 8, Hk, k, v, ks, vs, table, ints([14]), cos, sin)
        check_append(before, (k, v, ks, vs), q, qkv, 8, Hk, table, [14], [2], cos, sin, None, None)
        o, lse = paged_attention8(q, k, v, ks, vs, table, ints([45]), return_lse=True)
    check_attention(q, values(k, ks), values(v, vs), spread_scales(vs, ps), table, [45], D ** -0.5, None, o, lse)


def test_attention_bad_pages_and_lengths_are_flagged():
    g = gen(10)
    k, ks = cache_of(g, 4, 2, 16, 64, 16)
    v, vs = cache_of(g, 4, 2, 16, 64, 16)
    q = randn(g, 3, 1, 4, 64)
    table = ints([[0, 4], [1, -1], [2, 3]])                # two bad pages
    f = lambda q, t, n, **kw: paged_attention8(q, k, v, ks, vs, t, ints(n), **kw)  # noqa: E731
    with torch.inference_mode():
        o = f(q, table, [32, 32, 10])
        assert _lib.device_error() & _lib.DEV_ERR_BAD_INDEX
        _lib.clear_device_error()
        ref = f(q[2:], table[2:], [10])
        assert torch.equal(o[2:], ref) and _lib.device_error() == 0
        # a length past the table counts up to its end; a negative one counts as none
        o = f(q, table[2:].expand(3, 2), [33, 32, -5])
        assert _lib.device_error() & _lib.DEV_ERR_BAD_INDEX
        _lib.clear_device_error()
        assert torch.equal(o[:2], f(q[:2], table[2:].expand(2, 2), [32, 32])) and bool((o[2] == 0).all())
        # a bad page inside the window is flagged, one outside is not looked at
        f(q[:1], table[:1], [32], window=4)
        assert _lib.device_error() & _lib.DEV_ERR_BAD_INDEX
        _lib.clear_device_error()
        f(q[:1], ints([[4, 0]]), [32], window=4)
        assert _lib.device_error() == 0


def test_attention_is_repeatable_on_streams_and_in_graphs():
    """Equal bits on every call, on another stream, and from graphs replayed as the sequences grow."""
    g = gen(11)
    lens = [3000, 17, 900, 0]
    table, pages = tables(g, [4000] * 4, 16)
    k, ks = cache_of(g, pages, 8, 16, 128, 16)
    v, vs = cache_of(g, pages, 8, 16, 128, 16)
    q = randn(g, 4, 1, 32, 128)
    n = ints(lens)
    f = lambda **kw: paged_attention8(q, k, v, ks, vs, table, n, return_lse=True, **kw)  # noqa: E731
    with torch.inference_mode():
        first = [t.clone() for t in f()]
        for _ in range(3):
            again = f()
            assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
        streams = [torch.cuda.Stream() for _ in range(3)]
        outs = []
        for s in streams * 3:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(f())
        torch.cuda.synchronize()
        for a in outs:
            assert torch.equal(a[0], first[0]) and torch.equal(a[1], first[1])
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        held = []
        for graph, kw in zip(graphs, ({}, dict(window=200, sinks=4))):
            with torch.cuda.graph(graph):
                held.append(f(**kw))
        for more in (1, 400, 1000):
            n.copy_(ints(lens) + more)
            for graph in graphs:
                graph.replay()
            for got, kw in zip(held, ({}, dict(window=200, sinks=4))):
                now = f(**kw)
                assert torch.equal(now[0], got[0]) and torch.equal(now[1], got[1])


def test_attention_of_nothing():
    g = gen(12)
    k, ks = cache_of(g, 4, 2, 16, 64, 16)
    with torch.inference_mode():
        o = paged_attention8(randn(g, 0, 1, 4, 64), k, k, ks, ks, ints([]).view(0, 3), ints([]))
        assert o.shape == (0, 1, 4, 64)
        o = paged_attention8(randn(g, 2, 1, 4, 64), k, k, ks, ks, ints([]).view(2, 0), ints([0, 0]), window=5, sinks=1)
        assert bool((o == 0).all())


def test_inputs_at_odd_addresses_and_strides():
    g = gen(14)
    lens, ps, Hq, Hk, D = [50, 20], 16, 4, 2, 64
    table, pages = tables(g, lens, ps)
    wide = torch.full((2, table.shape[1] * 2), 9, dtype=torch.int32, device=DEV)
    wide[:, ::2] = table
    a, b = ([*cache_of(gen(1), pages, Hk, ps, D, 16), *cache_of(gen(2), pages, Hk, ps, D, 16)] for _ in range(2))
    cos, sin = rope_table(64, D, 1e4, DEV)
    qkv = randn(g, 2, 3, (Hq + 2 * Hk) * D)
    odd = torch.empty(qkv.numel() + 1, dtype=BF, device=DEV)[1:].view_as(qkv)
    odd.copy_(qkv)
    turn = qkv.transpose(0, 1).contiguous().transpose(0, 1)
    scales = torch.zeros(*a[1].shape, 3, device=DEV)
    with torch.inference_mode():
        want = paged_append8(qkv, Hq, Hk, a[0], a[2], a[1], a[3], table, ints(lens), cos, sin)
        for x in (odd, turn):
            c = [t.clone() for t in b]
            ks, vs = scales[..., 1], scales[..., 2]
            ks.copy_(c[1])
            vs.copy_(c[3])
            got = paged_append8(x, Hq, Hk, c[0], c[2], ks, vs, wide[:, ::2], ints([50, 0, 20, 0])[::2], cos, sin)
            assert torch.equal(got, want) and torch.equal(ks, a[1]) and torch.equal(vs, a[3])
            assert torch.equal(c[0].view(torch.uint8), a[0].view(torch.uint8))
            assert torch.equal(c[2].view(torch.uint8), a[2].view(torch.uint8))
            ref = paged_attention8(want, a[0], a[2], a[1], a[3], table, ints(lens))
            q = torch.empty(want.numel() + 1, dtype=BF, device=DEV)[1:].view_as(want)
            q.copy_(want)
            assert torch.equal(paged_attention8(q, c[0], c[2], ks, vs, wide[:, ::2], ints([50, 0, 20, 0])[::2]), ref)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("L", [1, 8])
@pytest.mark.parametrize("window", [None, 60])
def test_one_scale_for_all_and_pages_that_sequences_share(L, window):
    """Scales of stride 0; a prefix's pages in several rows, and one page many times in a row."""
    g = gen(L)
    k, _ = cache_of(g, 9, 2, 16, 64, 16, "hnd", BF)
    v, _ = cache_of(g, 9, 2, 16, 64, 16, "hnd", BF)
    one, two = (torch.full((1, 1, 1), s, device=DEV).expand(9, 2, 1) for s in (0.125, 0.5))
    table = ints([[0, 1, 2, 3, 4, 5], [0, 1, 2, 6, 7, 8], [3, 3, 3, 3, 3, 3]])
    lens = [95, 81, 96]
    q = randn(g, 3, L, 8, 64, dtype=BF)
    with torch.inference_mode():
        o, lse = paged_attention8(q, k, v, one, two, table, ints(lens), return_lse=True, window=window, sinks=3)
        apart = [table[b].long() for b in range(3)]
        k2, v2 = (torch.cat([c.view(torch.uint8)[t] for t in apart]).view(F8) for c in (k, v))
        own = torch.arange(18, dtype=torch.int32, device=DEV).view(3, 6)
        o2, lse2 = paged_attention8(q, k2, v2, one[:1].expand(18, 2, 1).contiguous(), two[:1].expand(18, 2, 1).contiguous(), own,
                                    ints(lens), return_lse=True, window=window, sinks=3)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    check_attention(q, values(k, one), values(v, two), spread_scales(two, 16), table, lens, 64 ** -0.5, None, o, lse, window, 3)
    assert _lib.device_error() == 0
