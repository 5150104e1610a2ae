"""Rules on logits (kernels/logit_rules.py) against a plain 64-bit implementation.

Tolerance.  u is half a step of the logits' type relative to the value (2^-8 bf16, 2^-11
fp16, 2^-24 fp32).  In 32 bits: the repetition step (a division or product), frequency
times count with the logit (one rounding more where it is not fused), presence, the sum of n
biases (n roundings) and its addition, each at most 2^-24 of the magnitudes that are
added so far: (4 + n) 2^-24 mag.  Then one rounding, u of the result, and fp16's smallest step.
"""
from __future__ import annotations

import math

import pytest
import torch

from kernels import _lib
from kernels.logit_rules import adjust_logits, count_tokens, token_bits

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP, FL = torch.bfloat16, torch.float16, torch.float32
U = {BF: 2.0 ** -8, FP: 2.0 ** -11, FL: 2.0 ** -24}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def bits(words, V):
    v = torch.arange(V, device=DEV)
    return (words[..., v // 32].long() >> (v % 32) & 1).bool()


def reference(x, counts=None, drafts=None, repetition=None, presence=None, frequency=None, seen=None, bias_ids=None,
              bias_values=None, allowed=None):
    """(value, magnitude) in 64 bits."""
    y = x.double().clone()
    B, R, V = y.shape
    mag = y.abs()
    for b in range(B):
        c = counts[b].double().clone() if counts is not None else torch.zeros(V, dtype=torch.float64, device=DEV)
        prompt = bits(seen[b], V) if seen is not None else torch.zeros(V, dtype=torch.bool, device=DEV)
        bias, size = torch.zeros(V, dtype=torch.float64, device=DEV), torch.zeros(V, dtype=torch.float64, device=DEV)
        if bias_ids is not None:
            for i, v in zip(bias_ids[b].tolist(), bias_values[b].double().tolist()):
                if 0 <= i < V:
                    bias[i] += v
                    size[i] += abs(v)
        for i in range(R):
            if i > 0 and drafts is not None and 0 <= int(drafts[b, i - 1]) < V:
                c[int(drafts[b, i - 1])] += 1
            z = y[b, i].clone()
            met = c > 0
            if any(t is not None for t in (repetition, presence, frequency)):
                r = float(repetition[b]) if repetition is not None else 1.0
                z = torch.where(met | prompt, torch.where(z > 0, z / r, z * r), z)
                f = float(frequency[b]) if frequency is not None else 0.0
                p = float(presence[b]) if presence is not None else 0.0
                mag[b, i] = torch.maximum(mag[b, i], z.abs()) + abs(f) * c + abs(p) * met
                z = z - f * c - p * met
            z = z + bias
            mag[b, i] += size
            if allowed is not None:
                z = z.masked_fill(~bits(allowed[b] if allowed.ndim == 2 else allowed[b, i], V), -math.inf)
            y[b, i] = z
    return y, mag


def check(got, x, n_bias=0, **rules):
    ref, mag = reference(x, **rules)
    assert got.shape == x.shape and got.dtype == x.dtype
    got = got.double()
    fine = ref.isfinite() & (ref.abs() < torch.finfo(x.dtype).max)
    assert torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got[ref.isinf()], ref[ref.isinf()])
    bound = U[x.dtype] * ref.abs() + (4 + n_bias) * 2.0 ** -24 * mag * (1 + U[x.dtype]) + (2.0 ** -25 if x.dtype == FP else 1e-40)
    err = (got - ref).abs()
    assert bool((err <= bound)[fine].all()), float((err / bound)[fine].max())
    assert _lib.device_error() == 0


def rules_of(g, B, R, V, penalties=True, seen=True, bias=20, mask="rows"):
    k = {}
    if penalties:
        k["counts"] = torch.randint(0, 4, (B, V), generator=g, device=DEV, dtype=torch.int32)
        k["counts"] *= torch.rand(B, V, generator=g, device=DEV) < 0.2
        k["drafts"] = torch.randint(0, V, (B, R - 1), generator=g, device=DEV)
        if R > 2:
            k["drafts"][:, 1] = k["drafts"][:, 0]           # drafted twice
        if R > 4:
            k["drafts"][0, 3] = -1
            k["drafts"][-1, 2] = V + 7
        k["repetition"] = torch.rand(B, generator=g, device=DEV) + 0.7
        k["presence"] = torch.randn(B, generator=g, device=DEV)
        k["frequency"] = torch.randn(B, generator=g, device=DEV)
        if seen:
            k["seen"] = token_bits(torch.randint(-3, V + 3, (B, 30), generator=g, device=DEV), V)
    if bias:
        k["bias_ids"] = torch.randint(-V // 4 - 1, V, (B, bias), generator=g, device=DEV, dtype=torch.int32)
        k["bias_ids"][:, -1] = k["bias_ids"][:, 0]           # the same token twice
        k["bias_ids"][0, 0] = V - 1
        k["bias_values"] = torch.randn(B, bias, generator=g, device=DEV) * 4
    if mask:
        shape = (B, R) if mask == "rows" else (B,)
        k["allowed"] = token_bits(torch.randint(0, V, (*shape, max(1, V // 3)), generator=g, device=DEV), V)
        k["allowed"].view(-1, k["allowed"].shape[-1])[-1] = 0        # a row that allows nothing
    return k


@pytest.mark.parametrize("B,R,V,dtype,kw", [
    (1, 1, 1, FL, {}), (1, 1, 7, BF, {}), (2, 3, 31, FP, {}), (3, 5, 32, BF, dict(mask="sequence")), (1, 4, 33, FL, {}),
    (2, 2, 2047, BF, {}), (2, 2, 2048, BF, {}), (2, 6, 2056, FP, {}), (1, 8, 4096, FL, dict(bias=600)),
    (3, 2, 5003, FL, dict(bias=1)), (2, 9, 32000, BF, dict(bias=300)), (1, 3, 50021, BF, dict(seen=False)),
    (2, 2, 8000, BF, dict(penalties=False)), (2, 2, 8000, FP, dict(bias=0, mask="")), (1, 1, 8008, FL, dict(penalties=False, bias=0)),
    (70, 2, 640, BF, {}), (1, 32, 2100, FP, {})])
def test_rules_match_64_bits(B, R, V, dtype, kw):
    g = gen(B * 7 + V)
    x = (torch.randn(B, R, V, generator=g, device=DEV) * 3).to(dtype)
    rules = rules_of(g, B, R, V, **kw)
    n = rules["bias_ids"].shape[1] if "bias_ids" in rules else 0
    with torch.inference_mode():
        y = adjust_logits(x, **rules)
        check(y, x, n, **rules)
        # the same bits in place, into rows apart, from rows apart
        z = x.clone()
        assert adjust_logits(z, **rules, out=z) is z and torch.equal(z.nan_to_num(7), y.nan_to_num(7))
        wide = torch.zeros(B, R, V + 3, dtype=dtype, device=DEV)
        assert torch.equal(adjust_logits(x, **rules, out=wide[..., :V]), y) and bool((wide[..., V:] == 0).all())
        wide[..., :V] = x
        assert torch.equal(adjust_logits(wide[..., :V], **rules), y)


def test_nothing_to_apply_and_nothing_at_all():
    g = gen(1)
    x = torch.randn(2, 3, 1000, generator=g, device=DEV).to(BF)
    with torch.inference_mode():
        assert torch.equal(adjust_logits(x), x)
        # counts, drafts and prompt do nothing without a penalty
        k = rules_of(g, 2, 3, 1000, bias=0, mask="")
        assert torch.equal(adjust_logits(x, counts=k["counts"], drafts=k["drafts"], seen=k["seen"]), x)
        assert adjust_logits(x[:0]).shape == (0, 3, 1000) and adjust_logits(x[:, :0]).shape == (2, 0, 1000)


@pytest.mark.parametrize("which", ["repetition", "presence", "frequency"])
def test_each_penalty_alone(which):
    g = gen(2)
    B, R, V = 2, 4, 3001
    x = torch.randn(B, R, V, generator=g, device=DEV)
    k = rules_of(g, B, R, V, bias=0, mask="")
    only = {which: k[which]}
    with torch.inference_mode():
        for more in (dict(counts=k["counts"]), dict(drafts=k["drafts"]), dict(seen=k["seen"]),
                     dict(counts=k["counts"], drafts=k["drafts"], seen=k["seen"])):
            check(adjust_logits(x, **only, **more), x, **only, **more)


def test_numbers_that_are_not_finite():
    """Masked NaN and infinities are -inf; allowed ones stay, and no neighbour is touched."""
    g = gen(3)
    B, R, V = 1, 2, 2050
    x = torch.randn(B, R, V, generator=g, device=DEV)
    low = torch.finfo(FL).min
    x[0, :, :8] = torch.tensor([math.nan, math.inf, -math.inf, low, math.nan, math.inf, -math.inf, low], device=DEV)
    allowed = token_bits(torch.arange(4, V, device=DEV)[None], V)
    rules = dict(allowed=allowed, counts=torch.ones(B, V, dtype=torch.int32, device=DEV),
                 repetition=torch.tensor([1.25], device=DEV), presence=torch.tensor([0.5], device=DEV))
    with torch.inference_mode():
        for t in (FL, BF, FP):
            y = adjust_logits(x.to(t), **rules)
            assert bool((y[0, :, :4] == -math.inf).all()) and bool(y[0, :, 4].isnan().all())
            assert bool((y[0, :, 5] == math.inf).all()) and bool((y[0, :, 6] == -math.inf).all())
            assert bool(y[0, :, 8:].isfinite().all())
            check(y[..., 8:], x.to(t)[..., 8:], counts=rules["counts"][:, 8:], repetition=rules["repetition"],
                  presence=rules["presence"])


def test_bad_ids_are_flagged():
    x = torch.zeros(2, 1, 100, device=DEV)
    ids = torch.tensor([[5, -1], [100, 7]], dtype=torch.int32, device=DEV)
    with torch.inference_mode():
        y = adjust_logits(x, bias_ids=ids, bias_values=torch.ones(2, 2, device=DEV))
    assert _lib.device_error() == _lib.DEV_ERR_BAD_INDEX
    _lib.clear_device_error()
    want = torch.zeros_like(x)
    want[0, 0, 5] = want[1, 0, 7] = 1
    assert torch.equal(y, want)


def test_counts():
    g = gen(4)
    B, N, V = 5, 300, 50
    counts = torch.randint(0, 9, (B, V + 2), generator=g, device=DEV, dtype=torch.int32)
    before = counts.clone()
    tokens = torch.randint(-5, V, (B, N), generator=g, device=DEV)
    count_tokens(counts[:, :V], tokens)
    want = before.clone()
    for b in range(B):
        t = tokens[b][tokens[b] >= 0]
        want[b, :V] += torch.bincount(t, minlength=V).to(torch.int32)
    assert torch.equal(counts, want) and _lib.device_error() == 0
    count_tokens(counts[:, :V], torch.full((B, 1), V, device=DEV))
    assert torch.equal(counts, want) and _lib.device_error() == _lib.DEV_ERR_BAD_INDEX
    _lib.clear_device_error()
    count_tokens(counts[:, :V], tokens[:, :0])
    count_tokens(counts[:, :V], tokens.t().contiguous().t()[:, ::2])
    assert torch.equal(counts.sum() - want.sum(), (tokens[:, ::2] >= 0).sum())


def test_token_bits():
    t = torch.tensor([[0, 31, 32, 63, 64, 31], [-1, 70, 69, 5, 5, 5]])
    w = token_bits(t, 70)
    assert w.dtype == torch.int32 and w.tolist() == [[-(1 << 31) + 1, -(1 << 31) + 1, 1], [32, 0, 32]]


def test_streams_and_graphs():
    g = gen(5)
    B, R, V = 3, 4, 9000
    x = torch.randn(B, R, V, generator=g, device=DEV).to(BF)
    k = rules_of(g, B, R, V)
    with torch.inference_mode():
        want = adjust_logits(x, **k)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = adjust_logits(x, **k)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = adjust_logits(x, **k)
            count_tokens(k["counts"], k["drafts"].clamp(max=V - 1))
        for _ in range(3):
            want = adjust_logits(x, **k)
            graph.replay()
            assert torch.equal(held, want)


@pytest.mark.parametrize("B,R,V,dtype,kw", [(1, 300, 2056, BF, {}), (2, 520, 37, FL, dict(bias=3)), (2, 3, 4096, FP, dict(bias=1500)),
                                            (1, 2, 50, FL, dict(bias=2100))])
def test_many_drafts_and_long_bias_lists(B, R, V, dtype, kw):
    g = gen(B + R + V)
    x = (torch.randn(B, R, V, generator=g, device=DEV) * 3).to(dtype)
    rules = rules_of(g, B, R, V, **kw)
    with torch.inference_mode():
        check(adjust_logits(x, **rules), x, rules["bias_ids"].shape[1], **rules)


def test_rows_in_another_order_and_the_same_row_for_all():
    g = gen(5)
    B, R, V = 3, 4, 2048
    rules = rules_of(g, B, R, V)
    with torch.inference_mode():
        x = torch.randn(1, R, V, generator=g, device=DEV).to(BF).expand(B, R, V)
        y = adjust_logits(x.contiguous(), **rules)
        assert torch.equal(adjust_logits(x, **rules), y)
        turned = torch.empty(R, B, V, dtype=BF, device=DEV).transpose(0, 1)
        assert adjust_logits(x, **rules, out=turned) is turned and torch.equal(turned, y)
        with pytest.raises(ValueError, match="share memory"):
            adjust_logits(x.contiguous(), **rules, out=x)
