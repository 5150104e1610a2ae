"""Verification of drafted tokens (kernels/spec_verify.py) against a plain 64-bit
implementation.

Decisions are compared where 32-bit arithmetic cannot turn them: an acceptance
whose two sides differ by less than 2^-14 of the larger, or a draw whose two best
races do, is left out (under 2 % of the sequences).  log p: the maximum, sum and
scaled difference each carry a few 2^-24, and the sum up to 2^-17 (dependent
additions), so 2^-16 + 2^-20 |log p|.
"""
from __future__ import annotations

import math

import pytest
import torch

from kernels import _lib
from kernels.spec_verify import speculative_verify

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def clean(x):
    x = x.double()
    return torch.where(x.isnan(), -math.inf, x).clamp(max=float(torch.finfo(F32).max))


def law(row, t):
    """(p, log p) of one row in 64 bits."""
    x = clean(row)
    if float(x.max()) == -math.inf:
        return torch.zeros_like(x), torch.full_like(x, -math.inf)
    if t == 0:
        p = torch.zeros_like(x)
        p[int((x == x.max()).nonzero()[0])] = 1.0
        return p, p.log()
    lp = torch.log_softmax((x - x.max()) / t, -1)
    return lp.exp(), lp


def reference(target, x, u, e, draft=None, temperature=None, n_draft=None):
    """Per sequence (tokens, accepted, logprobs, sure)."""
    out = []
    for b in range(target.shape[0]):
        t = 1.0 if temperature is None else float(temperature[b])
        d = x.shape[1] if n_draft is None else int(n_draft[b])
        toks, lps, sure, i = [], [], True, 0
        while True:
            p, lp = law(target[b, i], t)
            if i == d:
                left = p
                break
            xi = int(x[b, i])
            q = law(draft[b, i], t)[0] if draft is not None else \
                torch.nn.functional.one_hot(torch.tensor(xi, device=DEV), p.numel()).double()
            a, c = float(u[b, i]) * float(q[xi]), float(p[xi])
            sure &= abs(a - c) > 2.0 ** -14 * max(a, c) or (a == 0 and c == 0)
            if not a < c:
                left = (p - q).clamp(min=0)
                # a residual made of rounding only is as good as none
                sure &= float(left.max()) == 0 or float(left.sum()) > 1e-3
                left = left if float(left.max()) > 0 else p
                break
            toks.append(xi)
            lps.append(float(lp[xi]))
            i += 1
        race = left / e[b].double()
        top = race.topk(min(2, race.numel())).values
        new = int((race == race.max()).nonzero()[0])
        sure &= race.numel() == 1 or float(top[0] - top[1]) > 2.0 ** -14 * float(top[0]) or float(top[0]) == 0
        out.append((toks + [new], i, lps + [float(lp[new])], sure))
    return out


def check(got, ref, K, most=0.02):
    tokens, accepted, logprobs = (t.cpu() for t in got)
    unsure = 0
    for b, (toks, n, lps, sure) in enumerate(ref):
        if not sure:
            unsure += 1
            continue
        assert tokens[b].tolist() == toks + [-1] * (K + 1 - len(toks)), b
        assert int(accepted[b]) == n
        for i, r in enumerate(lps):
            v = float(logprobs[b, i])
            assert v == r if math.isinf(r) else abs(v - r) <= 2.0 ** -16 + 2.0 ** -20 * abs(r), (b, i, v, r)
        assert bool((logprobs[b, len(toks):] == 0).all())
    assert unsure <= most * len(ref) + 1


def inputs(seed, B, K, V, dtype=BF, spread=2.5, off=0.7):
    g = torch.Generator(device=DEV).manual_seed(seed)
    target = torch.randn(B, K + 1, V, generator=g, device=DEV) * spread
    target += 9.0 * (torch.rand(B, K + 1, V, generator=g, device=DEV) < 4.0 / V)
    draft = target[:, :K] + torch.randn(B, K, V, generator=g, device=DEV) * off
    e = torch.empty(B, K, V, device=DEV).exponential_(generator=g)
    x = (draft - e.log()).argmax(-1)
    return (target.to(dtype), x, torch.rand(B, K, generator=g, device=DEV),
            torch.empty(B, V, device=DEV).exponential_(generator=g).clamp_(min=1e-20), draft.to(dtype), g)


@pytest.mark.parametrize("B,K,V,dtype,drafted,temp,ragged", [
    (1, 4, 32000, BF, True, False, False), (40, 3, 1000, FP, True, True, True), (7, 1, 50021, F32, True, True, False),
    (25, 5, 333, BF, False, True, True), (3, 8, 151936, BF, True, False, True), (64, 2, 17, F32, False, False, False),
    (9, 0, 4097, BF, False, True, False), (5, 3, 1, FP, True, False, False), (30, 4, 8191, FP, False, False, False),
    (200, 2, 5, BF, True, True, True)])
def test_matches_64_bits(B, K, V, dtype, drafted, temp, ragged):
    target, x, u, e, draft, g = inputs(B + K + V, B, K, V, dtype)
    draft = draft if drafted and K else None
    t = n = None
    if temp:
        t = torch.rand(B, generator=g, device=DEV) + 0.3
        t[::4] = 0.0
    if ragged:
        n = torch.randint(0, K + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
        gone = torch.arange(K, device=DEV) >= n[:, None]
        x.masked_fill_(gone, -1)
        u.masked_fill_(gone, float("nan"))
        target[:, 1:].masked_fill_(gone[..., None], float("nan"))     # rows past the drafted ones hold anything
        if draft is not None:
            draft.masked_fill_(gone[..., None], float("nan"))
    with torch.inference_mode():
        got = speculative_verify(target, x, u, e, draft_logits=draft, temperature=t, n_draft=n)
        again = speculative_verify(target, x, u, e, draft_logits=draft, temperature=t, n_draft=n)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    assert _lib.device_error() == 0
    check(got, reference(target, x, u, e, draft, t, n), K)


def test_strided_inputs_and_another_stream():
    B, K, V = 6, 3, 1001
    target, x, u, e, draft, _ = inputs(3, B, K, V)
    wide = torch.full((B, K + 3, V + 6), float("nan"), dtype=BF, device=DEV)
    wide[:, 1:K + 2, 3:V + 3] = target
    noise = torch.full((B, V + 5), float("nan"), device=DEV)
    noise[:, 5:] = e
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.inference_mode(), torch.cuda.stream(s):
        got = speculative_verify(wide[:, 1:K + 2, 3:V + 3], x.t().contiguous().t(), u, noise[:, 5:],
                                 draft_logits=draft.transpose(0, 1).contiguous().transpose(0, 1))
    s.synchronize()
    check(got, reference(target, x, u, e, draft), K)


def test_infinities_nan_and_empty_rows():
    """Masked logits (-inf, the type's lowest value), NaN, +inf, a row that leaves nothing."""
    B, K, V = 8, 2, 700
    target, x, u, e, draft, _ = inputs(4, B, K, V, F32)
    target[0, :, 5:] = -math.inf                          # five tokens left
    target[1, :, 9:] = torch.finfo(F32).min
    target[2, :, ::2] = float("nan")
    target[3, 0, 77] = math.inf                           # takes all the weight
    target[4, 0] = -math.inf                              # nothing left: draft refused, token 0
    target[5, 0] = float("nan")
    draft[6, 0] = -math.inf                               # q = 0 everywhere: accepted where p > 0
    target[7, 0, 100] = target[7, 0, 200] = 60.0          # an exact tie
    draft[7, 0] = target[7, 0]
    for t in (None, torch.zeros(B, device=DEV), torch.full((B,), 0.7, device=DEV)):
        with torch.inference_mode():
            got = speculative_verify(target, x, u, e, draft_logits=draft, temperature=t)
        check(got, reference(target, x, u, e, draft, t), K, most=0.2)
        assert got[0][4].tolist() == [0, -1, -1] and float(got[2][4, 0]) == -math.inf


def test_bad_draft_tokens_are_refused_and_flagged():
    B, K, V = 3, 2, 400
    target, x, u, e, draft, _ = inputs(5, B, K, V)
    u.zero_()
    ok = [r for r in reference(target, x, u, e, draft)]
    x[0, 0], x[1, 1] = V, -1
    with torch.inference_mode():
        tokens, accepted, _ = speculative_verify(target, x, u, e, draft_logits=draft)
    assert _lib.device_error() & _lib.DEV_ERR_BAD_INDEX
    _lib.clear_device_error()
    assert accepted.tolist()[:2] == [0, 1] and int(accepted[2]) == ok[2][1]
    for b, i in ((0, 0), (1, 1)):                          # drawn from p
        assert int(tokens[b, i]) == int((law(target[b, i], 1.0)[0] / e[b].double()).argmax())


def test_greedy_is_the_framework_greedy_match():
    """Temperature 0 accepts exactly while the draft is the target's argmax."""
    from kernels.sdar_verify import greedy_match_verify
    B, K, V = 20, 4, 2000
    target, x, u, e, _, g = inputs(6, B, K, V)
    best = target.float().argmax(-1)
    x = torch.where(torch.rand(B, K, generator=g, device=DEV) < 0.7, best[:, :K], x)
    with torch.inference_mode():
        tokens, accepted, _ = speculative_verify(target, x, u, e, temperature=torch.zeros(B, device=DEV))
    for b in range(B):
        acc, n, bonus = greedy_match_verify(x[b].tolist(), best[b, :K].tolist())
        assert int(accepted[b]) == n
        assert tokens[b].tolist()[: len(acc)] == acc
        if bonus is None:
            assert int(tokens[b, K]) == int(best[b, K])


def test_emitted_tokens_follow_the_target():
    """First emitted token over 60000 sequences of one draft and target: every frequency
    within five standard deviations of the target's probability."""
    B, V = 60000, 11
    g = torch.Generator(device=DEV).manual_seed(7)
    target, draft = torch.randn(2, V, generator=g, device=DEV) * 1.5, torch.randn(1, V, generator=g, device=DEV) * 1.5
    x = torch.multinomial(torch.softmax(draft[0].double(), -1), B, replacement=True, generator=g).view(B, 1)
    u = torch.rand(B, 1, generator=g, device=DEV)
    e = torch.empty(B, V, device=DEV).exponential_(generator=g).clamp_(min=1e-20)
    with torch.inference_mode():
        tokens, accepted, _ = speculative_verify(target.expand(B, 2, V), x, u, e, draft_logits=draft.expand(B, 1, V))
    p = torch.softmax(target[0].double(), -1)
    f = torch.bincount(tokens[:, 0], minlength=V).double() / B
    assert bool(((f - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all())
    q = torch.softmax(draft[0].double(), -1)
    rate, kept = float(torch.minimum(p, q).sum()), float(accepted.double().mean())
    assert abs(kept - rate) <= 5 * math.sqrt(rate * (1 - rate) / B)


def test_in_a_graph():
    B, K, V = 4, 3, 5000
    target, x, u, e, draft, _ = inputs(8, B, K, V)
    with torch.inference_mode():
        speculative_verify(target, x, u, e, draft_logits=draft)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = speculative_verify(target, x, u, e, draft_logits=draft)
        for seed in (9, 10):
            new = inputs(seed, B, K, V)
            for a, b in zip((target, x, u, e, draft), new):
                a.copy_(b)
            graph.replay()
            check(held, reference(target, x, u, e, draft), K)


def test_no_sequences():
    with torch.inference_mode():
        t, a, l = speculative_verify(torch.empty(0, 3, 10, device=DEV), torch.empty(0, 2, dtype=torch.int64, device=DEV),
                                     torch.empty(0, 2, device=DEV), torch.empty(0, 10, device=DEV))
    assert t.shape == (0, 3) and a.shape == (0,) and l.shape == (0, 3)
