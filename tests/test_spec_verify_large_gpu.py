"""Verification at sizes where a warp takes several blocks of a row and a CTA several runs
of tokens, and the relative precision of log p of a likely token.

log p of a token that the other tokens' sum s - 1 falls short of: log p = -log1p(s - 1).
Every term exp(x - m) of that sum errs by the rounding of its argument, 2^-23 |x - m| (the
scale's and the product's), and by 2^-21 (the exponential, runs of 32-bit sums, the logarithm
and the result's rounding); |x - m| <= 22 here, so 2^-18 of |log p|.
"""
from __future__ import annotations

import pytest
import torch

from kernels import _lib
from kernels.spec_verify import speculative_verify
from test_spec_verify_gpu import BF, DEV, F32, FP, check, inputs, reference

pytestmark = pytest.mark.gpu


# more than 4 x 1024 logits for each of 32 warps on 148 SMs: 19.4 million with all rows
@pytest.mark.parametrize("B,K,V,dtype,drafted,temp,ragged", [
    (20, 4, 110001, BF, True, True, True), (44, 3, 64003, FP, True, False, True), (40, 1, 200003, F32, False, True, False),
    (64, 1, 110592, BF, False, True, True)])
def test_large_batches_match_64_bits(B, K, V, dtype, drafted, temp, ragged):
    assert B * (2 * K + 1) * V >= 148 * 32 * 4 * 1024 and B * V > 148 * 4 * 2048
    target, x, u, e, draft, g = inputs(B + V, B, K, V, dtype)
    # the row's maximum in its first, last and middle parts, so that sums are rescaled and not
    target[::3, :, 1], target[1::3, :, V - 2], target[2::3, :, V // 2 + 3] = 18.0, 18.0, 18.0
    draft = draft if drafted else None
    t = n = None
    if temp:
        t = torch.rand(B, generator=g, device=DEV) + 0.3
        t[::4] = 0.0
    if ragged:
        n = torch.randint(0, K + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
        gone = torch.arange(K, device=DEV) >= n[:, None]
        x.masked_fill_(gone, -1)
        target[:, 1:].masked_fill_(gone[..., None], float("nan"))
    with torch.inference_mode():
        got = speculative_verify(target, x, u, e, draft_logits=draft, temperature=t, n_draft=n)
    assert _lib.device_error() == 0
    check(got, reference(target, x, u, e, draft, t, n), K)


@pytest.mark.parametrize("B,V,dtype", [(3, 32000, BF), (5, 50021, F32), (3, 4001, FP), (64, 110001, BF)])
@pytest.mark.parametrize("gap", [9.0, 16.0])
def test_log_p_of_a_likely_token_keeps_its_relative_precision(B, V, dtype, gap):
    g = torch.Generator(device=DEV).manual_seed(V)
    target = torch.randn(B, 2, V, generator=g, device=DEV).clamp(-6, 6).to(dtype)
    x = torch.randint(0, V, (B, 1), generator=g, device=DEV)
    target[:, 0].scatter_(1, x, gap)
    u, e = torch.zeros(B, 1, device=DEV), torch.ones(B, V, device=DEV)
    with torch.inference_mode():
        tokens, accepted, logprobs = speculative_verify(target, x, u, e)
    assert accepted.tolist() == [1] * B and torch.equal(tokens[:, :1], x)
    l = target[:, 0].double()
    rest = (l - gap).exp().scatter(1, x, 0.0).sum(1)          # log_softmax would round 1 + rest
    ref = -torch.log1p(rest)
    err = ((logprobs[:, 0].double() - ref) / ref).abs()
    assert bool((err <= 2.0 ** -18).all()), float(err.max())
