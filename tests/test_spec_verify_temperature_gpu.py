"""Very large temperatures: softmax(x / T) tends to the uniform distribution over the tokens
whose logits are not -inf, and is that at T = inf.

Draws are compared where the two best races differ by more than 2^-14 of the larger; log p
within 2^-16 + 2^-20 |log p| (the maximum, sum and scaled difference carry a few 2^-24).
"""
from __future__ import annotations

import math

import pytest
import torch

from kernels.spec_verify import speculative_verify

pytestmark = pytest.mark.gpu
DEV = "cuda"


def law(row, t):
    x = row.double()
    x = torch.where(x.isnan(), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
    if math.isinf(t):
        return torch.where(x == -math.inf, 0.0, 1.0 / float((x != -math.inf).sum()))
    return torch.softmax((x - x.max()) / t, -1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [700, 4001])
@pytest.mark.parametrize("drafted", [False, True])
def test_temperatures_up_to_infinity(dtype, V, drafted):
    g = torch.Generator(device=DEV).manual_seed(V)
    temps = [math.inf, 1e6, 1e30, 3e38, math.inf, 50.0, math.inf, math.inf]
    B, K = len(temps), 2
    target = (torch.randn(B, K + 1, V, generator=g, device=DEV) * 4).to(dtype)
    draft = (torch.randn(B, K, V, generator=g, device=DEV) * 4).to(dtype)
    target[4, :, ::3] = -math.inf
    target[6, :, 100:] = float("nan")
    draft[7, :, 1::2] = -math.inf
    x = torch.randint(0, 99, (B, K), generator=g, device=DEV)
    u = torch.rand(B, K, generator=g, device=DEV) * 0.9
    if not drafted:
        u = u * 3.0 / V                                    # some kept against a probability of about 1 / V
    e = -torch.log1p(-torch.rand(B, V, generator=g, device=DEV)) + 1e-9
    with torch.inference_mode():
        tokens, accepted, logprobs = speculative_verify(target, x, u, e, draft if drafted else None,
                                                        torch.tensor(temps, device=DEV))
    one = lambda i: torch.nn.functional.one_hot(torch.tensor(i, device=DEV), V).double()  # noqa: E731
    left_out = 0
    for b, t in enumerate(temps):
        for i in range(K + 1):
            p = law(target[b, i], t)
            q = torch.zeros_like(p) if i == K else law(draft[b, i], t) if drafted else one(int(x[b, i]))
            if i < K:
                a, c = float(u[b, i]) * float(q[int(x[b, i])]), float(p[int(x[b, i])])
                if abs(a - c) <= 2.0 ** -14 * max(a, c) and max(a, c) > 0:
                    left_out += 1
                    break
                if a < c:
                    assert int(tokens[b, i]) == int(x[b, i])
                    ref = math.log(c)
                    assert abs(float(logprobs[b, i]) - ref) <= 2.0 ** -16 + 2.0 ** -20 * abs(ref), (b, i)
                    continue
            assert int(accepted[b]) == i, (b, i)
            left = (p - q).clamp(min=0)
            left = p if float(left.sum()) < 1e-3 else left
            race = left / e[b].double()
            top = race.topk(2).values
            if float(top[0] - top[1]) <= 2.0 ** -14 * float(top[0]) or 0 < float((p - q).clamp(min=0).sum()) < 1e-3:
                left_out += 1
                break
            new = int(race.argmax())
            assert int(tokens[b, i]) == new, (b, i, t)
            ref = math.log(float(p[new]))
            assert abs(float(logprobs[b, i]) - ref) <= 2.0 ** -16 + 2.0 ** -20 * abs(ref), (b, i)
            break
    assert left_out <= 2
