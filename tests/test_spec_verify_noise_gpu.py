"""Noise that no token wins with: a valid token comes out, the error word says so, and the
other sequences are as without it."""
import math

import pytest
import torch

from kernels import _lib
from kernels.spec_verify import speculative_verify

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1, 700, 4001])
@pytest.mark.parametrize("drafted", [False, True])
def test_noise_of_nan_draws_a_valid_token_and_is_flagged(dtype, V, drafted):
    g = torch.Generator(device=DEV).manual_seed(V)
    B, K = 5, 2
    target = torch.randn(B, K + 1, V, generator=g, device=DEV).to(dtype)
    draft = torch.randn(B, K, V, generator=g, device=DEV).to(dtype) if drafted else None
    x = torch.randint(0, V, (B, K), generator=g, device=DEV)
    u = torch.rand(B, K, generator=g, device=DEV)
    noise = torch.rand(B, V, generator=g, device=DEV) + 0.01
    t = torch.tensor([1.0, 0.7, 0.0, 1.0, 0.0], device=DEV)
    with torch.inference_mode():
        want = speculative_verify(target, x, u, noise, draft, t)
        assert _lib.device_error() == 0
        bad = noise.clone()
        bad[1] = bad[4] = math.nan                         # the greedy sequence 4 does not read it
        got = speculative_verify(target, x, u, bad, draft, t)
        assert _lib.device_error() == _lib.DEV_ERR_BAD_INDEX
        _lib.clear_device_error()
        for b in (0, 2, 3, 4):
            assert all(torch.equal(a[b], c[b]) for a, c in zip(got, want)), b
        assert torch.equal(got[1], want[1])
        n = int(got[1][1])
        assert got[0][1, :n].tolist() == x[1, :n].tolist() and int(got[0][1, n]) == 0
        # some of it NaN: those tokens are not drawn
        part = noise.clone()
        part[1, ::2] = math.nan
        if V > 1:
            got = speculative_verify(target, x, u, part, draft, t)
            n = int(got[1][1])
            if n == K:
                assert int(got[0][1, n]) % 2 == 1
            assert _lib.device_error() == 0
