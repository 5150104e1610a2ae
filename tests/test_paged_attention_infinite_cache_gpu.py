"""Long caches full of infinite values, at the numbers of rows that settle them key by key:
the call ends well inside the kernels' wait limit (no DEV_ERR_TIMEOUT) with infinities."""
import math

import pytest
import torch

from kernels import _lib
from kernels.paged_cache import paged_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("L,ps,dtype", [(8, 16, torch.bfloat16), (16, 1, torch.float16), (16, 64, torch.bfloat16)])
def test_a_long_cache_of_infinities(L, ps, dtype):
    B, n, Hk, D = 3, 131072, 2, 128
    g = torch.Generator(device=DEV).manual_seed(L)
    pages = n // ps
    kc = torch.randn(pages, Hk, ps, D, generator=g, device=DEV).mul_(0.3).to(dtype)
    vc = torch.full((pages, Hk, ps, D), math.inf, dtype=dtype, device=DEV)
    vc[..., D // 2:] = -math.inf
    table = torch.stack([torch.randperm(pages, generator=g, device=DEV).int() for _ in range(B)])    # pages may be shared
    q = torch.randn(B, L, 8, D, generator=g, device=DEV).to(dtype)
    lens = torch.tensor([n, 700, n - 5], dtype=torch.int32, device=DEV)
    with torch.inference_mode():
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        o, lse = paged_attention(q, kc, vc, table, lens, return_lse=True)
        b.record()
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    assert bool((o[..., : D // 2] == math.inf).all()) and bool((o[..., D // 2:] == -math.inf).all())
    assert bool(lse.isfinite().all()) and a.elapsed_time(b) < 1000
