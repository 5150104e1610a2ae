"""The serving operators without the native binding: the same bits."""
import pytest
import torch

from kernels import _lib
from kernels.paged_cache import paged_append, paged_attention, rope_table
from kernels.spec_verify import speculative_verify

pytestmark = pytest.mark.gpu
DEV = "cuda"


def calls():
    g = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    kc, vc = r(9, 2, 16, 128), r(9, 2, 16, 128)
    at = torch.arange(50, device=DEV)
    q = paged_append(r(50, 12 * 128), 8, 2, kc, vc, at, at, *rope_table(64, 128, 1e6, DEV), r(128), r(128))
    table = torch.randperm(9, generator=g, device=DEV).int()[:8].view(2, 4)
    lens = torch.tensor([50, 33], dtype=torch.int32, device=DEV)
    out = [q, kc, vc]
    for L in (1, 6):
        out += paged_attention(q[:2 * L].view(2, L, 8, 128), kc, vc, table, lens, return_lse=True)
    out.append(paged_attention(q[:2], kc, vc, table, lens))
    t, d = r(3, 5, 1001), r(3, 4, 1001)
    out += speculative_verify(t, torch.randint(0, 1001, (3, 4), generator=g, device=DEV), torch.rand(3, 4, generator=g, device=DEV),
                              torch.rand(3, 1001, generator=g, device=DEV) + 0.01, d)
    return out


def test_the_same_without_the_binding(monkeypatch):
    with torch.inference_mode():
        want = calls()
        monkeypatch.setattr(_lib, "_binding", _lib._CtypesOnly())
        got = calls()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and _lib.device_error() == 0
