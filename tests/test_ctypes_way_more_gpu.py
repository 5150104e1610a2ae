"""The 8-bit cache, the window, the page tables and the logit rules without the native binding: the same bits."""
import pytest
import torch

from kernels import _lib
from kernels.logit_rules import adjust_logits, count_tokens, token_bits
from kernels.paged_cache import paged_attention, rope_table
from kernels.paged_cache8 import cache8, paged_append8, paged_attention8
from kernels.paged_tables import page_pool, paged_release, paged_reserve

pytestmark = pytest.mark.gpu
DEV = "cuda"


def calls():
    g = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    c = cache8(9, 2, 16, 128, 8, DEV)
    table = torch.randperm(9, generator=g, device=DEV).int()[:8].view(2, 4)
    lens = i(50, 33)
    turn = rope_table(64, 128, 1e6, DEV)
    out = []
    for n, count in ((40, None), (10, i(10, 3))):
        out.append(paged_append8(r(2, n, 12 * 128), 8, 2, *c, table, i(40, 30) if n == 40 else lens, *turn, r(128), r(128), count=count))
    out += [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t.clone() for t in c]
    k, v = r(9, 2, 16, 128), r(9, 2, 16, 128)
    for L in (1, 6):
        q = r(2, L, 8, 128)
        out += [*paged_attention8(q, *c, table, lens, return_lse=True), paged_attention8(q, *c, table, lens, window=20, sinks=2)]
        out += paged_attention(q, k, v, table, lens, return_lse=True, window=9, sinks=1)
    pool = page_pool(3, 8, 20, DEV)
    out += paged_reserve(pool[0], i(0, 5, 9), *pool[1:], 7, 4, count=i(7, 2, 0))
    paged_release(*pool, i(3, 7, 0), 4)
    out += pool
    counts = torch.zeros(3, 1001, dtype=torch.int32, device=DEV)
    drafts = torch.randint(0, 1001, (3, 4), generator=g, device=DEV)
    count_tokens(counts, drafts)
    out += [counts, adjust_logits(r(3, 5, 1001), counts, drafts, repetition=torch.full((3,), 1.3, device=DEV),
                                  bias_ids=i(5, 6, 7).view(3, 1), bias_values=torch.ones(3, 1, device=DEV),
                                  allowed=token_bits(drafts, 1001))]
    return out


def test_the_same_without_the_binding(monkeypatch):
    with torch.inference_mode():
        want = calls()
        monkeypatch.setattr(_lib, "_binding", _lib._CtypesOnly())
        got = calls()
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
    # lengths 5 and 9 in a pool that is all free: the third row's pages were never taken from it, and it has no room for them
    assert _lib.device_error() == _lib.DEV_ERR_CAPACITY
    _lib.clear_device_error()
