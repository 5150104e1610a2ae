"""`PagedBatch.step` up to and past the end of a sequence's room.

A second batch of the same model with four times the room takes the same steps, with the
drafts cut by hand to what the small one has room for.  Lengths, launches and arithmetic
are then the same, so every output of a sequence that still has room is equal bit for bit.
"""
from __future__ import annotations

import pytest
import torch

from kernels import _lib
from kernels.sdar_paged import PagedBatch
from kernels.sdar_verify import SDARShape, SDARVerifyModel

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPE = SDARShape(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=128, intermediate=1024, vocab=4000)


def batches(lens, max_len, masked, K, page_size):
    m = SDARVerifyModel.random_init(SHAPE, DEV, torch.bfloat16, 0)
    g = torch.Generator().manual_seed(sum(lens))
    prompts = [torch.randint(0, SHAPE.vocab, (n,), generator=g).tolist() for n in lens]
    mask = torch.ones(K + 1, K + 1, dtype=torch.bool, device=DEV) if masked else None
    small, big = (PagedBatch(m, len(lens), n, page_size, tail_mask=mask) for n in (max_len, 4 * max_len))
    small.prefill(prompts)
    big.prefill(prompts)
    return small, big, g


@pytest.mark.parametrize("lens,K,masked,page_size", [([44, 48, 30], 4, False, 16), ([45, 47], 7, True, 16),
                                                     ([48, 47, 41], 1, False, 8), ([46, 40], 0, False, 24)])
def test_steps_to_the_end(lens, K, masked, page_size):
    limit = 48
    small, big, g = batches(lens, limit, masked, K, page_size)
    B = len(lens)
    for step in range(24):
        room = limit - small.lens
        live = room > 0
        drafts = torch.randint(0, SHAPE.vocab, (B, K), generator=g).to(DEV)
        u = torch.where(torch.rand(B, K, generator=g) < 0.3, 2.0, 0.0).to(DEV)          # refused or kept
        e = (torch.rand(B, SHAPE.vocab, generator=g) + 1e-3).to(DEV)
        held = (small.lens.clone(), small.last.clone())
        # a full sequence adds no keys to the small batch: the same lengths in the big one
        big.lens.copy_(torch.where(live, small.lens, small.lens - (K + 1)))
        big.last.copy_(small.last)
        got = small.step(drafts, u, e)
        want = big.step(drafts, u, e, n_draft=(room - 1).clamp(0, K).to(torch.int32))
        for a, b in zip(got, want):
            assert torch.equal(a[live], b[live]), step
        assert bool((got[0][~live] == -1).all()) and bool((got[1][~live] == 0).all()) and bool((got[2][~live] == 0).all())
        assert torch.equal(small.lens, torch.where(live, held[0] + (want[1] + 1).to(torch.int32), held[0]))
        assert torch.equal(small.last[~live], held[1][~live])
        assert int(small.lens.max()) <= limit and _lib.device_error() == 0
    assert not bool((small.lens < limit).any())                 # every sequence came to its end


def test_a_step_of_more_drafts_than_were_planned_for():
    """Where fewer than K more tokens have a place in the table, the sequence ends."""
    K = 6
    m = SDARVerifyModel.random_init(SHAPE, DEV, torch.bfloat16, 1)
    g = torch.Generator().manual_seed(5)
    batch = PagedBatch(m, 1, 32, 16, max_drafts=2)              # places for 48 tokens
    batch.prefill([torch.randint(0, SHAPE.vocab, (30,), generator=g).tolist()])
    cap = batch.page_table.shape[1] * batch.page_size
    while int(batch.lens) < 32 and int(batch.lens) + K + 1 <= cap:
        before = int(batch.lens)
        tokens, accepted, _ = batch.step(torch.zeros(1, K, dtype=torch.int64, device=DEV), torch.zeros(1, K, device=DEV),
                                         torch.ones(1, SHAPE.vocab, device=DEV))
        assert int(accepted) == min(K, 32 - before - 1) and int(batch.lens) == before + int(accepted) + 1
    tokens, accepted, _ = batch.step(torch.zeros(1, K, dtype=torch.int64, device=DEV), torch.zeros(1, K, device=DEV),
                                     torch.ones(1, SHAPE.vocab, device=DEV))
    assert bool((tokens == -1).all()) and int(accepted) == 0 and _lib.device_error() == 0


def test_counts_of_drafts_are_one_a_sequence():
    batch = PagedBatch(SDARVerifyModel.random_init(SHAPE, DEV, torch.bfloat16, 2), 2, 32)
    with pytest.raises(ValueError):
        batch.step(torch.zeros(2, 1, dtype=torch.int64, device=DEV), torch.zeros(2, 1, device=DEV),
                   torch.ones(2, SHAPE.vocab, device=DEV), n_draft=torch.ones(1, dtype=torch.int32, device=DEV))
