"""Token ids outside the vocabulary: drafted ones are refused and flagged, prompts refused."""
from __future__ import annotations

import pytest
import torch

from kernels import _lib
from kernels.sdar_paged import PagedBatch
from kernels.sdar_verify import SDARShape, SDARVerifyModel

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPE = SDARShape(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=128, intermediate=1024, vocab=1000)


def test_drafts_outside_the_vocabulary_are_refused():
    m = SDARVerifyModel.random_init(SHAPE, DEV, torch.bfloat16, 0)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, SHAPE.vocab, (n,), generator=g).tolist() for n in (10, 20, 5, 7)]
    drafts = torch.randint(0, SHAPE.vocab, (4, 3), generator=g).to(DEV)
    bad = drafts.clone()
    bad[0, 1], bad[1, 0], bad[3, 2] = SHAPE.vocab, 1 << 40, -5
    u, e = torch.zeros(4, 3, device=DEV), (torch.rand(4, SHAPE.vocab, generator=g) + 1e-3).to(DEV)
    batches = [PagedBatch(m, 4, 64) for _ in range(2)]
    for b in batches:
        b.prefill(prompts)
    want = batches[0].step(drafts, u, e)
    assert want[1].tolist() == [3] * 4 and _lib.device_error() == 0
    got = batches[1].step(bad, u, e)
    assert _lib.device_error() == _lib.DEV_ERR_BAD_INDEX
    _lib.clear_device_error()
    assert got[1].tolist() == [1, 0, 3, 2]
    assert all(torch.equal(a[2], b[2]) for a, b in zip(got, want))
    for b, n in enumerate(got[1].tolist()):
        assert got[0][b, :n].tolist() == drafts[b, :n].tolist() and 0 <= int(got[0][b, n]) < SHAPE.vocab
    assert batches[1].lens.tolist() == [len(p) - 1 + n + 1 for p, n in zip(prompts, got[1].tolist())]


@pytest.mark.parametrize("token", [SHAPE.vocab, -1])
def test_prompts_outside_the_vocabulary_are_refused(token):
    batch = PagedBatch(SDARVerifyModel.random_init(SHAPE, DEV, torch.bfloat16, 0), 2, 64)
    with pytest.raises(ValueError):
        batch.prefill([[1, 2, 3], [4, token, 5]])
