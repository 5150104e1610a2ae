"""The batched speculative step over a paged cache (kernels/sdar_paged.py).

Exactness of a bf16 forward is judged against the same weights in 64 bits: the paged
forward's logits may be off by at most twice what torch's own bf16 forward (the model's
`forward` with a causal mask) is, per row in the 2-norm.
"""
from __future__ import annotations

import pytest
import torch

from kernels import _lib
from kernels.sdar_paged import PagedBatch
from kernels.sdar_verify import SDARShape, SDARVerifyModel

pytestmark = pytest.mark.gpu
DEV = "cuda"


def model_of(head_dim, seed=0):
    s = SDARShape(hidden=512, layers=3, heads=8, kv_heads=2, head_dim=head_dim, intermediate=1024, vocab=4000)
    m = SDARVerifyModel.random_init(s, DEV, torch.bfloat16, seed)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if "proj" in n or "lm_head" in n:
                p.mul_(2.0)
    return m


def torch_logits(m, ids):
    """Causal logits [n, V] of one sequence by the model's own torch forward."""
    n = len(ids)
    mask = torch.ones(n, n, dtype=torch.bool, device=DEV).tril()[None, None]
    with torch.inference_mode():
        return m(torch.tensor(ids, device=DEV)[None], torch.arange(n, device=DEV), mask)[0][0]


def logits_64(m, ids):
    d = SDARVerifyModel(m.s).to(DEV, torch.float64)
    d.load_state_dict({k: v.double() for k, v in m.state_dict().items()})
    return torch_logits(d, ids)


@pytest.mark.parametrize("head_dim,page_size,lens", [(128, 16, [40, 1, 17, 33]), (64, 24, [5, 50, 100])])
def test_paged_forward_is_the_model(head_dim, page_size, lens):
    m = model_of(head_dim)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, m.s.vocab, (n,), generator=g).tolist() for n in lens]
    more = torch.randint(0, m.s.vocab, (len(lens), 4), generator=g).to(DEV)
    batch = PagedBatch(m, len(lens), 128, page_size)
    batch.page_table.copy_(batch.page_table.view(-1)[torch.randperm(batch.page_table.numel(), generator=g).to(DEV)]
                           .view_as(batch.page_table))
    batch.prefill(prompts)
    assert batch.lens.tolist() == [n - 1 for n in lens]
    with torch.inference_mode():
        x = batch.hidden(torch.cat([batch.last[:, None], more], 1))
        got = m.lm_head(x).double()
    for b, p in enumerate(prompts):
        ids = p + more[b].tolist()
        exact, plain = logits_64(m, ids)[len(p) - 1:], torch_logits(m, ids)[len(p) - 1:].double()
        err, ref = (got[b] - exact).norm(dim=-1), (plain - exact).norm(dim=-1)
        assert bool((err <= 2 * ref).all()), (b, (err / ref).tolist())
    assert _lib.device_error() == 0


def noise_of(m, B, K, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.rand(B, K, generator=g, device=DEV),
            torch.empty(B, m.s.vocab, device=DEV).exponential_(generator=g).clamp_(min=1e-20))


def test_greedy_steps_keep_right_drafts_and_move_on():
    m = model_of(128)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, m.s.vocab, (n,), generator=g).tolist() for n in (30, 9, 21)]
    B, K, V = 3, 4, m.s.vocab
    batch = PagedBatch(m, B, 128)
    batch.prefill(prompts)
    zero = torch.zeros(B, device=DEV)
    u, e = noise_of(m, B, K, 3)
    seqs = [list(p) for p in prompts]
    drafts = torch.randint(0, V, (B, K), generator=g).to(DEV)
    for step in range(6):
        before = batch.lens.clone()
        ids = torch.cat([batch.last[:, None], drafts], 1)
        with torch.inference_mode():
            want = m.lm_head(batch.hidden(ids)).float().argmax(-1)        # the step's own greedy tokens, without moving on
        tokens, accepted, _ = batch.step(drafts, u, e, temperature=zero)
        for b in range(B):
            n = 0
            while n < K and int(drafts[b, n]) == int(want[b, n]):
                n += 1
            assert int(accepted[b]) == n and tokens[b].tolist() == drafts[b, :n].tolist() + [int(want[b, n])] + [-1] * (K - n)
            assert int(batch.lens[b]) == int(before[b]) + n + 1 and int(batch.last[b]) == int(want[b, n])
            seqs[b] += tokens[b, : n + 1].tolist()
        # next drafts: two right ones (found one token at a time), then a wrong one
        lens, last = batch.lens.clone(), batch.last.clone()
        none = torch.empty(B, 0, dtype=torch.int64, device=DEV)
        for k in range(K):
            drafts[:, k] = batch.step(none, u[:, :0], e, temperature=zero)[0][:, 0]
        drafts[:, 2] = (drafts[:, 2] + 1) % V
        batch.lens.copy_(lens)
        batch.last.copy_(last)
    assert batch.lens.tolist() == [len(s) - 1 for s in seqs]
    # the cache the steps left behind is the one that the whole sequences give
    fresh = PagedBatch(m, B, 128)
    fresh.prefill(seqs)
    with torch.inference_mode():
        x, y = (b.hidden(b.last[:, None]) for b in (batch, fresh))
    # two bf16 forwards of other batch heights: a few roundings of 2^-9 a layer apart
    assert float((x.float() - y.float()).norm() / y.float().norm()) <= 2.0 ** -6


def test_step_replays_in_a_graph():
    m = model_of(64)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, m.s.vocab, (n,), generator=g).tolist() for n in (12, 25)]
    B, K = 2, 3
    u, e = noise_of(m, B, K, 5)
    drafts = torch.randint(0, m.s.vocab, (B, K), generator=g).to(DEV)
    eager, graphed = PagedBatch(m, B, 96), PagedBatch(m, B, 96)
    eager.prefill(prompts)
    graphed.prefill(prompts)
    lens, last = graphed.lens.clone(), graphed.last.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphed.step(drafts, u, e)                        # warm-up
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = graphed.step(drafts, u, e)
    graphed.lens.copy_(lens)
    graphed.last.copy_(last)
    for step in range(4):
        drafts.copy_(torch.randint(0, m.s.vocab, (B, K), generator=g))
        if step % 2:
            drafts[:, 0] = 7
        now = [t.clone() for t in eager.step(drafts, u, e)]
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(now, held))
        assert torch.equal(eager.lens, graphed.lens) and torch.equal(eager.last, graphed.last)


def test_prefill_refuses():
    m = model_of(64)
    batch = PagedBatch(m, 2, 32)
    with pytest.raises(ValueError):
        batch.prefill([[1, 2]])
    with pytest.raises(ValueError):
        batch.prefill([[1], []])
    with pytest.raises(ValueError):
        batch.prefill([[1], [0] * 33])


def test_example_runs(capsys):
    from kernels import sdar_paged
    sdar_paged.main(sequences=3, drafts=2, steps=4)
    assert "drafts kept per step" in capsys.readouterr().out
