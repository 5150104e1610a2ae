"""`PagedBatch` with a shared pool of pages, a cache in 8 bits, a window, and rules on the logits.

Where pages lie changes no number: with a pool every output equals bit for bit.  Over the 8-bit cache the
forward is compared with one in 64 bits that reads the batch's own stored keys and values: what is
left are the roundings of bf16 activations, some eight of 2^-9 a layer, under 2^-6 together
over three layers in the 2-norm.
"""
from __future__ import annotations

import pytest
import torch

from kernels import _lib
from kernels.paged_cache8 import F8
from kernels.sdar_paged import PagedBatch, main
from kernels.sdar_verify import SDARShape, SDARVerifyModel

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPE = SDARShape(hidden=512, layers=3, heads=8, kv_heads=2, head_dim=128, intermediate=1024, vocab=4000)


def model():
    return SDARVerifyModel.random_init(SHAPE, DEV, torch.bfloat16, 0)


def prompts_of(lens, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, SHAPE.vocab, (n,), generator=g).tolist() for n in lens]


def inputs(B, K, g):
    return (torch.randint(0, SHAPE.vocab, (B, K), generator=g).to(DEV), torch.where(torch.rand(B, K, generator=g) < 0.4, 2.0, 0.0).to(DEV),
            (torch.rand(B, SHAPE.vocab, generator=g) + 1e-3).to(DEV))


def pool_holds(batch):
    held, free, count = batch.pool
    want = [-(-n // batch.page_size) for n in batch.lens.tolist()]
    assert held.tolist() == want and int(count) == free.numel() - sum(want)
    used = [p for b, n in enumerate(want) for p in batch.page_table[b, :n].tolist()] + free[: int(count)].tolist()
    assert sorted(used) == list(range(free.numel()))


@pytest.mark.parametrize("kw", [{}, dict(cache_dtype=F8), dict(window=20, sinks=3), dict(cache_dtype=F8, window=20, sinks=3, block=4)])
def test_pages_from_a_pool_change_nothing(kw):
    m, lens, K = model(), [40, 1, 17, 33], 3
    own, shared = PagedBatch(m, 4, 96, **kw), PagedBatch(m, 4, 96, pages=18, **kw)
    for b in (own, shared):
        b.prefill(prompts_of(lens))
    pool_holds(shared)
    g = torch.Generator().manual_seed(2)
    for step in range(12):
        drafts, u, e = inputs(4, K, g)
        for a, b in zip(own.step(drafts, u, e), shared.step(drafts, u, e)):
            assert torch.equal(a, b), step
        assert torch.equal(own.lens, shared.lens) and torch.equal(own.last, shared.last)
        pool_holds(shared)
        if step == 6:
            done = torch.tensor([False, True, False, True], device=DEV)
            for b in (own, shared):
                b.finish(done)
            pool_holds(shared)
    assert _lib.device_error() == 0


def test_a_pool_that_runs_out():
    """The sequence that gets no page stays as it is; another's end lets it move on."""
    m, K = model(), 3
    batch = PagedBatch(m, 2, 64, pages=4)
    batch.prefill(prompts_of([33, 31]))                    # 2 pages each: full, and all but
    g = torch.Generator().manual_seed(3)
    drafts, u, e = inputs(2, K, g)
    tokens, accepted, logprobs = batch.step(drafts, u, e)
    assert _lib.device_error() == _lib.DEV_ERR_CAPACITY
    _lib.clear_device_error()
    assert tokens[0].tolist() == [-1] * (K + 1) and int(accepted[0]) == 0 and float(logprobs[0].abs().sum()) == 0.0
    assert int(batch.lens[0]) == 32
    pool_holds(batch)
    batch.finish(torch.tensor([False, True], device=DEV))
    tokens, accepted, _ = batch.step(drafts, u, e)
    assert int(tokens[0, 0]) >= 0 and int(batch.lens[0]) == 33 + int(accepted[0]) and _lib.device_error() == 0
    with pytest.raises(ValueError, match="pool"):
        batch.prefill(prompts_of([40, 40]))


def reference(m, batch, b, ids, kw):
    """Final-norm states in 64 bits of the last len(ids) tokens of sequence b, over the batch's stored keys and values."""
    n, L, s = int(batch.lens[b]) + len(ids), len(ids), SHAPE
    d = SDARVerifyModel(s).to(DEV, torch.float64)
    d.load_state_dict({k: v.double() for k, v in m.state_dict().items()})
    pos = torch.arange(n - L, n, device=DEV)
    cos, sin = batch.cos.double()[pos][:, None], batch.sin.double()[pos][:, None]
    norm = lambda x, w, eps: x * (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * w  # noqa: E731
    j = torch.arange(n, device=DEV)
    see = j <= pos[:, None]
    if kw.get("window"):
        see &= (j > pos[:, None] - kw["window"]) | (j < kw["sinks"])
    h = d.embed_tokens(torch.tensor(ids, device=DEV))
    pages = batch.page_table[b, : -(-n // batch.page_size)].long()
    for layer, (kc, vc, ks, vs) in zip(d.layers, batch.caches):
        a = layer.self_attn
        x = norm(h, layer.input_layernorm.weight, layer.input_layernorm.eps)
        q = norm(a.q_proj(x).view(L, s.heads, s.head_dim), a.q_norm.weight, a.q_norm.eps)
        y, z = q.chunk(2, -1)
        q = torch.cat([y * cos - z * sin, z * cos + y * sin], -1).view(L, s.kv_heads, -1, s.head_dim)
        value = lambda c, t: (c[pages].double() * t[pages].double().repeat_interleave(c.shape[2] // t.shape[2], 2)[..., None]  # noqa: E731
                              ).transpose(1, 2).reshape(-1, s.kv_heads, s.head_dim)[:n]
        w = torch.einsum("lhgd,nhd->lhgn", q, value(kc, ks)) * s.head_dim ** -0.5
        w = torch.softmax(w.masked_fill(~see[:, None, None], -torch.inf), -1)
        h = h + a.o_proj(torch.einsum("lhgn,nhd->lhgd", w, value(vc, vs)).reshape(L, -1))
        h = h + layer.mlp(norm(h, layer.post_attention_layernorm.weight, layer.post_attention_layernorm.eps))
    return norm(h, d.norm.weight, d.norm.eps)


@pytest.mark.parametrize("kw", [dict(), dict(window=24, sinks=2)])
def test_forward_over_the_8_bit_cache(kw):
    m, lens = model(), [40, 1, 70]
    batch = PagedBatch(m, 3, 128, page_size=32, cache_dtype=F8, **kw)
    batch.prefill(prompts_of(lens), chunk=7)
    more = torch.randint(0, SHAPE.vocab, (3, 4), generator=torch.Generator().manual_seed(5)).to(DEV)
    ids = torch.cat([batch.last[:, None], more], 1)
    with torch.inference_mode():
        x = batch.hidden(ids).double()
        for b in range(3):
            ref = reference(m, batch, b, ids[b].tolist(), kw)
            assert float((x[b] - ref).norm() / ref.norm()) <= 2.0 ** -6, b
    assert _lib.device_error() == 0


def test_rules_on_a_step():
    """Only allowed tokens come out, the counts are those of what came out, and repeated tokens give way."""
    m, K, B = model(), 2, 3
    batch = PagedBatch(m, B, 128)
    batch.prefill(prompts_of([9, 20, 5]))
    g = torch.Generator().manual_seed(6)
    some = torch.randperm(SHAPE.vocab, generator=g)[:40]
    from kernels.logit_rules import token_bits
    counts = torch.zeros(B, SHAPE.vocab, dtype=torch.int32, device=DEV)
    rules = dict(counts=counts, presence=torch.full((B,), 1e4, device=DEV),
                 allowed=token_bits(some.to(DEV)[None].expand(B, -1), SHAPE.vocab))
    seen = [[] for _ in range(B)]
    for step in range(10):
        drafts, u, e = inputs(B, K, g)
        tokens, accepted, _ = batch.step(drafts, u, e, temperature=torch.zeros(B, device=DEV), rules=rules)
        for b in range(B):
            seen[b] += tokens[b, : int(accepted[b]) + 1].tolist()
    for b in range(B):
        assert set(seen[b]) <= set(some.tolist()) and len(set(seen[b])) == len(seen[b])
        assert torch.equal(counts[b].cpu(), torch.bincount(torch.tensor(seen[b]), minlength=SHAPE.vocab).int())
    assert _lib.device_error() == 0


def test_all_of_it_replays_in_a_graph():
    m, K, B = model(), 3, 3
    eager, replayed = (PagedBatch(m, B, 96, pages=15, cache_dtype=F8, window=30, sinks=2) for _ in range(2))
    g = torch.Generator().manual_seed(7)
    drafts, u, e = inputs(B, K, g)
    rules = [dict(counts=torch.zeros(B, SHAPE.vocab, dtype=torch.int32, device=DEV),
                  frequency=torch.full((B,), 0.5, device=DEV)) for _ in range(2)]
    for b in (eager, replayed):
        b.prefill(prompts_of([20, 3, 31]))
    state = lambda b: (b.lens, b.last, b.page_table, *b.pool, *(t for c in b.caches for t in c))  # noqa: E731
    kept = [t.clone() for t in (*state(replayed), rules[1]["counts"])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        replayed.step(drafts, u, e, rules=rules[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = replayed.step(drafts, u, e, rules=rules[1])
    for t, k in zip((*state(replayed), rules[1]["counts"]), kept):
        t.copy_(k)
    for step in range(8):
        for t, n in zip((drafts, u, e), inputs(B, K, g)):
            t.copy_(n)
        want = eager.step(drafts, u, e, rules=rules[0])
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(want, held)), step
        assert all(torch.equal(a.view(torch.uint8) if a.dtype == F8 else a, b.view(torch.uint8) if b.dtype == F8 else b)
                   for a, b in zip(state(eager), state(replayed))), step
        assert torch.equal(rules[0]["counts"], rules[1]["counts"])
        pool_holds(replayed)
    assert _lib.device_error() == 0


def test_main_runs(capsys):
    main(sequences=3, drafts=2, steps=4)
    assert "drafts kept per step" in capsys.readouterr().out and _lib.device_error() == 0
