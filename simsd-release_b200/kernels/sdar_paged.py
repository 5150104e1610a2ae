"""Batched speculative decoding of an SDAR-shaped target over a paged key-value cache.

`PagedBatch` runs several sequences at once: every step appends each sequence's last
token and its K drafted ones to the cache (`paged_append`), attends over its pages
(`paged_attention`), takes the target's logits after each of them and keeps the drafts
that speculative sampling accepts (`speculative_verify`).  The layers around that are
the verify forward's (kernels/sdar_verify.py: `rmsnorm`, `thin_linear_cat` and the
model's own linears, which `fused_toggle.apply_to_model` may have swapped).

A step never waits for the host: lengths, slots and accepted tokens stay on the device,
so it can be captured in a CUDA graph and replayed with new drafts.

    batch = PagedBatch(model, sequences=8, max_len=4096)
    batch.prefill(prompts)                          # lists of token ids
    tokens, accepted, logprobs = batch.step(drafts, uniform, noise)

`python -m kernels.sdar_paged` runs a small random model this way.
"""
from __future__ import annotations

import torch

from .layer_ops import rmsnorm
from .paged_cache import paged_append, paged_attention, rope_table
from .sdar_verify import SDARShape, SDARVerifyModel
from .spec_verify import speculative_verify
from .thin_linear_fused import thin_linear_cat


class PagedBatch:
    """`sequences` sequences of up to `max_len` tokens (rounded up to whole pages) over one model.

    Pages are handed out at construction, `max_len` + `max_drafts` tokens' worth to each
    sequence: the places after `max_len` take the keys of drafted tokens that a step near
    the end has no room to keep, so that its queries and keys stay aligned.
    `page_table` may be edited between steps by a caller that allocates as it goes, as long
    as it covers `lens` + K + 1 tokens of every sequence that a step moves on.
    `lens` counts the tokens whose keys and values are in the cache; `last` is each
    sequence's newest token, which is not there yet.
    """

    def __init__(self, model: SDARVerifyModel, sequences: int, max_len: int, page_size: int = 16,
                 tail_mask: torch.Tensor | None = None, max_drafts: int = 31):
        s, p = model.s, next(model.parameters())
        self.model, self.page_size, self.tail_mask = model, page_size, tail_mask
        self.max_len = -(-max_len // page_size) * page_size
        per = -(-(self.max_len + max_drafts) // page_size)
        self.page_table = torch.arange(sequences * per, dtype=torch.int32, device=p.device).view(sequences, per)
        shape = (sequences * per, s.kv_heads, page_size, s.head_dim)
        self.caches = [(torch.zeros(shape, dtype=p.dtype, device=p.device), torch.zeros(shape, dtype=p.dtype, device=p.device))
                       for _ in model.layers]
        self.cos, self.sin = rope_table(per * page_size, s.head_dim, s.rope_theta, p.device)
        self.lens = torch.zeros(sequences, dtype=torch.int32, device=p.device)
        self.last = torch.zeros(sequences, dtype=torch.int64, device=p.device)

    def hidden(self, ids: torch.Tensor, count: torch.Tensor | None = None,
               tail_mask: torch.Tensor | None = None) -> torch.Tensor:
        """Final-norm hidden states [B, L, H] of ids [B, L], which go to the cache after the
        `lens` tokens that are there (`lens` itself is not moved).  count [B]: only the last
        count[b] of a row are tokens, those before them padding."""
        m, s = self.model, self.model.s
        B, L = ids.shape
        at = torch.arange(L, device=ids.device)
        new = torch.full_like(self.lens, L) if count is None else count.to(torch.int32)
        pos = self.lens[:, None].long() + at - (L - new[:, None].long())
        real = (at >= L - new[:, None]) & (pos < self.page_table.shape[1] * self.page_size)
        pos = pos.clamp(0, self.page_table.shape[1] * self.page_size - 1)
        page = self.page_table.gather(1, pos // self.page_size).long()
        slots = torch.where(real, page * self.page_size + pos % self.page_size, -1).view(-1)
        pos = pos.view(-1)
        total = self.lens + new
        h = m.embed_tokens(ids).view(B * L, -1)
        x = rmsnorm(h, m.layers[0].input_layernorm.weight, m.layers[0].input_layernorm.eps)
        for i, layer in enumerate(m.layers):
            a, (k_cache, v_cache) = layer.self_attn, self.caches[i]
            qkv = thin_linear_cat(x, [a.q_proj.weight, a.k_proj.weight, a.v_proj.weight], whole=True)
            q = paged_append(qkv, s.heads, s.kv_heads, k_cache, v_cache, slots, pos, self.cos, self.sin,
                             a.q_norm.weight, a.k_norm.weight, a.q_norm.eps)
            o = paged_attention(q.view(B, L, s.heads, s.head_dim), k_cache, v_cache, self.page_table, total,
                                tail_mask=tail_mask)
            n = layer.post_attention_layernorm
            h, x = rmsnorm(a.o_proj(o.view(B * L, -1)), n.weight, n.eps, residual=h)
            n = m.layers[i + 1].input_layernorm if i + 1 < len(m.layers) else m.norm
            h, x = rmsnorm(layer.mlp(x), n.weight, n.eps, residual=h)
        return x.view(B, L, -1)

    def prefill(self, prompts: list[list[int]], chunk: int = 16) -> None:
        """Put all but the last token of each prompt into the cache, `chunk` tokens of every
        sequence at a time; the last one starts the first step."""
        dev = self.lens.device
        if len(prompts) != self.lens.numel() or min(map(len, prompts)) < 1:
            raise ValueError(f"{self.lens.numel()} prompts of at least one token each")
        if max(map(len, prompts)) > self.max_len:
            raise ValueError("a prompt is longer than max_len")
        if not all(0 <= t < self.model.s.vocab for p in prompts for t in p):
            raise ValueError(f"a prompt has a token outside the vocabulary of {self.model.s.vocab}")
        self.lens.zero_()
        with torch.inference_mode():
            for c in range(0, max(map(len, prompts)) - 1, chunk):
                rows = [p[c: min(c + chunk, len(p) - 1)] for p in prompts]
                L = max(map(len, rows))
                ids = torch.tensor([[0] * (L - len(r)) + list(r) for r in rows], device=dev)
                count = torch.tensor([len(r) for r in rows], dtype=torch.int32, device=dev)
                self.hidden(ids, count)
                self.lens += count
            self.last.copy_(torch.tensor([p[-1] for p in prompts], device=dev))

    def step(self, drafts: torch.Tensor, uniform: torch.Tensor, noise: torch.Tensor,
             draft_logits: torch.Tensor | None = None, temperature: torch.Tensor | None = None,
             n_draft: torch.Tensor | None = None):
        """Verify drafts [B, K] (int64; see `speculative_verify` for the rest) and move on:
        (tokens [B, K + 1], accepted [B], logprobs [B, K + 1]).  K = 0 decodes plainly.

        A sequence keeps no more drafts than `max_len` leaves room for.  One that is full
        (lens = max_len, or fewer than K + 1 places left in the table, which only K >
        `max_drafts` brings about) stays as it is: its tokens are -1, accepted and logprobs 0."""
        with torch.inference_mode():
            # ids outside the vocabulary are speculative_verify's to refuse, not the embedding's to read
            ids = torch.cat([self.last[:, None], drafts.clamp(0, self.model.s.vocab - 1)], 1)
            B, L = ids.shape
            if n_draft is not None and n_draft.shape != (B,):
                raise ValueError(f"n_draft must be [{B}]")
            # with at most max_drafts drafts every sequence short of max_len has L places in the table
            full = self.lens >= min(self.max_len, self.page_table.shape[1] * self.page_size - L + 1)
            keep = self.max_len - 1 - self.lens              # speculative_verify takes 0 .. K of it
            keep = keep if n_draft is None else torch.minimum(keep, n_draft)
            x = self.hidden(ids, torch.where(full, 0, L), self.tail_mask)
            logits = self.model.lm_head(x.view(B * L, -1)).view(B, L, -1)
            tokens, accepted, logprobs = speculative_verify(logits, drafts, uniform, noise, draft_logits, temperature, keep)
            self.last.copy_(torch.where(full, self.last, tokens.gather(1, accepted[:, None])[:, 0]))
            accepted.masked_fill_(full, -1)
            self.lens += (accepted + 1).to(torch.int32)
            accepted.clamp_(min=0)
            tokens.masked_fill_(full[:, None], -1)
            logprobs.masked_fill_(full[:, None], 0.0)
        return tokens, accepted, logprobs


def main(sequences: int = 8, drafts: int = 3, steps: int = 20) -> None:
    """Decode a small random model; every other step's drafts are right."""
    dev = torch.device("cuda")
    shape = SDARShape(hidden=1024, layers=4, heads=16, kv_heads=4, head_dim=128, intermediate=2048, vocab=32000)
    model = SDARVerifyModel.random_init(shape, dev)
    g = torch.Generator(device=dev).manual_seed(0)
    prompts = [torch.randint(0, shape.vocab, (20 + 7 * i,), generator=g, device=dev).tolist() for i in range(sequences)]
    batch = PagedBatch(model, sequences, max_len=1024)
    batch.prefill(prompts)
    greedy = torch.zeros(sequences, device=dev)
    kept = 0
    for i in range(steps):
        u = torch.rand(sequences, drafts, generator=g, device=dev)
        e = torch.empty(sequences, shape.vocab, device=dev).exponential_(generator=g).clamp_(min=1e-20)
        guess = torch.randint(0, shape.vocab, (sequences, drafts), generator=g, device=dev)
        if i % 2:   # what the model itself would say, from a dry run without moving on
            lens, last = batch.lens.clone(), batch.last.clone()
            none = torch.empty(sequences, 0, dtype=torch.int64, device=dev)
            for k in range(drafts):
                guess[:, k] = batch.step(none, u[:, :0], e, temperature=greedy)[0][:, 0]
            batch.lens.copy_(lens)
            batch.last.copy_(last)
        tokens, accepted, _ = batch.step(guess, u, e, temperature=greedy)
        kept += int(accepted.sum())
    print(f"{sequences} sequences, {steps} steps of {drafts} drafts: {kept / (sequences * steps):.2f} drafts kept per step, "
          f"lengths {batch.lens.tolist()}")


if __name__ == "__main__":
    main()
