"""Verification of drafted tokens by speculative sampling, on libsimsd_b200.

`speculative_verify` keeps each sequence's drafted tokens while the target's
distribution accepts them and draws the token after them, so that the emitted
tokens are distributed as the target's own samples.  It is the batched form of
the reference's per-block modified rejection sampling
(speculative_decoding/mrs.py:14-108); temperature 0 is its greedy match
(:111-145).

Forward-only; CUDA tensors only (no CPU fallback).
"""
from __future__ import annotations

import torch

from . import _lib


_current_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _check(target_logits, draft_tokens, uniform, noise, draft_logits, temperature, n_draft) -> None:
    """Raise what is wrong with a request of speculative_verify."""
    _lib.dtype_code(target_logits.dtype)
    if target_logits.ndim != 3 or target_logits.shape[1] < 1 or target_logits.shape[2] < 1:
        raise ValueError(f"target_logits must be [B, K + 1, V], got {tuple(target_logits.shape)}")
    B, R, V = target_logits.shape
    K = R - 1
    if draft_tokens.dtype != torch.int64:
        raise TypeError("speculative_verify: draft_tokens are int64")
    if uniform.dtype != torch.float32 or noise.dtype != torch.float32:
        raise TypeError("speculative_verify: uniform and noise are fp32")
    if draft_tokens.shape != (B, K) or uniform.shape != (B, K) or noise.shape != (B, V):
        raise ValueError(f"draft_tokens and uniform must be [{B}, {K}] and noise [{B}, {V}], got "
                         f"{tuple(draft_tokens.shape)} / {tuple(uniform.shape)} / {tuple(noise.shape)}")
    if draft_logits is not None:
        if draft_logits.dtype != target_logits.dtype:
            raise TypeError(f"dtype mismatch: target {target_logits.dtype} draft {draft_logits.dtype}")
        if draft_logits.shape != (B, K, V):
            raise ValueError(f"draft_logits must be [{B}, {K}, {V}], got {tuple(draft_logits.shape)}")
    if temperature is not None:
        if temperature.dtype != torch.float32:
            raise TypeError("speculative_verify: temperature is fp32")
        if temperature.shape != (B,):
            raise ValueError(f"temperature must be [{B}]")
    if n_draft is not None:
        if n_draft.dtype != torch.int32:
            raise TypeError("speculative_verify: n_draft is int32")
        if n_draft.shape != (B,):
            raise ValueError(f"n_draft must be [{B}]")
    _lib.require_cuda(target_logits, draft_tokens, uniform, noise, draft_logits, temperature, n_draft)


def speculative_verify(target_logits: torch.Tensor, draft_tokens: torch.Tensor, uniform: torch.Tensor,
                       noise: torch.Tensor, draft_logits: torch.Tensor | None = None,
                       temperature: torch.Tensor | None = None, n_draft: torch.Tensor | None = None):
    """(tokens [B, K + 1] int64, accepted [B] int64, logprobs [B, K + 1] fp32).

    target_logits [B, K + 1, V]: row i is the target's after i drafted tokens.
    draft_tokens [B, K] int64.  draft_logits [B, K, V]: what they were drawn from
    (same type as target_logits, same temperature), or None for drafts without
    probabilities (greedy ones).  uniform [B, K] fp32 in [0, 1): accepts token i
    where uniform * q_i < p_i.  noise [B, V] fp32, positive, exponentially
    distributed: draws the token after the accepted ones from max(p - q, 0), or
    from p after the last one.  temperature [B] fp32: 1 when None, 0 = greedy,
    inf = uniform over the tokens whose logit is not -inf.
    n_draft [B] int32: drafted tokens of each sequence (K when None; cut to 0 .. K); the
    rows after them are not read.

    tokens: the accepted drafts, then the drawn token, then -1.  logprobs: the
    target's log probability of each, 0 after them.  Logits bf16, fp16 or fp32;
    NaN counts as -inf, +inf as the largest finite number; ties go to the lowest
    token.  A drafted token outside [0, V) is refused, the next one drawn from p,
    and DEV_ERR_BAD_INDEX raised in `_lib.device_error()`; so it is, with token 0, where
    no token wins (a noise row of NaN).
    """
    out = _lib.binding().speculative_verify(target_logits, draft_tokens, uniform, noise, draft_logits, temperature, n_draft)
    if out is not None:
        return out
    if torch.is_grad_enabled() and (target_logits.requires_grad
                                    or (draft_logits is not None and draft_logits.requires_grad)):
        raise RuntimeError("speculative_verify is a forward-only inference kernel.")
    _check(target_logits, draft_tokens, uniform, noise, draft_logits, temperature, n_draft)
    dev = target_logits.get_device()
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return speculative_verify(target_logits, draft_tokens, uniform, noise, draft_logits, temperature, n_draft)
    B, R, V = target_logits.shape
    K = R - 1
    if K == 0:
        draft_logits = None
    unit = lambda t: t if t is None or t.stride(-1) == 1 else t.contiguous()  # noqa: E731
    target_logits, draft_logits, draft_tokens, uniform, noise, temperature, n_draft = map(
        unit, (target_logits, draft_logits, draft_tokens, uniform, noise, temperature, n_draft))
    tokens = target_logits.new_empty((B, R), dtype=torch.int64)
    accepted = target_logits.new_empty((B,), dtype=torch.int64)
    logprobs = target_logits.new_empty((B, R), dtype=torch.float32)
    lib, stream = _lib.lib(), _current_stream(dev)
    # past the counters that paged_attention keeps zero in the stream's scratch
    skip = _lib.PAGED_COUNTER_BYTES
    ws, ws_bytes, _owner = _lib.stream_scratch(dev, stream,
                                               lib.simsd_speculative_verify_workspace_size(B, K, V) + skip, 0)
    rc = lib.simsd_speculative_verify(
        target_logits.data_ptr(), target_logits.stride(0), target_logits.stride(1),
        draft_logits.data_ptr() if draft_logits is not None else None,
        draft_logits.stride(0) if draft_logits is not None else 0,
        draft_logits.stride(1) if draft_logits is not None else 0, draft_tokens.data_ptr(), draft_tokens.stride(0),
        uniform.data_ptr(), uniform.stride(0), noise.data_ptr(), noise.stride(0),
        temperature.data_ptr() if temperature is not None else None, n_draft.data_ptr() if n_draft is not None else None,
        B, K, V, _lib.dtype_code(target_logits.dtype), tokens.data_ptr(), accepted.data_ptr(), logprobs.data_ptr(),
        ws + skip, ws_bytes - skip, _lib.error_ptr(dev), stream)
    _lib.check(rc, "speculative_verify")
    return tokens, accepted, logprobs
