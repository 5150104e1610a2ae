"""Rules on logits before a token is drawn, on libsimsd_b200: penalties for repeated
tokens, biases and grammar masks, for every drafted row of a sequence.

* `adjust_logits(logits, ...)` — the logits with the rules applied, as
  `speculative_verify` takes them.
* `count_tokens(counts, tokens)` — counts emitted tokens in.
* `token_bits(tokens, vocab)` — token ids as the bit lists that `seen` and `allowed` are.

Forward-only; CUDA tensors only (no CPU fallback).
"""
from __future__ import annotations

import torch

from . import _lib
from .paged_cache import _check_apart, _current_device, _current_stream


def token_bits(tokens: torch.Tensor, vocab: int) -> torch.Tensor:
    """int32 words [.., ceil(vocab / 32)] with the bits of token ids [.., n] (int64; those
    outside [0, vocab) are none): token v is bit v % 32 of word v // 32."""
    words = -(-vocab // 32)
    on = torch.zeros(*tokens.shape[:-1], words * 32 + 1, dtype=torch.int64, device=tokens.device)
    on.scatter_(-1, torch.where((tokens >= 0) & (tokens < vocab), tokens, words * 32), 1)
    w = (on[..., :-1].unflatten(-1, (words, 32)) << torch.arange(32, device=tokens.device)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _check_rules(logits, counts, drafts, repetition, presence, frequency, seen, bias_ids, bias_values, allowed, out) -> None:
    """Raise what is wrong with a request of adjust_logits."""
    _lib.dtype_code(logits.dtype)
    if logits.ndim != 3 or logits.shape[2] < 1:
        raise ValueError(f"logits must be [B, R, V], got {tuple(logits.shape)}")
    B, R, V = logits.shape
    if max(R, V) > 0x7fff0000:
        raise ValueError(f"adjust_logits: at most {0x7fff0000} rows and tokens, got {tuple(logits.shape)}")
    W = -(-V // 32)
    for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if t is not None:
            if t.dtype != torch.float32:
                raise TypeError(f"adjust_logits: {name} is fp32")
            if t.shape != (B,):
                raise ValueError(f"adjust_logits: {name} must be [{B}], got {tuple(t.shape)}")
    for name, t in (("counts", counts), ("seen", seen), ("bias_ids", bias_ids), ("allowed", allowed)):
        if t is not None and t.dtype != torch.int32:
            raise TypeError(f"adjust_logits: {name} is int32")
    if drafts is not None and drafts.dtype != torch.int64:
        raise TypeError("adjust_logits: drafts are int64")
    if counts is not None and counts.shape != (B, V):
        raise ValueError(f"counts must be [{B}, {V}], got {tuple(counts.shape)}")
    if drafts is not None and drafts.shape != (B, max(R - 1, 0)):
        raise ValueError(f"drafts must be [{B}, {max(R - 1, 0)}], got {tuple(drafts.shape)}")
    if seen is not None and seen.shape != (B, W):
        raise ValueError(f"seen must be [{B}, {W}] words of 32 tokens, got {tuple(seen.shape)}")
    if allowed is not None and allowed.shape != (B, W) and allowed.shape != (B, R, W):
        raise ValueError(f"allowed must be [{B}, {W}] or [{B}, {R}, {W}] words of 32 tokens, got {tuple(allowed.shape)}")
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("bias_ids and bias_values go together")
    if bias_ids is not None:
        if bias_values.dtype != torch.float32:
            raise TypeError("adjust_logits: bias_values are fp32")
        if bias_ids.ndim != 2 or bias_ids.shape[0] != B or bias_values.shape != bias_ids.shape:
            raise ValueError(f"bias_ids and bias_values must both be [{B}, n], got {tuple(bias_ids.shape)} / "
                             f"{tuple(bias_values.shape)}")
    if out is not None:
        if out.dtype != logits.dtype:
            raise TypeError(f"dtype mismatch: logits {logits.dtype} out {out.dtype}")
        if out.shape != logits.shape or (V > 1 and out.stride(2) != 1):
            raise ValueError(f"out must be {tuple(logits.shape)} with a unit last stride")
        _check_apart("adjust_logits", out=out)
    _lib.require_cuda(logits, counts, drafts, repetition, presence, frequency, seen, bias_ids, bias_values, allowed, out)


def adjust_logits(logits: torch.Tensor, counts: torch.Tensor | None = None, drafts: torch.Tensor | None = None,
                  repetition: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                  frequency: torch.Tensor | None = None, seen: torch.Tensor | None = None,
                  bias_ids: torch.Tensor | None = None, bias_values: torch.Tensor | None = None,
                  allowed: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """logits [B, R, V] (bf16, fp16 or fp32) with the rules applied; row i of a sequence follows
    i drafted tokens (R = K + 1, as `speculative_verify` takes them).  For token v, in fp32
    (what is added summed first), rounded once:

    * repetition [B] fp32 (positive): a logit over 0 is divided by it (multiplied by its fp32 reciprocal), another one multiplied,
      where v was answered, drafted before row i, or stands in the prompt;
    * frequency [B], presence [B] fp32: subtracted, times how often and once, where v was
      answered or drafted before row i;
    * bias_ids [B, n] int32, bias_values [B, n] fp32: the values whose id is v are added
      (negative ids are none: lists of different lengths);
    * allowed [B, W] or [B, R, W] int32, W = ceil(V / 32): tokens whose bit is not set get -inf.

    counts [B, V] int32: how often each token was answered (`count_tokens`).  drafts [B, R - 1]
    int64: the drafted tokens, those outside [0, V) counting nowhere.  seen [B, W] int32: bits of
    the prompt's tokens (`token_bits`).  None: none of it.  Without any of the three penalties
    counts, drafts and seen are not read.  A row whose mask allows nothing is -inf throughout.
    NaN stays NaN where it is allowed.  out: where to, `logits` itself among it (a new
    tensor when None); it must not overlap logits in another way.
    """
    y = _lib.binding().adjust_logits(logits, counts, drafts, repetition, presence, frequency, seen, bias_ids, bias_values,
                                     allowed, out)
    if y is not None:
        return y
    if torch.is_grad_enabled() and logits.requires_grad:
        raise RuntimeError("adjust_logits is a forward-only inference kernel.")
    _check_rules(logits, counts, drafts, repetition, presence, frequency, seen, bias_ids, bias_values, allowed, out)
    dev = logits.get_device()
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return adjust_logits(logits, counts, drafts, repetition, presence, frequency, seen, bias_ids, bias_values, allowed,
                                 out)
    B, R, V = logits.shape
    unit = lambda t: t if t is None or t.shape[-1] < 2 or t.stride(-1) == 1 else t.contiguous()  # noqa: E731
    logits, counts, drafts, repetition, presence, frequency, seen, bias_ids, bias_values, allowed = map(
        unit, (logits, counts, drafts, repetition, presence, frequency, seen, bias_ids, bias_values, allowed))
    if out is None:
        out = logits.new_empty((B, R, V))
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    ld = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    rc = _lib.lib().simsd_adjust_logits(
        logits.data_ptr(), logits.stride(0), logits.stride(1), out.data_ptr(), out.stride(0), out.stride(1), B, R, V,
        _lib.dtype_code(logits.dtype), ptr(counts), ld(counts), ptr(drafts), ld(drafts), ptr(seen), ld(seen), ptr(repetition),
        ptr(presence), ptr(frequency), ptr(bias_ids), ld(bias_ids), ptr(bias_values), ld(bias_values),
        0 if bias_ids is None else bias_ids.shape[1], ptr(allowed), ld(allowed),
        allowed.stride(1) if allowed is not None and allowed.ndim == 3 else 0, _lib.error_ptr(dev), _current_stream(dev))
    _lib.check(rc, "adjust_logits")
    return out


def count_tokens(counts: torch.Tensor, tokens: torch.Tensor) -> None:
    """counts [B, V] int32, in place: plus how often each token is among tokens [B, N] int64.
    Negative tokens are none (`speculative_verify` fills its rows with -1); one from V on is
    skipped and raises DEV_ERR_BAD_INDEX in `_lib.device_error()`."""
    if _lib.binding().count_tokens(counts, tokens) is not None:
        return
    if counts.dtype != torch.int32 or tokens.dtype != torch.int64:
        raise TypeError("count_tokens: counts are int32 and tokens int64")
    if counts.ndim != 2 or counts.shape[1] < 1 or tokens.ndim != 2 or tokens.shape[0] != counts.shape[0]:
        raise ValueError(f"counts must be [B, V] and tokens [B, N], got {tuple(counts.shape)} / {tuple(tokens.shape)}")
    if counts.shape[1] > 1 and counts.stride(1) != 1:
        raise ValueError("counts, which are written in place, must have a unit last stride")
    _check_apart("count_tokens", counts=counts)
    _lib.require_cuda(counts, tokens)
    dev = counts.get_device()
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return count_tokens(counts, tokens)
    if tokens.shape[1] > 1 and tokens.stride(1) != 1:
        tokens = tokens.contiguous()
    rc = _lib.lib().simsd_count_tokens(counts.data_ptr(), counts.stride(0), tokens.data_ptr(), tokens.stride(0), *tokens.shape,
                                       counts.shape[1], _lib.error_ptr(dev), _current_stream(dev))
    _lib.check(rc, "count_tokens")
