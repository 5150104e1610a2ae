"""A paged key-value cache held in 8 bits, on libsimsd_b200: half the bytes that a
decoding step reads, and room for twice the tokens.

Attention over it is faster than over the 16-bit cache up to 16 rows (query heads of a KV head times
tokens) and through a window, slower beyond that without one: 16 sequences of 1000 to 3000 tokens with 8 KV
heads take 32 us at 16 rows and 49 at 32 (16 bits: 36 and 37).

* `paged_append8(qkv, ...)` — q/k RMSNorm (optional), rotary embedding and the write of
  each sequence's new keys and values, quantised with a scale for each block of tokens
  and head.
* `paged_attention8(q, ...)` — attention over it, as `kernels/paged_cache.py` has it for
  the 16-bit cache, a sliding window included.
* `cache8(pages, ...)` — an empty cache.

The cache is a pair of float8_e4m3fn tensors [pages, kv_heads, page_size, head_dim] with a
unit last stride (a token-major one is passed as its `.transpose(1, 2)`) and a pair of
fp32 scales [pages, kv_heads, page_size // block]: a stored number stands for its
block's scale times itself.  Appends make scales that are powers of two, which costs
e4m3 no precision; a cache that was quantised otherwise may have any positive ones up to 2^64.

Forward-only; CUDA tensors only (no CPU fallback).  Streams, copies of inputs that the
kernels cannot read and flagged indices are as in `kernels/paged_cache.py`; the caches have to
start on 16 bytes and have page, head and token strides of multiples of 16.
"""
from __future__ import annotations

import torch

from . import _lib
from .paged_cache import (_HALF, _check_apart, _check_attention, _check_cache, _check_scales, _current_device, _current_stream,
                          _mask_strides, _on_16_bytes, _window)

F8 = torch.float8_e4m3fn


def cache8(pages: int, kv_heads: int, page_size: int, head_dim: int, block: int = 16, device=None):
    """(k_cache, v_cache, k_scale, v_scale) of zeros, a scale for each `block` tokens of a head."""
    if block < 1 or page_size % block:
        raise ValueError(f"a block of {block} tokens does not divide pages of {page_size}")
    shape, scales = (pages, kv_heads, page_size, head_dim), (pages, kv_heads, page_size // block)
    return (*(torch.zeros(shape, dtype=F8, device=device) for _ in range(2)),
            *(torch.zeros(scales, dtype=torch.float32, device=device) for _ in range(2)))


def _check_append8(qkv, heads, kv_heads, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cos, sin, q_weight, k_weight,
                   count) -> None:
    """Raise what is wrong with a request of paged_append8."""
    if qkv.dtype not in _HALF:
        raise TypeError(f"paged_append8 takes bf16 or fp16 activations, got {qkv.dtype}")
    _check_cache("paged_append8", k_cache, v_cache, kv_heads, F8)
    _check_scales("paged_append8", k_cache, k_scale, v_scale)
    _check_apart("paged_append8", k_cache=k_cache, k_scale=k_scale)
    D = k_cache.shape[3]
    if qkv.ndim not in (2, 3) or heads < 1 or kv_heads < 1 or qkv.shape[-1] != (heads + 2 * kv_heads) * D:
        raise ValueError(f"qkv must be [B, L, {(heads + 2 * kv_heads) * D}] or [B, ..], got {tuple(qkv.shape)}")
    B = qkv.shape[0]
    if page_table.dtype != torch.int32 or seq_lens.dtype != torch.int32 or (count is not None and count.dtype != torch.int32):
        raise TypeError("paged_append8: page_table, seq_lens and count are int32")
    if page_table.ndim != 2 or page_table.shape[0] != B or seq_lens.shape != (B,) or (count is not None and count.shape != (B,)):
        raise ValueError(f"page_table must be [{B}, max_pages], seq_lens and count [{B}], got {tuple(page_table.shape)} / "
                         f"{tuple(seq_lens.shape)}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("paged_append8: cos and sin are fp32")
    if cos.ndim != 2 or cos.shape != sin.shape or not cos.is_contiguous() or not sin.is_contiguous():
        raise ValueError("cos and sin must be contiguous [n, R / 2] tensors of the same shape")
    for w in (q_weight, k_weight):
        if w is not None:
            if w.dtype != qkv.dtype:
                raise TypeError("paged_append8: the norm weights must have qkv's dtype")
            if w.shape != (D,):
                raise ValueError(f"the norm weights must be [{D}]")
    _lib.require_cuda(qkv, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cos, sin, q_weight, k_weight, count)


def paged_append8(qkv: torch.Tensor, heads: int, kv_heads: int, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  k_scale: torch.Tensor, v_scale: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                  cos: torch.Tensor, sin: torch.Tensor, q_weight: torch.Tensor | None = None,
                  k_weight: torch.Tensor | None = None, eps: float = 1e-6, count: torch.Tensor | None = None) -> torch.Tensor:
    """qkv [B, L, (heads + 2 kv_heads) * D] (or [B, ..], L = 1; the merged projection's output)
    -> q [B, L, heads, D]; writes the new keys and values to the sequences' pages.

    seq_lens [B] int32: lengths with the new tokens, as `paged_attention8` takes them: row t
    of sequence b is the token at position seq_lens[b] - L + t.  count [B] int32: only the last
    count[b] rows are tokens, those before them padding (None: all L; positions before
    the sequence's start are padding anyway): their q is zero, nothing else of them is
    used.  After `paged_reserve` it is the tokens that were served, total - lens, not those that
    were asked for: seq_lens counts no others, and rows too many would be written over a
    sequence's older tokens.  page_table [B, max_pages] int32 as for `paged_attention`; no page is
    written by two sequences.  cos, sin, q_weight, k_weight, eps: as for `paged_append`.

    Where a call writes a block's first token, the block's scale is the smallest power of two
    (2^-64 to 2^64) that keeps the block's new numbers within 448; where it only adds
    to a block, the scale grows if need be, and the older tokens are rounded anew.  It does not come
    down before the block's first token is written again: where tokens are taken back (rejected drafts, a step
    undone by its lengths), the block that they ended in may keep a scale that only they needed, and the
    kept tokens' numbers under 2^-6 of it are 2^-9 of it apart.  Numbers that are not finite are
    stored as NaN and leave the scale alone.  Numbers are multiplied by the scale's reciprocal in fp32, which is
    exact for powers of two (a block may have another scale from elsewhere).  Computed in
    fp32, rounded once.  bf16 or fp16; D 64 or 128; R a multiple of 16.
    """
    q = _lib.binding().paged_append8(qkv, heads, kv_heads, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cos, sin,
                                     q_weight, k_weight, eps, count)
    if q is not None:
        return q
    if torch.is_grad_enabled() and (qkv.requires_grad or k_scale.requires_grad or v_scale.requires_grad):
        raise RuntimeError("paged_append8 is a forward-only inference kernel.")
    _check_append8(qkv, heads, kv_heads, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cos, sin, q_weight, k_weight,
                   count)
    dev, shape, strides = qkv.get_device(), k_cache.shape, k_cache.stride()
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return paged_append8(qkv, heads, kv_heads, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cos, sin,
                                 q_weight, k_weight, eps, count)
    one = qkv.ndim == 2
    if one:
        qkv = qkv[:, None]
    B, L = qkv.shape[:2]
    if qkv.stride(2) != 1 or qkv.stride(1) % 8 or qkv.stride(0) % 8 or qkv.stride(1) < qkv.shape[2] or qkv.stride(0) < 0:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    qkv, cos, sin, q_weight, k_weight = map(_on_16_bytes, (
        qkv, cos, sin, *(w.contiguous() if w is not None else None for w in (q_weight, k_weight))))
    seq_lens = seq_lens.contiguous()
    count = count.contiguous() if count is not None else None
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    q = qkv.new_empty((B, L, heads, shape[3]))
    rc = _lib.lib().simsd_paged_append8(
        qkv.data_ptr(), qkv.stride(0), qkv.stride(1), B, L, heads, kv_heads, shape[3], 2 * cos.shape[1],
        q_weight.data_ptr() if q_weight is not None else None, k_weight.data_ptr() if k_weight is not None else None, eps,
        cos.data_ptr(), sin.data_ptr(), cos.shape[0], page_table.data_ptr(), page_table.stride(0), page_table.shape[1],
        seq_lens.data_ptr(), count.data_ptr() if count is not None else None, q.data_ptr(), k_cache.data_ptr(),
        v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), shape[0], shape[2], shape[2] // k_scale.shape[2],
        strides[0], strides[1], strides[2], *k_scale.stride(), _HALF[qkv.dtype], _lib.error_ptr(dev), _current_stream(dev))
    _lib.check(rc, "paged_append8")
    return q[:, 0] if one else q


def paged_attention8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                     v_scale: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, scale: float | None = None,
                     tail_mask: torch.Tensor | None = None, return_lse: bool = False, window: int | None = None,
                     sinks: int = 0):
    """`paged_attention` over the 8-bit cache: q [B, L, heads, D] (or [B, heads, D], L = 1;
    bf16 or fp16) -> o of q's shape, or (o, lse).

    page_table, seq_lens, scale, tail_mask, window and sinks as there.  A key whose stored
    numbers or scale are NaN harms only the rows that see it.  fp32 scores, sums and sums of
    products; the weights, scaled by their block's value scale, are rounded to fp16 for the second
    product.
    """
    o = _lib.binding().paged_attention8(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, scale, tail_mask, return_lse,
                                        window, sinks)
    if o is not None:
        return o
    if torch.is_grad_enabled() and (q.requires_grad or k_scale.requires_grad or v_scale.requires_grad):
        raise RuntimeError("paged_attention8 is a forward-only inference kernel.")
    _check_attention(q, k_cache, v_cache, page_table, seq_lens, tail_mask, window, sinks, "paged_attention8", F8, (k_scale, v_scale))
    dev, shape, strides = q.get_device(), k_cache.shape, k_cache.stride()
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return paged_attention8(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, scale, tail_mask, return_lse,
                                    window, sinks)
    B, Hq, D = q.shape[0], q.shape[-2], q.shape[-1]
    L = q.shape[1] if q.ndim == 4 else 1
    tail_mask, ldm_b, ldm_t = _mask_strides(tail_mask)
    q, seq_lens = _on_16_bytes(q.contiguous()), seq_lens.contiguous()
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    o = torch.empty_like(q)
    lse = q.new_empty(q.shape[:-1], dtype=torch.float32) if return_lse else None
    lib, stream = _lib.lib(), _current_stream(dev)
    ws, ws_bytes, _owner = _lib.stream_scratch(dev, stream, lib.simsd_paged_attention8_workspace_size(L, Hq, shape[1], D),
                                               _lib.PAGED_COUNTER_BYTES)
    rc = lib.simsd_paged_attention8(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), shape[0], shape[2],
        shape[2] // k_scale.shape[2], strides[0], strides[1], strides[2], *k_scale.stride(), page_table.data_ptr(),
        page_table.stride(0), page_table.shape[1], seq_lens.data_ptr(), tail_mask.data_ptr() if tail_mask is not None else None,
        ldm_b, ldm_t, B, L, Hq, shape[1], D, D ** -0.5 if scale is None else scale, *_window(window, sinks), o.data_ptr(),
        lse.data_ptr() if return_lse else None, _HALF[q.dtype], ws, ws_bytes, _lib.error_ptr(dev), stream)
    _lib.check(rc, "paged_attention8")
    return (o, lse) if return_lse else o
