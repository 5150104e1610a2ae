"""A paged key-value cache for batched decoding, on libsimsd_b200.

* `paged_append(qkv, ...)` — q/k RMSNorm (optional), rotary embedding and the
  write of each token's key and value into its cache slot.
* `paged_attention(q, ...)` — attention of each sequence's newest token, or of
  its L drafted ones, over its pages.
* `rope_table(n, dim, theta)` — the fp32 cos/sin rows `paged_append` reads.

The cache is a pair of tensors [pages, kv_heads, page_size, head_dim] with a unit
last stride; a token-major cache [pages, page_size, kv_heads, head_dim] is passed
as its `.transpose(1, 2)`.  Slot s is token s % page_size of page s // page_size.
The reference keeps one static cache per sequence
(speculative_decoding/cache_aware.py:195-215); it has no paged form.

Forward-only; CUDA tensors only (no CPU fallback).  Every stream has scratch of its
own, so calls on several streams share none.
Inputs of other strides than the kernels read, or that do not start on 16 bytes, are
copied; the caches, which are written in place, have to start on 16 bytes and have page,
head and token strides of multiples of 8 elements.
Indices that the device finds out of range raise DEV_ERR_BAD_INDEX in
`_lib.device_error()`; nothing is read or written for them.
"""
from __future__ import annotations

import torch

from . import _lib

def rope_table(n: int, dim: int, theta: float = 1e6, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin [n, dim / 2] fp32 of positions 0 .. n - 1 (angles in fp64, rounded once)."""
    inv = theta ** (-torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim)
    a = torch.arange(n, device=device, dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


# What the kernels take, in the library's codes.
_HALF = {torch.bfloat16: _lib.SIMSD_BF16, torch.float16: _lib.SIMSD_F16}
_current_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _check_cache(what: str, k_cache: torch.Tensor, v_cache: torch.Tensor, kv_heads: int, dtype: torch.dtype) -> None:
    if k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise TypeError(f"{what}: the caches must have the activations' type {dtype}, got {k_cache.dtype} / {v_cache.dtype}")
    if k_cache.ndim != 4 or k_cache.shape != v_cache.shape or k_cache.shape[1] != kv_heads:
        raise ValueError(f"{what}: k_cache and v_cache must both be [pages, {kv_heads}, page_size, head_dim], got "
                         f"{tuple(k_cache.shape)} / {tuple(v_cache.shape)}")
    if k_cache.stride() != v_cache.stride() or k_cache.stride(3) != 1:
        raise ValueError(f"{what}: k_cache and v_cache must have the same strides, the last one 1")


def _on_16_bytes(t: torch.Tensor | None) -> torch.Tensor | None:
    """t, copied where the kernels' 16-byte loads cannot start at its first element."""
    return t if t is None or t.data_ptr() % 16 == 0 else t.clone()


def _check_append(qkv, heads, kv_heads, k_cache, v_cache, slots, positions, cos, sin, q_weight, k_weight) -> None:
    """Raise what is wrong with a request of paged_append."""
    if qkv.dtype not in _HALF:
        raise TypeError(f"paged_append takes bf16 or fp16 activations, got {qkv.dtype}")
    _check_cache("paged_append", k_cache, v_cache, kv_heads, qkv.dtype)
    D = k_cache.shape[3]
    if qkv.ndim != 2 or heads < 1 or kv_heads < 1 or qkv.shape[1] != (heads + 2 * kv_heads) * D:
        raise ValueError(f"qkv must be [T, {(heads + 2 * kv_heads) * D}], got {tuple(qkv.shape)}")
    T = qkv.shape[0]
    if slots.dtype != torch.int64 or positions.dtype != torch.int64:
        raise TypeError("paged_append: slots and positions are int64")
    if slots.shape != (T,) or positions.shape != (T,):
        raise ValueError(f"slots and positions must be [{T}], got {tuple(slots.shape)} / {tuple(positions.shape)}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("paged_append: cos and sin are fp32")
    if cos.ndim != 2 or cos.shape != sin.shape or not cos.is_contiguous() or not sin.is_contiguous():
        raise ValueError("cos and sin must be contiguous [n, R / 2] tensors of the same shape")
    for w in (q_weight, k_weight):
        if w is not None:
            if w.dtype != qkv.dtype:
                raise TypeError("paged_append: the norm weights must have qkv's dtype")
            if w.shape != (D,):
                raise ValueError(f"the norm weights must be [{D}]")
    _lib.require_cuda(qkv, k_cache, v_cache, slots, positions, cos, sin, q_weight, k_weight)


def paged_append(qkv: torch.Tensor, heads: int, kv_heads: int, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 slots: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                 eps: float = 1e-6) -> torch.Tensor:
    """qkv [T, (heads + 2 kv_heads) * D] (the merged projection's output) -> q
    [T, heads, D]; writes each token's key and value at its slot.

    slots [T] int64: where the token goes; a negative one leaves the cache as it
    is and gives a zero q row (padding; its position is not read).  Slots of one
    call are distinct.  positions [T] int64: row of cos/sin [n, R / 2] (fp32,
    contiguous); the first R <= D elements of a head are rotated in pairs (i, i +
    R / 2), the rest pass.  q_weight / k_weight [D]: RMSNorm over each q / k head
    before the rotation (sdar/modeling_sdar.py:197-302), or None.  Computed in
    fp32, rounded once.  bf16 or fp16; D 64 or 128; R a multiple of 16.
    """
    q = _lib.binding().paged_append(qkv, heads, kv_heads, k_cache, v_cache, slots, positions, cos, sin, q_weight, k_weight,
                                    eps)
    if q is not None:
        return q
    if torch.is_grad_enabled() and (qkv.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise RuntimeError("paged_append is a forward-only inference kernel.")
    _check_append(qkv, heads, kv_heads, k_cache, v_cache, slots, positions, cos, sin, q_weight, k_weight)
    dev, shape, strides = qkv.get_device(), k_cache.shape, k_cache.stride()
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return paged_append(qkv, heads, kv_heads, k_cache, v_cache, slots, positions, cos, sin, q_weight, k_weight, eps)
    if qkv.stride(1) != 1 or qkv.stride(0) % 8 or qkv.stride(0) < qkv.shape[1]:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    slots, positions = slots.contiguous(), positions.contiguous()
    qkv, cos, sin, q_weight, k_weight = map(_on_16_bytes, (
        qkv, cos, sin, *(w.contiguous() if w is not None else None for w in (q_weight, k_weight))))
    q = qkv.new_empty((qkv.shape[0], heads, shape[3]))
    rc = _lib.lib().simsd_paged_append(
        qkv.data_ptr(), qkv.stride(0), qkv.shape[0], heads, kv_heads, shape[3], 2 * cos.shape[1],
        q_weight.data_ptr() if q_weight is not None else None, k_weight.data_ptr() if k_weight is not None else None, eps,
        cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(), slots.data_ptr(), q.data_ptr(),
        k_cache.data_ptr(), v_cache.data_ptr(), shape[0], shape[2], strides[0], strides[1], strides[2], _HALF[qkv.dtype],
        _lib.error_ptr(dev), _current_stream(dev))
    _lib.check(rc, "paged_append")
    return q


def _check_attention(q, k_cache, v_cache, page_table, seq_lens, tail_mask) -> None:
    """Raise what is wrong with a request of paged_attention."""
    if q.dtype not in _HALF:
        raise TypeError(f"paged_attention takes bf16 or fp16 queries, got {q.dtype}")
    if q.ndim not in (3, 4):
        raise ValueError(f"q must be [B, L, heads, D] or [B, heads, D], got {tuple(q.shape)}")
    B, Hq, D = q.shape[0], q.shape[-2], q.shape[-1]
    L = q.shape[1] if q.ndim == 4 else 1
    Hk = k_cache.shape[1] if k_cache.ndim == 4 else 0
    _check_cache("paged_attention", k_cache, v_cache, Hk, q.dtype)
    if k_cache.shape[3] != D or Hk < 1 or Hq < 1 or Hq % Hk:
        raise ValueError(f"q heads {Hq} x {D} do not go with the cache's {Hk} x {k_cache.shape[3]}")
    if page_table.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise TypeError("paged_attention: page_table and seq_lens are int32")
    if page_table.ndim != 2 or page_table.shape[0] != B or seq_lens.shape != (B,):
        raise ValueError(f"page_table must be [{B}, max_pages] and seq_lens [{B}], got {tuple(page_table.shape)} / "
                         f"{tuple(seq_lens.shape)}")
    if tail_mask is not None:
        if tail_mask.dtype != torch.bool:
            raise TypeError("paged_attention: tail_mask is bool")
        if tail_mask.shape != (L, L) and tail_mask.shape != (B, L, L):
            raise ValueError(f"tail_mask must be [{L}, {L}] or [{B}, {L}, {L}], got {tuple(tail_mask.shape)}")
    _lib.require_cuda(q, k_cache, v_cache, page_table, seq_lens, tail_mask)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    seq_lens: torch.Tensor, scale: float | None = None, tail_mask: torch.Tensor | None = None,
                    return_lse: bool = False):
    """Attention of q [B, L, heads, D] (or [B, heads, D], L = 1) over each
    sequence's pages -> o of q's shape, or (o, lse) with lse [B, L, heads] (fp32,
    natural log of the softmax's denominator).

    page_table [B, max_pages] int32: sequence b's key j is token j % page_size of
    page page_table[b, j // page_size]; entries past its last page are not read.
    seq_lens [B] int32: its keys, the L queries' own included (they are the
    newest L); a negative one counts as 0, one past the table is cut to its end (and
    raises DEV_ERR_BAD_INDEX).  Keys before those are visible to all of its queries; among them
    query t sees key i where i <= t, or where tail_mask [L, L] or [B, L, L] (bool)
    is set.  A query that sees no key (an empty sequence, a mask without any) gets
    o = 0 and lse = -inf.  Only visible keys count: what stale cache memory or a
    masked key holds, NaN included, does not reach the output.  scale: D ** -0.5
    when None.  Lengths are read on the device, so the call can be captured in a
    CUDA graph and replayed as the sequences grow.
    """
    o = _lib.binding().paged_attention(q, k_cache, v_cache, page_table, seq_lens, scale, tail_mask, return_lse)
    if o is not None:
        return o
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise RuntimeError("paged_attention is a forward-only inference kernel.")
    _check_attention(q, k_cache, v_cache, page_table, seq_lens, tail_mask)
    dev, shape, strides = q.get_device(), k_cache.shape, k_cache.stride()
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return paged_attention(q, k_cache, v_cache, page_table, seq_lens, scale, tail_mask, return_lse)
    B, Hq, D = q.shape[0], q.shape[-2], q.shape[-1]
    L = q.shape[1] if q.ndim == 4 else 1
    ldm_b = ldm_t = 0
    if tail_mask is not None:
        if tail_mask.stride(-1) != 1:
            tail_mask = tail_mask.contiguous()
        ldm_t = tail_mask.stride(-2)
        ldm_b = tail_mask.stride(0) if tail_mask.ndim == 3 else 0
    q, seq_lens = _on_16_bytes(q.contiguous()), seq_lens.contiguous()
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    o = torch.empty_like(q)
    lse = q.new_empty(q.shape[:-1], dtype=torch.float32) if return_lse else None
    lib, stream = _lib.lib(), _current_stream(dev)
    ws, ws_bytes, _owner = _lib.stream_scratch(dev, stream, lib.simsd_paged_attention_workspace_size(L, Hq, shape[1], D),
                                               _lib.PAGED_COUNTER_BYTES)
    rc = lib.simsd_paged_attention(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), shape[0], shape[2], strides[0], strides[1], strides[2],
        page_table.data_ptr(), page_table.stride(0), page_table.shape[1], seq_lens.data_ptr(),
        tail_mask.data_ptr() if tail_mask is not None else None, ldm_b, ldm_t, B, L, Hq, shape[1], D,
        D ** -0.5 if scale is None else scale, o.data_ptr(), lse.data_ptr() if return_lse else None, _HALF[q.dtype], ws,
        ws_bytes, _lib.error_ptr(dev), stream)
    _lib.check(rc, "paged_attention")
    return (o, lse) if return_lse else o
