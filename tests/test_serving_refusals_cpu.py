"""What the batched serving operators refuse, before any device work: wrong types
and shapes in Python, wrong sizes, types, alignments and workspaces at the C entry
points."""
from __future__ import annotations

import ctypes

import pytest
import torch

from kernels import _lib
from kernels.paged_cache import paged_append, paged_attention, rope_table
from kernels.spec_verify import speculative_verify

BF = torch.bfloat16


def append_args(T=3, Hq=4, Hk=2, D=64, ps=16, dtype=BF):
    cos, sin = rope_table(32, D, 1e6)
    return dict(qkv=torch.zeros(T, (Hq + 2 * Hk) * D, dtype=dtype), heads=Hq, kv_heads=Hk,
                k_cache=torch.zeros(4, Hk, ps, D, dtype=dtype), v_cache=torch.zeros(4, Hk, ps, D, dtype=dtype),
                slots=torch.zeros(T, dtype=torch.int64), positions=torch.zeros(T, dtype=torch.int64), cos=cos, sin=sin)


@pytest.mark.parametrize("change,error", [
    (dict(qkv=torch.zeros(3, 512)), TypeError),                                      # fp32 activations
    (dict(qkv=torch.zeros(3, 500, dtype=BF)), ValueError),
    (dict(heads=5), ValueError),
    (dict(kv_heads=3), ValueError),
    (dict(k_cache=torch.zeros(4, 2, 16, 64)), TypeError),
    (dict(v_cache=torch.zeros(4, 2, 8, 64, dtype=BF)), ValueError),
    (dict(v_cache=torch.zeros(4, 16, 2, 64, dtype=BF).transpose(1, 2)), ValueError),  # other strides than k's
    (dict(slots=torch.zeros(3, dtype=torch.int32)), TypeError),
    (dict(slots=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(positions=torch.zeros(4, dtype=torch.int64)), ValueError),
    (dict(cos=torch.zeros(32, 32, dtype=BF)), TypeError),
    (dict(cos=torch.zeros(31, 32)), ValueError),
    (dict(q_weight=torch.ones(64)), TypeError),
    (dict(k_weight=torch.ones(32, dtype=BF)), ValueError),
    (dict(), RuntimeError),                                                          # CPU tensors
])
def test_append_refuses(change, error):
    with pytest.raises(error):
        paged_append(**{**append_args(), **change})


def attention_args(B=2, L=2, Hq=4, Hk=2, D=64, ps=16):
    return dict(q=torch.zeros(B, L, Hq, D, dtype=BF), k_cache=torch.zeros(4, Hk, ps, D, dtype=BF),
                v_cache=torch.zeros(4, Hk, ps, D, dtype=BF), page_table=torch.zeros(B, 2, dtype=torch.int32),
                seq_lens=torch.zeros(B, dtype=torch.int32))


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(2, 2, 4, 64)), TypeError),
    (dict(q=torch.zeros(2, 4 * 64, dtype=BF)), ValueError),
    (dict(q=torch.zeros(2, 2, 3, 64, dtype=BF)), ValueError),                        # 3 heads over 2
    (dict(q=torch.zeros(2, 2, 4, 128, dtype=BF)), ValueError),
    (dict(k_cache=torch.zeros(4, 2, 16, 64, dtype=torch.float16)), TypeError),
    (dict(k_cache=torch.zeros(4, 16, 64, dtype=BF)), ValueError),
    (dict(page_table=torch.zeros(2, 2, dtype=torch.int64)), TypeError),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int32)), ValueError),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(seq_lens=torch.zeros(1, dtype=torch.int32)), ValueError),
    (dict(tail_mask=torch.zeros(2, 2)), TypeError),
    (dict(tail_mask=torch.zeros(2, 3, dtype=torch.bool)), ValueError),
    (dict(), RuntimeError),
])
def test_attention_refuses(change, error):
    with pytest.raises(error):
        paged_attention(**{**attention_args(), **change})


def verify_args(B=2, K=3, V=10):
    return dict(target_logits=torch.zeros(B, K + 1, V), draft_tokens=torch.zeros(B, K, dtype=torch.int64),
                uniform=torch.zeros(B, K), noise=torch.ones(B, V))


@pytest.mark.parametrize("change,error", [
    (dict(target_logits=torch.zeros(2, 4, 10, dtype=torch.float64)), TypeError),
    (dict(target_logits=torch.zeros(8, 10)), ValueError),
    (dict(target_logits=torch.zeros(2, 4, 0)), ValueError),
    (dict(draft_tokens=torch.zeros(2, 3, dtype=torch.int32)), TypeError),
    (dict(draft_tokens=torch.zeros(2, 4, dtype=torch.int64)), ValueError),
    (dict(uniform=torch.zeros(2, 3, dtype=torch.float64)), TypeError),
    (dict(noise=torch.ones(2, 9)), ValueError),
    (dict(draft_logits=torch.zeros(2, 3, 10, dtype=BF)), TypeError),
    (dict(draft_logits=torch.zeros(2, 4, 10)), ValueError),
    (dict(temperature=torch.ones(2, dtype=torch.float64)), TypeError),
    (dict(temperature=torch.ones(3)), ValueError),
    (dict(n_draft=torch.ones(2, dtype=torch.int64)), TypeError),
    (dict(n_draft=torch.ones(1, dtype=torch.int32)), ValueError),
    (dict(), RuntimeError),
])
def test_verify_refuses(change, error):
    with pytest.raises(error):
        speculative_verify(**{**verify_args(), **change})


def test_forward_only():
    for f, args, name in ((paged_append, append_args(), "qkv"), (paged_attention, attention_args(), "q"),
                          (speculative_verify, verify_args(), "target_logits")):
        args[name].requires_grad_()
        with pytest.raises(RuntimeError, match="forward-only"):
            f(**args)


def test_c_entry_points_refuse():
    L = _lib.lib()
    buf = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(buf) + 15) & ~15

    def append(T=1, Hq=4, Hk=2, D=64, R=64, cache=p, ldqkv=512, pages=4, ps=16, ld_tok=64, dtype=0, qkv=p):
        return L.simsd_paged_append(qkv, ldqkv, T, Hq, Hk, D, R, None, None, 1e-6, p, p, 32, p, p, p, cache, p, pages, ps,
                                    2048, 1024, ld_tok, dtype, None, None)
    assert append(T=-1) == append(Hk=0) == append(pages=0) == append(ldqkv=511) == append(qkv=None) == _lib.SIMSD_ERR_SHAPE
    assert append(dtype=2) == _lib.SIMSD_ERR_DTYPE
    assert append(D=96) == append(R=24) == append(R=80) == _lib.SIMSD_ERR_UNSUPPORTED
    assert append(cache=p + 2) == append(ld_tok=68) == _lib.SIMSD_ERR_ALIGN
    assert append(T=0) == _lib.SIMSD_OK

    def attend(B=1, n=1, Hq=4, Hk=2, D=64, q=p, ld_table=2, ws=p, nbytes=1 << 30, dtype=0, ld_page=2048):
        return L.simsd_paged_attention(q, p, p, 4, 16, ld_page, 1024, 64, p, ld_table, 2, p, None, 0, 0, B, n, Hq, Hk, D,
                                       0.125, p, None, dtype, ws, nbytes, None, None)
    assert attend(Hq=5) == attend(q=None) == attend(ld_table=-1) == attend(B=-1) == _lib.SIMSD_ERR_SHAPE
    assert attend(dtype=2) == _lib.SIMSD_ERR_DTYPE
    assert attend(D=80) == _lib.SIMSD_ERR_UNSUPPORTED
    assert attend(q=p + 8) == attend(ld_page=2049) == _lib.SIMSD_ERR_ALIGN
    assert attend(ws=None) == attend(nbytes=0) == _lib.SIMSD_ERR_WORKSPACE
    assert attend(B=0) == attend(n=0) == _lib.SIMSD_OK

    def verify(B=1, K=2, V=10, dtype=0, target=p, x=p, ws=p, nbytes=1 << 30):
        return L.simsd_speculative_verify(target, 30, 10, None, 0, 0, x, 2, p, 2, p, 10, None, None, B, K, V, dtype, p, p, p,
                                          ws, nbytes, None, None)
    assert verify(V=0) == verify(K=-1) == verify(target=None) == verify(x=None) == _lib.SIMSD_ERR_SHAPE
    assert verify(dtype=3) == _lib.SIMSD_ERR_DTYPE
    assert verify(ws=None) == verify(nbytes=8) == _lib.SIMSD_ERR_WORKSPACE
    assert verify(B=0) == _lib.SIMSD_OK
