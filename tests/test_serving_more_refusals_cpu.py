"""What the 8-bit cache, the window, the page tables and the logit rules refuse, before any device work:
wrong types and shapes in Python, wrong sizes, types, alignments and workspaces at the C entry points."""
from __future__ import annotations

import ctypes

import pytest
import torch

from kernels import _lib
from kernels.logit_rules import adjust_logits, count_tokens
from kernels.paged_cache import paged_attention, rope_table
from kernels.paged_cache8 import F8, cache8, paged_append8, paged_attention8
from kernels.paged_tables import page_pool, paged_release, paged_reserve

BF = torch.bfloat16


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def cache(block=16, ps=16, Hk=2, D=64):
    return dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"), cache8(4, Hk, ps, D, block)))


def append_args(B=2, L=3, Hq=4, Hk=2, D=64):
    cos, sin = rope_table(32, D, 1e6)
    return dict(qkv=torch.zeros(B, L, (Hq + 2 * Hk) * D, dtype=BF), heads=Hq, kv_heads=Hk, **cache(), page_table=ints(B, 2),
                seq_lens=ints(B), cos=cos, sin=sin)


@pytest.mark.parametrize("change,error", [
    (dict(qkv=torch.zeros(2, 3, 512)), TypeError), (dict(qkv=torch.zeros(2, 3, 500, dtype=BF)), ValueError),
    (dict(qkv=torch.zeros(512, dtype=BF)), ValueError), (dict(heads=5), ValueError), (dict(kv_heads=3), ValueError),
    (dict(k_cache=torch.zeros(4, 2, 16, 64, dtype=BF)), TypeError), (dict(v_cache=torch.zeros(4, 2, 8, 64).to(F8)), ValueError),
    (dict(v_cache=torch.zeros(4, 16, 2, 64).to(F8).transpose(1, 2)), ValueError),
    (dict(k_scale=torch.zeros(4, 2, 1, dtype=BF)), TypeError), (dict(k_scale=torch.zeros(4, 2, 3)), ValueError),
    (dict(k_scale=torch.zeros(4, 2, 3), v_scale=torch.zeros(4, 2, 3)), ValueError),      # 3 does not divide 16
    (dict(k_scale=torch.zeros(4, 2, 0), v_scale=torch.zeros(4, 2, 0)), ValueError),
    (dict(v_scale=torch.zeros(4, 2, 2)[..., ::2]), ValueError),                          # other strides than k's
    (dict(page_table=torch.zeros(2, 2, dtype=torch.int64)), TypeError), (dict(page_table=ints(3, 2)), ValueError),
    (dict(seq_lens=torch.zeros(2)), TypeError), (dict(seq_lens=ints(3)), ValueError), (dict(count=torch.zeros(2)), TypeError),
    (dict(count=ints(1)), ValueError), (dict(cos=torch.zeros(32, 32, dtype=BF)), TypeError), (dict(cos=torch.zeros(31, 32)), ValueError),
    (dict(q_weight=torch.ones(64)), TypeError), (dict(k_weight=torch.ones(32, dtype=BF)), ValueError), (dict(), RuntimeError)])
def test_append8_refuses(change, error):
    with pytest.raises(error):
        paged_append8(**{**append_args(), **change})


def attention_args(B=2, L=2, Hq=4, D=64):
    return dict(q=torch.zeros(B, L, Hq, D, dtype=BF), **cache(), page_table=ints(B, 2), seq_lens=ints(B))


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(2, 2, 4, 64)), TypeError), (dict(q=torch.zeros(2, 256, dtype=BF)), ValueError),
    (dict(q=torch.zeros(2, 2, 3, 64, dtype=BF)), ValueError), (dict(q=torch.zeros(2, 2, 4, 128, dtype=BF)), ValueError),
    (dict(k_cache=torch.zeros(4, 2, 16, 64, dtype=BF)), TypeError), (dict(k_cache=torch.zeros(4, 16, 64).to(F8)), ValueError),
    (dict(k_scale=torch.zeros(4, 2, 1).double()), TypeError), (dict(v_scale=torch.zeros(4, 1, 1)), ValueError),
    (dict(page_table=ints(2, 2).long()), TypeError), (dict(seq_lens=ints(1)), ValueError), (dict(tail_mask=torch.zeros(2, 2)), TypeError),
    (dict(tail_mask=torch.zeros(2, 3, dtype=torch.bool)), ValueError), (dict(window=0), ValueError), (dict(window=-3), ValueError),
    (dict(sinks=-1), ValueError), (dict(), RuntimeError)])
def test_attention8_refuses(change, error):
    with pytest.raises(error):
        paged_attention8(**{**attention_args(), **change})


@pytest.mark.parametrize("change", [dict(window=0), dict(window=-1), dict(sinks=-1), dict(window=5, sinks=-2)])
def test_window_refuses(change):
    c = torch.zeros(4, 2, 16, 64, dtype=BF)
    with pytest.raises(ValueError):
        paged_attention(torch.zeros(2, 2, 4, 64, dtype=BF), c, c, ints(2, 2), ints(2), **change)


def test_cache8_refuses():
    for block in (0, 3, 32):
        with pytest.raises(ValueError):
            cache8(4, 2, 16, 64, block)


def reserve_args():
    table, held, free, count = page_pool(3, 4, 9)
    return dict(page_table=table, lens=ints(3), held=held, free_pages=free, free_count=count, L=2, page_size=16)


@pytest.mark.parametrize("change,error", [
    (dict(page_table=ints(3, 4).long()), TypeError), (dict(lens=ints(3).long()), TypeError), (dict(free_count=torch.zeros(1)), TypeError),
    (dict(page_table=ints(12)), ValueError), (dict(lens=ints(2)), ValueError), (dict(held=ints(4)), ValueError),
    (dict(count=ints(1)), ValueError), (dict(free_count=ints(2)), ValueError), (dict(free_pages=ints(3, 3)), ValueError),
    (dict(held=ints(6)[::2]), ValueError), (dict(free_pages=ints(18)[::2]), ValueError), (dict(page_table=ints(4, 3).t()), ValueError),
    (dict(page_size=0), ValueError), (dict(L=-1), ValueError), (dict(), RuntimeError)])
def test_reserve_refuses(change, error):
    with pytest.raises(error):
        paged_reserve(**{**reserve_args(), **change})


@pytest.mark.parametrize("change,error", [
    (dict(keep=ints(3).long()), TypeError), (dict(keep=ints(2)), ValueError), (dict(held=ints(6)[::2]), ValueError),
    (dict(page_size=0), ValueError), (dict(), RuntimeError)])
def test_release_refuses(change, error):
    args = {k: v for k, v in reserve_args().items() if k not in ("lens", "L")}
    with pytest.raises(error):
        paged_release(**{**args, "keep": ints(3), **change})


@pytest.mark.parametrize("change,error", [
    (dict(logits=torch.zeros(2, 3, 40).double()), TypeError), (dict(logits=torch.zeros(6, 40)), ValueError),
    (dict(logits=torch.zeros(2, 3, 0)), ValueError), (dict(counts=ints(2, 40).long()), TypeError), (dict(counts=ints(2, 39)), ValueError),
    (dict(drafts=ints(2, 2)), TypeError), (dict(drafts=ints(2, 3).long()), ValueError), (dict(repetition=torch.ones(2).double()), TypeError),
    (dict(presence=torch.ones(3)), ValueError), (dict(frequency=torch.ones(2, 1)), ValueError), (dict(seen=ints(2, 2).long()), TypeError),
    (dict(seen=ints(2, 1)), ValueError), (dict(bias_ids=ints(2, 3)), ValueError), (dict(bias_values=torch.zeros(2, 3)), ValueError),
    (dict(bias_ids=ints(2, 3).long(), bias_values=torch.zeros(2, 3)), TypeError),
    (dict(bias_ids=ints(2, 3), bias_values=torch.zeros(2, 3).double()), TypeError),
    (dict(bias_ids=ints(2, 3), bias_values=torch.zeros(2, 4)), ValueError), (dict(allowed=torch.ones(2, 3, 40, dtype=torch.bool)), TypeError),
    (dict(allowed=ints(2, 4, 2)), ValueError), (dict(allowed=ints(3, 2)), ValueError), (dict(out=torch.zeros(2, 3, 40, dtype=BF)), TypeError),
    (dict(out=torch.zeros(2, 40, 3).transpose(1, 2)), ValueError), (dict(out=torch.zeros(2, 3, 41)), ValueError), (dict(), RuntimeError)])
def test_rules_refuse(change, error):
    with pytest.raises(error):
        adjust_logits(**{"logits": torch.zeros(2, 3, 40), **change})


@pytest.mark.parametrize("counts,tokens,error", [
    (ints(2, 5).long(), ints(2, 3).long(), TypeError), (ints(2, 5), ints(2, 3), TypeError), (ints(2, 0), ints(2, 3).long(), ValueError),
    (ints(2, 5), ints(3, 3).long(), ValueError), (ints(2, 10)[:, ::2], ints(2, 3).long(), ValueError), (ints(2, 5), ints(2, 3).long(), RuntimeError)])
def test_counts_refuse(counts, tokens, error):
    with pytest.raises(error):
        count_tokens(counts, tokens)


def test_forward_only():
    for f, args, name in ((paged_append8, append_args(), "qkv"), (paged_attention8, attention_args(), "q"),
                          (adjust_logits, dict(logits=torch.zeros(1, 1, 8)), "logits")):
        args[name].requires_grad_()
        with pytest.raises(RuntimeError, match="forward-only"):
            f(**args)


def test_c_entry_points_refuse():
    L = _lib.lib()
    buf = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(buf) + 15) & ~15
    S, T, W, A, U = (_lib.SIMSD_ERR_SHAPE, _lib.SIMSD_ERR_DTYPE, _lib.SIMSD_ERR_WORKSPACE, _lib.SIMSD_ERR_ALIGN, _lib.SIMSD_ERR_UNSUPPORTED)

    def append(B=1, n=1, Hq=4, Hk=2, D=64, R=64, k=p, ldq_t=512, ldq_b=512, pages=4, ps=16, block=16, ld_tok=64, dtype=0, qkv=p, scale=p,
               max_pages=2, ld_table=2):
        return L.simsd_paged_append8(qkv, ldq_b, ldq_t, B, n, Hq, Hk, D, R, None, None, 1e-6, p, p, 32, p, ld_table, max_pages, p, None, p,
                                     k, p, scale, p, pages, ps, block, 2048, 1024, ld_tok, 2, 1, 1, dtype, None, None)
    assert append(B=-1) == append(Hk=0) == append(pages=0) == append(ldq_t=511) == append(qkv=None) == append(scale=None) == S
    assert append(block=0) == append(block=5) == append(ld_table=-1) == append(ldq_b=-8) == S
    assert append(dtype=2) == T
    assert append(D=96) == append(R=24) == append(R=80) == append(max_pages=1 << 28) == U
    assert append(k=p + 8) == append(ld_tok=72) == append(ldq_t=516) == A
    assert append(B=0) == append(n=0) == _lib.SIMSD_OK

    def attend(f, B=1, n=1, Hq=4, Hk=2, D=64, q=p, ld_table=2, ws=p, nbytes=1 << 30, dtype=0, ld_page=2048, window=0, sinks=0, block=16):
        eight = f is L.simsd_paged_attention8
        cache = (p, p, p, p, 4, 16, block, ld_page, 1024, 64, 2, 1, 1) if eight else (p, p, 4, 16, ld_page, 1024, 64)
        return f(q, *cache, p, ld_table, 2, p, None, 0, 0, B, n, Hq, Hk, D, 0.125, window, sinks, p, None, dtype, ws, nbytes, None, None)
    for f in (L.simsd_paged_attention8, L.simsd_paged_attention_window):
        assert attend(f, Hq=5) == attend(f, q=None) == attend(f, ld_table=-1) == attend(f, B=-1) == attend(f, window=-1) == S
        assert attend(f, sinks=-1) == S and attend(f, dtype=2) == T and attend(f, D=80) == U
        assert attend(f, q=p + 8) == attend(f, ld_page=2049) == A
        assert attend(f, ws=None) == attend(f, nbytes=0) == W
        assert attend(f, B=0) == attend(f, n=0) == _lib.SIMSD_OK
    assert attend(L.simsd_paged_attention8, block=5) == S
    assert L.simsd_paged_attention8_workspace_size(8, 32, 8, 128) > L.simsd_paged_attention8_workspace_size(0, 32, 8, 128)

    def reserve(B=1, n=1, ps=16, table=p, slots=p, lens=p, ws=p, nbytes=4096, max_pages=2, pool=4, ld=2):
        return L.simsd_paged_reserve(table, ld, max_pages, lens, None, p, p, pool, p, B, n, ps, slots, p, p, ws, nbytes, None, None)
    assert reserve(B=-1) == reserve(n=-1) == reserve(ps=0) == reserve(table=None) == reserve(slots=None) == reserve(lens=None) == S
    assert reserve(pool=-1) == reserve(ld=-1) == S and reserve(max_pages=1 << 28) == reserve(n=1 << 24) == U
    assert reserve(ws=None) == reserve(nbytes=8) == W and reserve(B=0) == _lib.SIMSD_OK

    def release(B=1, ps=16, table=p, keep=p, ws=p, nbytes=4096):
        return L.simsd_paged_release(table, 2, 2, p, p, 4, p, keep, B, ps, ws, nbytes, None, None)
    assert release(B=-1) == release(ps=0) == release(table=None) == release(keep=None) == S
    assert release(ws=None) == release(nbytes=8) == W and release(B=0) == _lib.SIMSD_OK

    def adjust(B=1, R=1, V=8, dtype=0, x=p, out=p, ids=None, n=0):
        return L.simsd_adjust_logits(x, 8, 8, out, 8, 8, B, R, V, dtype, None, 0, None, 0, None, 0, None, None, None, ids, 0, None, 0, n,
                                     None, 0, 0, None, None)
    assert adjust(B=-1) == adjust(V=0) == adjust(x=None) == adjust(out=None) == adjust(n=3) == adjust(n=-1) == S
    assert adjust(dtype=3) == T and adjust(B=65536) == U and adjust(B=0) == adjust(R=0) == _lib.SIMSD_OK
    assert L.simsd_count_tokens(None, 8, p, 1, 1, 1, 8, None, None) == L.simsd_count_tokens(p, 8, p, 1, 1, 1, 0, None, None) == S
    assert L.simsd_count_tokens(p, 8, p, 1, 1, 0, 8, None, None) == _lib.SIMSD_OK


def test_written_tensors_whose_elements_share_memory_are_refused():
    shared = torch.zeros(4, 1, 1).expand(4, 2, 1)
    with pytest.raises(ValueError, match="share memory"):
        paged_append8(**{**append_args(), "k_scale": shared, "v_scale": shared})
    wide = torch.zeros(1, 2, 16, 64).to(F8).expand(4, 2, 16, 64)
    with pytest.raises(ValueError, match="share memory"):
        paged_append8(**{**append_args(), "k_cache": wide, "v_cache": wide})
    with pytest.raises(ValueError, match="share memory"):
        paged_reserve(**{**reserve_args(), "page_table": ints(1, 4).expand(3, 4)})
    with pytest.raises(ValueError, match="share memory"):
        adjust_logits(torch.zeros(2, 3, 40), out=torch.zeros(2, 1, 40).expand(2, 3, 40))
    with pytest.raises(ValueError, match="share memory"):
        count_tokens(ints(1, 5).expand(2, 5), ints(2, 3).long())
    # rows in another order, rows with room between them and heads of a wider tensor are fine
    for out in (torch.zeros(3, 2, 40).transpose(0, 1), torch.zeros(2, 6, 48)[:, ::2, :40]):
        with pytest.raises(RuntimeError):                          # no CUDA tensors
            adjust_logits(torch.zeros(2, 3, 40), out=out)


def test_c_entry_points_refuse_shared_memory_and_lengths_past_30_bits():
    L = _lib.lib()
    buf = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(buf) + 15) & ~15
    S, U = _lib.SIMSD_ERR_SHAPE, _lib.SIMSD_ERR_UNSUPPORTED

    def append(strides=(2048, 1024, 64), scales=(2, 1, 1)):
        return L.simsd_paged_append8(p, 512, 512, 1, 1, 4, 2, 64, 64, None, None, 1e-6, p, p, 32, p, 2, 2, p, None, p, p, p, p, p, 4, 16,
                                     16, *strides, *scales, 0, None, None)
    for strides in ((2048, 0, 64), (0, 1024, 64), (2048, 1024, 48), (1024, 1024, 64), (1984, 1024, 64)):
        assert append(strides=strides) == S
    assert append(scales=(1, 1, 1)) == append(scales=(0, 1, 1)) == append(scales=(2, 0, 1)) == S

    def attend(f, pages, window):
        cache = (p, p, p, p, 4, 16, 16, 2048, 1024, 64, 2, 1, 1) if f is L.simsd_paged_attention8 else (p, p, 4, 16, 2048, 1024, 64)
        return f(p, *cache, p, pages, pages, p, None, 0, 0, 1, 1, 4, 2, 64, 0.125, window, 0, p, None, 0, p, 0, None, None)
    over, fits = (1 << 26) + 1, 1 << 26                            # pages of 16: 2^30 tokens
    assert attend(L.simsd_paged_attention8, over, 0) == attend(L.simsd_paged_attention8, over, 5) == U
    assert attend(L.simsd_paged_attention_window, over, 5) == U
    for f, pages, window in ((L.simsd_paged_attention8, fits, 0), (L.simsd_paged_attention_window, fits, 5),
                             (L.simsd_paged_attention_window, over, 0)):
        assert attend(f, pages, window) == _lib.SIMSD_ERR_WORKSPACE
    rows = lambda ld: L.simsd_paged_reserve(p, ld, 4, p, None, p, p, 4, p, 2, 1, 16, p, p, p, p, 0, None, None)  # noqa: E731
    assert rows(3) == S and rows(4) == _lib.SIMSD_ERR_WORKSPACE
    out = lambda b, r: L.simsd_adjust_logits(p, 8, 8, p, b, r, 2, 2, 8, 0, *[None, 0] * 3, None, None, None, *[None, 0] * 2, 0, None, 0, 0,  # noqa: E731
                                             None, None)
    assert out(8, 8) == out(16, 0) == out(8, 7) == S
    assert L.simsd_count_tokens(p, 7, p, 1, 2, 1, 8, None, None) == S


def test_numbers_past_32_bits_are_refused():
    for change in (dict(L=1 << 31), dict(page_size=1 << 31)):
        with pytest.raises(ValueError, match="2\\^31"):
            paged_reserve(**{**reserve_args(), **change})
    with pytest.raises(ValueError):
        paged_append8(**{**append_args(), "qkv": torch.zeros((), dtype=BF)})


@pytest.mark.parametrize("name", ["simsd_paged_attention_window", "simsd_paged_attention8", "simsd_paged_reserve", "simsd_paged_release"])
def test_calls_that_share_scratch_hold_the_gil(name):
    fn = getattr(_lib.lib(), name)
    assert type(fn)._flags_ & 4 and (fn.restype, list(fn.argtypes)) == (_lib.SIGNATURES[name][0], _lib.SIGNATURES[name][1])
