"""Inputs at odd offsets of a larger buffer and with odd row strides give what aligned
copies of them give."""
import pytest
import torch

from kernels import _lib
from kernels.paged_cache import paged_append, paged_attention, rope_table

pytestmark = pytest.mark.gpu
DEV = "cuda"


def odd(t, off=1):
    """t's values, `off` elements into a flat buffer."""
    buf = torch.empty(t.numel() + off, dtype=t.dtype, device=t.device)
    out = buf[off:].view(t.shape)
    out.copy_(t)
    assert out.data_ptr() % 16 and out.is_contiguous()
    return out


def setup(T, dtype=torch.bfloat16, D=64):
    g = torch.Generator(device=DEV).manual_seed(T)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)  # noqa: E731
    kc, vc = r(5, 2, 16, D), r(5, 2, 16, D)
    at = torch.randperm(80, generator=g, device=DEV)[:T]
    return dict(qkv=r(T, 8 * D), heads=4, kv_heads=2, k_cache=kc, v_cache=vc, slots=at, positions=at,
                **dict(zip(("cos", "sin"), rope_table(80, D, 1e6, DEV))), q_weight=r(D), k_weight=r(D))


def append(a):
    a = {**a, "k_cache": a["k_cache"].clone(), "v_cache": a["v_cache"].clone()}
    with torch.inference_mode():
        return paged_append(**a), a["k_cache"], a["v_cache"]


@pytest.mark.parametrize("name", ["qkv", "cos", "sin", "q_weight", "k_weight", "slots", "positions"])
def test_append_of_an_odd_offset(name):
    a = setup(7)
    assert all(torch.equal(x, y) for x, y in zip(append(a), append({**a, name: odd(a[name])})))


@pytest.mark.parametrize("T", [1, 7])
def test_append_of_odd_rows(T):
    a = setup(T)
    want, qkv = append(a), a["qkv"]
    wide = torch.empty(T, qkv.shape[1] + 3, dtype=qkv.dtype, device=DEV)
    wide[:, :-3] = qkv
    same = a["qkv"][:1].expand(T, -1)                      # rows 0 apart
    for x in (wide[:, :-3], qkv.t().contiguous().t(), qkv.repeat_interleave(2, 1)[:, ::2]):
        assert all(torch.equal(x_, y) for x_, y in zip(want, append({**a, "qkv": x})))
    assert all(torch.equal(x, y) for x, y in zip(append({**a, "qkv": same.contiguous()}), append({**a, "qkv": same})))
    assert _lib.device_error() == 0


@pytest.mark.parametrize("L", [1, 8])
def test_attention_of_an_odd_offset(L):
    a = setup(60)
    append(a)
    g = torch.Generator(device=DEV).manual_seed(L)
    q = torch.randn(2, L, 16, 64, generator=g, device=DEV).to(torch.bfloat16)
    table = torch.tensor([[0, 1, 2], [4, 3, 2]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([40, 33], dtype=torch.int32, device=DEV)
    with torch.inference_mode():
        want = paged_attention(q, a["k_cache"], a["v_cache"], table, lens, return_lse=True)
        for qq, tt, ll in ((odd(q), table, lens), (q, odd(table), lens), (q, table, odd(lens)),
                           (q.transpose(1, 2).contiguous().transpose(1, 2), table.t().contiguous().t(), lens)):
            got = paged_attention(qq, a["k_cache"], a["v_cache"], tt, ll, return_lse=True)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_caches_that_cannot_be_written_in_place_are_refused():
    a = setup(3)
    with pytest.raises(RuntimeError):
        paged_append(**{**a, "k_cache": odd(a["k_cache"]), "v_cache": odd(a["v_cache"])})
