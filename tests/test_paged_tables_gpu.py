"""Page tables and slot maps (kernels/paged_tables.py) against plain Python: whole numbers, equal."""
from __future__ import annotations

import random

import pytest
import torch

from kernels import _lib
from kernels.paged_tables import page_pool, paged_release, paged_reserve

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Pool:
    """The same in plain Python."""

    def __init__(self, table, held, free):
        self.table, self.held, self.free = [list(r) for r in table], list(held), list(free)

    def reserve(self, lens, count, L, ps):
        slots, positions, totals, short, bad = [], [], [], False, False
        wanted, size = 0, len(self.free)
        taken = 0
        for b, n in enumerate(lens):
            c = max(0, min(count[b], L))
            if n < 0:
                bad, n, c = True, 0, 0
                have = max(self.held[b], 0)
                take = 0
            else:
                have = max(self.held[b], -(-n // ps))
                take = max(0, -(-(n + c) // ps) - have)
                if have + take > len(self.table[b]):
                    short, c, take = True, 0, 0
            wanted += take
            if take and wanted > size:
                short, c, take = True, 0, 0
            for i in range(take):
                self.table[b][have + i] = self.free[size - 1 - taken - i]
            taken += take
            self.held[b] = have + take
            row = [(-1, 0)] * (L - c)
            for x in range(n, n + c):
                page = self.table[b][x // ps]
                row.append((page * ps + x % ps if page >= 0 else -1, x))
            slots.append([s for s, _ in row])
            positions.append([p for _, p in row])
            totals.append(n + c)
        self.free = self.free[: size - taken]
        return slots, positions, totals, (short, bad)

    def release(self, keep, ps, room):
        wanted, short, back = 0, False, []
        for b, k in enumerate(keep):
            kept = min(self.held[b], -(-max(k, 0) // ps))
            wanted += self.held[b] - kept
            if self.held[b] > kept and len(self.free) + wanted > room:
                short = True
                continue
            back += self.table[b][kept: self.held[b]]
            self.held[b] = kept
        self.free += back
        return short


def state(pool, pages, spare=0):
    """The device's copy of a Pool."""
    free = pool.free + [-7] * (pages - len(pool.free) + spare)
    return ints(pool.table), ints(pool.held), ints(free), ints([len(pool.free)])


def same(pool, dev):
    table, held, free, count = (t.tolist() for t in dev)
    assert table == pool.table and held == pool.held and count == [len(pool.free)]
    assert free[: count[0]] == pool.free


def errors():
    e = _lib.device_error()
    _lib.clear_device_error()
    return bool(e & _lib.DEV_ERR_CAPACITY), bool(e & _lib.DEV_ERR_BAD_INDEX)


@pytest.mark.parametrize("B,L,ps,most,lack", [
    (1, 1, 16, 50, False), (1, 5, 1, 20, False), (3, 4, 16, 0, False), (32, 4, 16, 4096, False), (7, 300, 24, 100, False),
    (256, 2, 8, 60, False), (257, 3, 16, 40, False), (700, 1, 4, 33, True), (64, 33, 16, 200, True), (5, 2048, 64, 3, False),
    (300, 9, 1, 12, True), (2, 0, 16, 40, False), (40, 1, 128, 9000, True)])
def test_reserve_and_release_match_plain_python(B, L, ps, most, lack):
    r = random.Random(B * 31 + L)
    lens = [r.randint(0, most) for _ in range(B)]
    held = [-(-n // ps) + r.choice([0, 0, 0, 1, 2]) for n in lens]         # drafts that were not kept leave pages behind
    width = -(-(most + L) // ps) + 3
    pages = sum(held) + B * (-(-L // ps) + 1)
    order = list(range(pages))
    r.shuffle(order)
    table, at = [], 0
    for h in held:
        table.append(order[at: at + h] + [-1] * (width - h))
        at += h
    pool = Pool(table, held, order[at: at + (pages - at) // (3 if lack else 1)])
    dev = state(pool, pages)
    for turn in range(3):
        count = [r.choice([L, L, r.randint(0, L), L + 5, -2]) for _ in range(B)]
        if turn == 0:
            count = [L] * B
        slots, positions, total, (short, bad) = pool.reserve(lens, count, L, ps)
        with torch.inference_mode():
            got = paged_reserve(dev[0], ints(lens), dev[1], dev[2], dev[3], L, ps, count=None if turn == 0 else ints(count))
        assert got[0].tolist() == slots and got[1].tolist() == positions and got[2].tolist() == total
        same(pool, dev)
        assert errors() == (short, bad)
        kept = [r.randint(min(a, b), b) for a, b in zip(lens, total)]      # some of the new tokens, some sequences done
        keep = [r.choice([k, k, k, 0, -1]) for k in kept]
        short = pool.release(keep, ps, pages)
        with torch.inference_mode():
            assert paged_release(dev[0], dev[1], dev[2], dev[3], ints(keep), ps) is None
        same(pool, dev)
        assert errors() == (short, False)
        lens = [max(k, 0) for k in keep]


def test_refused_sequences_and_lengths():
    """A stack that runs out, a row that is too short, a negative length; the others are served."""
    pool = Pool([[0, 1, -1, -1], [2, -1, -1, -1], [3, -1, -1, -1], [4, -1, -1, -1], [5, 6, 7, 8]], [2, 1, 1, 1, 4], [9, 10])
    lens, count = [32, 16, -3, 10, 64], [1, 17, 4, 6, 1]
    dev = state(pool, 11)
    want = pool.reserve(lens, count, 17, 16)
    got = paged_reserve(dev[0], ints(lens), dev[1], dev[2], dev[3], 17, 16, count=ints(count))
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1] and got[2].tolist() == want[2] == [33, 16, 0, 16, 64]
    same(pool, dev)
    assert errors() == (True, True)
    # a stack that is full takes no page of a sequence whose pages do not all fit
    pool = Pool([[0, 1, 2], [3, 4, 5]], [3, 3], [6, 7])
    dev = state(pool, 6)
    assert pool.release([0, 0], 16, 6)
    paged_release(dev[0], dev[1], dev[2], dev[3], ints([0, 0]), 16)
    same(pool, dev)
    assert dev[1].tolist() == [0, 3] and errors() == (True, False)


def test_pages_are_taken_once():
    """Many sequences at once: every page in one place at most, on the stack or in a row."""
    B, ps, pages = 300, 16, 4000
    table, held, free, count = page_pool(B, 40, pages, DEV)
    r = random.Random(1)
    lens = [0] * B
    for step in range(6):
        new = [r.randint(0, 40) for _ in range(B)]
        slots, _, total = paged_reserve(table, ints(lens), held, free, count, 40, ps, count=ints(new))
        used = slots[slots >= 0]
        assert used.numel() == sum(new) == used.unique().numel()
        lens = [0 if r.random() < 0.2 else n for n in total.tolist()]
        paged_release(table, held, free, count, ints(lens), ps)
        mine = [p for b in range(B) for p in table[b, : int(held[b])].tolist()]
        assert sorted(mine + free[: int(count)].tolist()) == list(range(pages))
    assert errors() == (False, False)


def test_streams_and_graphs():
    """Two captured graphs replayed in turn, and calls on another stream, give what eager calls give."""
    B, L, ps = 9, 6, 4
    lens = ints([0, 3, 9, 1, 0, 0, 20, 7, 2])
    want, dev = page_pool(B, 20, 200, DEV), page_pool(B, 20, 200, DEV)
    graphs, out = [torch.cuda.CUDAGraph() for _ in range(2)], []

    def step(s, n):
        got = paged_reserve(s[0], n, s[1], s[2], s[3], L, ps)
        paged_release(s[0], s[1], s[2], s[3], n, ps)
        return got
    step(page_pool(B, 20, 200, DEV), lens)
    for graph in graphs:
        with torch.cuda.graph(graph):
            out.append(step(dev, lens))
    side = torch.cuda.Stream()
    for turn in range(4):
        lens += turn
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ref = step(want, lens)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ref, out[turn % 2]))
        assert all(torch.equal(a, b) for a, b in zip(want, dev))
    assert errors() == (False, False)


def test_nothing():
    table, held, free, count = page_pool(0, 4, 5, DEV)
    none = ints([])
    assert [t.shape for t in paged_reserve(table, none, held, free, count, 3, 16)] == [(0, 3), (0, 3), (0,)]
    paged_release(table, held, free, count, none, 16)
    table, held, free, count = page_pool(2, 0, 0, DEV)                     # no pages at all
    slots, _, total = paged_reserve(table, ints([0, 0]), held, free, count, 2, 16)
    assert bool((slots == -1).all()) and total.tolist() == [0, 0]
    assert errors() == (True, False)


def test_a_length_past_its_row_takes_and_keeps_nothing():
    """Two pages of 16 a row: 40 tokens are not in the row, and what it holds stays its own."""
    table, held, free, count = ints([[5, -1], [6, 7]]), ints([1, 2]), ints([0, 1, 2, 3, 4, -1, -1, -1]), ints([5])
    slots, positions, total = paged_reserve(table, ints([40, 20]), held, free, count, 3, 16)
    assert slots.tolist() == [[-1] * 3, [7 * 16 + 4 + i for i in range(3)]] and total.tolist() == [40, 23]
    assert held.tolist() == [1, 2] and count.tolist() == [5] and errors() == (True, False)
    paged_release(table, held, free, count, ints([0, 0]), 16)
    assert held.tolist() == [0, 0] and free.tolist() == [0, 1, 2, 3, 4, 5, 6, 7] and count.tolist() == [8]
    assert errors() == (False, False)
