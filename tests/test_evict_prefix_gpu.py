"""Eviction of sequences that have a prefix (GPU): their first rows are counted from
their own first position, which lies behind the prefix."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.gpuutil import bits
from tests.pageddata import assert_within, evict_ref, rounding
from tests.spandata import spans64
from tests.test_paged_gpu import _freqs, _tracked
from ttspipe_amd import pagedcache as pc

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _served(seed, lens=((20, 0), (30, None), (5, 0), (26, 1))):
    """A tracked cache of four streams, three behind prefixes of 33 and 90 rows."""
    g = torch.Generator().manual_seed(seed)
    table = pc.PageTable(4, 100, 60, 16, prefixes=2, max_prefix=100)
    cache = pc.PagedKVCache(table, 2, 64, tracked=True)
    rows = lambda n: [torch.randn(n, 2, 64, generator=g).to(BF).cuda() for _ in "kv"]  # noqa: E731
    for n in (33, 90):
        assert cache.store_prefix(table.admit_prefix(n), *rows(n))
    for n, p in lens:
        assert cache.store(table.admit(n, prefix=p), *rows(n))
    freqs = _freqs(300, 64)

    def step():
        table.step()
        q = cache.qk_rope_kv((torch.randn(4, 12 * 64, generator=g)).to(BF).cuda(), 8, freqs)
        y = cache.attention(q)
        ref, _, yb, _ = spans64(q, cache.k_pages, cache.v_pages, table.block_table, table.slots, prefix=table.prefix)
        assert_within(y, ref, rounding(ref, BF) * (1 + 2**-7) + yb)

    return table, cache, step


def _cut(table, cache, budget, sinks, recent, run):
    """`run`s the eviction and holds it to the definition, its positions counted from each sequence's first."""
    cache.scores[:, :, :6] = 0.0  # the first rows have gathered least
    s, sp = cache.scores.cpu().numpy().copy(), cache.slot_pos.cpu().numpy().copy()
    k, v = cache.k_pages.clone(), cache.v_pages.clone()
    rows = [table.rows(b) for b in range(4)]
    run()
    torch.cuda.synchronize()
    bt = table.block_table.cpu()
    for b, n in enumerate(rows):
        first = table.first_position(b)
        for h in range(2):
            for src, dst in evict_ref(s[b, h], sp[b, h] - first, n, int(table.positions[b]) - first, budget, sinks, recent):
                s[b, h, dst], sp[b, h, dst] = s[b, h, src], sp[b, h, src]
                at, to = (int(bt[b, src // 16]), h, src % 16), (int(bt[b, dst // 16]), h, dst % 16)
                k[to], v[to] = k[at], v[at]
            if n > budget:
                assert set(range(first, first + sinks)) <= set(cache.slot_pos[b, h, :budget].tolist()), (b, h)
    assert np.array_equal(cache.slot_pos.cpu().numpy(), sp) and np.array_equal(cache.scores.cpu().numpy(), s)
    assert np.array_equal(bits(cache.k_pages), bits(k)) and np.array_equal(bits(cache.v_pages), bits(v))
    table.evicted(budget)


def test_a_stream_behind_a_prefix_keeps_its_own_first_rows():
    table, cache, step = _served(1)
    for _ in range(3):
        step()
    _cut(table, cache, 16, 4, 3, lambda: cache.evict(16, sinks=4, recent=3))
    for i in range(6):
        step()
        if i % 2:
            _cut(table, cache, 16, 4, 3, lambda: cache.evict(16, sinks=4, recent=3))


def test_a_captured_eviction_follows_streams_that_change_their_prefix():
    table, cache, step = _served(2)
    step()
    work = torch.zeros(max(1, pc.evict_work(4, 2, table.block_table.shape[1], 16, 16)), dtype=torch.int32, device="cuda")
    before = [t.clone() for t in (cache.k_pages, cache.v_pages, cache.scores, cache.slot_pos)]
    cache.evict(16, sinks=4, recent=3, work=work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.evict(16, sinks=4, recent=3, work=work)
    for t, old in zip((cache.k_pages, cache.v_pages, cache.scores, cache.slot_pos), before):
        t.copy_(old)
    for change in (None, (0, 1, 25), (3, None, 40), (1, 0, 18)):
        if change is not None:
            seq, prefix, n = change
            table.release(seq)
            assert table.admit(n, prefix=prefix) == seq
            assert cache.store(seq, *[torch.randn(n, 2, 64, device="cuda").to(BF) for _ in "kv"])
            step()
        _cut(table, cache, 16, 4, 3, graph.replay)


@pytest.mark.parametrize("lens,budget,cols", [([300, 290, 5], 288, None), ([2000, 700, 1500], 600, None), ([2050, 300, 2048], 2047, None),
                                              ([20000, 9000, 100], 5000, None), ([300, 290], 200, 600)])
def test_positions_that_start_anywhere_move_the_same_rows(lens, budget, cols):
    """Narrow, listed and long caches: as without first positions where all positions are counted from them."""
    got = []
    off = torch.tensor([1000, 2**31 - 2**16, 7][: len(lens)], device="cuda")
    for first in (None, off):
        c, s, sp = _tracked(lens, 2, 64, 16, FP, seed=budget, cols=cols)
        newest = torch.tensor([n - 1 for n in lens], device="cuda")
        if first is not None:
            sp += first.to(torch.int32)[:, None, None]
            newest = newest + first
        assert pc.evict(*c.pools(), c.slots, s, sp, newest, budget, sinks=40, recent=30, first=first)
        torch.cuda.synchronize()
        got.append((c.k, c.v, s, sp if first is None else sp - first.to(torch.int32)[:, None, None]))
    for a, b in zip(*got):
        assert np.array_equal(bits(a), bits(b)) if a.dtype is FP else torch.equal(a, b)


def test_first_positions_that_do_not_fit_are_declined():
    c, s, sp = _tracked([100, 90], 2, 64, 16, FP, seed=1)
    pos = torch.tensor([99, 89], device="cuda")
    for bad in (pos.int(), pos[:1], pos.cpu(), pos.repeat(2)[::2]):
        assert pc.evict(*c.pools(), c.slots, s, sp, pos, 50, sinks=3, first=bad) is None
