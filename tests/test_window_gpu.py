"""One-token attention through a sliding window with sinks over the paged cache
(GPU): against its formula in 64 bits, at the lengths, windows, pages and holes
where it can go wrong. Tolerances are those of `tests/pageddata.py`."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.gpuutil import bits
from tests.pageddata import Case
from tests.spandata import slid, spans_check
from ttspipe_amd import pagedcache as pc

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
EDGES = [0, 1, 2, 15, 16, 17, 31, 33, 48, 64, 65, 100, 127, 128, 129, 257, 700]


def _attend(c, window, sinks, **kw):
    before = None if c.scores is None else c.scores.clone()
    y = pc.attention(c.q, *c.pools(), c.slots, scores=c.scores, window=window, sinks=sinks, **kw)
    assert y is not None
    torch.cuda.synchronize()
    return y, before


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 4), (15, 0), (16, 16), (17, 15), (31, 17), (32, 0), (33, 33),
                                          (64, 4), (100, 64), (255, 1), (600, 100), (1000, 4), (10**6, 10**6), (5, 10**9)])
@pytest.mark.parametrize("tracked", [False, True])
@pytest.mark.parametrize("page", [16, 64])
def test_windows_of_ragged_sequences(window, sinks, tracked, page):
    c = Case(EDGES, 8, 2, 128, page, BF, seed=window % 1000 + sinks % 1000, tracked=tracked)
    slid(c, window, sinks)
    y, before = _attend(c, window, sinks)
    assert not y[0].any()
    spans_check(c, y, c.scores, before, window=window, sinks=sinks)


@pytest.mark.parametrize("nh,nkv,hd,page,dtype", [(32, 8, 128, 64, BF), (8, 2, 64, 16, FP), (7, 7, 64, 32, BF), (20, 4, 128, 128, FP),
                                                  (24, 1, 64, 256, BF), (40, 2, 128, 32, FP), (1, 1, 128, 4096, BF)])
@pytest.mark.parametrize("tracked", [False, True])
def test_windows_of_other_heads(nh, nkv, hd, page, dtype, tracked):
    for window, sinks in ((40, 3), (777, 20)):
        c = Case([5, 0, 41, 900, 1301, 60], nh, nkv, hd, page, dtype, seed=nh + hd, tracked=tracked)
        y, before = _attend(c, window, sinks)
        spans_check(c, y, c.scores, before, window=window, sinks=sinks)


@pytest.mark.parametrize("n,window,sinks", [(5000, 4096, 4), (20011, 1024, 64), (20011, 15000, 0), (3001, 497, 0), (3001, 481, 16),
                                            (3001, 482, 16)])
def test_window_of_one_long_sequence(n, window, sinks):
    c = Case([n], 32, 8, 128, 64, FP, seed=n + window)
    slid(c, window, sinks)
    y, before = _attend(c, window, sinks)
    spans_check(c, y, c.scores, before, window=window, sinks=sinks)


def test_a_window_wider_than_the_sequences_changes_no_bit():
    c = Case([3, 300, 1000, 0], 32, 8, 128, 16, BF, seed=4)
    plain = pc.attention(c.q, *c.pools(), c.slots)
    y, _ = _attend(c, 1008, 0)
    assert np.array_equal(bits(plain), bits(y))


def test_one_row_windows_give_its_value():
    c = Case([70, 17, 1], 4, 2, 64, 16, BF, seed=8, tracked=False)
    y, _ = _attend(c, 1, 0)
    for b, n in enumerate(c.lens):
        v = c.v[c.table[b, (n - 1) // 16].long(), :, (n - 1) % 16]
        assert torch.equal(y[b], v.repeat_interleave(2, 0))


def test_infinities_behind_the_window_are_not_seen():
    c = Case([200, 333], 8, 2, 128, 16, BF, seed=12)
    for b, n in enumerate(c.lens):
        for j in range(7, n - 50):
            c.k[c.table[b, j // 16], :, j % 16] = math.inf if j % 2 else math.nan
            c.v[c.table[b, j // 16], :, j % 16] = -math.inf if j % 3 else math.nan
    y, before = _attend(c, 50, 7)
    assert torch.isfinite(y).all()
    spans_check(c, y, c.scores, before, window=50, sinks=7)
    for b, n in enumerate(c.lens):
        assert torch.equal(c.scores[b, :, 7:n - 50], before[b, :, 7:n - 50])
        assert torch.equal(c.scores[b, :, n:], before[b, :, n:])


def test_holes_in_the_window_and_slots_past_the_table():
    c = Case([300, 300, 300, 300], 8, 2, 128, 16, FP, seed=14)
    c.table[0, 18] = -1
    c.table[1, 0] = 10**6
    c.table[2, 17:] = -1
    c.table[3] = -1
    c.slots[1] = 10**12
    y, before = _attend(c, 40, 10)
    assert not y[3].any()
    c.slots[1] = c.cap - 1
    c.k[c.table[1, 18].long(), :, 12:] = 0  # (rows past the case's 300, NaN so far)
    c.v[c.table[1, 18].long(), :, 12:] = 0
    c.slots[1] = 299
    y, before = _attend(c, 40, 10)
    spans_check(c, y, c.scores, before, window=40, sinks=10)


@pytest.mark.parametrize("tracked", [False, True])
def test_many_sequences(tracked):
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 900, (130,), generator=g).tolist()
    c = Case(lens, 4, 2, 64, 16, BF, seed=5, tracked=tracked)
    for window, sinks in ((30, 4), (600, 4)):
        y, before = _attend(c, window, sinks)
        spans_check(c, y, c.scores, before, window=window, sinks=sinks)


def test_workspaces_and_refusals():
    c = Case([400, 3000], 8, 2, 128, 16, BF, seed=6)
    cols = c.table.shape[1]
    assert pc.attention_work(2, 8, 2, 128, cols, 16, window=100, sinks=4) == 0  # one chunk a sequence
    need = pc.attention_work(2, 8, 2, 128, cols, 16, True, window=1000, sinks=4)
    assert need > 0
    work = torch.empty(need, device="cuda")
    y, before = _attend(c, 1000, 4, work=work)
    spans_check(c, y, c.scores, before, window=1000, sinks=4)
    with pytest.raises(ValueError):
        _attend(c, 1000, 4, work=work[:-256])
    for kw in (dict(window=0), dict(window=-1), dict(window=5, sinks=-1), dict(sinks=2)):
        with pytest.raises(ValueError):
            pc.attention(c.q, *c.pools(), c.slots, **kw)


def test_a_captured_window_follows_the_rows():
    c = Case([900, 40, 500], 8, 2, 128, 16, BF, seed=7)
    out = torch.empty_like(c.q)
    work = torch.empty(pc.attention_work(3, 8, 2, 128, c.table.shape[1], 16, True, window=600, sinks=4), device="cuda")
    run = lambda: pc.attention(c.q, *c.pools(), c.slots, scores=c.scores, out=out, work=work, window=600, sinks=4)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for cut in (0, 1, 39, 200, 0):
        slots = c.slots.clone()
        c.slots -= cut
        before = c.scores.clone()
        graph.replay()
        torch.cuda.synchronize()
        spans_check(c, out, c.scores, before, window=600, sinks=4)
        c.slots.copy_(slots)
