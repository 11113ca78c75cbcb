"""One-token attention over prefixes that sequences share (GPU): against its
formula in 64 bits, and against the plain attention over tables that hold the
prefix's pages first. Tolerances are those of `tests/pageddata.py`."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.gpuutil import bits
from tests.pageddata import assert_within, rounding
from tests.spandata import PrefixCase, slid, spans64, spans_check
from ttspipe_amd import pagedcache as pc

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _attend(c, **kw):
    before = None if c.scores is None else c.scores.clone()
    y = pc.attention(c.q, *c.pools(), c.slots, scores=c.scores, prefix=c.prefix(), **kw)
    assert y is not None
    torch.cuda.synchronize()
    return y, before


def _check(c, y, before=None, **kw):
    spans_check(c, y, c.scores, before, prefix=c.prefix(), **kw)


HEADS = [(32, 8, 128, 64, BF), (8, 2, 128, 16, FP), (8, 2, 64, 16, BF), (4, 2, 64, 32, FP), (7, 7, 64, 16, BF),
         (20, 4, 128, 128, BF), (32, 2, 128, 16, FP), (24, 1, 64, 256, BF), (40, 2, 128, 32, BF), (1, 1, 128, 4096, FP),
         (70, 1, 64, 16, BF)]


@pytest.mark.parametrize("nh,nkv,hd,page,dtype", HEADS)
@pytest.mark.parametrize("tracked", [False, True])
def test_shared_prefixes_match_the_formula(nh, nkv, hd, page, dtype, tracked):
    """Prefixes of none to a few chunks, of one sequence to many, with sequences of
    no own rows and of no prefix."""
    far = [300, 0, 1, 33, 700]
    of = [0, 4, 0, -1, 2, 3, 4, 4, 0, 1, -1, 5, 4, -7, 0, 2]
    lens = [5, 0, 17, 40, 1, 130, 700, 0, 33, 20, 0, 9, 64, 0, 1, 0]
    c = PrefixCase(lens, far, of, nh, nkv, hd, page, dtype, seed=nh + hd, tracked=tracked)
    y, before = _attend(c)
    assert not y[10].any() and not y[13].any()  # neither rows nor a prefix
    _check(c, y, before)


@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 513, 5000])
@pytest.mark.parametrize("seqs", [1, 4, 5, 8, 9, 17])
def test_one_prefix_of_all_lengths(n, seqs):
    """32 query and 8 KV heads: 4 to 68 query rows a KV head, the tiles' edges."""
    dtype = BF if n % 2 else FP
    c = PrefixCase([(7 * i) % 40 for i in range(seqs)], [n], [0] * seqs, 32, 8, 128, 16, dtype, seed=n + seqs, tracked=seqs == 5)
    y, before = _attend(c)
    _check(c, y, before)


@pytest.mark.parametrize("seqs,prefixes", [(70, 3), (300, 40), (520, 256)])
@pytest.mark.parametrize("tracked", [False, True])
def test_many_sequences_and_prefixes(seqs, prefixes, tracked):
    g = torch.Generator().manual_seed(seqs)
    lens = torch.randint(0, 60, (seqs,), generator=g).tolist()
    far = torch.randint(0, 200, (prefixes,), generator=g).tolist()
    of = torch.randint(-1, prefixes, (seqs,), generator=g).tolist()
    c = PrefixCase(lens, far, of, 4, 2, 64, 16, FP, seed=prefixes, tracked=tracked)
    y, before = _attend(c)
    _check(c, y, before)


@pytest.mark.parametrize("tracked", [False, True])
def test_long_prefixes_and_long_own_rows(tracked):
    c = PrefixCase([3000, 2, 900, 0], [9000, 4000], [0, 0, 1, 1], 32, 8, 128, 64, BF, seed=3, tracked=tracked)
    y, before = _attend(c)
    _check(c, y, before)


def test_own_rows_through_a_window():
    """The prefix stays visible; own rows slide out behind their sinks."""
    for tracked in (False, True):
        for window, sinks in ((1, 0), (40, 4), (300, 17), (10**9, 5)):
            c = PrefixCase([0, 1, 50, 700, 333, 41], [250, 60], [0, 1, -1, 0, 1, 0], 8, 2, 128, 16, BF, seed=window % 97, tracked=tracked)
            slid(c, window, sinks)
            y, before = _attend(c, window=window, sinks=sinks)
            _check(c, y, before, window=window, sinks=sinks)


def test_it_is_the_attention_over_the_pages_one_after_the_other():
    """Prefixes of whole pages, put before the own pages in a table of the plain call."""
    c = PrefixCase([40, 1, 77, 500], [256, 320], [0, 1, 1, 0], 32, 8, 128, 64, BF, seed=11, tracked=False)
    y, _ = _attend(c)
    cols = c.table.shape[1] + c.far_table.shape[1]
    table = torch.full((4, cols), -1, dtype=torch.int32, device="cuda")
    far_pages = [4, 5]
    for b in range(4):
        p = int(c.of[b])
        table[b, :far_pages[p]] = c.far_table[p, :far_pages[p]]
        table[b, far_pages[p]:far_pages[p] + c.table.shape[1]] = c.table[b]
    plain = pc.attention(c.q, c.k, c.v, table, c.slots + torch.tensor([256, 320, 320, 256], device="cuda"))
    ref, _, yb, _ = spans64(c.q, c.k, c.v, c.table, c.slots, prefix=c.prefix())
    assert_within(y, plain, 2 * (rounding(ref, BF) * (1 + 2**-7) + yb))


def test_holes_and_slots_past_the_tables():
    c = PrefixCase([100, 100, 100], [200, 200], [0, 1, 0], 8, 2, 128, 16, BF, seed=21)
    c.far_table[0, 3] = -1
    c.far_table[0, 12] = 10**8
    c.far_table[1] = -5
    c.table[2, 0] = -1
    y, before = _attend(c)
    _check(c, y, before)
    c.far_slots[0] = 207  # the last page's rows are NaN behind the prefix's 200: that page is a hole
    y, before = _attend(c)
    _check(c, y, before)
    c.far_slots[0] = 10**14
    y, before = _attend(c)
    _check(c, y, before)


def test_infinities_in_the_prefix_and_nan_behind_it():
    c = PrefixCase([20, 30], [100], [0, 0], 8, 2, 64, 16, BF, seed=23, tracked=False)
    c.v[c.far_table[0, 2].long(), 0, 3, 5] = math.inf
    c.v[c.far_table[0, 2].long(), 1, 3, 6] = -math.inf
    c.k[c.far_table[0, 1].long(), 1, 2] = 0
    y, _ = _attend(c)
    ref, *_ = spans64(c.q, c.k, c.v, c.table, c.slots, prefix=c.prefix())
    assert torch.equal(torch.isinf(y.cpu()), torch.isinf(ref)) and not torch.isnan(y).any()
    c.k[c.far_table[0, 1].long(), 0, 2, 0] = math.nan  # a key of KV head 0: its heads' outputs are NaN, the others' not
    y, _ = _attend(c)
    assert torch.isnan(y[:, :4]).all() and not torch.isnan(y[:, 4:]).any()


def test_strides_and_a_view_of_the_tables():
    c = PrefixCase([60, 5, 130], [90, 40], [1, 0, 1], 8, 2, 128, 16, FP, seed=31)
    wide = torch.full((2, c.far_table.shape[1] + 7), -3, dtype=torch.int32, device="cuda")
    wide[:, 5:5 + c.far_table.shape[1]] = c.far_table
    c.far_table = wide[:, 5:5 + c.far_table.shape[1]]
    q = torch.zeros(3, 10 * 128, dtype=FP, device="cuda")
    q[:, 128:9 * 128] = c.q.view(3, -1)
    before = c.scores.clone()
    y = pc.attention(q[:, 128:9 * 128].view(3, 8, 128), *c.pools(), c.slots, scores=c.scores, prefix=c.prefix())
    torch.cuda.synchronize()
    _check(c, y, before)


def test_refusals_and_workspaces():
    c = PrefixCase([60, 5, 130], [90, 40], [1, 0, 1], 8, 2, 128, 16, FP, seed=31)
    good = c.prefix()
    cols, far_cols = c.table.shape[1], c.far_table.shape[1]
    for bad in (good._replace(table=good.table.long()), good._replace(table=good.table[0]), good._replace(slots=good.slots[:1]),
                good._replace(slots=good.slots.int()), good._replace(of=good.of[:2]), good._replace(of=good.of.long()),
                good._replace(table=good.table.cpu()), good._replace(table=good.table.t().contiguous().t()),
                pc.Prefix(good.table.expand(2, -1)[:0], good.slots[:0], good.of),
                pc.Prefix(good.table[:1].repeat(257, 1), good.slots[:1].repeat(257), good.of)):
        assert pc.attention(c.q, *c.pools(), c.slots, prefix=bad) is None
    for kw in (dict(window=0), dict(sinks=3), dict(window=4, sinks=-1)):
        with pytest.raises(ValueError):
            pc.attention(c.q, *c.pools(), c.slots, prefix=good, **kw)
    need = pc.attention_work(3, 8, 2, 128, cols, 16, True, prefixes=2, prefix_columns=far_cols)
    work = torch.full((need,), math.nan, device="cuda")
    out = torch.empty_like(c.q)
    y, before = _attend(c, work=work, out=out)
    assert y is out
    _check(c, y, before)
    with pytest.raises(ValueError):
        _attend(c, work=work[:-256])


def test_a_captured_call_follows_lengths_and_prefixes():
    c = PrefixCase([400, 40, 300, 0, 7], [500, 90, 1200], [0, 1, 0, 2, -1], 8, 2, 128, 16, BF, seed=41)
    work = torch.empty(pc.attention_work(5, 8, 2, 128, c.table.shape[1], 16, True, prefixes=3,
                                         prefix_columns=c.far_table.shape[1]), device="cuda")
    out = torch.empty_like(c.q)
    run = lambda: pc.attention(c.q, *c.pools(), c.slots, scores=c.scores, out=out, work=work, prefix=c.prefix())  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    slots, far = c.slots.clone(), c.far_slots.clone()
    for cut, of in ((0, [0, 1, 0, 2, -1]), (6, [2, 2, 2, 2, 2]), (39, [-1] * 5), (0, [1, 0, 1, 0, 1]), (200, [0, 0, 2, 9, 0])):
        c.slots.copy_(slots - cut)
        c.far_slots.copy_(far - cut)
        c.of.copy_(torch.tensor(of, dtype=torch.int32))
        before = c.scores.clone()
        graph.replay()
        torch.cuda.synchronize()
        _check(c, out, before)
        again = pc.attention(c.q, *c.pools(), c.slots, prefix=c.prefix())
        assert np.array_equal(bits(again), bits(out))  # the sums' order is fixed


def test_two_streams_at_once():
    cs = [PrefixCase([200, 7, 90], [800], [0, 0, 0], 32, 8, 128, 16, BF, seed=50 + i, tracked=False) for i in range(2)]
    want = [_attend(c)[0] for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    got = [[], []]
    for _ in range(5):
        for c, st, g in zip(cs, streams, got):
            with torch.cuda.stream(st):
                g.append(pc.attention(c.q, *c.pools(), c.slots, prefix=c.prefix()))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(np.array_equal(bits(w), bits(x)) for x in g)
