"""Shared prefixes and windows on the host (no GPU calls): `PageTable`'s account of
prefixes and of pages that a window has left, what the C entries refuse before any
launch, and the mirrored argument block."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tests.test_paged import P, _at, _cache
from ttspipe_amd import _lib, fastpath
from ttspipe_amd import pagedcache as pc


def table(**kw):
    return pc.PageTable(3, 100, 20, 16, device="cpu", **{**dict(prefixes=2, max_prefix=50), **kw})


def test_sequences_behind_a_prefix():
    t = table()
    assert t.prefix.table.shape == (2, 4) and t.prefix.of.tolist() == [-1] * 3
    p = t.admit_prefix(33)
    assert p == 0 and t.free_pages == 17 and t.prefix_rows(0) == 33 and t.prefix.slots.tolist() == [32, -1]
    assert t.admit(5, prefix=p) == 0 and t.admit(16) == 1 and t.admit(1, prefix=p) == 2
    assert t.prefix.of.tolist() == [0, -1, 0]
    assert t.slots.tolist() == [4, 15, 0] and t.positions.tolist() == [37, 15, 33]
    assert (t.first_position(0), t.first_position(1)) == (33, 0) and t.positions_used == 38
    t.step()
    assert t.slots.tolist() == [5, 16, 1] and t.positions.tolist() == [38, 16, 34]
    pages = [x for x in [*t.block_table.flatten().tolist(), *t.prefix.table.flatten().tolist()] if x >= 0]
    assert len(pages) == len(set(pages)) == 20 - t.free_pages
    with pytest.raises(ValueError):
        t.release_prefix(0)
    t.release(0)
    assert t.prefix.of.tolist() == [-1, -1, 0] and t.positions.tolist()[0] == -1
    t.release(2)
    t.release_prefix(0)
    assert t.prefix.table.tolist() == [[-1] * 4] * 2 and t.prefix.slots.tolist() == [-1, -1] and t.free_pages == 18
    t.release(1)
    assert t.free_pages == 20


def test_prefixes_that_do_not_fit():
    t = table(max_position=60)
    for rows in (0, 51, -1):
        with pytest.raises(ValueError):
            t.admit_prefix(rows)
    assert t.admit_prefix(50) == 0 and t.admit_prefix(1) == 1 and t.admit_prefix(1) is None
    for kw in (dict(rows=11, prefix=0), dict(rows=1, prefix=2), dict(rows=1, prefix=-1)):
        with pytest.raises(ValueError):
            t.admit(**kw)
    t.release_prefix(1)
    with pytest.raises(ValueError):
        t.admit(1, prefix=1)
    with pytest.raises(ValueError):
        t.release_prefix(5)
    assert t.admit(10, prefix=0) == 0
    with pytest.raises(ValueError):
        t.step()  # position 60
    assert t.rows(0) == 10
    small = pc.PageTable(1, 16, 2, 16, device="cpu", prefixes=1, max_prefix=100)
    with pytest.raises(MemoryError):
        small.admit_prefix(33)
    assert small.free_pages == 2 and small.prefix.slots.tolist() == [-1]
    plain = pc.PageTable(1, 16, 2, 16, device="cpu")
    assert plain.prefix is None
    with pytest.raises(ValueError):
        plain.admit_prefix(3)
    for kw in (dict(prefixes=257), dict(prefixes=-1), dict(max_prefix=0)):
        with pytest.raises(ValueError):
            table(**kw)


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (20, 4), (33, 17), (1000, 3)])
def test_a_window_gives_pages_back(window, sinks):
    t = pc.PageTable(2, 400, 60, 16, device="cpu")
    t.admit(100), t.admit(7)
    for _ in range(150):
        t.step()
        t.slide(window, sinks)
        for b in range(2):
            n, row = t.rows(b), t.block_table[b].tolist()
            assert n == int(t.slots[b]) + 1
            for j in range(n):
                # what this step's token or the next one's may see is there; whole pages that neither sees are not
                seen = j < sinks or j > n - 1 - window
                assert row[j // 16] >= 0 or not seen
            for c in range(-(-n // 16)):
                whole = c * 16 >= sinks and (c + 1) * 16 <= n - window
                assert (row[c] < 0) == whole
        held = [x for x in t.block_table.flatten().tolist() if x >= 0]
        assert len(held) == len(set(held)) == 60 - t.free_pages
    t.release(0), t.release(1)
    assert t.free_pages == 60
    for kw in (dict(window=0), dict(window=3, sinks=-1)):
        with pytest.raises(ValueError):
            t.slide(**kw)


def test_a_cache_with_a_window():
    t = table()
    for kw in (dict(window=0), dict(sinks=2), dict(window=2, sinks=-1)):
        with pytest.raises(ValueError):
            pc.PagedKVCache(t, 2, 64, **kw)
    c = pc.PagedKVCache(t, 2, 64, tracked=True, window=30, sinks=4)
    with pytest.raises(ValueError):
        c.evict(20)
    t.admit_prefix(10)
    k = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    for kw in (dict(prefix=1), dict(prefix=0, start=6), dict(prefix=0, start=-1), dict(prefix=2)):
        with pytest.raises(ValueError):
            c.store_prefix(k=k, v=k, **kw)
    assert c.store_prefix(0, k, k) is None  # (in range: declined, off the GPU)
    assert c.attention(torch.zeros(3, 4, 64, dtype=torch.bfloat16)) is None


def test_the_prefix_block_is_the_one_that_is_packed():
    assert ctypes.sizeof(_lib.PagedPrefix) == pc._PREFIX.size
    values = list(range(1, 7))
    block = _lib.PagedPrefix.from_buffer_copy(pc._PREFIX.pack(*values))
    assert [getattr(block, name) for name, _ in _lib.PagedPrefix._fields_] == values


def _window(lib, c, **kw):
    a = dict(Q=P, qs=1024, SLOT=P, Y=P, nh=8, scale=0.1, window=5, sinks=2, work=P)
    a.update(kw)
    return lib.ttsp_paged_attention_window(_at(c), *a.values(), None)


def _prefix(lib, c, pre=None, **kw):
    a = dict(Q=P, qs=1024, SLOT=P, Y=P, nh=8, scale=0.1, window=0, sinks=0, work=P)
    a.update(kw)
    pre = _lib.PagedPrefix(**{**dict(table=P, SLOT=P, OF=P, table_stride=4, count=2, cols=4), **(pre or {})})
    return lib.ttsp_paged_attention_prefix(_at(c), ctypes.byref(pre), *a.values(), None)


BAD = [dict(Q=None), dict(Q=P + 8), dict(qs=1020), dict(qs=1016), dict(SLOT=None), dict(Y=None), dict(Y=P + 2), dict(nh=0), dict(nh=7),
       dict(nh=65540), dict(sinks=-1), dict(window=-1)]


@pytest.mark.parametrize("kw", BAD + [dict(window=0), dict(work=None), dict(work=P + 4)])
def test_bad_windows_are_refused(kw):
    lib = _lib.load()
    assert _window(lib, _cache(), **kw) == 1
    assert _window(lib, _cache(K=None)) == 1 and _window(lib, None) == 1


@pytest.mark.parametrize("kw", BAD + [dict(work=None), dict(work=P + 8)])
def test_bad_calls_over_prefixes_are_refused(kw):
    lib = _lib.load()
    assert _prefix(lib, _cache(scores=None, slot_pos=None), **kw) == 1


@pytest.mark.parametrize("pre", [dict(table=None), dict(table=P + 2), dict(SLOT=None), dict(SLOT=P + 4), dict(OF=None), dict(OF=P + 1),
                                 dict(count=0), dict(count=257), dict(cols=0), dict(cols=5), dict(cols=(1 << 20) + 1, table_stride=1 << 21)])
def test_bad_prefixes_are_refused(pre):
    lib = _lib.load()
    assert _prefix(lib, _cache(), pre=pre) == 1
    assert lib.ttsp_paged_attention_prefix(_at(_cache()), None, P, 1024, P, P, 8, 0.1, 0, 0, P, None) == 1


def test_workspace_queries():
    lib = _lib.load()
    w, x = lib.ttsp_paged_attention_window_work_kib, lib.ttsp_paged_attention_prefix_work_kib
    assert w(4, 8, 2, 128, 100, 16, 100, 4, 0) == 0 and w(4, 8, 2, 128, 100, 16, 2000, 4, 0) > 0
    assert w(4, 8, 2, 128, 100, 16, 100, 4, 1) > 0
    for bad in ((4, 8, 2, 128, 100, 16, 0, 4, 0), (4, 8, 2, 128, 100, 16, 5, -1, 0), (65536, 8, 2, 128, 1, 16, 5, 1, 0)):
        assert w(*bad) == -1
    assert x(4, 8, 2, 128, 100, 16, 2, 50, 0, 0, 0) > 0
    big = 2**31 - 1
    for bad in ((4, 8, 2, 128, 100, 16, 0, 50, 0, 0, 0), (4, 8, 2, 128, 100, 16, 257, 50, 0, 0, 0), (4, 8, 2, 128, 100, 16, 2, 0, 0, 0, 0),
                (4, 8, 2, 128, 100, 16, 2, (1 << 20) + 1, 0, 0, 0), (4, 8, 2, 128, 100, 16, 2, 5, -1, 0, 0), (65535, 256, 1, 64, 1, 16, 1, 1, 0, 0, 0),
                (65535, 128, 1, 64, 1, 16, 256, 1 << 20, 0, 0, 0), (big,) * 8 + (0, 0, 0), (big,) * 11):
        assert x(*bad) == -1, bad
    with pytest.raises(ValueError):
        pc.attention_work(4, 8, 2, 128, 100, 16, prefixes=300, prefix_columns=4)


def test_window_masks():
    pos = torch.tensor([0, 5, 9, 30, -1])
    m = fastpath.window_mask(pos, 12, 3, 2)
    assert m.shape == (1, 1, 5, 12)
    for i, p in enumerate(pos.tolist()):
        assert m[0, 0, i].tolist() == [j <= p and (j < 2 or j > p - 3) for j in range(12)]


@pytest.mark.parametrize("kw", [dict(Q=None), dict(K=None), dict(pos=None), dict(Y=P + 2), dict(Q=P + 8), dict(pos=P + 4), dict(qs=4),
                                dict(kh=-8), dict(S=0), dict(S=(1 << 20) + 1), dict(nh=7), dict(nh=0), dict(nh=65544), dict(L=0), dict(window=0),
                                dict(sinks=-1), dict(dtype=2), dict(splits=0), dict(splits=17), dict(splits=2, work=None),
                                dict(splits=2, work=P + 8), dict(ks=1 << 24, L=1 << 10), dict(vs=1 << 30, L=3)])
def test_bad_windowed_prompts_are_refused(kw):
    a = dict(Q=P, qs=1024, qh=128, K=P, ks=128, kh=4096, V=P, vs=128, vh=4096, pos=P, Y=P, S=20, nh=8, nkv=2, L=30, window=5, sinks=1,
             scale=0.1, dtype=1, work=P, splits=1)
    a.update(kw)
    assert _lib.load().ttsp_prefill_attention_window(*a.values(), None) == 1


def test_splits_of_windowed_prompts():
    f = _lib.load().ttsp_prefill_attention_window_splits
    assert f(9, 32, 8, 2000, 1024, 4) == 8 and f(512, 32, 8, 2512, 1024, 4) == 1 and f(8000, 32, 8, 8000, 2048, 16) == 1
    assert f(9, 32, 8, 300, 1024, 4) == 1 and f(1, 1, 1, 1 << 20, 1 << 20, 0) == 16
    assert f(0, 8, 2, 10, 5, 0) == f(4, 1, 2, 10, 5, 0) == f(4, 8, 2, 10, 0, 0) == 1
    with pytest.raises(ValueError):
        fastpath.prefill_attention(torch.zeros(1), None, None, None, 8, 2, 128, window=5)
