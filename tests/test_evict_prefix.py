"""Eviction behind a prefix on the host (no GPU calls): the first positions that
`PageTable` keeps on the device, and what the C entry refuses before any launch."""

from __future__ import annotations

import pytest
import torch

from tests.test_paged import P, _at, _cache
from ttspipe_amd import _lib
from ttspipe_amd import pagedcache as pc


def test_first_positions_follow_the_sequences():
    t = pc.PageTable(3, 100, 30, 16, device="cpu", prefixes=2, max_prefix=50)
    assert t.starts.dtype is torch.int64 and t.starts.tolist() == [0, 0, 0]
    a, b = t.admit_prefix(33), t.admit_prefix(50)
    t.admit(5, prefix=a), t.admit(7), t.admit(9, prefix=b)
    kept = t.starts
    assert kept.tolist() == [33, 0, 50]
    t.step()
    assert kept.tolist() == [t.first_position(i) for i in range(3)] == [33, 0, 50]
    t.evicted(4)
    t.release(0)
    assert kept.tolist() == [0, 0, 50]
    t.release(1)
    assert t.admit(3, prefix=b) == 0 and t.admit(1, prefix=a) == 1
    assert kept.tolist() == [50, 33, 50] and t.starts is kept  # (a captured call's tensor)
    assert pc.PageTable(3, 100, 30, 16, device="cpu").starts is None


def _evict(lib, c, **kw):
    a = dict(SLOT=P, POS=P, FIRST=P, budget=20, sinks=2, recent=3, work=P)
    a.update(kw)
    return lib.ttsp_paged_evict_from(_at(c), *a.values(), None)


@pytest.mark.parametrize("kw", [dict(SLOT=None), dict(POS=None), dict(FIRST=P + 4), dict(budget=0), dict(sinks=-1), dict(recent=-1),
                                dict(sinks=10, recent=11)])
def test_bad_calls_are_refused_before_any_launch(kw):
    lib = _lib.load()
    assert _evict(lib, _cache(), **kw) == 1
    assert _evict(lib, None) == 1 and _evict(lib, _cache(scores=None)) == 1 and _evict(lib, _cache(slot_pos=None)) == 1
    assert _evict(lib, _cache(), budget=64, work=None) == 0  # nothing to do: no launch
