"""The paged cache's refusals and host parts (no GPU calls), beside `test_paged.py`."""

from __future__ import annotations

import pytest

from tests.test_paged import _attention, _cache, _evict, _rope, _store
from ttspipe_amd import _lib


@pytest.mark.parametrize("kw", [dict(score_seq=64), dict(score_seq=192), dict(score_head=63), dict(pos_seq=64, pos_head=65),
                                dict(score_seq=100, score_head=100), dict(pos_seq=255, pos_head=64),
                                dict(score_seq=1 << 62, score_head=(1 << 62) - 1)])
def test_scores_and_positions_of_several_heads_in_one_place_are_refused(kw):
    """(sequence, head) pairs whose words overlap: two sequences of four heads of 64 slots."""
    lib, c = _lib.load(), _cache(**kw)
    for call in (_rope, _store, _attention, _evict):
        assert call(lib, c) == 1


def test_scores_whose_heads_lie_apart_are_taken():
    lib = _lib.load()
    for kw in (dict(score_seq=64, score_head=128), dict(pos_seq=70, pos_head=140), dict(score_head=1000, score_seq=64),
               dict(score_seq=3 * 80 + 64, score_head=80), dict(seqs=1, score_seq=0, pos_seq=5),
               dict(n_kv=1, score_head=0, pos_head=3)):
        c = _cache(**kw)
        assert _evict(lib, c, budget=64) == 0 and _rope(lib, c, rows=0, rs=4096) == 0  # (nothing to launch)
