"""The paged cache's refusals and host parts (no GPU calls), beside `test_paged.py`."""

from __future__ import annotations

import pytest
import torch

from tests.test_paged import _attention, _cache, _evict, _rope, _store
from ttspipe_amd import _lib
from ttspipe_amd import pagedcache as pc


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


def test_workspace_queries_of_sizes_that_no_call_takes():
    lib = _lib.load()
    for seqs, nh, nkv, hd, cols, page, tracked in (
            (65535, 256, 1, 64, 1, 16, 0), (65535, 4096, 8, 128, 1, 16, 0), (20000, 840, 1, 128, 100, 16, 0),  # workgroups
            (1, 65535, 1, 64, 1 << 20, 16, 1),  # 4 TiB of scores
            (65535, 1, 1, 64, 1 << 20, 16, 0), (1, 1, 1, 64, (1 << 20) + 1, 16, 0), (65536, 1, 1, 64, 1, 16, 0),
            (1, 65536, 1, 64, 1, 16, 0), (1, 1, 1, 256, 1, 16, 0), (1, 5000, 5000, 64, 1, 16, 0), *[(2**31 - 1,) * 6 + (t,) for t in (0, 1)],
            (2**31 - 1, 2**31 - 1, 1, 128, 2**31 - 1, 16, 1)):
        assert lib.ttsp_paged_attention_work_kib(seqs, nh, nkv, hd, cols, page, tracked) == -1, (seqs, nh, cols)
        with pytest.raises(ValueError):
            pc.attention_work(seqs, nh, nkv, hd, cols, page, bool(tracked))
    assert lib.ttsp_paged_attention_work_kib(65535, 128, 1, 64, 1, 16, 0) == 0
    for seqs, nkv, cols, page, budget in ((65536, 1, 64, 16, 5), (1, 4097, 64, 16, 5), (1, 1, (1 << 20) + 1, 16, 5),
                                          (2**31 - 1, 2**31 - 1, 2**31 - 1, 2**31 - 1, 5)):
        assert lib.ttsp_paged_evict_work_kib(seqs, nkv, cols, page, budget) == -1, (seqs, nkv, cols)


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.to(torch.float16), lambda m: m.to("cpu", torch.float16)])
def test_a_cast_cache_keeps_its_scores_in_32_bits(cast):
    """(In 16 bits every call on the cache would be declined.)"""
    c = pc.PagedKVCache(pc.PageTable(2, 40, 5, 16, device="cpu"), 2, 64, tracked=True)
    c.scores.copy_(torch.rand(c.scores.shape))
    want = c.scores.clone()
    assert cast(c) is c
    assert c.k_pages.dtype is c.v_pages.dtype is torch.float16 and c.slot_pos.dtype is torch.int32
    assert c.scores.dtype is torch.float32 and torch.equal(c.scores, want) and "scores" in dict(c.named_buffers())
    plain = cast(pc.PagedKVCache(c.table, 2, 64))
    assert plain.scores is None and plain.k_pages.dtype is torch.float16


def test_a_position_past_the_rotary_table_is_refused_before_its_row_is_left_out():
    t = pc.PageTable(2, 64, 8, 16, device="cpu")
    c = pc.PagedKVCache(t, 2, 64)
    t.admit(30)
    qkv = torch.zeros(2, 8 * 64, dtype=torch.bfloat16)
    for n in (0, 29):
        with pytest.raises(ValueError):
            c.qk_rope_kv(qkv, 4, torch.zeros(n, 32, 2))
    assert c.qk_rope_kv(qkv, 4, torch.zeros(30, 32, 2)) is None  # (in range: declined, off the GPU)
