"""The paged cache on the host (no GPU calls): what the C entries refuse before
any launch, the kernels' own index checks, the mirrored argument block, the
calls' declines without a GPU, and `PageTable`'s account of pages and rows."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from ttspipe_amd import _lib
from ttspipe_amd import pagedcache as pc

ROOT = Path(__file__).resolve().parent.parent
P = 1 << 20  # an address that is aligned and never followed: every call here is refused first


def _cache(**kw):
    base = dict(K=P, V=P, table=P, scores=P, slot_pos=P, k_page=8192, k_head=2048, k_row=128, v_page=8192, v_head=2048,
                v_row=128, table_stride=4, score_seq=256, score_head=64, pos_seq=256, pos_head=64, seqs=2, cols=4, pages=9,
                page_size=16, n_kv=4, head_dim=128, dtype=_lib.DT_BF16)
    return _lib.PagedCache(**{**base, **kw})


def _at(c):
    return None if c is None else ctypes.byref(c)


BAD_CACHES = [dict(K=None), dict(V=None), dict(table=None), dict(K=P + 8), dict(V=P + 2), dict(table=P + 1), dict(k_page=-8),
              dict(k_head=4), dict(v_row=129), dict(k_row=(1 << 24) + 8), dict(v_row=1 << 30), dict(table_stride=3), dict(seqs=0), dict(seqs=65536), dict(cols=0),
              dict(pages=0), dict(page_size=8), dict(page_size=24), dict(page_size=8192), dict(page_size=0), dict(n_kv=0),
              dict(n_kv=5000), dict(head_dim=96), dict(head_dim=256), dict(dtype=_lib.DT_F32), dict(dtype=7),
              dict(cols=(1 << 24) // 16 + 1, table_stride=1 << 30), dict(scores=P + 2), dict(score_seq=-1),
              dict(slot_pos=P + 1), dict(pos_head=-4)]


def _rope(lib, c, **kw):
    a = dict(QKV=P, rs=1536, QW=P, KW=P, eps=1e-6, F=P, ftype=1, n=10, POS=P, SEQ=P, SLOT=P, Q=P, nh=4, rows=3, **{})
    a.update(kw)
    return lib.ttsp_paged_qk_rope_kv(_at(c), *(a[k] for k in ("QKV", "rs", "QW", "KW", "eps", "F", "ftype", "n", "POS", "SEQ",
                                                         "SLOT", "Q", "nh", "rows")), None)


def _store(lib, c, **kw):
    a = dict(K=P, krs=512, khs=128, V=P, vrs=512, vhs=128, POS=P, SEQ=P, SLOT=P, rows=3)
    a.update(kw)
    return lib.ttsp_paged_store(_at(c), *a.values(), None)


def _attention(lib, c, **kw):
    a = dict(Q=P, qs=1024, SLOT=P, Y=P, nh=8, scale=0.1, work=P)
    a.update(kw)
    return lib.ttsp_paged_attention(_at(c), *a.values(), None)


def _evict(lib, c, **kw):
    a = dict(SLOT=P, POS=P, budget=20, sinks=2, recent=3, work=P)
    a.update(kw)
    return lib.ttsp_paged_evict(_at(c), *a.values(), None)


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda b: next(iter(b)) + str(next(iter(b.values()))))
def test_bad_caches_are_refused_before_any_launch(bad):
    lib = _lib.load()
    c = _cache(**bad)
    for call in (_rope, _store, _attention, _evict):
        assert call(lib, c) == 1
    for call in (_rope, _store, _attention, _evict):
        assert call(lib, None) == 1


def test_bad_arguments_are_refused_before_any_launch():
    lib, c = _lib.load(), _cache()
    for kw in (dict(QKV=None), dict(QKV=P + 2), dict(rs=1535), dict(rs=1528), dict(F=None), dict(F=P + 4), dict(ftype=3),
               dict(ftype=-1), dict(n=0), dict(SLOT=None), dict(Q=None), dict(Q=P + 8), dict(nh=0), dict(nh=5000), dict(rows=-1),
               dict(rows=(1 << 24) + 1), dict(QW=P + 2), dict(KW=P + 8), dict(POS=None), dict(SEQ=None)):
        assert _rope(lib, c, **kw) == 1, kw
    no_pos = _cache(slot_pos=None)
    assert _rope(lib, no_pos, POS=None, n=2) == 1  # fewer rotary rows than rows
    for kw in (dict(K=None), dict(V=None), dict(K=P + 8), dict(V=P + 4), dict(krs=-8), dict(khs=4), dict(vrs=3), dict(vhs=-1),
               dict(POS=None), dict(SEQ=None), dict(SLOT=None), dict(rows=-2), dict(rows=1 << 25)):
        assert _store(lib, c, **kw) == 1, kw
    for kw in (dict(Q=None), dict(Q=P + 2), dict(qs=1023), dict(qs=1016), dict(SLOT=None), dict(Y=None), dict(Y=P + 8), dict(nh=0),
               dict(nh=6), dict(nh=65540)):
        assert _attention(lib, c, **kw) == 1, kw
    for big in (_cache(cols=100, table_stride=100, scores=None), c):  # partial sums, or scores to gather
        for kw in (dict(work=None), dict(work=P + 4)):
            assert _attention(lib, big, **kw) == 1, kw
    for kw in (dict(SLOT=None), dict(POS=None), dict(budget=0), dict(budget=-3), dict(sinks=-1), dict(recent=-1),
               dict(sinks=10, recent=11), dict(sinks=2**31 - 1, recent=2**31 - 1)):
        assert _evict(lib, c, **kw) == 1, kw
    wide = _cache(cols=100, table_stride=100)
    for kw in (dict(work=None, budget=800), dict(work=P + 2, budget=800)):
        assert _evict(lib, wide, **kw) == 1, kw
    for kw in (dict(score_seq=0), dict(pos_seq=0), dict(score_head=0), dict(pos_head=0)):  # one row for several
        assert _evict(lib, _cache(**kw)) == 1, kw
    assert _evict(lib, _cache(scores=None)) == 1 and _evict(lib, _cache(slot_pos=None)) == 1
    # nothing to do: no launch either
    assert _rope(lib, c, rows=0) == 0 and _store(lib, c, rows=0) == 0
    assert _evict(lib, c, budget=64, work=None) == 0 and _evict(lib, c, budget=1 << 24, work=None) == 0


def test_calls_of_more_workgroups_than_a_launch_counts_are_refused_before_it():
    lib, c = _lib.load(), _cache()
    rows, rs = 1 << 24, 4096 * 128 + 8 * 128
    assert _rope(lib, c, rows=rows, nh=64, rs=rs) == 1 and _rope(lib, c, rows=rows, nh=4096, rs=rs) == 1
    assert _store(lib, _cache(n_kv=16), rows=rows) == 1
    assert _attention(lib, _cache(seqs=65535, scores=None, pages=1 << 20), nh=512, qs=512 * 128) == 1


def test_attention_refuses_scores_that_several_share():
    lib = _lib.load()
    for kw in (dict(score_seq=0), dict(score_head=0)):
        assert _attention(lib, _cache(**kw)) == 1, kw


def test_workspace_queries():
    lib = _lib.load()
    assert pc.attention_work(1, 1, 1, 64, 1, 16) >= 0
    assert lib.ttsp_paged_attention_work_kib(0, 8, 2, 128, 4, 16, 0) == 0
    assert lib.ttsp_paged_attention_work_kib(65535, 4096, 1, 128, 1 << 20, 16, 1) == -1
    with pytest.raises(ValueError):
        pc.attention_work(65535, 4096, 1, 128, 1 << 20, 16, True)
    assert pc.evict_work(3, 2, 4, 16, 64) == 0 and pc.evict_work(3, 2, 4, 16, 20) == 0
    assert pc.evict_work(3, 2, 100, 16, 1300) >= 3 * 2 * (1 + 2 * 300) and pc.evict_work(1, 1, 100, 16, 257) >= 515
    assert lib.ttsp_paged_evict_work_kib(65535, 4096, 1 << 20, 16, 1 << 23) == -1


def test_the_kernels_index_checks(tmp_path):
    """`Paged::page` and `Paged::rows`, which every kernel's addresses go
    through, on table entries, slots and lengths of every kind (compiled for
    the host)."""
    src = tmp_path / "check.hip"
    src.write_text('''
#include <cstdio>
#include <climits>
#include "paged_common.h"
using namespace ttsp;
int main() {
  int table[2][6] = {{3, -1, 4, 5, INT_MIN, 0}, {INT_MAX, 2, -2, 1, 4, 7}};
  ttsp_paged_cache c{};
  c.K = c.V = (void*)4096;
  c.table = &table[0][0];
  c.k_page = c.v_page = 4096, c.k_head = c.v_head = 2048, c.k_row = c.v_row = 128;
  c.table_stride = 6, c.seqs = 2, c.cols = 5, c.pages = 5, c.page_size = 16, c.n_kv = 2, c.head_dim = 128, c.dtype = 1;
  Paged p;
  if (!paged_args(&c, &p)) return 2;
  for (int b = 0; b < 2; ++b)
    for (int j = 0; j < p.cap(); j += 15) printf("%d ", p.page(b, j));
  printf("| ");
  for (long long s : {LLONG_MIN, -2LL, -1LL, 0LL, 14LL, 78LL, 79LL, 80LL, 1LL << 31, 1LL << 32, LLONG_MAX}) printf("%d ", p.rows(s));
  printf("\\n");
}''')
    exe = tmp_path / "check"
    subprocess.run(["/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "-std=c++17", "-O1",
                    f"-I{ROOT / 'ttspipe_amd' / 'csrc'}", str(src), "-o", str(exe)], check=True, capture_output=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("|")
    pages = [3, -1, 4, -1, -1], [-1, 2, -1, 1, 4]
    assert [int(x) for x in out[0].split()] == [pages[b][j // 16] for b in range(2) for j in range(0, 80, 15)]
    assert [int(x) for x in out[1].split()] == [0, 0, 0, 1, 15, 79, 80, 80, 80, 80, 80]


def test_the_argument_block_matches_the_header(tmp_path):
    names = [n for n, _ in _lib.PagedCache._fields_]
    src = tmp_path / "layout.c"
    src.write_text("#define TTSP_HIP_TYPES_ONLY\n#include <stddef.h>\n#include <stdio.h>\n#include \"ttsp_hip.h\"\nint main(void) {"
                   + "".join(f'printf("%zu ", offsetof(ttsp_paged_cache, {n}));' for n in names)
                   + 'printf("%zu %d", sizeof(ttsp_paged_cache), TTSP_PAGED_MAX_SLOTS); return 0; }')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert pc._BLOCK.size == ctypes.sizeof(_lib.PagedCache)  # the calls pack the block by itself
    block = _lib.PagedCache.from_buffer_copy(pc._BLOCK.pack(*range(1, len(names) + 1)))
    assert [getattr(block, n) for n in names] == list(range(1, len(names) + 1))
    assert got == [getattr(_lib.PagedCache, n).offset for n in names] + [ctypes.sizeof(_lib.PagedCache), _lib.PAGED_MAX_SLOTS]


def test_calls_decline_tensors_off_the_gpu():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    t, s = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    sc, sp = torch.zeros(2, 2, 32), torch.zeros(2, 2, 32, dtype=torch.int32)
    assert pc.attention(torch.zeros(2, 4, 64, dtype=torch.bfloat16), k, k, t, s) is None
    assert pc.store(k[:2, :, 0], k[:2, :, 0], k, k, t, s) is None
    assert pc.qk_rope_kv(torch.zeros(2, 8 * 64, dtype=torch.bfloat16), 4, k, k, t, s, torch.zeros(9, 32, 2), s) is None
    assert pc.evict(k, k, t, s, sc, sp, s, 8) is None


@pytest.mark.parametrize("kw", [dict(budget=0), dict(budget=4, sinks=-1), dict(budget=4, recent=-1),
                                dict(budget=4, sinks=2, recent=3), dict(budget=(1 << 24) + 1)])
def test_bad_budgets_raise(kw):
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        pc.evict(k, k, None, None, None, None, None, **kw)


# ------------------------------------------------------------------ PageTable


def _consistent(t):
    """Every page is free or held once, the device table says what the host holds, and the slots fit."""
    held = [p for row in t._held for p in row]
    assert sorted(held + t._free) == list(range(t.pages))
    for i, row in enumerate(t._held):
        assert t.block_table[i].tolist() == row + [-1] * (t.block_table.shape[1] - len(row))
        assert len(row) * t.page_size >= t.rows(i) == int(t.slots[i]) + 1


def test_page_table_hands_pages_out_and_takes_them_back():
    t = pc.PageTable(3, 100, 12, 16, device="cpu")
    assert t.block_table.shape == (3, 7)
    a, b = t.admit(33), t.admit(16)
    assert (a, b) == (0, 1) and t.free_pages == 12 - 3 - 1
    assert t.slots.tolist() == [32, 15, -1] and t.positions.tolist() == [32, 15, -1]
    _consistent(t)
    t.step()
    assert t.slots.tolist() == [33, 16, -1] and t.free_pages == 12 - 3 - 2  # b's 17th row: a page
    _consistent(t)
    for _ in range(20):
        t.step()
    assert t.rows(0) == 54 and t.rows(1) == 37
    t.evicted(40)  # the 41st row's page stays
    assert t.slots.tolist() == [39, 36, -1] and t.positions.tolist() == [53, 36, -1] and len(t._held[0]) == 3
    _consistent(t)
    t.step()
    assert t.slots.tolist() == [40, 37, -1] and t.positions.tolist() == [54, 37, -1]
    t.release(0)
    assert t.slots.tolist() == [-1, 37, -1]
    _consistent(t)
    assert t.admit(1) == 0 and t.admit(2) == 2 and t.admit(1) is None
    _consistent(t)


def test_page_table_refuses_what_does_not_fit():
    for kw in (dict(page_size=8), dict(page_size=48), dict(page_size=8192), dict(seqs=0), dict(pages=0), dict(max_len=0)):
        with pytest.raises(ValueError):
            pc.PageTable(**{**dict(seqs=2, max_len=64, pages=5, page_size=16, device="cpu"), **kw})
    t = pc.PageTable(3, 64, 5, 16, device="cpu")
    for rows in (0, 65):
        with pytest.raises(ValueError):
            t.admit(rows)
    assert t.admit(48) == 0 and t.admit(17) == 1
    with pytest.raises(MemoryError):
        t.admit(1)
    _consistent(t)
    before = t.slots.tolist()
    with pytest.raises(MemoryError):  # sequence 0 needs a page
        t.step()
    assert t.slots.tolist() == before
    _consistent(t)
    t.release(1)
    for _ in range(16):
        t.step()
    with pytest.raises(ValueError):  # 64 rows are the table's width
        t.step()
    _consistent(t)


def test_page_table_keeps_at_least_a_row_of_each_sequence():
    t = pc.PageTable(2, 64, 8, 16, device="cpu")
    t.admit(20)
    for budget in (0, -1):
        with pytest.raises(ValueError):
            t.evicted(budget)
    assert t.rows(0) == 20 and t.slots.tolist() == [19, -1]
    _consistent(t)


def test_page_table_keeps_positions_below_their_end():
    with pytest.raises(ValueError):
        pc.PageTable(1, 64, 4, 16, device="cpu", max_position=0)
    t = pc.PageTable(2, 64, 8, 16, device="cpu", max_position=20)
    with pytest.raises(ValueError):
        t.admit(21)
    assert t.admit(18) == 0 and t.positions_used == 18
    t.step()
    t.evicted(10)
    t.step()
    assert t.rows(0) == 11 and t.positions.tolist() == [19, -1] and t.positions_used == 20
    with pytest.raises(ValueError):
        t.step()
    assert t.positions.tolist() == [19, -1] and t.rows(0) == 11
    _consistent(t)
    t.release(0)
    assert t.positions_used == 0 and t.admit(20) == 0


def test_paged_cache_shapes():
    t = pc.PageTable(3, 100, 12, 16, device="cpu")
    c = pc.PagedKVCache(t, 2, 64, dtype=torch.float16, tracked=True)
    assert c.k_pages.shape == c.v_pages.shape == (12, 2, 16, 64) and c.scores.shape == c.slot_pos.shape == (3, 2, 112)
    plain = pc.PagedKVCache(t, 2)
    assert plain.scores is None and plain.k_pages.shape == (12, 2, 16, 128)
    with pytest.raises(ValueError):
        plain.evict(20)
    for seq in (0, -1, 3):
        with pytest.raises(ValueError):
            c.store(seq, torch.zeros(1, 2, 64), torch.zeros(1, 2, 64))
    for seq in (-1, 3):
        with pytest.raises(ValueError):
            t.release(seq)
