"""Streams that decode together: a paged key-value cache, and the attention,
writes and eviction that work on it.

The reference decodes one sequence over one contiguous cache
(app/engine/fusedlayer.py:162-306); a server of several streams keeps their
keys and values in pages of one pool instead, so that a stream takes the pages
it needs and gives them back. For D-wide heads (64 or 128) and 16-bit caches:

* pools `k_pages`, `v_pages` (pages, n_local_heads, page size, D), the last
  axis contiguous, any other strides that keep rows 16-byte aligned and
  apart; the page size a power of two from 16 to 4096;
* `block_table` int32 (sequences, columns): row b names sequence b's pages, and
  slot j of the sequence is row j % page size of its page j // page size. An
  entry that is no page of the pool (-1) is a hole: its slots do not exist;
* `slots` int64 (sequences,): the newest slot of each sequence, -1 for one that
  holds nothing;
* `scores` fp32 and `slot_pos` int32 (sequences, n_local_heads, columns * page
  size), where a cache is evicted from: the attention weight each slot has
  gathered and the position its row came from; a head's slots contiguous, any
  strides that keep the heads apart.

`qk_rope_kv` and `store` write rows, `attention` reads them, `evict` cuts a
sequence down to a budget. `PageTable` hands the pages out and keeps the device
tensors above; `PagedKVCache` is one layer's pools with the four calls as
methods; `fusedlayer.decode_batch` runs a transformer block on them.

As elsewhere in the package a call the kernels cannot take returns None (and is
counted in `stats()`), a wrong `out`, `work` or budget raises ValueError and a
failed launch RuntimeError. Work is queued on the current stream of the
tensors' device; nothing is synchronised, and with `out=` and `work=` given
nothing is allocated, so that calls can be captured. Calls that may overlap
(two streams, two graphs) need workspaces of their own. These are calls of a
decode: they have no gradients.
"""

from __future__ import annotations

import functools
import struct

import torch
from torch import nn

from ttspipe_amd import _lib

#: Head dims, and bounds of the page size (a power of two).
HEAD_DIMS = (64, 128)
MIN_PAGE, MAX_PAGE = 16, 4096

_stats = {"rows": 0, "attention": 0, "evict": 0, "declined": 0}


def stats() -> dict:
    return dict(_stats)


def _declined():
    _stats["declined"] += 1


#: `ttsp_paged_cache`'s fields in order (`_lib.PagedCache` names them).
_BLOCK = struct.Struct("@5P11q7i4x")


def _strides_ok(s, nkv, pages, hd) -> bool:
    return (s[3] == 1 and not (s[0] % 8 or s[1] % 8 or s[2] % 8) and hd <= s[2] <= _lib.PAGED_MAX_ROW_STRIDE
            and (nkv == 1 or s[1] >= hd) and (pages == 1 or s[0] >= hd))


def _words_ok(s0, s1, last, seqs, nkv, cap) -> bool:
    """Whether the cap words of every (sequence, head) are contiguous and lie apart, by their strides."""
    if last != 1 or (seqs > 1 and s0 < cap) or (nkv > 1 and s1 < cap):
        return False
    return seqs == 1 or nkv == 1 or s0 >= (nkv - 1) * s1 + cap or s1 >= (seqs - 1) * s0 + cap


def _pool(k_pages, v_pages, block_table, scores=None, slot_pos=None):
    """(the C-ABI's argument block, n_kv, page size, head dim, sequences, columns,
    the cache's dtype, its device's index) of these tensors, or None where the
    kernels do not take them. On every call's host path: plain integers, each
    tensor asked for a thing once."""
    dev, dtype, shape, table = k_pages.get_device(), k_pages.dtype, k_pages.shape, block_table.shape
    if dtype is torch.bfloat16:
        dt = _lib.DT_BF16
    elif dtype is torch.float16:
        dt = _lib.DT_F16
    else:
        return None
    if (dev < 0 or v_pages.get_device() != dev or block_table.get_device() != dev or v_pages.dtype is not dtype
            or block_table.dtype is not torch.int32 or len(shape) != 4 or len(table) != 2 or v_pages.shape != shape):
        return None
    pages, nkv, page, hd = shape
    seqs, cols = table
    if (hd not in HEAD_DIMS or not MIN_PAGE <= page <= MAX_PAGE or page & (page - 1) or not pages or not 1 <= nkv <= 4096
            or not 1 <= seqs <= 65535 or not 1 <= cols <= _lib.PAGED_MAX_SLOTS // page):
        return None
    ks, vs, (t0, t1) = k_pages.stride(), v_pages.stride(), block_table.stride()
    if not _strides_ok(ks, nkv, pages, hd) or (vs != ks and not _strides_ok(vs, nkv, pages, hd)):
        return None
    kp, vp = k_pages.data_ptr(), v_pages.data_ptr()
    if kp % 16 or vp % 16 or (t1 != 1 and cols > 1) or (seqs > 1 and t0 < cols):
        return None
    scp = spp = sc0 = sc1 = sp0 = sp1 = 0
    cap = cols * page
    if scores is not None:
        if scores.dtype is not torch.float32 or scores.get_device() != dev or scores.shape != (seqs, nkv, cap):
            return None
        sc0, sc1, last = scores.stride()
        if not _words_ok(sc0, sc1, last, seqs, nkv, cap):
            return None
        scp = scores.data_ptr()
    if slot_pos is not None:
        if slot_pos.dtype is not torch.int32 or slot_pos.get_device() != dev or slot_pos.shape != (seqs, nkv, cap):
            return None
        sp0, sp1, last = slot_pos.stride()
        if not _words_ok(sp0, sp1, last, seqs, nkv, cap):
            return None
        spp = slot_pos.data_ptr()
    block = _BLOCK.pack(kp, vp, block_table.data_ptr(), scp, spp, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                        t0 if t0 > cols else cols, sc0 or 1, sc1, sp0 or 1, sp1, seqs, cols, pages, page, nkv, hd, dt)
    return block, nkv, page, hd, seqs, cols, dtype, dev


def _vector(t, dtype, n, dev) -> bool:
    """Whether `t` is a contiguous vector of n values of `dtype` on `dev`."""
    return t.dtype is dtype and t.dim() == 1 and t.numel() == n and t.is_contiguous() and t.get_device() == dev


def _launch(what, dev, *args):
    """`what` of the library on the current stream of device `dev`."""
    fn = getattr(_lib.lib(), what)
    if dev == torch._C._cuda_getDevice():
        rc = fn(*args, _lib.stream())
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _lib.stream())
    if rc:
        raise RuntimeError(f"{what} failed: hipError_t {rc}")


def _out_ok(out, shape, dtype, dev) -> bool:
    return (out.shape == shape and out.dtype is dtype and out.get_device() == dev and out.is_contiguous()
            and not out.data_ptr() % 16)


def _rows_ok(rows, width, seqs_of, slots, positions, seqs, dev) -> bool:
    # (a thread takes eight of a row's `width` elements, and a launch is counted in 32 bits)
    if rows > 1 << 24 or rows * width > 0xffffff << 11 or not _vector(slots, torch.int64, rows, dev):
        return False
    if positions is not None and not _vector(positions, torch.int64, rows, dev):
        return False
    return rows <= seqs if seqs_of is None else _vector(seqs_of, torch.int32, rows, dev)


def qk_rope_kv(qkv, n_head, k_pages, v_pages, block_table, slots, freqs_cis, positions=None, *, q_weight=None,
               k_weight=None, eps: float = 1e-6, seqs=None, scores=None, slot_pos=None, out=None):
    """New rows from the wqkv output: qkv (rows, (n_head + 2 n_local_heads) D),
    rows 16-byte aligned. Row t belongs to sequence `seqs[t]` (int32; None: to
    sequence t), slot `slots[t]` (int64). Its q and k heads are normed with
    `q_weight` / `k_weight` (None: no norm) and `eps` and rotated at
    `positions[t]` (int64; None: row t) of `freqs_cis` (positions, D / 2, 2),
    rounded once; k and v go to the slot, whose score becomes 0 and whose
    `slot_pos` becomes the position. Returns q (rows, n_head, D), in `out` if
    given, or None when declined.

    A row whose slot has no page (or lies outside the table: -1 for a padding
    row) is not written; a position outside `freqs_cis` makes its q zeros, too.
    No two rows may name one slot, and `out` must not overlap qkv. Without norms
    the result has the bits of the contiguous cache's kernel, which with norms
    also rounds between the two."""
    if not _lib.gpu_present():
        return _declined()
    c = _pool(k_pages, v_pages, block_table, scores, slot_pos)
    if c is None or qkv.dim() != 2:
        return _declined()
    block, nkv, _, hd, n_seqs, _, dtype, dev = c
    rows, width = qkv.shape
    step, last = qkv.stride()
    n_freqs, ftype = freqs_cis.shape[0] if freqs_cis.dim() == 3 else 0, _lib.dtype_code(freqs_cis.dtype)
    qp, fp = qkv.data_ptr(), freqs_cis.data_ptr()
    if (not 1 <= n_head <= 4096 or width != (n_head + 2 * nkv) * hd or qkv.dtype is not dtype or qkv.get_device() != dev or last != 1
            or (rows > 1 and (step < width or step % 8)) or qp % 16 or ftype is None or freqs_cis.get_device() != dev
            or not 0 < n_freqs < 1 << 31 or freqs_cis.shape != (n_freqs, hd // 2, 2) or not freqs_cis.is_contiguous()
            or fp % 16 or not _rows_ok(rows, width, seqs, slots, positions, n_seqs, dev)):
        return _declined()
    if positions is None and (n_freqs < rows or slot_pos is not None):
        return _declined()
    qw = kw = 0
    if q_weight is not None:
        qw = q_weight.data_ptr()
        if not _out_ok(q_weight, (hd,), dtype, dev):
            return _declined()
    if k_weight is not None:
        kw = k_weight.data_ptr()
        if not _out_ok(k_weight, (hd,), dtype, dev):
            return _declined()
    if out is None:
        out = qkv.new_empty((rows, n_head, hd))
    elif not _out_ok(out, (rows, n_head, hd), dtype, dev):
        raise ValueError("out must be a contiguous, 16-byte aligned (rows, n_head, head_dim) tensor of the cache's dtype")
    if rows:
        _launch("ttsp_paged_qk_rope_kv", dev, block, qp, step if rows > 1 else width, qw, kw, eps, fp, ftype, n_freqs,
                0 if positions is None else positions.data_ptr(), 0 if seqs is None else seqs.data_ptr(),
                slots.data_ptr(), out.data_ptr(), n_head, rows)
        _stats["rows"] += 1
    return out


def store(k, v, k_pages, v_pages, block_table, slots, *, positions=None, seqs=None, scores=None, slot_pos=None):
    """Finished rows into the pages: k, v (rows, n_local_heads, D), the last axis
    contiguous and rows 16-byte aligned (a contiguous cache's slice, transposed,
    is taken in place). `seqs`, `slots`, `positions` (needed with `slot_pos`) and
    the slots' scores as `qk_rope_kv`; positions are noted as 32-bit integers.
    True, or None when declined."""
    if not _lib.gpu_present():
        return _declined()
    c = _pool(k_pages, v_pages, block_table, scores, slot_pos)
    shape = k.shape
    if c is None or len(shape) != 3 or v.shape != shape:
        return _declined()
    block, nkv, _, hd, n_seqs, _, dtype, dev = c
    rows = shape[0]
    if (shape[1] != nkv or shape[2] != hd or k.dtype is not dtype or v.dtype is not dtype or k.get_device() != dev
            or v.get_device() != dev or not _rows_ok(rows, 2 * nkv * hd, seqs, slots, positions, n_seqs, dev)
            or (slot_pos is not None and positions is None)):
        return _declined()
    (kr, kh, kl), (vr, vh, vl) = k.stride(), v.stride()
    kp, vp = k.data_ptr(), v.data_ptr()
    if kl != 1 or vl != 1 or kr % 8 or kh % 8 or vr % 8 or vh % 8 or kp % 16 or vp % 16:
        return _declined()
    if rows:
        _launch("ttsp_paged_store", dev, block, kp, kr, kh, vp, vr, vh, 0 if positions is None else positions.data_ptr(),
                0 if seqs is None else seqs.data_ptr(), slots.data_ptr(), rows)
        _stats["rows"] += 1
    return True


@functools.lru_cache(maxsize=256)
def _attention_kib(seqs, n_head, n_local_heads, head_dim, columns, page_size, tracked) -> int:
    return _lib.lib().ttsp_paged_attention_work_kib(seqs, n_head, n_local_heads, head_dim, columns, page_size,
                                                    int(tracked))


def attention_work(seqs: int, n_head: int, n_local_heads: int, head_dim: int, columns: int, page_size: int,
                   tracked: bool = False) -> int:
    """fp32 elements of `attention`'s workspace; ValueError where `attention` declines sizes like these."""
    kib = _attention_kib(seqs, n_head, n_local_heads, head_dim, columns, page_size, tracked)
    if kib < 0:
        raise ValueError("too many heads or slots for one call, or the workspace would take more than 2 TiB")
    return kib * 256


def _workspace(work, need, dtype, like):
    """`work`, checked, or a new workspace of `need` elements on the device of `like` (None: none is needed)."""
    if work is None:
        return like.new_empty(need, dtype=dtype) if need else None
    if (work.dtype is not dtype or work.device != like.device or not work.is_contiguous() or work.numel() < need
            or work.data_ptr() % 16):
        raise ValueError(f"work must be a contiguous, 16-byte aligned {dtype} tensor of at least {need} elements")
    return work


def attention(q, k_pages, v_pages, block_table, slots, *, scale: float | None = None, scores=None, out=None,
              work=None):
    """One new token of each sequence over its cached rows: q (sequences, n_head,
    D), a sequence's heads contiguous, over slots 0 .. slots[b] (cut to the
    table's width), query head h with KV head h // (n_head / n_local_heads), the
    scores scaled by `scale` (D^-0.5). Returns (sequences, n_head, D), in `out`
    if given (which must not overlap q), or None when declined. A sequence
    without a row gives zeros; a row's infinities and NaN give what the formula gives, but for an infinite
    value in an fp16 cache, which may give NaN, and scores beyond 2e38, which
    count as infinite.

    With `scores`, each slot's weight, summed over the query heads of its KV
    head, is added to it (what `evict` ranks by). `work`: an fp32 workspace of
    `attention_work(...)` elements, else allocated per call; with `scores` it holds
    sequences * n_head * the table's slots, whatever the sequences hold."""
    if not _lib.gpu_present():
        return _declined()
    c = _pool(k_pages, v_pages, block_table, scores)
    shape = q.shape
    if c is None or len(shape) != 3:
        return _declined()
    block, nkv, page, hd, n_seqs, cols, dtype, dev = c
    seqs, nh, d = shape
    step, head_step, last = q.stride()
    qp = q.data_ptr()
    if (seqs != n_seqs or d != hd or nh < 1 or nh % nkv or nh > 65535 or q.dtype is not dtype or q.get_device() != dev
            or last != 1 or (nh > 1 and head_step != hd) or (seqs > 1 and (step < nh * hd or step % 8)) or qp % 16
            or not _vector(slots, torch.int64, seqs, dev)):
        return _declined()
    kib = _attention_kib(seqs, nh, nkv, hd, cols, page, scores is not None)
    if kib < 0:
        return _declined()
    if out is None:
        out = q.new_empty(shape)
    elif not _out_ok(out, shape, dtype, dev):
        raise ValueError("out must be a contiguous, 16-byte aligned (sequences, n_head, head_dim) tensor of q's dtype")
    work = _workspace(work, kib * 256, torch.float32, q)
    _launch("ttsp_paged_attention", dev, block, qp, step if seqs > 1 else nh * hd, slots.data_ptr(), out.data_ptr(), nh,
            hd**-0.5 if scale is None else scale, 0 if work is None else work.data_ptr())
    _stats["attention"] += 1
    return out


@functools.lru_cache(maxsize=256)
def evict_work(seqs: int, n_local_heads: int, columns: int, page_size: int, budget: int) -> int:
    """int32 elements of `evict`'s workspace."""
    kib = _lib.lib().ttsp_paged_evict_work_kib(seqs, n_local_heads, columns, page_size, budget)
    if kib < 0:
        raise ValueError("the workspace would take more than 2 TiB")
    return kib * 256


def evict(k_pages, v_pages, block_table, slots, scores, slot_pos, positions, budget: int, *, sinks: int = 0,
          recent: int = 0, work=None):
    """Cut every sequence of more than `budget` rows down to it, in place and in
    each KV head by itself: kept are rows of the first `sinks` positions and of
    the last `recent` ones (up to `positions[b]`, int64, the newest), then those
    of the largest scores (+inf is as good as protected, NaN counts as -inf), ties
    to the lowest slot. Rows that no step has attended to yet, a prompt's after
    `store`, have a score of 0: of those the lowest slots stay. A kept
    row below `budget` stays; the others move, in order, into the free slots
    below it with their score and position. Slots from `budget` on are left as
    they were, and so are `slots`: the caller's next slot is `budget`
    (`PageTable.evicted`). True, or None when declined.

    The pages of a sequence that is cut belong to it alone, and it has no holes up
    to its newest slot (as `PageTable` keeps it): a hole's slots would be ranked by
    what their scores hold, and a row that would move from or into one stays where
    it is, with its score and position. `work`: an int32
    workspace of `evict_work(...)` elements, else allocated per call."""
    if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget or budget > _lib.PAGED_MAX_SLOTS:
        raise ValueError("evict needs a budget of at least one row, 0 <= sinks, 0 <= recent and sinks + recent <= budget")
    if not _lib.gpu_present():
        return _declined()
    c = None if scores is None or slot_pos is None else _pool(k_pages, v_pages, block_table, scores, slot_pos)
    if c is None:
        return _declined()
    block, nkv, page, _, seqs, cols, _, dev = c
    if not _vector(slots, torch.int64, seqs, dev) or not _vector(positions, torch.int64, seqs, dev):
        return _declined()
    if cols * page > budget:  # else no sequence can be longer
        work = _workspace(work, evict_work(seqs, nkv, cols, page, budget), torch.int32, k_pages)
        _launch("ttsp_paged_evict", dev, block, slots.data_ptr(), positions.data_ptr(), budget, sinks, recent,
                0 if work is None else work.data_ptr())
    _stats["evict"] += 1
    return True


class PageTable:
    """Pages of the pools handed to sequences, and the device tensors that the
    calls read: `block_table`, `slots` and `positions` (the newest slot and
    position of each sequence, -1: none). One table serves every layer's pools.

    The host knows each sequence's row count and position without asking the
    device, and changes the tensors by work queued on the current stream, which it
    does not wait for: `admit` and `step` add rows, `evicted` cuts them, `release`
    drops them. Running out of pages raises MemoryError and changes nothing; so does,
    with ValueError, a row past `max_len` rows or past `max_position` positions
    (the rotary table's rows: a sequence that is evicted from runs on while its
    rows stay few; None: not checked here)."""

    def __init__(self, seqs: int, max_len: int, pages: int, page_size: int = 64, device="cuda",
                 max_position: int | None = None):
        if not MIN_PAGE <= page_size <= MAX_PAGE or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from {MIN_PAGE} to {MAX_PAGE}")
        if seqs < 1 or pages < 1 or max_len < 1 or (max_position is not None and max_position < 1):
            raise ValueError("seqs, max_len, pages and max_position must be positive")
        self.page_size, self.pages, self.max_len, self.max_position = page_size, pages, max_len, max_position
        columns = -(-max_len // page_size)
        self.block_table = torch.full((seqs, columns), -1, dtype=torch.int32, device=device)
        self.slots = torch.full((seqs,), -1, dtype=torch.int64, device=device)
        self.positions = torch.full((seqs,), -1, dtype=torch.int64, device=device)
        self._active = torch.zeros(seqs, dtype=torch.int64, device=device)
        self._free = list(range(pages - 1, -1, -1))
        self._held: list[list[int]] = [[] for _ in range(seqs)]
        self._rows, self._next = [0] * seqs, [0] * seqs  # rows held, the next position

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def positions_used(self) -> int:
        """Positions the furthest sequence has used (its newest one and those before it)."""
        return max(self._next)

    def rows(self, seq: int) -> int:
        """Rows sequence `seq` holds."""
        return self._rows[seq]

    def _missing(self, seq: int, rows: int) -> int:
        return max(0, -(-rows // self.page_size) - len(self._held[seq]))

    def _grow(self, wanted) -> None:
        """The pages that `wanted`, (sequence, rows) pairs, are missing (there are as many free), in one upload."""
        new = []
        for seq, rows in wanted:
            held = self._held[seq]
            for _ in range(self._missing(seq, rows)):
                new.append((seq, len(held), self._free.pop()))
                held.append(new[-1][2])
        if not new:
            return
        dev = self.block_table.device
        up = torch.tensor(list(zip(*new)), dtype=torch.int64, pin_memory=dev.type == "cuda").to(dev, non_blocking=True)
        self.block_table[up[0], up[1]] = up[2].to(torch.int32)

    def _place(self, seq: int, newest: int, active: int) -> None:
        # (fill_: a number assigned to one element is uploaded, and waited for)
        self.slots[seq].fill_(newest)
        self.positions[seq].fill_(newest)
        self._active[seq].fill_(active)

    def admit(self, rows: int):
        """A free sequence with pages for `rows` rows (a prompt's, at positions
        0 .. rows - 1): its index, or None when every sequence is taken."""
        if not 1 <= rows <= self.max_len or rows > (self.max_position or rows):
            raise ValueError(f"a sequence holds 1 to {self.max_len} rows, at positions below {self.max_position}")
        seq = next((i for i, n in enumerate(self._rows) if n == 0), None)
        if seq is None:
            return None
        if self._missing(seq, rows) > len(self._free):
            raise MemoryError(f"{self._missing(seq, rows)} pages needed, {len(self._free)} free")
        self._grow([(seq, rows)])
        self._rows[seq] = self._next[seq] = rows
        self._place(seq, rows - 1, 1)
        return seq

    def step(self) -> None:
        """One more row for every sequence: its page, slot and position."""
        live = [i for i, n in enumerate(self._rows) if n]
        if any(self._rows[i] == self.max_len for i in live):
            raise ValueError(f"a sequence holds at most {self.max_len} rows")
        if self.max_position is not None and any(self._next[i] >= self.max_position for i in live):
            raise ValueError(f"positions end at {self.max_position}")
        need = sum(self._missing(i, self._rows[i] + 1) for i in live)
        if need > len(self._free):
            raise MemoryError(f"{need} pages needed, {len(self._free)} free")
        self._grow((i, self._rows[i] + 1) for i in live)
        for i in live:
            self._rows[i] += 1
            self._next[i] += 1
        self.slots += self._active
        self.positions += self._active

    def evicted(self, budget: int) -> None:
        """After `evict` on every layer: no sequence holds more than `budget`
        rows. Pages past those (and the next row's) go back to the pool."""
        if budget < 1:
            raise ValueError("a sequence keeps at least one row")
        self.slots.clamp_(max=budget - 1)
        keep = -(-(budget + 1) // self.page_size)
        free = len(self._free)
        for seq, n in enumerate(self._rows):
            if n > budget:
                self._rows[seq] = budget
                held = self._held[seq]
                self._free += held[keep:][::-1]
                del held[keep:]
        if len(self._free) > free:  # (no sequence holds more than `keep` pages now)
            self.block_table[:, keep:].fill_(-1)

    def release(self, seq: int) -> None:
        """Sequence `seq` ends: its pages go back to the pool."""
        if not 0 <= seq < len(self._rows):
            raise ValueError(f"there is no sequence {seq}")
        self._free += self._held[seq][::-1]
        self._held[seq], self._rows[seq], self._next[seq] = [], 0, 0
        self.block_table[seq].fill_(-1)
        self._place(seq, -1, 0)


class PagedKVCache(nn.Module):
    """One layer's pools on a `PageTable`. `tracked`: with the scores and slot
    positions that `evict` needs."""

    def __init__(self, table: PageTable, n_heads: int, head_dim: int = 128, dtype=torch.bfloat16, tracked: bool = False):
        super().__init__()
        dev = table.block_table.device
        self.table = table
        shape = (table.pages, n_heads, table.page_size, head_dim)
        self.register_buffer("k_pages", torch.zeros(shape, dtype=dtype, device=dev))
        self.register_buffer("v_pages", torch.zeros(shape, dtype=dtype, device=dev))
        slots = (table.block_table.shape[0], n_heads, table.block_table.shape[1] * table.page_size)
        self.register_buffer("scores", torch.zeros(slots, dtype=torch.float32, device=dev) if tracked else None)
        self.register_buffer("slot_pos", torch.zeros(slots, dtype=torch.int32, device=dev) if tracked else None)

    def _apply(self, fn, *args, **kw):
        # a module's cast to 16 bits is for the pools: the gathered weights stay fp32
        scores = self.scores
        super()._apply(fn, *args, **kw)
        if scores is not None and self.scores.dtype is not torch.float32:
            self.scores = scores.to(self.scores.device)
        return self

    def qk_rope_kv(self, qkv, n_head, freqs_cis, *, q_weight=None, k_weight=None, eps: float = 1e-6, out=None):
        """`qk_rope_kv` of each sequence's newest row (qkv: one row a sequence).
        ValueError where one's position lies past `freqs_cis`: its slot would stay
        unwritten, and `attention` would read it."""
        t = self.table
        if t.positions_used > freqs_cis.shape[0]:
            raise ValueError(f"position {t.positions_used - 1} lies past the rotary table")
        return qk_rope_kv(qkv, n_head, self.k_pages, self.v_pages, t.block_table, t.slots, freqs_cis, t.positions,
                          q_weight=q_weight, k_weight=k_weight, eps=eps, scores=self.scores, slot_pos=self.slot_pos,
                          out=out)

    def store(self, seq: int, k, v, start: int = 0):
        """Rows start .. start + rows - 1 of sequence `seq` from k, v (rows, n_heads,
        head_dim), their slots also their positions."""
        t, rows = self.table, k.shape[0]
        if not 0 <= seq < t.slots.shape[0] or start < 0 or start + rows > t.rows(seq):
            raise ValueError(f"sequence {seq} has no rows {start} to {start + rows - 1}")
        slots = torch.arange(start, start + rows, dtype=torch.int64, device=t.slots.device)
        seqs = torch.full((rows,), seq, dtype=torch.int32, device=t.slots.device)
        return store(k, v, self.k_pages, self.v_pages, t.block_table, slots, positions=slots, seqs=seqs,
                     scores=self.scores, slot_pos=self.slot_pos)

    def attention(self, q, *, out=None, work=None):
        """`attention` of each sequence's newest token; a tracked cache gathers its weights."""
        t = self.table
        return attention(q, self.k_pages, self.v_pages, t.block_table, t.slots, scores=self.scores, out=out, work=work)

    def evict(self, budget: int, *, sinks: int = 0, recent: int = 0, work=None):
        """`evict` on this layer (then, once for all layers, `PageTable.evicted`)."""
        if self.scores is None:
            raise ValueError("only a tracked cache is evicted from")
        t = self.table
        return evict(self.k_pages, self.v_pages, t.block_table, t.slots, self.scores, self.slot_pos, t.positions, budget,
                     sinks=sinks, recent=recent, work=work)
