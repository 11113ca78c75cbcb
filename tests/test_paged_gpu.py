"""The paged cache's operators (GPU): against their formulas in 64 bits, at
the lengths, pages, strides and values where they can go wrong, and their
refusals. Tolerances are those of `tests/pageddata.py`: half a step of the
output's type plus what fp32 arithmetic may add; copies and positions are
equal bit for bit."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.gpuutil import bits
from tests.pageddata import Case, assert_within, attention64, attention_check, evict_ref, rounding
from ttspipe_amd import pagedcache as pc

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
EDGES = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257]


def _attend(c, **kw):
    before = None if c.scores is None else c.scores.clone()
    y = pc.attention(c.q, *c.pools(), c.slots, scores=c.scores, **kw)
    assert y is not None
    torch.cuda.synchronize()
    return y, before


@pytest.mark.parametrize("nh,nkv,hd,page,dtype", [
    (32, 8, 128, 64, BF), (32, 8, 128, 16, FP), (8, 2, 128, 16, BF), (4, 2, 64, 32, FP), (7, 7, 64, 16, BF),
    (20, 4, 128, 128, BF), (32, 2, 128, 16, FP), (24, 1, 64, 256, BF), (40, 2, 128, 32, BF), (1, 1, 128, 4096, FP)])
@pytest.mark.parametrize("tracked", [False, True])
def test_attention_matches_the_formula(nh, nkv, hd, page, dtype, tracked):
    lens = [0] + EDGES + [700, 0, 1300]
    c = Case(lens, nh, nkv, hd, page, dtype, seed=nh + hd + page, tracked=tracked)
    y, before = _attend(c)
    assert not y[0].any() and not y[-2].any()  # sequences without a row
    attention_check(c, y, c.scores, before)


@pytest.mark.parametrize("n", [1, 5, 300, 2304, 5000, 20011])
@pytest.mark.parametrize("dtype,page,hd", [(BF, 64, 128), (FP, 16, 128), (BF, 256, 64)])
def test_attention_of_one_sequence(n, dtype, page, hd):
    c = Case([n], 32, 8, hd, page, dtype, seed=n)
    y, before = _attend(c)
    attention_check(c, y, c.scores, before)


@pytest.mark.parametrize("nh,nkv,hd,dtype", [(8, 2, 128, BF), (40, 2, 64, FP), (3, 3, 64, BF)])
@pytest.mark.parametrize("cap", [16, 512, 528])
@pytest.mark.parametrize("tracked", [False, True])
def test_attention_at_the_width_of_short_caches(nh, nkv, hd, dtype, cap, tracked):
    """Tables one slot group below, at and above the width up to which a
    sequence is never cut."""
    lens = [cap, 0, 1, max(1, cap - 15), cap // 2 + 1]
    c = Case(lens, nh, nkv, hd, 16, dtype, seed=cap + nh, tracked=tracked)
    y, before = _attend(c)
    assert not y[1].any()
    attention_check(c, y, c.scores, before)


@pytest.mark.parametrize("seqs,hi", [(65, 40), (130, 700), (200, 16), (200, 600)])
@pytest.mark.parametrize("tracked", [False, True])
def test_attention_of_many_sequences(seqs, hi, tracked):
    """More sequences than a wave has lanes, with empty ones among them, at the
    ends, and 64 in a row."""
    g = torch.Generator().manual_seed(seqs)
    lens = torch.randint(0, hi + 1, (seqs,), generator=g).tolist()
    lens[0] = lens[-1] = lens[64] = 0
    lens[-2] = hi
    if seqs > 190:
        lens[64:128] = [0] * 64
    c = Case(lens, 4, 2, 64, 16, BF, seed=seqs, tracked=tracked)
    y, before = _attend(c)
    attention_check(c, y, c.scores, before)


def test_attention_on_two_streams_at_once():
    cs = [Case([2000, 700, 3], 32, 8, 128, 16, BF, seed=50 + i) for i in range(2)]
    want = []
    for c in cs:
        s = c.scores.clone()
        want.append((pc.attention(c.q, *c.pools(), c.slots, scores=s), s))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    got = [[] for _ in cs]
    for _ in range(4):
        for c, stream, out in zip(cs, streams, got):
            with torch.cuda.stream(stream):
                s = c.scores.clone()
                out.append((pc.attention(c.q, *c.pools(), c.slots, scores=s), s))
    torch.cuda.synchronize()
    for (y, s), outs in zip(want, got):
        for y2, s2 in outs:
            assert np.array_equal(bits(y), bits(y2)) and torch.equal(s, s2)


@pytest.mark.parametrize("tracked", [False, True])
def test_attention_of_one_long_sequence_among_short_ones(tracked):
    c = Case([3, 9000, 1, 0, 40], 8, 2, 128, 32, BF, seed=5, tracked=tracked)
    y, before = _attend(c)
    attention_check(c, y, c.scores, before)


def test_attention_reads_only_the_rows_of_each_sequence():
    """slots behind the table are cut to it; -1 and less hold nothing."""
    c = Case([64, 64, 64, 64], 8, 2, 128, 16, BF, seed=6)
    c.slots = torch.tensor([10**12, 63, -7, 0], device="cuda")
    y, before = _attend(c)
    attention_check(c, y, c.scores, before)
    assert torch.equal(c.scores[2], before[2]) and torch.equal(c.scores[3, :, 1:], before[3, :, 1:])


@pytest.mark.parametrize("page", [16, 64])
def test_attention_leaves_holes_out(page):
    """Table entries outside the pool are holes: their slots are no keys, and a
    sequence of holes alone gives zeros and gathers nothing."""
    c = Case([300, 300, 200, 33], 8, 2, 128, page, FP, seed=7)
    c.table[0, 1], c.table[0, 3] = -1, c.pages
    c.table[1, 0] = 2**31 - 1
    c.table[2] = -(2**31)
    y, before = _attend(c)
    assert not y[2].any() and torch.equal(c.scores[2], before[2])
    attention_check(c, y, c.scores, before)


def test_attention_takes_strided_pools_heads_and_tables():
    """Pools with the heads inside the page and K and V side by side, q cut out
    of the wqkv rows, a table cut out of a wider one, scores of another order."""
    base = Case([100, 1, 513, 0, 77], 8, 2, 128, 32, BF, seed=8)
    y0, before = _attend(base)
    c = base
    kv = torch.full((c.pages, c.page, 2, c.nkv, 2 * 128 + 8), math.nan, dtype=BF, device="cuda")
    k, v = kv[:, :, 0, :, 8:136].transpose(1, 2), kv[:, :, 1, :, 128:256].transpose(1, 2)
    k.copy_(c.k), v.copy_(c.v)
    qkv = torch.full((5, 8 + 4, 128), math.nan, dtype=BF, device="cuda")
    qkv[:, :8] = c.q
    wide = torch.full((5, c.table.shape[1] + 5), 10**9, dtype=torch.int32, device="cuda")
    wide[:, 2:-3] = c.table
    scores = torch.zeros(2, 5, c.cap + 3, device="cuda")[:, :, 3:].transpose(0, 1)
    scores.copy_(before)
    y = pc.attention(qkv[:, :8], k, v, wide[:, 2:-3], c.slots, scores=scores)
    torch.cuda.synchronize()
    assert np.array_equal(bits(y), bits(y0)) and torch.equal(scores, c.scores)


def test_attention_with_large_and_infinite_values():
    """One key far above the others, scores that all are -inf, and infinite and
    NaN values: what the formula gives, in the heads that see them only."""
    c = Case([130, 130, 130, 130], 8, 2, 128, 16, BF, seed=9, tracked=False)
    c.q *= 40
    p1, p2, p3 = int(c.table[1, 5]), int(c.table[2, 3]), int(c.table[3, 0])
    for b in (1, 2):
        c.q[b] = c.q[b].abs()
    c.q[2] /= 40  # weights that do not vanish beside the infinite value
    c.k[c.table[1, :9].long(), 0] = -math.inf  # every score of sequence 1's first KV head: -inf
    c.v[p2, 1, 4, 7] = math.inf
    c.k[p3, 0, 2, 3] = math.nan
    y, _ = _attend(c)
    ref, _, yb, _ = attention64(c.q, c.k, c.v, c.table, c.slots)
    assert torch.isnan(ref[1, :4]).all() and torch.isnan(ref[3, :4]).all() and not torch.isnan(ref[3, 4:]).any()
    got = y.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))
    fine = torch.isfinite(ref)
    assert ((got - ref)[fine].abs() <= (rounding(ref, BF) * (1 + 2**-7) + yb)[fine]).all()
    assert p1 >= 0


def test_attention_with_a_minus_infinite_key_among_finite_ones():
    c = Case([70], 4, 2, 128, 16, FP, seed=10)
    c.q.abs_()
    c.k[c.table[0, 0].long(), :, 0] = -math.inf
    c.k[c.table[0, 4].long(), :, 5] = -math.inf  # the newest slot, too
    y, before = _attend(c)
    ref, p, yb, _ = attention64(c.q, c.k, c.v, c.table, c.slots)
    # the bound's magnitudes are infinite here: the finite keys' alone
    c.k[torch.isinf(c.k)] = 0
    yb = attention64(c.q, c.k, c.v, c.table, c.slots)[2] * 2
    assert torch.equal(c.scores[0, :, 0], before[0, :, 0]) and torch.equal(c.scores[0, :, 69], before[0, :, 69])
    assert_within(y, ref, rounding(ref, FP) * (1 + 2**-7) + yb)


@pytest.mark.parametrize("gap", [9, 14, 17, 21])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_keeps_a_long_tail_of_small_weights(dtype, first, gap):
    """16380 rows e^-gap of the four largest weights each (one in the share of
    each wave of a sequence that is not cut), whose values alone count: weights of
    2^-13 to 2^-30. Relative to y: 2 (D + 4) 2^-24 gap for the scores, 2^-23 (n / 8
    + 64) for the sums, 2^-16 for the weights' parts (and, in fp16, 2^-38 of the
    largest weight)."""
    n, hd, heads, seqs = 16384, 64, 64, 16
    k, v = torch.zeros(n // 64, heads, 64, hd), torch.ones(n // 64, heads, 64, hd)
    for j in (0, 32, 64, 96):
        j += 0 if first else n - 128
        k[j // 64, :, j % 64, 0] = gap
        v[j // 64, :, j % 64] = 0.0
    q = torch.zeros(seqs, heads, hd)
    q[:, :, 0] = 1.0
    k, v, q = (x.to(dtype).cuda() for x in (k, v, q))
    table = torch.arange(n // 64, dtype=torch.int32, device="cuda").expand(seqs, -1).contiguous()
    y = pc.attention(q, k, v, table, torch.full((seqs,), n - 1, device="cuda"), scale=1.0)
    tail = (n - 4) * math.exp(-gap) / 4
    ref = torch.full((seqs, heads, hd), tail / (1 + tail), dtype=torch.float64)
    e = 2 * (hd + 4) * 2.0**-24 * gap + 2.0**-20 + 2.0**-23 * (n / 8 + 64) + 2.0**-16 + 2.0**-38 * math.exp(gap)
    assert_within(y, ref, rounding(ref, dtype) * (1 + 2**-7) + ref * e, "tail")


def test_attention_scale_out_and_work():
    c = Case([90, 33], 8, 2, 64, 16, BF, seed=11)
    need = pc.attention_work(2, 8, 2, 64, c.table.shape[1], 16, tracked=True)
    out = torch.full((2, 8, 64), math.nan, dtype=BF, device="cuda")
    y, before = _attend(c, scale=0.31, out=out, work=torch.full((need,), math.nan, device="cuda"))
    assert y is out
    attention_check(c, y, c.scores, before, scale=0.31)


def test_attention_past_32_bit_offsets():
    """A pool of over 2^32 bytes and 2^31 elements, the sequence's pages at its end."""
    pages, nkv, page, hd = 2200, 8, 1024, 128
    k = torch.empty(pages, nkv, page, hd, dtype=BF, device="cuda")
    assert k.numel() > 1 << 31
    v = torch.empty_like(k)
    k[:3], v[:3] = math.nan, math.nan
    table = torch.tensor([[pages - 1, 0, pages - 3], [pages - 2, 1, 2]], dtype=torch.int32, device="cuda")
    table[0, 1] = pages - 4
    small = Case([2100, 900], 16, 8, hd, page, BF, seed=12, cols=3, tracked=False)
    for b, n in enumerate((2100, 900)):
        for col in range(-(-n // page)):
            k[table[b, col].long()] = small.k[small.table[b, col].long()]
            v[table[b, col].long()] = small.v[small.table[b, col].long()]
    y = pc.attention(small.q, k, v, table, small.slots)
    ys = pc.attention(small.q, *small.pools(), small.slots)
    assert np.array_equal(bits(y), bits(ys))
    attention_check(small, y)
    # the write and the eviction, to and from the last pages
    rows = torch.randn(1, nkv, hd, device="cuda").to(BF)
    assert pc.store(rows, -rows, k, v, table, torch.tensor([2100], device="cuda"),
                    seqs=torch.tensor([0], dtype=torch.int32, device="cuda"))
    assert torch.equal(k[pages - 3, :, 2100 - 2048], rows[0]) and torch.equal(v[pages - 3, :, 2100 - 2048], -rows[0])
    sc = torch.zeros(2, nkv, 3 * page, device="cuda")
    sc[0, :, 2100] = 1.0
    sp = torch.arange(3 * page, dtype=torch.int32, device="cuda").expand(2, nkv, -1).contiguous()
    slots = torch.tensor([2100, 899], device="cuda")
    assert pc.evict(k, v, table, slots, sc, sp, slots.clone(), 2100)
    # slot 2099 has score 0 and the highest index of those: the new row takes its place
    assert torch.equal(k[pages - 3, :, 2099 - 2048], rows[0]) and (sp[0, :, 2099] == 2100).all()


def test_attention_is_deterministic_on_any_stream():
    c = Case([1000, 3, 0, 250], 32, 8, 128, 16, BF, seed=13)
    y, before = _attend(c)
    side = torch.cuda.Stream()
    for _ in range(3):
        scores = before.clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y2 = pc.attention(c.q, *c.pools(), c.slots, scores=scores)
        side.synchronize()
        assert np.array_equal(bits(y), bits(y2)) and torch.equal(scores, c.scores)


def test_captured_attention_follows_its_slots():
    """Two graphs with workspaces of their own, replayed in turn at growing
    lengths: every replay equals the eager call."""
    c = Case([700, 700, 700], 8, 2, 128, 16, BF, seed=14)
    need = pc.attention_work(3, 8, 2, 128, c.table.shape[1], 16, tracked=True)
    slots = [c.slots.clone(), c.slots.clone()]
    outs = [torch.empty_like(c.q) for _ in range(2)]
    scores = [torch.zeros_like(c.scores) for _ in range(2)]
    works = [torch.empty(need, device="cuda") for _ in range(2)]
    graphs = []
    for i in range(2):
        call = lambda: pc.attention(c.q, *c.pools(), slots[i], scores=scores[i], out=outs[i], work=works[i])  # noqa: E731
        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)
    for step, lens in enumerate([(1, 2, 3), (0, 700, 64), (129, 0, 1), (699, 300, 16), (5, 5, 5)]):
        for i in range(2):
            slots[i].copy_(torch.tensor([n - 1 - i * (n > 1) for n in lens]))
            scores[i].fill_(0.25 * step)
            graphs[i].replay()
        expect = []
        for i in range(2):
            s = torch.full_like(scores[i], 0.25 * step)
            expect.append((pc.attention(c.q, *c.pools(), slots[i], scores=s), s))
        torch.cuda.synchronize()
        for i in range(2):
            assert np.array_equal(bits(outs[i]), bits(expect[i][0])) and torch.equal(scores[i], expect[i][1]), (step, i)


# ------------------------------------------------------------------- the rows


def _freqs(n, hd, dtype=BF):
    ang = torch.outer(torch.arange(n).double(), 1.0 / 1e6 ** (torch.arange(0, hd, 2).double() / hd))
    return torch.stack([ang.cos(), ang.sin()], -1).to(dtype).cuda()


def _rope64(x, w, cs, eps):
    """x (..., D) normed with w and turned by cs, in 64 bits, and the bound of fp32
    arithmetic before the last rounding: the norm's D-term sum, root and
    quotients ((D + 12) 2^-24) and the rotation's products and sum (4 2^-24),
    of |a c| + |b s|."""
    x, cs = x.double().cpu(), cs.double().cpu()
    D, e = x.shape[-1], 4 * 2.0**-24
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double().cpu()
        e += (D + 12) * 2.0**-24
    a, b, c, s = x[..., 0::2], x[..., 1::2], cs[..., 0], cs[..., 1]
    y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    m = torch.stack([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1).flatten(-2)
    return y, m * e


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("nh,nkv,hd,page,dtype,ftype", [
    (32, 8, 128, 64, BF, BF), (8, 2, 128, 16, FP, torch.float32), (7, 7, 64, 32, BF, FP), (24, 1, 64, 16, FP, BF),
    (5, 5, 128, 16, BF, torch.float32)])
@pytest.mark.parametrize("rows", [1, 3, 64, 257])
def test_rows_match_the_formula(nh, nkv, hd, page, dtype, ftype, rows, norm):
    """Every row's q, k and v, and nothing else in the pools touched."""
    g = torch.Generator().manual_seed(rows + nh)
    B = 3
    c = Case([rows] * B, nh, nkv, hd, page, dtype, seed=rows, cols=-(-rows // page) + 1)
    qkv = (torch.randn(rows, (nh + 2 * nkv) * hd, generator=g) * 2).to(dtype).cuda()
    freqs = _freqs(1000, hd, ftype)
    pos = torch.randint(0, 1000, (rows,), generator=g).cuda()
    seqs = torch.randint(0, B, (rows,), generator=g).to(torch.int32).cuda()
    slots = torch.randperm(rows, generator=g).cuda()
    qw, kw = ((torch.rand(hd, generator=g) + 0.5).to(dtype).cuda() if norm else None for _ in "qk")
    sp = torch.full(c.scores.shape, -5, dtype=torch.int32, device="cuda")
    k0, v0, s0 = c.k.clone(), c.v.clone(), c.scores.clone()
    q = pc.qk_rope_kv(qkv, nh, *c.pools(), slots, freqs, pos, q_weight=qw, k_weight=kw, eps=1e-5, seqs=seqs,
                      scores=c.scores, slot_pos=sp)
    assert q is not None
    x = qkv.view(rows, -1, hd)
    cs = freqs[pos][:, None]
    ref, b = _rope64(x[:, :nh], qw, cs, 1e-5)
    assert_within(q, ref, rounding(ref, dtype) * (1 + 2**-7) + b, "q")
    ref, b = _rope64(x[:, nh:nh + nkv], kw, cs, 1e-5)
    page_of = c.table[seqs.long(), slots // page].long()
    assert_within(c.k[page_of, :, slots % page], ref, rounding(ref, dtype) * (1 + 2**-7) + b, "k")
    assert torch.equal(c.v[page_of, :, slots % page], x[:, nh + nkv:])
    # exactly those rows
    k0[page_of, :, slots % page] = c.k[page_of, :, slots % page]
    v0[page_of, :, slots % page] = x[:, nh + nkv:]
    assert np.array_equal(bits(k0), bits(c.k)) and np.array_equal(bits(v0), bits(c.v))
    s0[seqs.long(), :, slots] = 0
    p0 = torch.full_like(sp, -5)
    p0[seqs.long(), :, slots] = pos.to(torch.int32)[:, None]
    assert torch.equal(s0, c.scores) and torch.equal(p0, sp)


@pytest.mark.parametrize("dtype,ftype", [(BF, BF), (FP, torch.float32)])
def test_rows_without_norms_have_the_contiguous_kernels_bits(hip, dtype, ftype):
    from ttspipe_amd import _lib

    nh, nkv, hd, rows, L = 8, 2, 128, 70, 96
    qkv = (torch.randn(rows, (nh + 2 * nkv) * hd, generator=torch.Generator().manual_seed(3)) * 2).to(dtype).cuda()
    freqs, pos = _freqs(L, hd, ftype), torch.arange(10, 10 + rows, device="cuda")
    kc, vc = (torch.zeros(nkv, L, hd, dtype=dtype, device="cuda") for _ in "kv")
    q1 = torch.empty(rows, nh, hd, dtype=dtype, device="cuda")
    rc = hip.ttsp_qk_rope_kv_rows(qkv.data_ptr(), qkv.shape[1], 0, 0, 0.0, freqs[pos].contiguous().data_ptr(),
                                  _lib.dtype_code(ftype), pos.data_ptr(), q1.data_ptr(), kc.data_ptr(), vc.data_ptr(),
                                  nh, nkv, L, rows, _lib.dtype_code(dtype), _lib.stream())
    assert rc == 0
    kp, vp = (torch.zeros(6, nkv, 16, hd, dtype=dtype, device="cuda") for _ in "kv")
    table = torch.arange(6, dtype=torch.int32, device="cuda").view(1, 6)
    q2 = pc.qk_rope_kv(qkv, nh, kp, vp, table, pos, freqs, pos, seqs=torch.zeros(rows, dtype=torch.int32, device="cuda"))
    assert np.array_equal(bits(q1), bits(q2))
    for a, b in ((kc, kp), (vc, vp)):
        assert np.array_equal(bits(a), bits(b.transpose(0, 1).reshape(nkv, L, hd)))


def test_rows_that_have_no_place_are_not_written():
    """Padding rows, holes, sequences, slots and positions outside what there is."""
    c = Case([40, 40], 4, 2, 128, 16, BF, seed=20)
    c.table[1, 1] = c.pages
    qkv = torch.randn(8, 8 * 128, device="cuda").to(BF)
    freqs = _freqs(50, 128)
    slots = torch.tensor([-1, 48, 10**15, 20, 5, 6, 7, 8], device="cuda")
    seqs = torch.tensor([0, 0, 0, 1, 2, -1, 0, 1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([3, 3, 3, 3, 3, 3, 50, -1], device="cuda")
    k0, v0, s0 = c.k.clone(), c.v.clone(), c.scores.clone()
    sp = torch.zeros(c.scores.shape, dtype=torch.int32, device="cuda")
    q = pc.qk_rope_kv(qkv, 4, *c.pools(), slots, freqs, pos, seqs=seqs, scores=c.scores, slot_pos=sp)
    assert np.array_equal(bits(k0), bits(c.k)) and np.array_equal(bits(v0), bits(c.v))
    assert torch.equal(s0, c.scores) and not sp.any()
    assert not q[6:].any()
    ref, b = _rope64(qkv.view(8, -1, 128)[:6, :4], None, freqs[pos[:6]][:, None], 0)
    assert_within(q[:6], ref, rounding(ref, BF) * (1 + 2**-7) + b)


def test_store_copies_rows_of_a_contiguous_cache():
    nkv, rows, hd = 4, 130, 64
    cache = torch.randn(2, 1, nkv, 200, hd, device="cuda").to(FP)
    k, v = (t[0, :, 7:7 + rows].transpose(0, 1) for t in cache)
    c = Case([rows, 20], 4, nkv, hd, 32, FP, seed=21)
    k0, v0 = c.k.clone(), c.v.clone()
    slots = torch.arange(rows, device="cuda")
    sp = torch.full(c.scores.shape, -1, dtype=torch.int32, device="cuda")
    seqs = torch.zeros(rows, dtype=torch.int32, device="cuda")
    assert pc.store(k, v, *c.pools(), slots, positions=slots + 5, seqs=seqs, scores=c.scores, slot_pos=sp)
    pg = c.table[0, slots // 32].long()
    assert torch.equal(c.k[pg, :, slots % 32], k) and torch.equal(c.v[pg, :, slots % 32], v)
    k0[pg, :, slots % 32], v0[pg, :, slots % 32] = k, v
    assert np.array_equal(bits(k0), bits(c.k)) and np.array_equal(bits(v0), bits(c.v))
    assert (c.scores[0, :, :rows] == 0).all() and (sp[0, :, :rows] == slots + 5).all() and (sp[1] == -1).all()
    # without scores and positions
    assert pc.store(v, k, *c.pools(), slots, seqs=seqs)
    assert torch.equal(c.k[pg, :, slots % 32], v)


# --------------------------------------------------------------- the eviction


def _evict(c, scores, sp, positions, budget, **kw):
    k0, v0 = c.k.clone(), c.v.clone()
    s0, p0 = scores.clone(), sp.clone()
    assert pc.evict(*c.pools(), c.slots, scores, sp, positions, budget, **kw)
    torch.cuda.synchronize()
    moved = 0
    table, ps, pp = c.table.cpu(), s0.cpu().numpy(), p0.cpu().numpy()
    for b in range(len(c.lens)):
        n = max(0, min(int(c.slots[b]) + 1, c.cap))
        for h in range(c.nkv):
            moves = evict_ref(ps[b, h], pp[b, h], n, int(positions[b]), budget, kw.get("sinks", 0), kw.get("recent", 0))
            moved += len(moves)
            for src, dst in moves:
                s, d = (int(table[b, src // c.page]), src % c.page), (int(table[b, dst // c.page]), dst % c.page)
                k0[d[0], h, d[1]], v0[d[0], h, d[1]] = k0[s[0], h, s[1]], v0[s[0], h, s[1]]
                s0[b, h, dst], p0[b, h, dst] = s0[b, h, src], p0[b, h, src]
    assert torch.equal(sp, p0)
    assert torch.equal(scores.view(torch.int32), s0.view(torch.int32))
    assert np.array_equal(bits(c.k), bits(k0)) and np.array_equal(bits(c.v), bits(v0))
    return moved


def _tracked(lens, nkv, hd, page, dtype, seed, kind="exp", cols=None):
    c = Case(lens, nkv, nkv, hd, page, dtype, seed=seed, cols=cols)
    g = torch.Generator().manual_seed(seed)
    shape = c.scores.shape
    if kind == "exp":
        s = torch.empty(shape).exponential_(generator=g).pow_(3)
    elif kind == "few":  # many equal scores, signed zeros among them
        s = torch.randint(-1, 3, shape, generator=g).float() * -0.0 + torch.randint(0, 3, shape, generator=g).float()
        s[torch.rand(shape, generator=g) < 0.2] = -0.0
    elif kind == "same":
        s = torch.full(shape, 0.5)
    else:  # every kind of value
        s = torch.randn(shape, generator=g)
        r = torch.rand(shape, generator=g)
        s[r < 0.1], s[(r >= 0.1) & (r < 0.15)], s[(r >= 0.15) & (r < 0.2)] = math.nan, math.inf, -math.inf
        s[(r >= 0.2) & (r < 0.25)] = 1e-42
    sp = torch.stack([torch.randperm(shape[2], generator=g) for _ in range(shape[0] * shape[1])]).view(shape)
    return c, s.cuda(), sp.to(torch.int32).cuda()


@pytest.mark.parametrize("kind", ["exp", "few", "same", "every"])
@pytest.mark.parametrize("hd,page,dtype", [(128, 16, BF), (64, 64, FP)])
@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (16, 4, 4), (100, 0, 100), (255, 16, 30), (299, 3, 9)])
def test_evict_matches_the_definition(kind, hd, page, dtype, budget, sinks, recent):
    lens = [300, 301, 0, 1, 255, 256, 100, 3000]
    c, s, sp = _tracked(lens, 2, hd, page, dtype, seed=budget, kind=kind)
    newest = sp.amax((1, 2)).long()
    moved = _evict(c, s, sp, newest, budget, sinks=sinks, recent=recent)
    assert moved or budget == 1  # (budget 1: the kept row may be slot 0)


@pytest.mark.parametrize("n,budget", [(1025, 1024), (1030, 1024), (1100, 1024), (5000, 4999), (8192, 4096), (20000, 19990), (20000, 5000),
                                      (65530, 70), (70001, 20000),
                                      (70001, 69000)])
@pytest.mark.parametrize("kind", ["exp", "every"])
def test_evict_of_long_sequences(n, budget, kind):
    c, s, sp = _tracked([n, n - 1, budget], 2, 64, 64, BF, seed=n, kind=kind)
    _evict(c, s, sp, sp.amax((1, 2)).long(), budget, sinks=4, recent=64)


@pytest.mark.parametrize("cap", [1056, 8192, 20000, 70000])
@pytest.mark.parametrize("kind", ["exp", "few", "same", "every"])
def test_evict_of_a_few_rows(cap, kind):
    """1 to 6 rows over the budget, in every ranking variant."""
    budget = cap - 20
    lens = [budget + i for i in range(7)]
    c, s, sp = _tracked(lens, 2, 64, 16, BF, seed=cap, kind=kind, cols=-(-cap // 16))
    _evict(c, s, sp, sp.amax((1, 2)).long(), budget, sinks=3, recent=8)


def test_evict_of_many_sequences():
    g = torch.Generator().manual_seed(60)
    lens = torch.randint(0, 300, (90,), generator=g).tolist()
    c, s, sp = _tracked(lens, 3, 64, 16, FP, seed=60, cols=20)
    assert _evict(c, s, sp, sp.amax((1, 2)).long(), 100, sinks=2, recent=9) > 0


def test_evict_of_the_newest_rows_themselves():
    """The lowest keys past the budget: nothing moves, or only what stays of them."""
    c, s, sp = _tracked([104, 103, 102, 101], 2, 128, 16, FP, seed=34, cols=8)
    s[:, :, 100:] = -1.0
    assert _evict(c, s, sp, sp.amax((1, 2)).long() + 1000, 100) == 0
    s[:, :, 101:103] = 10.0
    s[:, :, 103] = -2.0
    s[:, :, 7], s[:, :, 55] = -3.0, -4.0
    assert _evict(c, s, sp, sp.amax((1, 2)).long() + 1000, 100) > 0


def test_evict_leaves_short_sequences_and_wide_budgets_alone():
    c, s, sp = _tracked([50, 0, 64], 2, 64, 16, FP, seed=30)
    pos = sp.amax((1, 2)).long()
    assert _evict(c, s, sp, pos, 64) == 0
    assert _evict(c, s, sp, pos, 10**6) == 0
    c.slots = torch.tensor([-1, -9, -1], device="cuda")
    assert _evict(c, s, sp, pos, 8) == 0
    c.slots = torch.tensor([49, -1, 10**14], device="cuda")  # cut to the table's 64
    assert _evict(c, s, sp, pos, 20) > 0


def test_evict_with_equal_positions():
    """More protected rows than the budget holds (positions that repeat): the lowest slots of them."""
    c, s, sp = _tracked([200, 90], 2, 64, 16, BF, seed=31)
    sp.fill_(7)
    assert _evict(c, s, sp, torch.tensor([7, 7], device="cuda"), 60, sinks=5, recent=50) == 0
    sp[:, :, ::3] = 3
    _evict(c, s, sp, torch.tensor([7, 7], device="cuda"), 60, sinks=4, recent=0)


def test_evict_takes_strided_scores_and_pools():
    c, s, sp = _tracked([300, 280, 100], 2, 64, 16, BF, seed=32)
    pos = sp.amax((1, 2)).long()
    want_s, want_p = s.clone(), sp.clone()
    k1, v1 = c.k.clone(), c.v.clone()
    assert pc.evict(k1, v1, c.table, c.slots, want_s, want_p, pos, 120, sinks=2, recent=9)
    kv = torch.zeros(c.pages, 16, 2, 2, 80, dtype=BF, device="cuda")
    k, v = kv[:, :, 0, :, 8:72].transpose(1, 2), kv[:, :, 1, :, 16:].transpose(1, 2)
    k.copy_(c.k), v.copy_(c.v)
    ts = torch.zeros(2, 3, c.cap + 1, device="cuda")[:, :, 1:].transpose(0, 1)
    tp = torch.zeros(2, 3, c.cap + 5, dtype=torch.int32, device="cuda")[:, :, :-5].transpose(0, 1)
    ts.copy_(s), tp.copy_(sp)
    work = torch.full((pc.evict_work(3, 2, c.table.shape[1], 16, 120),), -1, dtype=torch.int32, device="cuda")
    assert pc.evict(k, v, c.table, c.slots, ts, tp, pos, 120, sinks=2, recent=9, work=work)
    assert torch.equal(ts, want_s) and torch.equal(tp, want_p)
    assert np.array_equal(bits(k), bits(k1)) and np.array_equal(bits(v), bits(v1))


def test_captured_evict_follows_its_slots():
    c, s, sp = _tracked([400, 400], 2, 64, 16, BF, seed=33)
    k0, v0, s0, p0 = c.k.clone(), c.v.clone(), s.clone(), sp.clone()
    pos = sp.amax((1, 2)).long()
    work = torch.zeros(pc.evict_work(2, 2, c.table.shape[1], 16, 128), dtype=torch.int32, device="cuda")
    call = lambda: pc.evict(*c.pools(), c.slots, s, sp, pos, 128, sinks=2, recent=16, work=work)  # noqa: E731
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for lens in ((400, 129), (100, 400), (130, 300), (128, 1), (399, 398)):
        for a, b in ((c.k, k0), (c.v, v0), (s, s0), (sp, p0)):
            a.copy_(b)
        c.slots.copy_(torch.tensor([n - 1 for n in lens]))
        g.replay()
        k1, v1, s1, p1 = k0.clone(), v0.clone(), s0.clone(), p0.clone()
        assert pc.evict(k1, v1, c.table, c.slots, s1, p1, pos, 128, sinks=2, recent=16)
        torch.cuda.synchronize()
        assert torch.equal(s, s1) and torch.equal(sp, p1)
        assert np.array_equal(bits(c.k), bits(k1)) and np.array_equal(bits(c.v), bits(v1))


# --------------------------------------------------------------- the refusals


def test_calls_that_are_declined():
    c = Case([40, 40], 8, 2, 128, 16, BF, seed=40)
    k, v, t = c.pools()
    sp = torch.zeros(c.scores.shape, dtype=torch.int32, device="cuda")
    ok = dict(q=c.q, k=k, v=v, t=t, slots=c.slots)

    def attend(**kw):
        a = {**ok, **kw}
        return pc.attention(a["q"], a["k"], a["v"], a["t"], a["slots"], scores=a.get("scores"))

    assert attend() is not None and attend(scores=c.scores) is not None
    before = pc.stats()["declined"]
    bad = [
        dict(q=c.q.float()), dict(q=c.q.to(FP)), dict(k=k.to(FP)), dict(k=k.float(), v=v.float(), q=c.q.float()),
        dict(q=c.q[:1]), dict(q=c.q[:, :7]), dict(q=c.q[..., :64]), dict(q=c.q[0]), dict(q=c.q.cpu()),
        dict(q=c.q.transpose(1, 2).contiguous().transpose(1, 2)), dict(v=v[:-1]), dict(v=v[:, :1]),
        dict(k=k[..., :96], v=v[..., :96], q=c.q[..., :96]), dict(k=k[:, :, :12], v=v[:, :, :12]),
        dict(k=k[:, :, :8], v=v[:, :, :8]), dict(k=k[0]), dict(k=k[:0], v=v[:0]), dict(k=k[:1].expand(9, -1, -1, -1)),
        dict(t=t.long()), dict(t=t[0]), dict(t=t[:1]), dict(t=t[:, :0]), dict(t=t.t().contiguous().t()), dict(t=t.cpu()),
        dict(slots=c.slots.int()), dict(slots=c.slots[:1]), dict(slots=c.slots.cpu()), dict(slots=c.slots.view(2, 1)),
        dict(slots=torch.zeros(4, dtype=torch.int64, device="cuda")[::2]), dict(scores=c.scores.half()),
        dict(scores=c.scores[:, :, :-1]), dict(scores=c.scores[:, :1].expand(-1, 2, -1)), dict(scores=c.scores.cpu()),
    ]
    for kw in bad:
        assert attend(**kw) is None, kw.keys()
    # rows off a 16-byte boundary
    flat = torch.zeros(k.numel() + 4, dtype=BF, device="cuda")
    assert attend(k=flat[4:].view(k.shape)) is None
    qkv = torch.zeros(2, 12 * 128, dtype=BF, device="cuda")
    f = _freqs(64, 128)

    def rope(qkv=qkv, n_head=8, slots=c.slots, freqs=f, pos=c.slots, **kw):
        return pc.qk_rope_kv(qkv, n_head, k.clone(), v.clone(), t, slots, freqs, pos, **kw)

    assert rope() is not None
    w = torch.ones(128, dtype=BF, device="cuda")
    for kw in (dict(qkv=qkv[:, :-128]), dict(qkv=qkv.float()), dict(n_head=7), dict(n_head=0), dict(freqs=f[:, :32]),
               dict(freqs=f.double()), dict(freqs=f.cpu()), dict(freqs=f[::2]), dict(pos=c.slots.int()), dict(slots=c.slots[:1]),
               dict(q_weight=w[:64]), dict(k_weight=w.float()), dict(k_weight=w.cpu()), dict(pos=None, slot_pos=sp),
               dict(pos=None, freqs=f[:1]), dict(seqs=c.slots), dict(qkv=torch.zeros(3, 12 * 128, dtype=BF, device="cuda"),
                                                                     slots=torch.zeros(3, dtype=torch.int64, device="cuda"), pos=None)):
        assert rope(**kw) is None, kw.keys()
    r = torch.zeros(2, 2, 128, dtype=BF, device="cuda")
    for a, b, kw in ((r, r[:1], {}), (r.float(), r.float(), {}), (r[:, :1], r[:, :1], {}), (r, r, dict(slot_pos=sp)),
                     (r.transpose(1, 2).contiguous().transpose(1, 2), r, {})):
        assert pc.store(a, b, k, v, t, c.slots, **kw) is None
    for a in ((c.scores.half(), sp, c.slots), (c.scores, sp.long(), c.slots), (c.scores, sp, c.slots.int()),
              (c.scores, sp[:, :1], c.slots), (None, sp, c.slots)):
        assert pc.evict(k, v, t, c.slots, a[0], a[1], a[2], 20) is None
    assert pc.stats()["declined"] > before


def test_calls_that_raise():
    c = Case([40, 40], 8, 2, 128, 16, BF, seed=41)
    sp = torch.zeros(c.scores.shape, dtype=torch.int32, device="cuda")
    for out in (torch.empty(2, 8, 64, dtype=BF, device="cuda"), torch.empty(2, 8, 128, device="cuda"),
                torch.empty(2, 8, 128, dtype=BF)):
        with pytest.raises(ValueError):
            pc.attention(c.q, *c.pools(), c.slots, out=out)
    need = pc.attention_work(2, 8, 2, 128, 3, 16)
    for work in (torch.empty(max(need - 1, 0), device="cuda"), torch.empty(need, dtype=torch.float64, device="cuda"),
                 torch.empty(need + 1, device="cuda")[1:]):
        if need:
            with pytest.raises(ValueError):
                pc.attention(c.q, *c.pools(), c.slots, work=work)
    w = Case([900, 40], 2, 2, 64, 16, BF, seed=41)
    wp = torch.zeros(w.scores.shape, dtype=torch.int32, device="cuda")
    need = pc.evict_work(2, 2, w.table.shape[1], 16, 400)
    for work in (torch.empty(0, dtype=torch.int32, device="cuda"), torch.empty(need, device="cuda"),
                 torch.empty(need, dtype=torch.int32), torch.empty(need - 1, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError):
            pc.evict(*w.pools(), w.slots, w.scores, wp, w.slots, 400, work=work)
    with pytest.raises(ValueError):
        pc.qk_rope_kv(torch.zeros(2, 12 * 128, dtype=BF, device="cuda"), 8, *c.pools(), c.slots, _freqs(64, 128), c.slots,
                      out=torch.empty(2, 8, 64, dtype=BF, device="cuda"))


def test_no_rows_at_all():
    c = Case([40], 8, 2, 128, 16, BF, seed=42)
    k0 = c.k.clone()
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    q = pc.qk_rope_kv(torch.zeros(0, 12 * 128, dtype=BF, device="cuda"), 8, *c.pools(), none, _freqs(64, 128), none,
                      seqs=none.int())
    assert q.shape == (0, 8, 128)
    r = torch.zeros(0, 2, 128, dtype=BF, device="cuda")
    assert pc.store(r, r, *c.pools(), none, seqs=none.int())
    assert np.array_equal(bits(k0), bits(c.k))
