"""The paged cache's operators in forms and at sizes that lie between those of
`test_paged_gpu.py` (GPU): each against its definition in 64 bits, with the
bounds of `tests/pageddata.py` unless a test derives its own."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.gpuutil import bits
from tests.pageddata import Case, assert_within, attention64, attention_check, evict_ref, rounding
from tests.test_paged_gpu import _evict, _freqs, _rope64, _tracked
from ttspipe_amd import pagedcache as pc

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def cancelling(seqs, cols, hd=64, page=16):
    """bf16 caches of three rows whose scores are 0, 0 and -s and whose values are
    what bf16 holds of w = exp(-s), what it holds of the rest, both negative, and
    1: y = (w - hi - mid) / (2 + w), 2^-18 w and less, so that the bits of w
    beyond two parts of eight are all that is left."""
    s = torch.linspace(0.03, 2.0, seqs).to(BF)
    w = torch.exp(-s.double())
    hi = w.to(BF)
    mid = (w - hi.double()).to(BF)
    k, v = torch.zeros(seqs, 1, page, hd, dtype=BF), torch.zeros(seqs, 1, page, hd, dtype=BF)
    k[:, 0, 2, 0] = -s
    v[:, 0, 0], v[:, 0, 1], v[:, 0, 2] = -hi[:, None], -mid[:, None], 1.0
    q = torch.zeros(seqs, 1, hd, dtype=BF)
    q[:, :, 0] = 1.0
    table = torch.full((seqs, cols), -1, dtype=torch.int32)
    table[:, 0] = torch.arange(seqs)
    return q, k, v, table, w, (w - hi.double() - mid.double()) / (2 + w)


@pytest.mark.parametrize("cols", [1, 64])
def test_attention_holds_a_bf16_weight_whole(cols):
    """Of w, a weight is off by its argument's two roundings (at most 2 of 2^-24 of
    2 log2(e), as a factor 2^-22), exp2's step (2^-23) and three products' sums at w's
    size (3 (2^-23 + 2^-24)): less than 2^-19 together."""
    q, k, v, table, w, y = cancelling(70, cols)
    got = pc.attention(q.cuda(), k.cuda(), v.cuda(), table.cuda(), torch.full((70,), 2, device="cuda"), scale=1.0)
    ref = y.view(-1, 1, 1).expand(got.shape)
    assert_within(got, ref, rounding(ref, BF) * (1 + 2**-7) + (w / (2 + w)).view(-1, 1, 1) * 2.0**-19)


def test_scores_and_positions_that_overlap_are_declined():
    """Strides of at least a head's slots each, and sequence 1's first head in the place of sequence 0's second."""
    c = Case([40, 40], 4, 2, 64, 16, BF, seed=1)
    over, apart, wrong = (torch.zeros(6 * c.cap, dtype=t, device="cuda").as_strided((2, 2, c.cap), (c.cap, n * c.cap, 1))
                          for t, n in ((torch.float32, 1), (torch.float32, 2), (torch.int32, 1)))
    sp, pos = torch.zeros(c.scores.shape, dtype=torch.int32, device="cuda"), c.slots.clone()
    assert pc.attention(c.q, *c.pools(), c.slots, scores=over) is None
    assert pc.attention(c.q, *c.pools(), c.slots, scores=apart) is not None
    assert pc.evict(*c.pools(), c.slots, over, sp, pos, 20) is None
    assert pc.evict(*c.pools(), c.slots, c.scores, wrong, pos, 20) is None
    rows = torch.zeros(2, 2, 64, dtype=BF, device="cuda")
    assert pc.store(rows, rows, *c.pools(), c.slots, scores=over) is None
    assert not over.any()


def test_calls_of_more_heads_than_a_launch_has_workgroups_are_declined():
    """65535 sequences of 256 heads (2 GB of q): sizes that every check of a tensor lets pass."""
    seqs, nh, hd = 65535, 256, 64
    k = torch.zeros(1, 1, 16, hd, dtype=BF, device="cuda")
    table = torch.zeros(seqs, 1, dtype=torch.int32, device="cuda")
    slots = torch.zeros(seqs, dtype=torch.int64, device="cuda")
    q = torch.empty(seqs, nh, hd, dtype=BF, device="cuda")
    before = pc.stats()["declined"]
    assert pc.attention(q, k, k, table, slots) is None and pc.stats()["declined"] == before + 1
    y = pc.attention(torch.zeros(seqs, 1, hd, dtype=BF, device="cuda"), k, k, table, slots)
    assert y is not None and not y.any()


@pytest.mark.parametrize("lens,track", [([131072], True), ([130941, 5], False), ([261000], False), ([196613, 0, 5], True)])
def test_attention_of_one_kv_head_in_a_thousand_chunks(lens, track):
    """One KV head, which its own chunks must fill the GPU with: 1024, 1023, 1020 and 769 to a sequence."""
    c = Case(lens, 3, 1, 64, 4096, BF, seed=lens[0] % 97, tracked=track)
    before = c.scores.clone() if track else None
    y = pc.attention(c.q, *c.pools(), c.slots, scores=c.scores)
    attention_check(c, y, c.scores, before)


@pytest.mark.parametrize("seqs", [63, 64, 65, 256, 257, 300, 1000])
@pytest.mark.parametrize("tracked", [False, True])
def test_attention_counts_the_chunks_of_many_sequences(seqs, tracked):
    """Tables wide enough to be cut, one sequence a lane of a wave and one to four a
    thread of the workgroup, the last of them uneven; empty ones at both ends, in a
    run of 70 and alone, a few long ones among short ones."""
    g = torch.Generator().manual_seed(seqs)
    lens = torch.randint(0, 25, (seqs,), generator=g).tolist()
    for b, n in zip(torch.randperm(seqs, generator=g).tolist(), (1023, 700, 513, 129, 128, 400)):
        lens[b] = n
    lens[0] = lens[-1] = lens[seqs // 2] = 0
    lens[-2] = 640
    if seqs > 200:
        lens[100:170] = [0] * 70
    c = Case(lens, 4, 2, 64, 16, BF, seed=seqs, cols=64, tracked=tracked)
    before = c.scores.clone() if tracked else None
    y = pc.attention(c.q, *c.pools(), c.slots, scores=c.scores)
    attention_check(c, y, c.scores, before)


@pytest.mark.parametrize("nh,nkv,hd,dtype", [(65, 1, 64, BF), (132, 2, 128, FP), (200, 1, 64, FP)])
@pytest.mark.parametrize("cols", [20, 130])
def test_weights_of_more_query_heads_than_are_gathered_at_once(nh, nkv, hd, dtype, cols):
    """Over 64 query heads a KV head: their weights are added to a score in rounds."""
    c = Case([300, 0, 1, 129, min(cols * 16, 2000)], nh, nkv, hd, 16, dtype, seed=nh, cols=cols)
    before = c.scores.clone()
    y = pc.attention(c.q, *c.pools(), c.slots, scores=c.scores)
    attention_check(c, y, c.scores, before)


@pytest.mark.parametrize("page", [16, 64])
def test_attention_of_pages_that_sequences_share(page):
    """A prefix of pages that three sequences read, one of them with a page twice:
    each gathers weights of its own."""
    c = Case([600, 600, 600], 8, 2, 128, page, FP, seed=page)
    n = 320 // page
    c.table[1, :n] = c.table[2, :n] = c.table[0, :n]
    c.table[2, n] = c.table[2, 1]
    before = c.scores.clone()
    y = pc.attention(c.q, *c.pools(), c.slots, scores=c.scores)
    attention_check(c, y, c.scores, before)


def _longest():
    """One sequence of the most slots there may be, pages in falling order."""
    n, page, hd = 1 << 24, 4096, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(n // page, 1, page, hd, generator=g, device="cuda", dtype=FP) for _ in "kv")
    table = torch.arange(n // page - 1, -1, -1, dtype=torch.int32, device="cuda").view(1, -1)
    return n, page, hd, g, k, v, table


def test_attention_of_the_longest_sequence():
    """2^24 slots, 64 bits on the GPU. The bounds are those of `attention64`."""
    n, page, hd, g, k, v, table = _longest()
    q = torch.randn(1, 2, hd, generator=g, device="cuda", dtype=FP) * 3
    scores = torch.zeros(1, 1, n, device="cuda")
    y = pc.attention(q, k, v, table, torch.tensor([n - 1], device="cuda"), scores=scores)
    K, V = (t.flip(0).reshape(n, hd) for t in (k, v))
    dots, mag = torch.empty(2, n, dtype=torch.float64, device="cuda"), torch.zeros((), dtype=torch.float64, device="cuda")
    step = 1 << 20
    for i in range(0, n, step):
        rows = K[i:i + step].double()
        dots[:, i:i + step] = (rows @ q[0].double().t()).t() * hd**-0.5
        mag = torch.maximum(mag, (rows.abs() @ q[0].double().abs().t()).max() * hd**-0.5)
    w = torch.softmax(dots, 1)
    ref, absolute, total = (torch.zeros(2, hd, dtype=torch.float64, device="cuda") for _ in "yab")
    for i in range(0, n, step):
        rows = V[i:i + step].double()
        ref += w[:, i:i + step] @ rows
        absolute += w[:, i:i + step] @ rows.abs()
        total += rows.abs().sum(0)
    e = 2 * (hd + 4) * 2.0**-24 * mag + 2.0**-20 + 2.0**-23 * (n / 8 / 1024 + 64)  # (1024 chunks' sums, then theirs)
    assert_within(y[0], ref, rounding(ref, FP) * (1 + 2**-7) + absolute * (e + 2.0**-16) + 2.0**-38 * total, "y")
    assert_within(scores[0, 0], w.sum(0), w.sum(0) * (e + 2.0**-23), "scores")


@pytest.mark.parametrize("kind", ["exp", "same"])
def test_evict_of_the_longest_sequence(kind):
    n, page, hd, g, k, v, table = _longest()
    budget, sinks, recent = (1 << 23) + 77, 100, 1000
    s = torch.rand(1, 1, n, generator=g, device="cuda") if kind == "exp" else torch.ones(1, 1, n, device="cuda")
    sp = torch.arange(n, dtype=torch.int32, device="cuda").view(1, 1, n).clone()
    key = s[0, 0].clone()
    key[:sinks] = key[n - recent:] = math.inf
    kept = torch.zeros(n, dtype=torch.bool, device="cuda")
    kept[torch.sort(key, descending=True, stable=True).indices[:budget]] = True
    src = kept[budget:].nonzero()[:, 0] + budget
    dst = (~kept[:budget]).nonzero()[:, 0]
    want = [t.flip(0).reshape(n, hd) for t in (k, v)] + [s[0, 0].clone(), sp[0, 0].clone()]
    for t in want:
        t[dst] = t[src]
    assert pc.evict(k, v, table, torch.tensor([n - 1], device="cuda"), s, sp, torch.tensor([n - 1], device="cuda"), budget,
                    sinks=sinks, recent=recent)
    assert len(src) and torch.equal(s[0, 0], want[2]) and torch.equal(sp[0, 0], want[3])
    for t, w in zip((k, v), want):
        assert torch.equal(t.flip(0).reshape(n, hd).view(torch.int16), w.view(torch.int16))


# --------------------------------------------------------------- the eviction


@pytest.mark.parametrize("n,budget,cols", [(103, 100, 8), (140, 100, 9), (700, 300, 44), (9000, 8000, 563), (2500, 1200, 157)])
def test_evict_moves_nothing_from_or_into_a_hole(n, budget, cols):
    """A hole among the slots below the budget and one above it, in every variant (a
    few rows over, moved while ranking, listed, in parts): each move between pages
    is whole, and of the others neither the row nor its score or position goes."""
    c = Case([n], 2, 2, 64, 16, BF, seed=n, cols=cols)
    g = torch.Generator().manual_seed(n)
    s = torch.rand(1, 2, c.cap, generator=g)
    low, high = 2, budget // 16 + 1 if n - budget > 16 else (n - 1) // 16
    s[:, :, 16 * low:16 * low + 3] = -1.0  # some of the free slots are the hole's, and some movers
    s[:, :, budget:][:, :, :2] += 2.0
    sp = torch.arange(c.cap, dtype=torch.int32).expand(1, 2, -1).contiguous()
    moves = [evict_ref(s[0, h].numpy(), sp[0, h].numpy(), n, n - 1, budget, 0, 0) for h in range(2)]
    c.table[0, low] = c.table[0, high] = -1
    holes = [sum(src // 16 == high or dst // 16 == low for src, dst in m) for m in moves]
    assert all(holes), holes
    k, v, s1, sp1 = c.k.clone(), c.v.clone(), s.clone(), sp.clone()
    table = c.table.cpu().tolist()[0]
    for h, m in enumerate(moves):
        for src, dst in m:
            p, q = table[src // 16], table[dst // 16]
            if p < 0 or q < 0:
                continue
            for t in (k, v):
                t[q, h, dst % 16] = t[p, h, src % 16]
            s1[0, h, dst], sp1[0, h, dst] = s[0, h, src], sp[0, h, src]
    s, sp = s.cuda(), sp.cuda()
    assert pc.evict(*c.pools(), c.slots, s, sp, torch.tensor([n - 1], device="cuda"), budget)
    assert torch.equal(s.cpu(), s1) and torch.equal(sp.cpu(), sp1)
    assert np.array_equal(bits(c.k), bits(k)) and np.array_equal(bits(c.v), bits(v))


@pytest.mark.parametrize("cap", [2048, 2064])
@pytest.mark.parametrize("budget", [257, 1024, -257])
@pytest.mark.parametrize("hd,dtype", [(64, FP), (128, BF)])
@pytest.mark.parametrize("kind", ["exp", "few", "same", "every"])
def test_evict_lists_the_moves_of_whole_caches(cap, budget, hd, dtype, kind):
    """More moves than the ranking workgroup does by itself, at the last width of its
    256-thread form and the first of its 1024-thread one."""
    budget = budget if budget > 0 else cap + budget
    lens = [cap, cap - 1, budget, budget + 1, budget + 4, budget + 5, 0, 1, (cap + budget) // 2]
    c, s, sp = _tracked(lens, 2, hd, 16, dtype, seed=cap + budget, kind=kind, cols=cap // 16)
    assert pc.evict_work(len(lens), 2, cap // 16, 16, budget) > 0
    assert _evict(c, s, sp, sp.amax((1, 2)).long(), budget, sinks=3, recent=17)


@pytest.mark.parametrize("n,budget", [(700, 300), (3000, 1000), (9000, 2000)])
def test_captured_evict_in_every_form(n, budget):
    """Moves listed by 256 and by 1024 threads and in parts, replayed at other lengths: a workspace that
    earlier replays have used."""
    c, s, sp = _tracked([n, n], 2, 64, 16, BF, seed=n)
    first = [t.clone() for t in (c.k, c.v, s, sp)]
    pos = sp.amax((1, 2)).long()
    work = torch.full((pc.evict_work(2, 2, c.table.shape[1], 16, budget),), -1, dtype=torch.int32, device="cuda")
    call = lambda: pc.evict(*c.pools(), c.slots, s, sp, pos, budget, sinks=2, recent=16, work=work)  # noqa: E731
    assert len(work) and call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for lens in ((n, budget + 1), (5, n), (budget, budget + 40), (n - 1, n), (0, 1), (budget + 2, n // 2)):
        for a, b in zip((c.k, c.v, s, sp), first):
            a.copy_(b)
        c.slots.copy_(torch.tensor([x - 1 for x in lens]))
        g.replay()
        k, v, s1, sp1 = (t.clone() for t in first)
        assert pc.evict(k, v, c.table, c.slots, s1, sp1, pos, budget, sinks=2, recent=16)
        torch.cuda.synchronize()
        assert torch.equal(s, s1) and torch.equal(sp, sp1), lens
        assert np.array_equal(bits(c.k), bits(k)) and np.array_equal(bits(c.v), bits(v)), lens


# ------------------------------------------------------------------ the table


def test_the_page_table_waits_for_nothing():
    """Streams that grow page by page, are cut and end while the GPU is still busy
    with what was queued before: no call waits, and the tensors end up as the host has them."""
    table = pc.PageTable(24, 400, 24 * 12, 16)
    cache = pc.PagedKVCache(table, 1, 64)
    rows = torch.zeros(20, 1, 64, dtype=BF, device="cuda")
    a = torch.randn(4096, 4096, device="cuda")
    states = []
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        for _ in range(20):
            a = a @ a
        for i in range(20):
            assert table.admit(14 + i) == i
        assert cache.store(3, rows[:17], rows[:17])
        for step in range(90):
            table.step()
            if step in (40, 70):
                table.evicted(30)
            if step == 50:
                table.release(5)
                assert table.admit(33) == 5
            states.append((table.block_table.clone(), table.slots.clone(), [list(x) for x in table._held], list(table._rows)))
    finally:
        torch.cuda.set_sync_debug_mode("default")
    for t, slots, held, n in states:
        assert t.tolist() == [x + [-1] * (t.shape[1] - len(x)) for x in held] and slots.tolist() == [x - 1 for x in n]


# ------------------------------------------------------------------ the block


def _streams(nkv, hd, lens, dtype, layers=1, **kw):
    """A table with a stream of each length, and `layers` caches with seeded rows."""
    table = pc.PageTable(len(lens) + 1, 128, 60, 16)
    caches = [pc.PagedKVCache(table, nkv, hd, dtype=dtype, **kw) for _ in range(layers)]
    for b, n in enumerate(lens):
        assert table.admit(n) == b
        for i, cache in enumerate(caches):
            g = torch.Generator().manual_seed(100 * n + i)
            assert cache.store(b, *(torch.randn(n, nkv, hd, generator=g).to(dtype).cuda() for _ in "kv"))
    return table, caches


def _same(a, b, what):
    for name in ("k_pages", "v_pages", "scores", "slot_pos"):
        x, y = getattr(a, name), getattr(b, name)
        if x is None and y is None:
            continue
        assert torch.equal(x.view(torch.int16), y.view(torch.int16)), (what, name)


@pytest.mark.parametrize("lens,dtype", [((70,), BF), ((3, 47, 17, 64), FP), (tuple(range(1, 20)), BF)])
@pytest.mark.parametrize("tracked", [False, True])
def test_decode_batch_is_its_parts(lens, dtype, tracked):
    """The block on a cache, tracked or not, against its steps called one by one on
    a twin, bit for bit; of those steps the rows, the attention and the gathered
    weights against 64 bits."""
    from tests.test_fused_gpu import _block
    from ttspipe_amd import fusedlayer, fusedops, nf4gemv

    assert nf4gemv.install() and fusedops.install()
    block, _ = _block(dtype, True, seed=len(lens))
    a, ff, an, fn = block.attention, block.feed_forward, block.attention_norm, block.ffn_norm
    nh, nkv, hd, rows = 4, 2, 128, len(lens) + 1
    (ta, (ca,)), (tb, (cb,)) = (_streams(nkv, hd, lens, dtype, tracked=tracked) for _ in "ab")
    ta.step(), tb.step()
    x = torch.randn(rows, 1, 512, generator=torch.Generator().manual_seed(7)).to(dtype).cuda()
    freqs = _freqs(128, hd)
    got = fusedlayer.decode_batch(block, x, freqs, ca)
    # the steps
    if rows <= nf4gemv.FUSED_MAX_ROWS:
        qkv = nf4gemv.matmul_fused(a.wqkv, x, norm_weight=an.weight, eps=an.eps)
    else:
        qkv = nf4gemv.matmul(a.wqkv, fusedops.rms_norm(x, an.weight, an.eps))
    qkv = qkv.view(rows, -1)
    q = cb.qk_rope_kv(qkv, nh, freqs, q_weight=a.q_norm.weight, k_weight=a.k_norm.weight, eps=a.q_norm.eps)
    head = qkv.view(rows, -1, hd)
    for b, n in enumerate(lens):
        ref, bound = _rope64(head[b, :nh], a.q_norm.weight, freqs[n], 1e-6)
        assert_within(q[b], ref, rounding(ref, dtype) * (1 + 2**-7) + bound, f"q {b}")
        at, off = int(tb.block_table[b, n // 16]), n % 16
        ref, bound = _rope64(head[b, nh:nh + nkv], a.k_norm.weight, freqs[n], 1e-6)
        assert_within(cb.k_pages[at, :, off], ref, rounding(ref, dtype) * (1 + 2**-7) + bound, f"k {b}")
        assert torch.equal(cb.v_pages[at, :, off], head[b, nh + nkv:])
    before = cb.scores.clone() if tracked else None
    y = cb.attention(q)
    ref, p, yb, pb = attention64(q, cb.k_pages, cb.v_pages, tb.block_table, tb.slots)
    assert_within(y, ref, rounding(ref, dtype) * (1 + 2**-7) + yb, "y")
    if tracked:
        new = before.double().cpu() + p
        assert_within(cb.scores, new, new.abs() * 2.0**-24 + pb, "scores")
        for b, n in enumerate(lens):
            assert (ca.slot_pos[b, :, : n + 1].cpu() == torch.arange(n + 1)).all()
    y = y.view(rows, 1, nh * hd)
    hh = nf4gemv.matmul_norm(a.wo, y, fn.weight, fn.eps, epi=nf4gemv.EPI_RESIDUAL, operand=x)
    h, hn = hh if hh is not None else (nf4gemv.matmul(a.wo, y, epi=nf4gemv.EPI_RESIDUAL, operand=x), None)
    h, u = h.view(x.shape), None
    if hn is None and rows <= nf4gemv.FUSED_MAX_ROWS:
        u = nf4gemv.matmul_fused(ff.w1, h, norm_weight=fn.weight, eps=fn.eps, module3=ff.w3)
    if u is None:
        hn = fusedops.rms_norm(h, fn.weight, fn.eps) if hn is None else hn.view(x.shape)
        u = nf4gemv.matmul_swiglu(ff.w1, ff.w3, hn)
        if u is None:
            u = nf4gemv.matmul(ff.w3, hn, epi=nf4gemv.EPI_SILU_GATE, operand=nf4gemv.matmul(ff.w1, hn))
    want = nf4gemv.matmul(ff.w2, u, epi=nf4gemv.EPI_RESIDUAL, operand=h)
    assert np.array_equal(bits(got).reshape(-1), bits(want).reshape(-1))
    _same(ca, cb, "cache")


def test_captured_decode_batch_equals_eager_steps():
    """Two blocks on tracked caches and their eviction in one graph, replayed as the
    streams grow past the budget and one ends, the table's own steps between."""
    from tests.test_fused_gpu import _block
    from ttspipe_amd import fusedlayer, fusedops, nf4gemv

    assert nf4gemv.install() and fusedops.install()
    blocks = [_block(BF, True, seed=i)[0] for i in (3, 4)]
    budget, freqs = 30, _freqs(128, 128)
    (ta, la), (tb, lb) = (_streams(2, 128, (20, 1, 29), BF, layers=2, tracked=True) for _ in "ab")

    def step(caches, x):
        for block, cache in zip(blocks, caches):
            x = fusedlayer.decode_batch(block, x, freqs, cache)
        for cache in caches:
            assert cache.evict(budget, sinks=1, recent=6)
        return x

    g = torch.Generator().manual_seed(2)
    xs = [torch.randn(4, 1, 512, generator=g).to(BF).cuda() for _ in range(18)]
    x = xs[0].clone()
    ta.step(), tb.step()
    assert np.array_equal(bits(step(la, x)), bits(step(lb, xs[0])))
    ta.evicted(budget), tb.evicted(budget)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(la, x)
    for i, new in enumerate(xs[1:]):
        if i == 7:
            ta.release(2), tb.release(2)
        ta.step(), tb.step()
        x.copy_(new)
        graph.replay()
        assert np.array_equal(bits(got), bits(step(lb, new))), i
        for p, q in zip(la, lb):
            _same(p, q, i)
        ta.evicted(budget), tb.evicted(budget)
    assert ta.rows(0) == budget and ta.rows(1) == 19 and ta.rows(2) == 0
