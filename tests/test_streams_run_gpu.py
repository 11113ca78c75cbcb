"""Streams that share a voice's prompt, slide through a window and have their logits
penalised, together as a server's decode uses them (GPU): the paged cache's
bookkeeping and kernels against 64 bits at every step, the transformer block on
such caches, prompts through a window, and a captured step against an eager one."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.gpuutil import bits
from tests.pageddata import assert_within, rounding
from tests.spandata import spans64
from tests.test_paged_gpu import _freqs
from tests.test_penalize_gpu import check as penalized_check
from ttspipe_amd import fastpath, fusedsample
from ttspipe_amd import pagedcache as pc

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _block(dtype, seed):
    from tests.test_fused_gpu import _block as make
    from ttspipe_amd import fusedops, nf4gemv

    assert nf4gemv.install() and fusedops.install()
    return make(dtype, True, seed=seed)[0]


def _rel(a, b):
    a, b = a.double(), b.double()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("dtype,page,window,sinks", [(BF, 16, None, 0), (FP, 32, None, 0), (BF, 16, 24, 3)])
def test_streams_behind_prefixes_that_come_and_go(dtype, page, window, sinks):
    """Voices admitted and released, streams behind them and without one, pages
    given back by the window, each step's attention against 64 bits."""
    nh, nkv, hd, seqs = 8, 2, 128, 4
    g = torch.Generator().manual_seed(page)
    table = pc.PageTable(seqs, 120, 60, page, prefixes=2, max_prefix=200)
    cache = pc.PagedKVCache(table, nkv, hd, dtype=dtype, window=window, sinks=sinks)
    freqs = _freqs(512, hd)

    def rows(n):
        return torch.randn(n, nkv, hd, generator=g).to(dtype).cuda(), torch.randn(n, nkv, hd, generator=g).to(dtype).cuda()

    def voice(n):
        p = table.admit_prefix(n)
        k, v = rows(n)
        assert cache.store_prefix(p, k[:n // 2], v[:n // 2]) and cache.store_prefix(p, k[n // 2:], v[n // 2:], start=n // 2)
        return p

    def stream(n, p=None):
        b = table.admit(n, prefix=p)
        assert cache.store(b, *rows(n))
        return b

    a, b = voice(150), voice(33)
    assert [stream(20, a), stream(7, b), stream(1), stream(12, a)] == [0, 1, 2, 3]
    for step in range(60):
        if step == 15:
            table.release(1)
            table.release_prefix(b)
            b = voice(90)
            assert stream(30, b) == 1
        if step == 30:
            table.release(2)
            assert stream(3, b) == 2
        table.step()
        qkv = (torch.randn(seqs, (nh + 2 * nkv) * hd, generator=g) * 2).to(dtype).cuda()
        q = cache.qk_rope_kv(qkv, nh, freqs)
        y = cache.attention(q)
        for s in range(seqs):
            assert int(table.positions[s]) == table.first_position(s) + table.rows(s) - 1
        ref, _, yb, _ = spans64(q, cache.k_pages, cache.v_pages, table.block_table, table.slots, window=window, sinks=sinks,
                                prefix=table.prefix)
        assert_within(y, ref, rounding(ref, dtype) * (1 + 2**-7) + yb, f"step {step}")
        if window is not None:
            table.slide(window, sinks)
    if window is not None:
        assert (table.block_table[0, :4] < 0).any()


def test_decode_batch_behind_a_prefix_is_decode_batch_with_its_rows_copied():
    block = _block(BF, 3)
    x = torch.randn(3, 1, 512, device="cuda").to(BF)
    freqs = _freqs(512, 128)
    voice = [torch.randn(100, 2, 128, device="cuda").to(BF) for _ in "kv"]
    own = [[torch.randn(n, 2, 128, device="cuda").to(BF) for _ in "kv"] for n in (5, 40)]
    shared = pc.PageTable(3, 100, 40, 16, prefixes=1)
    c1 = pc.PagedKVCache(shared, 2)
    assert c1.store_prefix(shared.admit_prefix(100), *voice)
    copied = pc.PageTable(3, 200, 40, 16)
    c2 = pc.PagedKVCache(copied, 2)
    for k, v in own:
        assert c1.store(shared.admit(len(k), prefix=0), k, v)
        assert c2.store(copied.admit(100 + len(k)), torch.cat([voice[0], k]), torch.cat([voice[1], v]))
    shared.step(), copied.step()
    assert torch.equal(shared.positions, copied.positions)
    from ttspipe_amd import fusedlayer

    y1, y2 = fusedlayer.decode_batch(block, x, freqs, c1), fusedlayer.decode_batch(block, x, freqs, c2)
    assert _rel(y1, y2) < 5e-3 and _rel(y1[2], y2[2]) < 5e-3  # (the last row holds no stream)


def test_decode_batch_through_a_window_is_decode_batch_over_the_rows_it_sees():
    from ttspipe_amd import fusedlayer

    block = _block(FP, 4)
    window, sinks, lens = 30, 4, (100, 12)
    x = torch.randn(2, 1, 512, device="cuda").to(FP)
    freqs = _freqs(512, 128)
    t1, t2 = pc.PageTable(2, 200, 40, 16), pc.PageTable(2, 200, 40, 16)
    c1, c2 = pc.PagedKVCache(t1, 2, dtype=FP, window=window, sinks=sinks), pc.PagedKVCache(t2, 2, dtype=FP)
    for n in lens:
        k, v = (torch.randn(n, 2, 128, device="cuda").to(FP) for _ in "kv")
        assert c1.store(t1.admit(n), k, v)
        seen = torch.tensor([j for j in range(n) if j < sinks or j > n - window], device="cuda")  # (the step's token is row n)
        assert c2.store(t2.admit(len(seen)), k[seen], v[seen])
    t1.slide(window, sinks)
    t1.step(), t2.step()
    t2.positions.copy_(t1.positions)
    y1, y2 = fusedlayer.decode_batch(block, x, freqs, c1), fusedlayer.decode_batch(block, x, freqs, c2)
    assert _rel(y1, y2) < 5e-3


@pytest.mark.parametrize("n,start,window,sinks", [(40, 0, 9, 2), (70, 60, 50, 4), (2, 100, 30, 0), (33, 20, 1000, 1)])
def test_prefill_block_through_a_window(n, start, window, sinks):
    """Against the same block with the window's mask."""
    from ttspipe_amd import fusedlayer

    block = _block(BF, 5)
    kv = block.attention.kv_cache
    past = [torch.randn_like(kv.k_cache) for _ in "kv"]
    x = torch.randn(1, n, 512, device="cuda").to(BF)
    freqs, pos = _freqs(512, 128)[start:start + n].contiguous(), torch.arange(start, start + n, device="cuda")
    width = start + n
    pad = -(-width // 16) * 16
    mask = torch.zeros(1, 1, n, pad, dtype=torch.bool, device="cuda")
    mask[..., :width] = fastpath.window_mask(pos, width, window, sinks)
    got = []
    for kw, m in ((dict(window=window, sinks=sinks), mask[..., :width]), (dict(), mask[..., :width])):
        kv.k_cache.copy_(past[0]), kv.v_cache.copy_(past[1])
        got.append(fusedlayer.prefill_block(block, x, freqs, m, pos, **kw))
        got.append(kv.k_cache.clone())
    assert _rel(got[0], got[2]) < 5e-3 and torch.equal(got[1], got[3])
    for kw in (dict(window=5, causal=True), dict(window=0), dict(sinks=2)):
        with pytest.raises(ValueError):
            fusedlayer.prefill_block_chain(block, x, freqs, mask[..., :width], pos, **kw)


def test_a_servers_step_captured_and_eager():
    """Two layers behind a shared prompt, a head, penalties after each stream's
    tokens and a draw a stream: a captured step, replayed between the table's own
    steps, against an eager one bit for bit; the logits against 64 bits."""
    from ttspipe_amd import fusedlayer

    blocks = [_block(BF, s) for s in (6, 7)]
    seqs, vocab, steps = 3, 700, 12
    g = torch.Generator().manual_seed(8)
    freqs = _freqs(512, 128)
    head = (torch.randn(512, vocab, generator=g) * 0.2).to(BF).cuda()
    embed = torch.randn(vocab, 512, generator=g).to(BF).cuda()
    rep, freq, pres = (torch.full((seqs,), v, device="cuda") for v in (1.3, 0.1, 0.4))
    mask = fusedsample.pack_mask(torch.rand(vocab, generator=g) < 0.7).cuda()
    temp, topp, topk = torch.full((1,), 0.8, dtype=BF, device="cuda"), torch.full((1,), 0.9, dtype=BF, device="cuda"), torch.tensor([20], device="cuda")
    uniforms = torch.rand(steps, seqs, vocab, generator=g).cuda()

    class Server:
        def __init__(self):
            r = torch.Generator().manual_seed(9)
            self.table = pc.PageTable(seqs, 100, 40, 16, prefixes=1)
            self.caches = [pc.PagedKVCache(self.table, 2, window=16, sinks=2) for _ in blocks]
            rows = lambda n: [torch.randn(n, 2, 128, generator=r).to(BF).cuda() for _ in "kv"]  # noqa: E731
            p = self.table.admit_prefix(70)
            first = [self.table.admit(n, prefix=q) for n, q in ((20, p), (3, p), (11, None))]
            for c in self.caches:
                assert c.store_prefix(p, *rows(70))
                for b, n in zip(first, (20, 3, 11)):
                    assert c.store(b, *rows(n))
            self.tokens = torch.zeros(seqs, 1, dtype=torch.int64, device="cuda")
            self.history = torch.full((seqs, 64), -1, dtype=torch.int32, device="cuda")
            self.lengths = torch.zeros(seqs, dtype=torch.int32, device="cuda")
            self.uniform = torch.zeros(seqs, vocab, device="cuda")
            self.raw = self.logits = None

        def step(self):
            x = embed[self.tokens]
            for block, cache in zip(blocks, self.caches):
                x = fusedlayer.decode_batch(block, x, freqs, cache)
            self.raw = x.view(seqs, -1) @ head
            self.logits = fusedsample.penalize(self.raw, self.history, lengths=self.lengths, repetition=rep, frequency=freq,
                                               presence=pres, mask=mask)
            drawn = [fusedsample.sample(self.logits[b], temp, topp, topk, uniform=self.uniform[b]) for b in range(seqs)]
            tokens = torch.stack(drawn).view(seqs, 1)
            self.history.scatter_(1, self.lengths.view(seqs, 1).long(), tokens)
            self.lengths += 1
            self.tokens.copy_(tokens)

        def advance(self, i):
            self.table.slide(16, 2)
            self.table.step()
            self.uniform.copy_(uniforms[i])

    one, two = Server(), Server()
    for s in (one, two):
        s.advance(0)
        s.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    one.advance(1)
    with torch.cuda.graph(graph):
        one.step()
    for i in range(1, steps):
        if i > 1:
            one.advance(i)
        two.advance(i)
        before = two.history.clone(), two.lengths.clone()
        graph.replay()
        two.step()
        torch.cuda.synchronize()
        assert np.array_equal(bits(one.logits), bits(two.logits)), i
        assert torch.equal(one.tokens, two.tokens) and torch.equal(one.history, two.history), i
        penalized_check(two.logits, two.raw, *before, rep, freq, pres, None, mask)
        allowed = (mask.long()[two.tokens.view(-1) // 32] >> (two.tokens.view(-1) % 32)) & 1
        assert allowed.all()
    assert len(torch.unique(two.history[:, :steps])) > 3


def test_other_streams_than_the_tensors_own():
    """Calls on a side stream after the tensors were made on the default one, and
    back: the results are the default stream's."""
    from tests.spandata import PrefixCase

    c = PrefixCase([200, 7, 90], [300], [0, 0, -1], 8, 2, 128, 16, BF, seed=60, tracked=False)
    want = pc.attention(c.q, *c.pools(), c.slots, prefix=c.prefix(), window=50, sinks=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pc.attention(c.q, *c.pools(), c.slots, prefix=c.prefix(), window=50, sinks=3)
    torch.cuda.current_stream().wait_stream(side)
    assert np.array_equal(bits(want), bits(got))
