"""The paged cache's operators together, as a server's decode uses them (GPU):
several streams that come and go, each step writing a row per stream, attending
and, past a budget, evicting - against a plain restatement in 64 bits that
keeps each head's rows in lists; the same steps captured in a graph against
eager ones, bit for bit; and the transformer block on a paged cache
(`fusedlayer.decode_batch`) against the block's definition in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.gpuutil import bits
from tests.pageddata import assert_within, attention64, evict_ref, rounding
from tests.test_paged_gpu import _freqs, _rope64
from ttspipe_amd import pagedcache as pc

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


class Plain:
    """One layer's cache as lists: rows[seq][head] of [k, v, score, position], in slot order."""

    def __init__(self, seqs, nkv):
        self.rows = [[[] for _ in range(nkv)] for _ in range(seqs)]

    def evict(self, positions, budget, sinks, recent):
        for b, heads in enumerate(self.rows):
            for rows in heads:
                n = len(rows)
                moves = evict_ref([r[2] for r in rows], [r[3] for r in rows], n, positions[b], budget, sinks, recent)
                for src, dst in moves:
                    rows[dst] = rows[src]
                del rows[budget:]


@pytest.mark.parametrize("nh,nkv,hd,dtype,page", [(8, 2, 128, BF, 16), (6, 3, 64, FP, 32)])
def test_streams_that_come_and_go(nh, nkv, hd, dtype, page):
    """Prompts stored from contiguous rows, steps, evictions every step past
    the budget, a stream released and another admitted into its pages."""
    g = torch.Generator().manual_seed(nh)
    budget, sinks, recent, steps = 48, 2, 8, 40
    table = pc.PageTable(3, 80, 12 if page == 16 else 7, page)
    cache = pc.PagedKVCache(table, nkv, hd, dtype=dtype, tracked=True)
    freqs = _freqs(256, hd)
    qw, kw = ((torch.rand(hd, generator=g) + 0.5).to(dtype).cuda() for _ in "qk")
    plain = Plain(3, nkv)

    def admit(n):
        seq = table.admit(n)
        k, v = (torch.randn(1, nkv, n + 3, hd, generator=g).to(dtype).cuda() for _ in "kv")
        assert cache.store(seq, k[0, :, :n].transpose(0, 1), v[0, :, :n].transpose(0, 1))
        for h in range(nkv):
            plain.rows[seq][h] = [[k[0, h, j].cpu(), v[0, h, j].cpu(), 0.0, j] for j in range(n)]
        return seq

    assert admit(30) == 0 and admit(5) == 1
    for step in range(steps):
        if step == 15:
            table.release(0)
            plain.rows[0] = [[] for _ in range(nkv)]
            assert admit(47) == 0
        if step == 20:
            assert admit(1) == 2
        table.step()
        qkv = (torch.randn(3, (nh + 2 * nkv) * hd, generator=g) * 2).to(dtype).cuda()
        q = cache.qk_rope_kv(qkv, nh, freqs, q_weight=qw, k_weight=kw, eps=1e-6)
        y = cache.attention(q)
        # what was written, and the attention over it
        pos = table.positions.tolist()
        x = qkv.view(3, -1, hd)
        scores = cache.scores.cpu()
        for b in range(3):
            rows = plain.rows[b]
            if pos[b] < 0:
                assert not rows[0] and not y[b].any() and not q[b].any()
                continue
            cs = freqs[pos[b]]
            ref, bound = _rope64(x[b, :nh], qw, cs, 1e-6)
            assert_within(q[b], ref, rounding(ref, dtype) * (1 + 2**-7) + bound, f"step {step} q {b}")
            j = len(rows[0])
            assert j == table.rows(b) - 1 == int(table.slots[b])
            at, off = int(table.block_table[b, j // page]), j % page
            ref, bound = _rope64(x[b, nh:nh + nkv], kw, cs, 1e-6)
            assert_within(cache.k_pages[at, :, off], ref, rounding(ref, dtype) * (1 + 2**-7) + bound, f"step {step} k {b}")
            for h in range(nkv):
                # (the kernel's own K row from here on: its rounding is checked above)
                rows[h].append([cache.k_pages[at, h, off].cpu(), x[b, nh + nkv + h].cpu(), 0.0, pos[b]])
                K, V = torch.stack([r[0] for r in rows[h]]), torch.stack([r[1] for r in rows[h]])
                n, group = len(rows[h]), nh // nkv
                heads = slice(h * group, (h + 1) * group)
                ref, p, yb, pb = attention64(q[b:b + 1, heads], K.view(1, 1, n, hd), V.view(1, 1, n, hd),
                                             torch.zeros(1, 1, dtype=torch.int32), torch.tensor([n - 1]))
                assert_within(y[b:b + 1, heads], ref, rounding(ref, dtype) * (1 + 2**-7) + yb, f"step {step} y {b} {h}")
                new = torch.tensor([r[2] for r in rows[h]], dtype=torch.float64) + p[0, 0]
                got = scores[b, h, :n]
                assert_within(got, new, new.abs() * 2.0**-24 + pb[0, 0], f"step {step} scores {b} {h}")
                for r, s in zip(rows[h], got.tolist()):
                    r[2] = s
        if max(table.rows(b) for b in range(3)) > budget:
            assert cache.evict(budget, sinks=sinks, recent=recent)
            plain.evict(pos, budget, sinks, recent)
            table.evicted(budget)
            for b in range(3):
                for h in range(nkv):
                    n = len(plain.rows[b][h])
                    assert n == table.rows(b)
                    assert cache.slot_pos[b, h, :n].tolist() == [r[3] for r in plain.rows[b][h]]
                    assert cache.scores[b, h, :n].tolist() == [r[2] for r in plain.rows[b][h]]
    assert max(table.rows(b) for b in range(3)) == budget


def test_captured_steps_equal_eager_ones():
    """Write, attention and eviction of two layers in one graph, replayed as the
    streams grow past the budget, with the table's own steps between."""
    nh, nkv, hd, budget = 8, 2, 128, 40
    g = torch.Generator().manual_seed(1)
    freqs = _freqs(128, hd)
    qkv = torch.zeros(4, (nh + 2 * nkv) * hd, dtype=BF, device="cuda")
    rows = [(torch.randn(4, (nh + 2 * nkv) * hd, generator=g) * 2).to(BF).cuda() for _ in range(24)]

    def make():
        table = pc.PageTable(4, 64, 16, 16)
        layers = [pc.PagedKVCache(table, nkv, hd, tracked=True) for _ in range(2)]
        for n in (25, 1, 38):
            seq = table.admit(n)
            for i, layer in enumerate(layers):
                k = torch.randn(n, nkv, hd, generator=torch.Generator().manual_seed(10 * n + i)).to(BF).cuda()
                assert layer.store(seq, k, -k)
        return table, layers

    def step(layers, x):
        out = []
        for layer in layers:
            out.append(layer.attention(layer.qk_rope_kv(x, nh, freqs)))
            assert layer.evict(budget, sinks=1, recent=6)
        return out

    (ta, la), (tb, lb) = make(), make()
    qkv.copy_(rows[0])
    ta.step(), tb.step()
    first = step(la, qkv), step(lb, rows[0])
    for p, q in zip(*first):
        assert np.array_equal(bits(p), bits(q))
    ta.evicted(budget), tb.evicted(budget)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(la, qkv)
    for i, r in enumerate(rows[1:]):
        if i == 9:
            ta.release(1), tb.release(1)
        ta.step(), tb.step()
        qkv.copy_(r)
        graph.replay()
        want = step(lb, r)
        for a, b in zip(la, lb):
            for name in ("k_pages", "v_pages", "scores", "slot_pos"):
                x, y = getattr(a, name), getattr(b, name)
                assert torch.equal(x.view(torch.int16) if x.dtype == BF else x, y.view(torch.int16) if y.dtype == BF else y), (i, name)
        for p, q in zip(got, want):
            assert np.array_equal(bits(p), bits(q)), i
        ta.evicted(budget), tb.evicted(budget)
    assert ta.rows(0) == ta.rows(2) == budget and ta.rows(1) == 0


# ------------------------------------------------------------------ the block


def _weights(layers):
    from oracle import oracle as o
    from tests.nf4data import dequant_numpy

    return {n: o.to_f32(dequant_numpy(L, o.DT_BF16), o.DT_BF16).reshape(L["M"], L["K"]).astype(np.float64)
            for n, L in layers.items()}


@pytest.mark.parametrize("qk_norm", [True, False])
@pytest.mark.parametrize("lens", [(70,), (3, 200), (1, 64, 65, 130, 17), tuple(range(1, 41))])
def test_decode_batch_matches_the_blocks_definition(qk_norm, lens):
    """Each sequence's output and its new K/V row against `refblock`, whose
    roundings the block keeps except one of q and k, within the bar of the
    prefill block against it (2e-2 of the norm); the caches' other rows, and
    what stands behind the last sequence, stay."""
    from tests.refblock import block_fp64, rel_norm
    from tests.test_fused_gpu import _block
    from ttspipe_amd import fusedlayer, fusedops, nf4gemv

    assert nf4gemv.install() and fusedops.install()
    block, layers = _block(BF, qk_norm, seed=len(lens))
    nh, nkv, hd, D = 4, 2, 128, 512
    B = len(lens) + 1  # the last row of the table holds nothing
    table = pc.PageTable(B, 256, 200, 16)
    cache = pc.PagedKVCache(table, nkv, hd)
    g = torch.Generator().manual_seed(len(lens))
    past = []
    for n in lens:
        k, v = (torch.randn(n, nkv, hd, generator=g).to(BF).cuda() for _ in "kv")
        seq = table.admit(n)
        assert cache.store(seq, k, v)
        past.append((k, v))
    table.step()
    x = torch.randn(B, 1, D, generator=g).to(BF).cuda()
    freqs = _freqs(256, hd)
    k0, v0 = cache.k_pages.clone(), cache.v_pages.clone()
    before = fusedlayer.stats()["batch"]
    out = fusedlayer.decode_batch(block, x, freqs, cache)
    assert out is not None and fusedlayer.stats()["batch"] == before + 1 and out.shape == x.shape
    W = _weights(layers)
    a = block.attention
    norms = {"attention_norm": block.attention_norm.weight, "ffn_norm": block.ffn_norm.weight}
    if qk_norm:
        norms |= {"q_norm": a.q_norm.weight, "k_norm": a.k_norm.weight}
    norms = {n: w.detach().double().cpu().numpy() for n, w in norms.items()}
    rnd = lambda t: torch.from_numpy(t).to(BF).double().numpy()  # noqa: E731
    for b, n in enumerate(lens):
        kc, vc = (torch.cat([t, torch.zeros(1, nkv, hd, dtype=BF, device="cuda")]).double().cpu().numpy().transpose(1, 0, 2).copy()
                  for t in past[b])
        ref, kr, vr = block_fp64(W, norms, x[b].double().cpu().numpy(), freqs[n:n + 1].double().cpu().numpy(), kc, vc, [n],
                                 nh, nkv, qk_norm, rnd=rnd)
        assert rel_norm(out[b].double().cpu().numpy(), ref) < 2e-2
        at, off = int(table.block_table[b, n // 16]), n % 16
        assert rel_norm(cache.k_pages[at, :, off].double().cpu().numpy(), kr[0]) < 2e-2
        assert rel_norm(cache.v_pages[at, :, off].double().cpu().numpy(), vr[0]) < 2e-2
        k0[at, :, off], v0[at, :, off] = cache.k_pages[at, :, off], cache.v_pages[at, :, off]
    assert np.array_equal(bits(k0), bits(cache.k_pages)) and np.array_equal(bits(v0), bits(cache.v_pages))
    assert torch.isfinite(out).all()


def test_decode_batch_of_one_is_close_to_the_decode_block():
    from tests.test_fused_gpu import _block
    from ttspipe_amd import fusedlayer, fusedops, nf4gemv

    assert nf4gemv.install() and fusedops.install()
    block, _ = _block(FP, True, seed=9)
    kc, vc = block.attention.kv_cache.k_cache, block.attention.kv_cache.v_cache
    kc.normal_(), vc.normal_()
    table = pc.PageTable(1, 256, 16, 16)
    cache = pc.PagedKVCache(table, 2, dtype=FP)
    assert table.admit(100) == 0 and cache.store(0, kc[0, :, :100].transpose(0, 1), vc[0, :, :100].transpose(0, 1))
    table.step()
    freqs = _freqs(256, 128)
    x = torch.randn(1, 1, 512, device="cuda").to(FP)
    ip = torch.tensor([100], device="cuda")
    mask = torch.ones(1, 1, 1, 256, dtype=torch.bool, device="cuda")
    ours = fusedlayer.decode_batch(block, x, freqs, cache)
    theirs = fusedlayer.decode_block(block, x, freqs[100:101].contiguous(), mask, ip)
    got, ref = ours.double(), theirs.double()
    assert (got - ref).norm() / ref.norm() < 5e-3


def test_decode_batch_takes_head_norms_without_an_epsilon_as_the_decode_block_does():
    from tests.test_fused_gpu import _block
    from ttspipe_amd import fusedlayer

    block, _ = _block(BF, True)
    x = torch.randn(2, 1, 512, device="cuda").to(BF)
    got = []
    for eps in (None, 1e-6):
        table = pc.PageTable(2, 64, 8, 16)
        cache = pc.PagedKVCache(table, 2)
        table.admit(3), table.step()
        block.attention.q_norm.eps = block.attention.k_norm.eps = eps
        got += [fusedlayer.decode_batch(block, x, _freqs(64, 128), cache), cache.k_pages]
    assert np.array_equal(bits(got[0]), bits(got[2])) and np.array_equal(bits(got[1]), bits(got[3]))


def test_decode_batch_declines():
    from tests.test_fused_gpu import _block
    from ttspipe_amd import fusedlayer

    block, _ = _block(BF, True)
    table = pc.PageTable(2, 64, 8, 16)
    cache = pc.PagedKVCache(table, 2)
    x = torch.zeros(2, 1, 512, dtype=BF, device="cuda")
    freqs = _freqs(64, 128)
    assert fusedlayer.decode_batch(block, x, freqs, cache) is not None
    for args in ((x[:1], freqs, cache), (x.to(FP), freqs, cache), (x.float(), freqs, cache), (x.cpu(), freqs, cache),
                 (x.expand(2, 3, 512), freqs, cache), (x.view(2, 512), freqs, cache), (x, freqs[:, :16], cache),
                 (x, freqs, pc.PagedKVCache(table, 4)), (x, freqs, pc.PagedKVCache(table, 2, 64)),
                 (x, freqs, pc.PagedKVCache(table, 2, dtype=FP))):
        assert fusedlayer.decode_batch(block, *args) is None


def test_decode_batch_refuses_positions_past_the_rotary_table():
    from tests.test_fused_gpu import _block
    from ttspipe_amd import fusedlayer

    block, _ = _block(BF, True)
    table = pc.PageTable(2, 64, 8, 16)
    cache = pc.PagedKVCache(table, 2)
    table.admit(30)
    table.step()
    x = torch.zeros(2, 1, 512, dtype=BF, device="cuda")
    k0 = cache.k_pages.clone()
    with pytest.raises(ValueError):
        fusedlayer.decode_batch(block, x, _freqs(30, 128), cache)
    assert torch.equal(k0, cache.k_pages)
    assert fusedlayer.decode_batch(block, x, _freqs(31, 128), cache) is not None
