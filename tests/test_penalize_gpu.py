"""Penalties on logits (GPU): against the formula in 64 bits at the sizes, types,
histories and masks where they can go wrong, and the refusals.

Bar: an operation in 32 bits is off by at most half a step, 2^-24 of its result; a
row's value is a division or product, a product and two sums of penalties and a
sum with the bias, so it is off by 2^-24 of what each of them comes to (counted
below with the next power's room, 2^-23), and half a step of the logits' type."""

from __future__ import annotations

import math

import pytest
import torch

from ttspipe_amd import fusedsample

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def reference(logits, history, lengths, rep, freq, pres, bias, mask):
    """(the formula in 64 bits, its bound before the last rounding), on the CPU; rows (rows, V)."""
    x = logits.double().cpu()
    rows, vocab = x.shape
    off = torch.zeros_like(x)
    per_row = lambda t, i: None if t is None else float(t.reshape(-1)[i if t.numel() > 1 else 0])  # noqa: E731
    for i in range(rows):
        if history is not None:
            h = (history if history.dim() == 1 else history[min(i, history.shape[0] - 1)]).cpu().long()
            if lengths is not None:
                h = h[: min(max(int(lengths[i]), 0), len(h))]
            h = h[(h >= 0) & (h < vocab)]
            t, c = torch.unique(h, return_counts=True)
            r, f, p = (per_row(v, i) for v in (rep, freq, pres))
            if r is not None:
                x[i, t] = torch.where(x[i, t] > 0, x[i, t] / r, x[i, t] * r)
                off[i, t] += x[i, t].abs()
            if f is not None or p is not None:
                f, p = f or 0.0, p or 0.0
                x[i, t] -= f * c + p
                off[i, t] += f * c + abs(f * c + p) + x[i, t].abs()
        if bias is not None:
            x[i] += (bias if bias.dim() == 1 else bias[min(i, bias.shape[0] - 1)]).double().cpu()
            off[i] += x[i].abs()
        if mask is not None:
            m = (mask if mask.dim() == 1 else mask[min(i, mask.shape[0] - 1)]).cpu().long()
            t = torch.arange(vocab)
            gone = (m[t // 32] >> (t % 32)) & 1 == 0
            x[i, gone] = -math.inf
            off[i, gone] = 0.0
    return x, off * 2.0**-23


def check(got, logits, *parts):
    rows = logits.reshape(-1, logits.shape[-1])
    want, off = reference(rows, *parts)
    got = got.reshape(rows.shape).double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    f = torch.finfo(logits.dtype)
    fine = ~inf & ~torch.isnan(want)
    bad = ((got - want).abs() > want.abs() * (f.eps / 2) * (1 + 2**-7) + off + f.tiny * f.eps) & fine
    assert not bad.any(), f"{int(bad.sum())} off, first {bad.nonzero()[0].tolist()}"


def make(rows, vocab, hist, dtype, seed, parts="rfpbm", h64=False):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(rows, vocab, generator=g) * 4).to(dtype).cuda()
    history = torch.randint(-2, vocab + 2, (rows, hist), generator=g)
    history[:, ::3] = (history[:, ::3] % 7).clamp(max=vocab - 1)  # some come often
    history = history.to(torch.int64 if h64 else torch.int32).cuda()
    lengths = torch.randint(0, hist + 1, (rows,), generator=g).to(torch.int64 if not h64 else torch.int32).cuda()
    lengths[-1] = hist
    vec = lambda lo, hi: (torch.rand(rows, generator=g) * (hi - lo) + lo).cuda()  # noqa: E731
    rep, freq, pres = vec(0.7, 1.8), vec(-0.2, 0.6), vec(0.0, 1.0)
    bias = torch.randn(vocab, generator=g).cuda()
    mask = fusedsample.pack_mask(torch.rand(rows, vocab, generator=g) < 0.6).cuda()
    pick = lambda c, t: t if c in parts else None  # noqa: E731
    return (logits, history, lengths, pick("r", rep), pick("f", freq), pick("p", pres), pick("b", bias), pick("m", mask))


def call(logits, history, lengths, rep, freq, pres, bias, mask, **kw):
    y = fusedsample.penalize(logits, history, lengths=lengths, repetition=rep, frequency=freq, presence=pres, bias=bias,
                             mask=mask, **kw)
    assert y is not None
    torch.cuda.synchronize()
    return y


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 32, 33, 500, 1023, 1024, 1025, 2049, 4096, 4097, 8191, 8200, 16385, 40003])
def test_every_part_at_the_slices_edges(vocab, dtype):
    a = make(3, vocab, 50, dtype, seed=vocab)
    check(call(*a), *a)


@pytest.mark.parametrize("parts", ["", "r", "f", "p", "fp", "b", "m", "rb", "rm", "rfpbm"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_parts_by_themselves(parts, dtype):
    a = make(2, 777, 33, dtype, seed=len(parts), parts=parts, h64=True)
    y = call(*a)
    check(y, *a)
    if not parts:
        assert torch.equal(y, a[0])


@pytest.mark.parametrize("hist", [1, 63, 255, 256, 257, 1000, 5001])
@pytest.mark.parametrize("rows,vocab", [(1, 4096), (5, 9001), (67, 300)])
def test_histories_of_all_lengths(hist, rows, vocab):
    for h64 in (False, True):
        a = make(rows, vocab, hist, FP, seed=hist + rows, parts="rfp", h64=h64)
        check(call(*a), *a)
        a = (*a[:2], None, *a[3:])  # all entries count
        check(call(*a), *a)


@pytest.mark.parametrize("rows,vocab", [(1, 160001), (300, 4099), (40, 50003)])
def test_large_calls(rows, vocab):
    a = make(rows, vocab, 300, BF, seed=rows)
    check(call(*a), *a)


def test_extreme_tokens_and_lengths():
    logits = torch.randn(4, 100, device="cuda")
    history = torch.tensor([[2**63 - 1, -2**63, 100, -1, 99, 0, 2**32, 2**32 + 5]] * 4, device="cuda")
    lengths = torch.tensor([2**40, -5, 5, 0], device="cuda")
    a = (logits, history, lengths, torch.full((1,), 2.0, device="cuda"), None, None, None, None)
    y = call(*a)
    check(y, *a)
    assert torch.equal(y[1], logits[1]) and torch.equal(y[3], logits[3]) and y[0, 99] != logits[0, 99]


def test_a_token_that_fills_the_history_is_counted_whole():
    logits = torch.zeros(1, 64, device="cuda")
    history = torch.full((1, 200000), 5, dtype=torch.int32, device="cuda")
    y = call(logits, history, None, None, torch.ones(1, device="cuda"), None, None, None)
    assert y[0, 5] == -200000 and y.count_nonzero() == 1


def test_infinities_and_nan():
    inf, nan = math.inf, math.nan
    logits = torch.tensor([[inf, -inf, nan, 0.0, -0.0, 1.0, -1.0, nan, inf]], device="cuda")
    mask = fusedsample.pack_mask(torch.tensor([1, 1, 1, 1, 1, 1, 1, 0, 0], dtype=torch.bool)).cuda()
    a = (logits, torch.arange(9, device="cuda"), None, torch.full((1,), 1.5, device="cuda"),
         torch.full((1,), 0.25, device="cuda"), None, torch.zeros(9, device="cuda"), mask)
    y = call(*a)
    check(y, *a)
    assert y[0, 7] == -inf and y[0, 8] == -inf and y[0, 0] == inf and y[0, 1] == -inf and torch.isnan(y[0, 2])
    lowest = torch.full((2, 40), torch.finfo(BF).min, dtype=BF, device="cuda")
    a = (lowest, torch.arange(40, device="cuda"), None, torch.full((2,), 3.0, device="cuda"), None, None, None, None)
    assert torch.isinf(call(*a)).all()  # beyond bf16's range: -inf, as the formula's rounding


def test_a_mask_that_allows_nothing_leaves_minus_infinity():
    a = make(2, 300, 10, FP, seed=1)
    a = (*a[:7], torch.zeros(2, 10, dtype=torch.int32, device="cuda"))
    assert torch.equal(call(*a), torch.full((2, 300), -math.inf, dtype=FP, device="cuda"))


@pytest.mark.parametrize("dtype", [FP, BF])
def test_a_grammar_of_few_tokens_is_what_is_drawn_from(dtype):
    """Fewer tokens allowed than the sampler's top-k takes: none of the others is drawn."""
    g = torch.Generator().manual_seed(21)
    logits = (torch.randn(24, 4096, generator=g) * 4).to(dtype).cuda()
    allowed = torch.zeros(24, 4096, dtype=torch.bool)
    for r in range(24):
        allowed[r, torch.randperm(4096, generator=g)[: 1 + r % 6]] = True
    y = fusedsample.penalize(logits, mask=fusedsample.pack_mask(allowed).cuda())
    temp, topp = torch.full((1,), 0.9, dtype=dtype, device="cuda"), torch.full((1,), 0.95, dtype=dtype, device="cuda")
    for top_k in (1, 30, 64):
        uniform = (torch.rand(24, 4096, generator=g) * 0.998 + 0.001).cuda()
        for r in range(24):
            t = fusedsample.sample(y[r], temp, topp, torch.tensor([top_k], device="cuda"), uniform=uniform[r])
            assert allowed[r, int(t)], (r, top_k, int(t))


def test_one_row_and_shared_parts():
    """(V,) logits; a bias, a mask and a history of one row for all; a bias of the logits' type."""
    g = torch.Generator().manual_seed(3)
    v = 500
    history = torch.randint(0, v, (20,), generator=g).cuda()
    bias = torch.randn(1, v, generator=g).to(FP).cuda()
    mask = fusedsample.pack_mask(torch.rand(v, generator=g) < 0.5).cuda()
    for shape in ((v,), (1, v), (6, v)):
        logits = torch.randn(shape, generator=g).to(FP).cuda()
        a = (logits, history, None, torch.tensor(1.3, device="cuda"), None, torch.full((1,), 0.5, device="cuda"), bias, mask)
        y = call(*a)
        assert y.shape == logits.shape
        check(y, *a)


@pytest.mark.parametrize("dtype,step", [(BF, 1001), (FP, 1003), (F32, 1001)])
def test_strided_rows_in_place_and_beside_others(dtype, step):
    """Rows of any stride and alignment: nothing between them is touched."""
    a = make(5, 1000, 40, dtype, seed=9, h64=True)
    wide = torch.full((5, step), 7.0, dtype=dtype, device="cuda")
    wide[:, :1000] = a[0]
    bias = torch.randn(5, 1234, device="cuda")[:, 3:1003]
    mask = torch.randint(-2**31, 2**31 - 1, (5, 50), dtype=torch.int32, device="cuda")[:, 1:33]
    hist = torch.cat([a[1], a[1]], 1)[:, 7:47]
    a = (a[0], hist, *a[2:6], bias, mask)
    for first in (0, 1):
        big = torch.full((6 * step,), 7.0, dtype=dtype, device="cuda")
        view = big[first:first + 5 * step].view(5, step)[:, :1000]
        view.copy_(a[0])
        before = big.clone()
        y = call(view, *a[1:], out=view)
        assert y is view
        check(y, *a)
        rest = torch.ones_like(big, dtype=torch.bool)
        rest[first:first + 5 * step].view(5, step)[:, :1000] = False
        assert torch.equal(big[rest], before[rest])
        fresh = torch.full((5, step + 2), 3.0, dtype=dtype, device="cuda")
        call(a[0], *a[1:], out=fresh[:, 1:1001])
        check(fresh[:, 1:1001], *a)
        assert (fresh[:, 0] == 3).all() and (fresh[:, 1001:] == 3).all()


def test_refusals():
    x = torch.zeros(3, 100, dtype=BF, device="cuda")
    h = torch.zeros(3, 5, dtype=torch.int64, device="cuda")
    one = torch.ones(3, device="cuda")
    for kw in (dict(history=h.float()), dict(history=h[:2]), dict(history=h.t()), dict(history=h.cpu()), dict(history=h[None]),
               dict(history=h, lengths=one), dict(history=h, lengths=torch.zeros(2, dtype=torch.int32, device="cuda")),
               dict(repetition=one.double()), dict(frequency=one[:2]), dict(presence=one.cpu()), dict(repetition=one[:, None]),
               dict(bias=torch.zeros(99, device="cuda")), dict(bias=torch.zeros(100, dtype=FP, device="cuda")),
               dict(bias=torch.zeros(200, device="cuda")[::2]), dict(mask=torch.zeros(3, 3, dtype=torch.int32, device="cuda")),
               dict(mask=torch.zeros(3, 4, device="cuda")), dict(mask=torch.zeros(3, 100, dtype=torch.bool, device="cuda")),
               dict(out=torch.zeros(3, 100, device="cuda")), dict(out=torch.zeros(3, 101, dtype=BF, device="cuda")),
               dict(out=torch.zeros(1, 100, dtype=BF, device="cuda").expand(3, 100))):
        with pytest.raises(ValueError):
            fusedsample.penalize(x, **kw)
    flat = torch.zeros(1000, dtype=BF, device="cuda")
    rows = flat[:300].view(3, 100)
    for out in (flat[1:301].view(3, 100), flat[100:400].view(3, 100), flat[:600].view(3, 200)[:, :100]):
        with pytest.raises(ValueError):
            fusedsample.penalize(rows, out=out)
    assert fusedsample.penalize(rows, out=flat[300:600].view(3, 100)) is not None
    for bad in (x.double(), x.to(torch.int32), x.t(), x[None], x.cpu()):
        assert fusedsample.penalize(bad) is None
    for empty in (x[:0], x[:, :0]):
        assert fusedsample.penalize(empty, mask=None).shape == empty.shape


def test_a_captured_call_follows_its_inputs():
    """The history, its lengths and the penalties change in place between replays."""
    a = make(4, 3000, 64, BF, seed=5)
    out = torch.empty_like(a[0])
    call(*a, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fusedsample.penalize(a[0], a[1], lengths=a[2], repetition=a[3], frequency=a[4], presence=a[5], bias=a[6], mask=a[7],
                             out=out)
    for i in range(4):
        b = make(4, 3000, 64, BF, seed=20 + i)
        for x, y in zip(a, b):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        check(out, *b)


def test_two_streams():
    cases = [make(8, 20000, 500, FP, seed=i) for i in range(2)]
    want = [call(*a) for a in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for a, st, g in zip(cases, streams, got):
            with torch.cuda.stream(st):
                g.append(fusedsample.penalize(a[0], a[1], lengths=a[2], repetition=a[3], frequency=a[4], presence=a[5],
                                              bias=a[6], mask=a[7]))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)
