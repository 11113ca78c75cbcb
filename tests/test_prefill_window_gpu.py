"""A prompt's attention through a sliding window with sinks (GPU): against its
formula in 64 bits at the spans, windows, sinks and widths where it can go wrong.

Bar: scores are fp32 sums (relative error e of the weights as
`tests/pageddata.py` counts it); a weight is rounded to the cache's type before it
meets V, half a step of it; the output is rounded once."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.gpuutil import bits
from tests.pageddata import assert_within, rounding
from ttspipe_amd import fastpath

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def make(S, L, nh, nkv, dtype, seed, start=None, pad=0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(1, S, nh, 128, generator=g) * 1.5).to(dtype).cuda().transpose(1, 2)
    cache = torch.full((2, 1, nkv, L + pad, 128), math.nan)
    cache[:, :, :, :L] = torch.randn(2, 1, nkv, L, 128, generator=g)
    cache = cache.to(dtype).cuda()
    k, v = cache[0][:, :, :L], cache[1][:, :, :L]
    start = L - S if start is None else start
    return q, k, v, torch.arange(start, start + S, device="cuda")


def reference(q, k, v, pos, window, sinks):
    dtype = k.dtype
    q, k, v, pos = q[0].double(), k[0].double(), v[0].double(), pos.cuda()[:, None]  # (64-bit products on the GPU)
    nh, S, D = q.shape
    nkv, L = k.shape[:2]
    key = torch.arange(L, device=pos.device)
    seen = (key <= pos) & ((key < sinks) | (key > pos - window))
    y, yb = torch.empty(nh, S, D, dtype=torch.float64), torch.empty(nh, S, D, dtype=torch.float64)
    n = seen.sum(1, keepdim=True)
    for h in range(nh):
        K, V = k[h * nkv // nh], v[h * nkv // nh]
        w = torch.softmax((q[h] @ K.t() * D**-0.5).masked_fill(~seen, -math.inf), 1)
        mag = (q[h].abs() @ K.abs().t()).masked_fill(~seen, 0.0).amax(1, keepdim=True) * D**-0.5
        e = 2 * (D + 4) * 2.0**-24 * mag + 2.0**-20 + 2.0**-23 * (n / 8 + 64) + torch.finfo(dtype).eps / 2
        # (fp16 weights below 2^-14 of the row's reference, which lies within 2^8 of its largest, lose up to 2^-25)
        tail = (dtype is FP) * 2.0**-24 * (seen.double() @ V.abs())
        y[h], yb[h] = (w @ V).cpu(), ((w @ V.abs()) * e + tail).cpu()
    return y[None], yb[None]


def run(q, k, v, pos, window, sinks, **kw):
    nh, nkv = q.shape[1], k.shape[1]
    y = fastpath.prefill_attention(q, k, v, None, nh, nkv, 128, positions=pos, window=window, sinks=sinks, **kw)
    assert y is not None
    torch.cuda.synchronize()
    return y


def check(q, k, v, pos, window, sinks, y, what=""):
    ref, bound = reference(q, k, v, pos, window, sinks)
    assert_within(y, ref, rounding(ref, k.dtype) * (1 + 2**-7) + bound, what)


@pytest.mark.parametrize("S", [1, 2, 9, 31, 32, 33, 64, 65, 127, 200])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (31, 0), (32, 32), (33, 31), (64, 65), (100, 4), (1000, 17),
                                          (10**9, 10**9)])
def test_spans_and_windows(S, window, sinks):
    for L in (S, S + 1, S + 77, S + 300):
        a = make(S, L, 8, 2, BF, seed=S + L, pad=13)
        check(*a, window, sinks, run(*a, window, sinks), f"L {L}")


@pytest.mark.parametrize("nh,nkv", [(1, 1), (2, 1), (3, 1), (32, 8), (5, 1), (12, 2), (7, 7), (14, 2), (8, 1), (16, 8), (24, 1), (70, 1)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_other_heads(nh, nkv, dtype):
    for S, L, window, sinks in ((100, 100, 40, 3), (70, 1200, 300, 16), (40, 900, 800, 0)):
        a = make(S, L, nh, nkv, dtype, seed=nh + S)
        check(*a, window, sinks, run(*a, window, sinks))


@pytest.mark.parametrize("S,L,window,sinks", [(512, 2512, 1024, 4), (1500, 1500, 256, 64), (2300, 2300, 1, 0), (130, 9000, 4000, 100),
                                              (600, 700, 33, 0), (4100, 4100, 700, 4)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_long_spans(S, L, window, sinks, dtype):
    a = make(S, L, 32, 8, dtype, seed=S + window)
    check(*a, window, sinks, run(*a, window, sinks))


def test_a_window_wider_than_the_span_is_the_causal_attention():
    for S, L in ((100, 100), (64, 1000), (512, 512), (600, 2000)):
        q, k, v, pos = a = make(S, L, 32, 8, BF, seed=S)
        causal = fastpath.prefill_attention(q, k, v, None, 32, 8, 128, positions=pos)
        ref, bound = reference(*a, L, 0)
        y = run(*a, L, 0)
        check(*a, L, 0, y)
        assert_within(y, causal, 2 * (rounding(ref, BF) * (1 + 2**-7) + bound))


def test_one_key_windows_give_its_value():
    q, k, v, pos = a = make(300, 400, 8, 2, BF, seed=6)
    y = run(*a, 1, 0)
    assert torch.equal(y[0], v[0, :, 100:].repeat_interleave(4, 0))


def test_positions_in_any_order_and_past_the_keys():
    """A row past the keys sees its window's rest and the sinks, or nothing (NaN); a
    row below 0 nothing."""
    for window, sinks in ((40, 3), (40, 0), (200, 50)):
        q, k, v, _ = make(70, 500, 8, 2, FP, seed=window)
        g = torch.Generator().manual_seed(window)
        pos = torch.randint(0, 500, (70,), generator=g)
        pos[:8] = torch.tensor([499, 0, 510, 539, 540, 10**15, -1, -2**40])
        a = (q, k, v, pos.cuda())
        y = run(*a, window, sinks)
        check(*a, window, sinks, y)
        assert torch.isnan(y[0, :, 6:8]).all() and (sinks > 0) != bool(torch.isnan(y[0, 0, 5]).any())


@pytest.mark.parametrize("S", [20, 600])
def test_causal_rows_far_below_zero_see_nothing(S):
    """(A position below -2^31 lost its high bits and saw the first key.)"""
    q, k, v, _ = make(S, 700, 8, 2, BF, seed=2)
    for low in (-2**32, -2**40, -2**63):
        y = fastpath.prefill_attention(q, k, v, None, 8, 2, 128, positions=torch.full((S,), low, device="cuda"))
        assert torch.isnan(y).all()


def test_infinities_and_nan_behind_the_window_are_not_seen():
    q, k, v, pos = a = make(20, 600, 8, 2, BF, seed=9)
    k[:, :, 10:500:2] = math.nan
    k[:, :, 11:500:2] = math.inf
    y = run(*a, 81, 10)  # rows 580 .. 599 see 0 .. 9 and from 500 on
    assert torch.isfinite(y).all()
    clean = (q, torch.where(torch.isfinite(k), k, 0.0), v, pos)
    check(*clean, 81, 10, y)


@pytest.mark.parametrize("S", [20, 300, 3000])
def test_values_that_no_row_sees_may_be_nan(S):
    """(Those of the window's first tile that lie before it, and of the sinks' last behind them.)"""
    L = 3300
    q, k, v, pos = make(S, L, 8, 2, BF, seed=11)
    low = L - S - 100  # the first row's window starts behind it
    clean = v.clone()
    v[:, :, 10:low + 1] = math.nan
    v[:, :, 10:low + 1:3] = math.inf
    y = run(q, k, v, pos, 100, 10)
    assert torch.isfinite(y).all()
    clean[:, :, 10:low + 1] = 0.0
    check(q, k, clean, pos, 100, 10, y)


def test_rows_without_a_key_among_split_ones():
    q, k, v, pos = make(9, 3000, 8, 2, BF, seed=12)
    assert fastpath.prefill_splits(9, 8, 2, 3000, 2000, 0) > 1
    pos[3], pos[5] = -1, 3000 + 2000
    y = run(q, k, v, pos, 2000, 0)
    assert torch.isnan(y[0, :, [3, 5]]).all()
    for rows in (slice(0, 3), slice(4, 5), slice(6, 9)):
        check(q[:, :, rows], k, v, pos[rows], 2000, 0, y[:, :, rows])


def test_strides_workspaces_and_out():
    q, k, v, pos = make(40, 3000, 32, 8, BF, seed=10, pad=72)
    splits = fastpath.prefill_splits(40, 32, 8, 3000, 2500, 4)
    need = fastpath.prefill_work_floats(40, 32, splits)
    work, out = torch.full((max(need, 4),), math.nan, device="cuda"), torch.empty(1, 40, 4096, dtype=BF, device="cuda")
    y = run(q, k, v, pos, 2500, 4, out=out, work=work)
    assert y.data_ptr() == out.data_ptr()
    check(q, k, v, pos, 2500, 4, y)
    heads_last = torch.randn(1, 3000, 8, 2, 128, dtype=BF, device="cuda")
    k, v = heads_last[:, :, :, 0].transpose(1, 2), heads_last[:, :, :, 1].transpose(1, 2)
    check(q, k, v, pos, 700, 4, run(q, k, v, pos, 700, 4))
    if splits > 1:
        with pytest.raises(ValueError):
            run(q, k, v, pos, 2500, 4, work=work[:-1])


def test_refusals():
    q, k, v, pos = make(20, 100, 8, 2, BF, seed=1)
    att = fastpath.prefill_attention
    for kw in (dict(window=0), dict(window=-3), dict(window=4, sinks=-1), dict(sinks=4)):
        with pytest.raises(ValueError):
            att(q, k, v, None, 8, 2, 128, positions=pos, **kw)
    with pytest.raises(ValueError):
        att(q, k, v, torch.ones(1, 1, 20, 112, dtype=torch.bool, device="cuda")[..., :100], 8, 2, 128, window=5)
    for bad in (pos.int(), pos[:19], pos.cpu()):
        assert att(q, k, v, None, 8, 2, 128, positions=bad, window=5) is None
    assert att(q.float(), k.float(), v.float(), None, 8, 2, 128, positions=pos, window=5) is None
    assert att(q.repeat(1, 3, 1, 1), k[:, :1], v[:, :1], None, 24, 1, 64, positions=pos, window=5) is None
    assert att(q[:, :7], k, v, None, 7, 2, 128, positions=pos, window=5) is None
    for odd in (q[..., 4:], torch.randn(1, 8, 20, 132, dtype=BF, device="cuda")[..., :128]):
        assert att(odd, k, v, None, 8, 2, 128, positions=pos, window=5) is None
    for kw in (dict(out=torch.empty(1, 20, 1000, dtype=BF, device="cuda")), dict(out=torch.empty(1, 20, 1024, device="cuda"))):
        with pytest.raises(ValueError):
            att(q, k, v, None, 8, 2, 128, positions=pos, window=5, **kw)


def test_a_captured_call_follows_the_positions():
    q, k, v, pos = make(64, 1500, 8, 2, BF, seed=12)
    out = torch.empty(1, 64, 1024, dtype=BF, device="cuda")
    splits = fastpath.prefill_splits(64, 8, 2, 1500, 500, 4)
    work = torch.empty(max(4, fastpath.prefill_work_floats(64, 8, splits)), device="cuda")
    step = lambda: fastpath.prefill_attention(q, k, v, None, 8, 2, 128, positions=pos, window=500, sinks=4, out=out, work=work)  # noqa: E731
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for start in (1436, 0, 300, 900):
        pos.copy_(torch.arange(start, start + 64))
        graph.replay()
        torch.cuda.synchronize()
        check(q, k, v, pos, 500, 4, out.view(1, 64, 8, 128).transpose(1, 2))
        again = run(q, k, v, pos, 500, 4)
        assert np.array_equal(bits(again.contiguous()), bits(out.view(1, 64, 8, 128).transpose(1, 2).contiguous()))
