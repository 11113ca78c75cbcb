"""Forms that only large calls take (GPU): penalties in large slices (long histories
of many rows), and prefixes whose chunks have the most rows a chunk may have."""

from __future__ import annotations

import math

import pytest
import torch

from tests.pageddata import assert_within, rounding
from tests.test_penalize_gpu import call, make, reference
from ttspipe_amd import fusedsample
from ttspipe_amd import pagedcache as pc

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def check(got, logits, *parts):
    """`tests/test_penalize_gpu.py`'s check with its bar in full where a frequency is
    negative. That bar counts 2^-23 of what each operation comes to, and of
    frequency * c by its value, not its size: for f < 0 it takes |f c| off the sum where it
    is to add it. So |f c| is 2 |f c| short there, 2^-23 of which are added: a product f c
    is off by 2^-24 |f c|, whatever its sign. (With long histories c is large, and the
    formula in fp32 on the CPU leaves the short bar at the same elements.)"""
    want, off = reference(logits, *parts)
    history, lengths, freq = parts[0].cpu().long(), parts[1], parts[3]
    if freq is not None:
        for i in range(len(want)):
            h = history if history.dim() == 1 else history[i]
            h = h if lengths is None else h[: min(max(int(lengths[i]), 0), len(h))]
            c = torch.bincount(h[(h >= 0) & (h < want.shape[1])], minlength=want.shape[1])
            off[i] += 2.0**-23 * 2 * max(-float(freq[i]), 0.0) * c
    got, f = got.double().cpu(), torch.finfo(logits.dtype)
    assert not torch.isnan(got).any() and torch.equal(torch.isinf(got), torch.isinf(want))
    fine = ~torch.isinf(want)
    assert (got[~fine] == want[~fine]).all()
    bad = ((got - want).abs() > want.abs() * (f.eps / 2) * (1 + 2**-7) + off + f.tiny * f.eps) & fine
    assert not bad.any(), f"{int(bad.sum())} off, first {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("rows,vocab,hist", [(256, 300, 1025), (256, 16383, 1100), (256, 16384, 1025), (130, 16385, 1500),
                                             (86, 40003, 2047), (52, 65537, 1200)])
def test_large_slices(rows, vocab, hist, dtype):
    """Over 1024 tokens of history and 256 slices of 16384: their edges and ends, every part on."""
    a = make(rows, vocab, hist, dtype, seed=rows + vocab, h64=rows % 3 == 0)
    check(call(*a), *a)


@pytest.mark.parametrize("dtype,step", [(BF, 16391), (FP, 16389), (F32, 16387)])
def test_large_slices_of_strided_rows_in_place(dtype, step):
    """Rows of any alignment: nothing between them is touched."""
    vocab = 16386
    a = make(128, vocab, 1030, dtype, seed=step)
    mask = torch.randint(-2**31, 2**31 - 1, (128, vocab // 32 + 5), dtype=torch.int32, device="cuda")[:, 3:3 + vocab // 32 + 1]
    bias = torch.randn(128, vocab + 9, device="cuda").to(dtype)[:, 5:5 + vocab]
    a = (*a[:6], bias, mask)
    big = torch.full((129 * step,), 7.0, dtype=dtype, device="cuda")
    view = big[1:1 + 128 * step].view(128, step)[:, :vocab]
    view.copy_(a[0])
    assert call(view, *a[1:], out=view) is view
    check(view, *a)
    rest = torch.ones_like(big, dtype=torch.bool)
    rest[1:1 + 128 * step].view(128, step)[:, :vocab] = False
    assert (big[rest] == 7).all()


def test_large_slices_of_a_shared_history():
    a = make(300, 700, 3000, FP, seed=5, parts="rf")
    history = a[1][0].contiguous()
    a = (a[0], history, None, *a[3:])
    check(call(*a), *a)
    y = fusedsample.penalize(a[0], history[:0], repetition=a[3], frequency=a[4])
    assert torch.equal(y, a[0])


@pytest.mark.parametrize("n", [16379, 16384, 20011])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_chunks_of_the_most_rows(n, dtype):
    """32 KV heads, five tiles of query rows: eight chunks a head would be over 8192 rows each.
    Against 64 bits on the GPU, head by head; the bounds are those of `tests/spandata.py`."""
    B, nkv, group, D, page = 80, 32, 8, 64, 256
    g = torch.Generator(device="cuda").manual_seed(n)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    cols = -(-n // page)
    order = torch.randperm(cols + B, generator=g, device="cuda").to(torch.int32)
    pools = []
    for _ in "kv":
        pool = torch.full((cols + B, nkv, page, D), math.nan, dtype=dtype, device="cuda")
        pool[order[:cols].long()] = rand(cols, nkv, page, D).to(dtype)
        pool[order[cols - 1].long(), :, (n - 1) % page + 1:] = math.nan
        pool[order[cols:].long(), :, :2] = rand(B, nkv, 2, D).to(dtype)  # own: none, one or two rows
        pools.append(pool)
    k, v = pools
    q = (rand(B, nkv * group, D) * 1.5).to(dtype)
    own, far = order[cols:][:, None].contiguous(), order[None, :cols].contiguous()
    slots = torch.arange(B, device="cuda") % 3 - 1
    prefix = pc.Prefix(far, torch.tensor([n - 1], device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda"))
    y = pc.attention(q, k, v, own, slots, prefix=prefix)
    assert y is not None
    ref, bound = torch.empty(B, nkv * group, D, dtype=torch.float64, device="cuda"), torch.empty(B, nkv * group, D, dtype=torch.float64, device="cuda")
    for h in range(nkv):
        heads = slice(h * group, (h + 1) * group)
        qq = q[:, heads].double()
        K, V = (p[far[0].long(), h].reshape(-1, D)[:n].double() for p in (k, v))
        ko, vo = (p[own[:, 0].long(), h, :2].double() for p in (k, v))  # (B, 2, D)
        there = torch.arange(2, device="cuda") <= slots[:, None, None]
        s = torch.cat([qq.reshape(-1, D) @ K.t(), (qq[:, :, None] * ko[:, None]).sum(-1).view(-1, 2)], 1) * D**-0.5
        s[:, n:] = s[:, n:].masked_fill(~there.expand(B, group, 2).reshape(-1, 2), -math.inf)
        w = torch.softmax(s, 1)
        mag = (qq.abs().reshape(-1, D) @ K.abs().t()).amax(1)
        mag = torch.maximum(mag, (qq.abs()[:, :, None] * ko.abs()[:, None]).sum(-1).view(-1, 2).amax(1)) * D**-0.5
        e = 2 * (D + 4) * 2.0**-24 * mag[:, None] + 2.0**-20 + 2.0**-23 * ((n + 2) / 8 + 64)
        near = lambda x, t: (x.view(B, group, 2, 1) * t[:, None]).sum(2).view(-1, D)  # noqa: E731
        ref[:, heads] = (w[:, :n] @ V + near(w[:, n:], vo)).view(B, group, D)
        top = w[:, :n] @ V.abs() + near(w[:, n:], vo.abs())
        tail = (dtype is FP) * 2.0**-38 * (V.abs().sum(0) + vo.abs().sum(1).amax(0))
        bound[:, heads] = (top * (e + 2.0**-16) + tail).view(B, group, D)
    ref, bound = ref.cpu(), bound.cpu()
    assert_within(y, ref, rounding(ref, dtype) * (1 + 2**-7) + bound)
