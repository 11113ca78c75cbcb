"""A paged cache's test inputs and its operators in 64 bits, slot by slot."""

from __future__ import annotations

import math

import torch


class Case:
    """Pools whose every unused row is NaN, with shuffled pages: a kernel that
    reads a row it must not read, or multiplies one by zero, shows it."""

    def __init__(self, lens, nh, nkv, hd, page, dtype, seed, cols=None, device="cuda", tracked=True):
        g = torch.Generator().manual_seed(seed)
        self.g, self.lens, self.nh, self.nkv, self.hd, self.page, self.dtype = g, list(lens), nh, nkv, hd, page, dtype
        self.device = device
        cols = cols or max(1, -(-max(lens) // page))
        used = [min(-(-n // page), cols) for n in lens]
        order = torch.randperm(sum(used) + 3, generator=g)
        self.pages = len(order)
        table = torch.full((len(lens), cols), -1, dtype=torch.int32)
        at = 0
        for b, u in enumerate(used):
            table[b, :u] = order[at:at + u].to(torch.int32)
            at += u
        self.table = table.to(device)
        nan = torch.full((self.pages, nkv, page, hd), math.nan)
        self.k, self.v = nan.clone(), nan.clone()
        for b, n in enumerate(lens):
            for c in range(used[b]):
                r = min(page, n - c * page)
                self.k[table[b, c], :, :r] = torch.randn(nkv, r, hd, generator=g)
                self.v[table[b, c], :, :r] = torch.randn(nkv, r, hd, generator=g)
        self.k, self.v = self.k.to(dtype).to(device), self.v.to(dtype).to(device)
        self.slots = torch.tensor([n - 1 for n in lens], device=device)
        self.q = (torch.randn(len(lens), nh, hd, generator=g) * 1.5).to(dtype).to(device)
        self.cap = cols * page
        self.scores = torch.rand(len(lens), nkv, self.cap, generator=g).to(device) if tracked else None

    def pools(self):
        return self.k, self.v, self.table


def attention64(q, k, v, table, slots, scale=None):
    """(y, p, y's bound, p's bound): the attention in 64 bits, the weights summed
    over each KV head's query heads [B, nkv, cap], and how far the kernels'
    arithmetic may take them before y's last rounding.

    A score is a sum of D fp32 products, scaled, off by at most (D + 4) 2^-24
    sum |q||k| scale; an error d in every score moves the weights by a factor
    within 1 +- 2d; exp2 and the sums of n terms, 32 and more at a time, add
    2^-20 + 2^-23 (n / 8 + 64): together the weights' relative error e. For y the
    matrix cores take each term exp(s - m) in two parts of the cache's type,
    together within 2^-16 of it, and 2^-25 where an fp16 part is subnormal; the
    largest term of each partial sum in fp16 is at least 2^13, so that is at most
    2^-38 of the denominator."""
    fp16 = k.dtype == torch.float16
    q, k, v, table = q.double().cpu(), k.cpu(), v.cpu(), table.cpu()
    B, nh, D = q.shape
    nkv, page = k.shape[1], k.shape[2]
    cap, group = table.shape[1] * page, nh // nkv
    scale = D**-0.5 if scale is None else scale
    y, p = torch.zeros(B, nh, D, dtype=torch.float64), torch.zeros(B, nkv, cap, dtype=torch.float64)
    yb, pb = torch.zeros_like(y), torch.zeros_like(p)
    for b in range(B):
        n = min(int(slots[b]) + 1, cap)
        there = [j for j in range(max(n, 0)) if 0 <= int(table[b, j // page]) < k.shape[0]]
        if not there:
            continue
        j = torch.tensor(there)
        pg, off = table[b, j // page].long(), j % page
        for h in range(nkv):
            K, V = k[pg, h, off].double(), v[pg, h, off].double()
            qq = q[b, h * group:(h + 1) * group]
            w = torch.softmax(qq @ K.t() * scale, 1)
            mag = (qq.abs() @ K.abs().t()).max(1, keepdim=True).values * scale
            e = 2 * (D + 4) * 2.0**-24 * mag + 2.0**-20 + 2.0**-23 * (n / 8 + 64)
            y[b, h * group:(h + 1) * group] = w @ V
            yb[b, h * group:(h + 1) * group] = (w @ V.abs()) * (e + 2.0**-16) + fp16 * 2.0**-38 * V.abs().sum(0)
            p[b, h, j] = w.sum(0)
            pb[b, h, j] = (w * e).sum(0)
    return y, p, yb, pb


def rounding(y, dtype):
    """Half a step of `dtype` at y."""
    f = torch.finfo(dtype)
    return y.abs() * f.eps / 2 + f.tiny * f.eps


def assert_within(got, ref, bound, what=""):
    got, ref, bound = got.double().cpu(), ref.double().cpu(), bound.double().cpu()
    assert got.shape == ref.shape
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    bad = (got - ref).abs() > bound
    if bad.any():
        i = bad.nonzero()[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first {i}: {got[tuple(i)]} for "
                             f"{ref[tuple(i)]}, bound {bound[tuple(i)]}")


def attention_check(case, y, scores=None, before=None, slots=None, scale=None, what=""):
    slots = case.slots if slots is None else slots
    ref, p, yb, pb = attention64(case.q, case.k, case.v, case.table, slots, scale)
    assert_within(y, ref, rounding(ref, case.dtype) * (1 + 2**-7) + yb, what + " y")
    if scores is not None:
        new = before.double().cpu() + p
        assert_within(scores, new, new.abs() * 2.0**-24 + pb, what + " scores")


def evict_ref(scores, slot_pos, n, position, budget, sinks, recent):
    """[(source, destination)] of one (sequence, kv head), from lists."""
    if n <= budget:
        return []

    def key(j):
        if slot_pos[j] < sinks or slot_pos[j] > position - recent:
            return math.inf
        return -math.inf if math.isnan(scores[j]) else scores[j]

    rank = sorted(range(n), key=lambda j: (-key(j), j))
    kept = set(rank[:budget])
    return list(zip([j for j in range(budget, n) if j in kept], [j for j in range(budget) if j not in kept]))
