"""One-token attention through a window and over shared prefixes, in 64 bits, row by row."""

from __future__ import annotations

import math

import torch

from tests.pageddata import Case, assert_within, rounding


def _keys(table, n, page, pages, window=None, sinks=0):
    """Slots below n that lie in a page and that the newest row sees."""
    n = min(n, len(table) * page)
    return [j for j in range(max(n, 0)) if 0 <= int(table[j // page]) < pages
            and (window is None or j < sinks or j > n - 1 - window)]


def spans64(q, k, v, table, slots, window=None, sinks=0, prefix=None, scale=None):
    """(y, p, y's bound, p's bound) as `pageddata.attention64` (the bounds are its,
    for the same arithmetic): each sequence's keys are the rows of its prefix,
    `prefix` = (table, slots, of), and those of its own that the window leaves; p is
    the weights of the own slots."""
    fp16 = k.dtype == torch.float16
    q, k, v, table = q.double().cpu(), k.cpu(), v.cpu(), table.cpu()
    B, nh, D = q.shape
    pages, nkv, page = k.shape[:3]
    cap, group = table.shape[1] * page, nh // nkv
    scale = D**-0.5 if scale is None else scale
    y, p = torch.zeros(B, nh, D, dtype=torch.float64), torch.zeros(B, nkv, cap, dtype=torch.float64)
    yb, pb = torch.zeros_like(y), torch.zeros_like(p)
    for b in range(B):
        j = _keys(table[b], int(slots[b]) + 1, page, pages, window, sinks)
        near = torch.tensor(j, dtype=torch.long)
        at = [(int(table[b, i // page]), i % page) for i in j]
        if prefix is not None and 0 <= int(prefix[2][b]) < prefix[0].shape[0]:
            far = prefix[0][int(prefix[2][b])].cpu()
            at = [(int(far[i // page]), i % page) for i in _keys(far, int(prefix[1][int(prefix[2][b])]) + 1, page, pages)] + at
        if not at:
            continue
        pg, off = torch.tensor(at).t()
        n = len(at)
        for h in range(nkv):
            K, V = k[pg, h, off].double(), v[pg, h, off].double()
            qq = q[b, h * group:(h + 1) * group]
            w = torch.softmax(qq @ K.t() * scale, 1)
            mag = (qq.abs() @ K.abs().t()).max(1, keepdim=True).values * scale
            e = 2 * (D + 4) * 2.0**-24 * mag + 2.0**-20 + 2.0**-23 * (n / 8 + 64)
            y[b, h * group:(h + 1) * group] = w @ V
            yb[b, h * group:(h + 1) * group] = (w @ V.abs()) * (e + 2.0**-16) + fp16 * 2.0**-38 * V.abs().sum(0)
            p[b, h, near] = w.sum(0)[n - len(j):]
            pb[b, h, near] = (w * e).sum(0)[n - len(j):]
    return y, p, yb, pb


def spans_check(case, y, scores=None, before=None, what="", slots=None, **kw):
    ref, p, yb, pb = spans64(case.q, case.k, case.v, case.table, case.slots if slots is None else slots, **kw)
    assert_within(y, ref, rounding(ref, case.dtype) * (1 + 2**-7) + yb, what + " y")
    if scores is not None:
        new = before.double().cpu() + p
        assert_within(scores, new, new.abs() * 2.0**-24 + pb, what + " scores")


def slid(case, window, sinks):
    """Give back the pages no token sees through the window: their rows become NaN, their table entries -1."""
    table = case.table.cpu()
    for b, n in enumerate(case.lens):
        for c in range(table.shape[1]):
            if c * case.page >= sinks and (c + 1) * case.page <= n - window:
                page = int(table[b, c])
                case.k[page] = math.nan
                case.v[page] = math.nan
                table[b, c] = -1
    case.table.copy_(table)


class PrefixCase(Case):
    """A case whose sequences have prefixes: `far` rows each, in pages of the same
    pools; `of` names each sequence's (-1: none)."""

    def __init__(self, lens, far, of, nh, nkv, hd, page, dtype, seed, tracked=True, cols=None, far_cols=None):
        super().__init__(lens, nh, nkv, hd, page, dtype, seed, cols=cols, tracked=tracked)
        other = Case(far, nh, nkv, hd, page, dtype, seed + 1000, cols=far_cols, tracked=False)
        self.far_table = torch.where(other.table >= 0, other.table + self.pages, other.table)
        self.pages += other.pages
        self.k, self.v = torch.cat([self.k, other.k]), torch.cat([self.v, other.v])
        self.far_slots = other.slots
        self.of = torch.tensor(of, dtype=torch.int32, device=self.device)

    def prefix(self):
        from ttspipe_amd import pagedcache

        return pagedcache.Prefix(self.far_table, self.far_slots, self.of)
