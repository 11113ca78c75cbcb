"""`PageTable.slide` on the host (no GPU calls): what it looks at, and what it gives
back when windows, sinks and sequences change."""

from __future__ import annotations

import random

import pytest

from ttspipe_amd import pagedcache as pc


class Counted(list):
    """A list that counts the elements read from it."""

    reads = 0

    def __getitem__(self, i):
        self.reads += 1
        return super().__getitem__(i)


def test_a_step_looks_at_no_column_twice():
    """A stream of 10,000 rows whose window has left 600 pages of 16: sixteen more
    steps, of which one leaves a page behind."""
    t = pc.PageTable(2, 20000, 1300, 16, device="cpu")
    t.admit(10000), t.admit(9000)
    t.slide(400, 20)
    free = t.free_pages
    held = t._held[:] = [Counted(h) for h in t._held]
    for _ in range(16):
        t.step()
        t.slide(400, 20)
    assert t.free_pages == free  # (a page given back by each, and one taken)
    assert all(h.reads <= 8 for h in held), [h.reads for h in held]


def _left(n, window, sinks, page):
    """Columns that no row of the newest token's window, or a later one's, lies in."""
    return {c for c in range(-(-n // page)) if c * page >= sinks and (c + 1) * page <= n - window}


@pytest.mark.parametrize("seed", range(12))
def test_windows_sinks_and_sequences_that_change(seed):
    """Each call gives back what its own window has left, whatever the calls before
    it were for; sequences are cut, released and admitted in between."""
    rng = random.Random(seed)
    page = rng.choice([16, 32])
    t = pc.PageTable(3, 600, 200, page, device="cpu")
    gone = [set(), set(), set()]
    for _ in range(120):
        what = rng.choice(["step"] * 8 + ["slide"] * 4 + ["jump", "cut", "release"])
        live = [b for b in range(3) if t.rows(b)]
        if what == "jump" and len(live) < 3:
            b = t.admit(rng.randint(1, 300))
            gone[b] = set()
        elif what == "release" and live:
            b = rng.choice(live)
            t.release(b)
            gone[b] = set()
        elif what == "cut" and rng.random() < 0.4:
            budget = rng.randint(20, 300)
            t.evicted(budget)
            keep = -(-(budget + 1) // page)
            gone = [{c for c in g if c < keep} for g in gone]
        elif what == "slide":
            window, sinks = rng.choice([(1, 0), (30, 4), (30, 40), (100, 0), (100, 17), (250, 4)])
            t.slide(window, sinks)
            for b in range(3):
                gone[b] |= _left(t.rows(b), window, sinks, page)
        elif all(t.rows(b) < 600 for b in range(3)):
            t.step()
        held = []
        for b in range(3):
            row = t.block_table[b].tolist()
            n = -(-t.rows(b) // page)
            assert {c for c in range(n) if row[c] < 0} == gone[b], (what, b)
            held += [x for x in row if x >= 0]
        assert len(held) == len(set(held)) == 200 - t.free_pages
    for b in range(3):
        t.release(b)
    assert t.free_pages == 200
