"""Windows whose newest slot lies past the table's end (GPU): the slot is cut to the
table first, so the window is of the table's last rows, as one that ends there."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.gpuutil import bits
from tests.spandata import PrefixCase, slid, spans_check
from ttspipe_amd import pagedcache as pc

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 10), (299, 3), (1000, 0), (10**6, 10**6)])
@pytest.mark.parametrize("behind", [False, True])
def test_slots_past_the_table_are_its_last(window, sinks, behind):
    c = PrefixCase([304, 304, 120, 304], [70], [0, -1, 0, 0], 8, 2, 128, 16, FP, seed=window % 89)
    assert c.cap == 304
    slid(c, window, sinks)
    kw = dict(window=window, sinks=sinks, **(dict(prefix=c.prefix()) if behind else {}))
    last = c.slots.clone()
    before = c.scores.clone()
    want = pc.attention(c.q, *c.pools(), c.slots, scores=c.scores, **kw)
    torch.cuda.synchronize()
    spans_check(c, want, c.scores, before, **kw)
    scores = c.scores.clone()
    for over in (1, 17, 304, 10**12):
        c.slots.copy_(torch.where(last == c.cap - 1, last + over, last))
        c.scores.copy_(before)
        y = pc.attention(c.q, *c.pools(), c.slots, scores=c.scores, **kw)
        assert np.array_equal(bits(y), bits(want)) and torch.equal(c.scores, scores), over
