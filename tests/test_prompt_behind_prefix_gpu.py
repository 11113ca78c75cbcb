"""A stream's own prompt behind a prefix, prefilled over a contiguous cache that holds
the prefix's rows first (GPU): with `sinks` counted from the prefix's end, its rows
see what one-token attention over the prefix and the same window sees."""

from __future__ import annotations

import pytest
import torch

from tests.spandata import PrefixCase, spans64, spans_check
from tests.test_prefill_window_gpu import check as prompt_check
from tests.test_prefill_window_gpu import reference
from ttspipe_amd import fastpath
from ttspipe_amd import pagedcache as pc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,m,window,sinks", [(100, 60, 20, 4), (33, 130, 50, 0), (300, 40, 7, 40), (64, 64, 64, 3)])
def test_prompts_and_later_tokens_see_the_same_rows(n, m, window, sinks):
    nh, nkv = 8, 2
    # m sequences that are the stream at each of its rows: the same pages, slots 0 .. m - 1
    c = PrefixCase([m], [n], [0], nh, nkv, 128, 16, torch.bfloat16, seed=n + m, tracked=False)
    c.table, c.lens = c.table.repeat(m, 1), [m] * m
    c.slots, c.of = torch.arange(m, device="cuda"), torch.zeros(m, dtype=torch.int32, device="cuda")
    c.q = (torch.randn(m, nh, 128, generator=c.g) * 1.5).to(c.dtype).cuda()
    y = pc.attention(c.q, *c.pools(), c.slots, window=window, sinks=sinks, prefix=c.prefix())
    spans_check(c, y, window=window, sinks=sinks, prefix=c.prefix())
    rows = []
    for pages in (c.k, c.v):
        far, own = pages[c.far_table[0].long()], pages[c.table[0].long()]
        far, own = (t.transpose(0, 1).reshape(nkv, -1, 128) for t in (far, own))
        rows.append(torch.cat([far[:, :n], own[:, :m]], 1)[None].contiguous())
    q, pos = c.q.transpose(0, 1)[None], torch.arange(n, n + m, device="cuda")
    p = fastpath.prefill_attention(q, *rows, None, nh, nkv, 128, positions=pos, window=window, sinks=n + sinks)
    prompt_check(q, *rows, pos, window, n + sinks, p)
    # both meet their bars, of one value
    ref, seen = spans64(c.q, c.k, c.v, c.table, c.slots, window=window, sinks=sinks, prefix=c.prefix())[0], reference(q, *rows, pos, window, n + sinks)[0]
    assert float((ref - seen[0].transpose(0, 1)).abs().max()) < 1e-12
    # and with the decode's own number of sinks a prompt's rows miss the prefix
    short = fastpath.prefill_attention(q, *rows, None, nh, nkv, 128, positions=pos, window=window, sinks=sinks)
    if n - sinks > window:
        assert float((short.float() - p.float()).abs().max()) > 0.1
