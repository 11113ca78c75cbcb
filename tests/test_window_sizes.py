"""Windowed prompts whose sizes or strides leave the kernel's arithmetic are refused
before any launch (no GPU calls): keys in 32-bit numbers, a KV head's in 2 GiB."""

from __future__ import annotations

import pytest

from tests.test_paged import P
from ttspipe_amd import _lib


def _call(**kw):
    a = dict(Q=P, qs=1024, qh=128, K=P, ks=128, kh=4096, V=P, vs=128, vh=4096, pos=P, Y=P, S=20, nh=8, nkv=2, L=30, window=5, sinks=1,
             scale=0.1, dtype=1, work=P, splits=1)
    a.update(kw)
    return _lib.load().ttsp_prefill_attention_window(*a.values(), None)


@pytest.mark.parametrize("kw", [dict(L=2**31 - 1), dict(L=2**31 - 64), dict(L=2**31 - 127)])
def test_more_keys_than_are_counted(kw):
    """(All of them one row: no stride makes them too large.)"""
    assert _call(ks=0, vs=0, **kw) == 1


@pytest.mark.parametrize("kw", [dict(ks=1 << 61, L=9), dict(vs=1 << 61, L=9), dict(ks=1 << 62, L=5), dict(ks=(1 << 63) - 8, L=3),
                                dict(vs=1 << 60, L=17), dict(ks=1 << 30, L=2)])
def test_strides_whose_products_leave_64_bits(kw):
    assert _call(**kw) == 1
