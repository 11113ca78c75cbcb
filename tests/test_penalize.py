"""Penalties on logits on the host (no GPU calls): what the C entry refuses before
any launch, the mirrored argument block, the packed masks, and the call without a
GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from ttspipe_amd import _lib, fusedsample

P = 1 << 20  # an address that is aligned and never followed


def _call(block=None, **kw):
    a = dict(X=P, xs=100, Y=P, ys=100, rows=3, vocab=100, dtype=_lib.DT_BF16)
    a.update(kw)
    block = _lib.Penalties() if block is None else block
    return _lib.load().ttsp_penalize(ctypes.byref(block) if block else None, *a.values(), None)


def test_the_argument_block_is_the_one_that_is_packed():
    assert ctypes.sizeof(_lib.Penalties) == fusedsample._PENALTIES.size
    values = list(range(1, 18))
    block = _lib.Penalties.from_buffer_copy(fusedsample._PENALTIES.pack(*values))
    assert [getattr(block, name) for name, _ in _lib.Penalties._fields_] == values


@pytest.mark.parametrize("kw", [dict(X=None), dict(Y=None), dict(X=P + 1), dict(Y=P + 1), dict(xs=-1), dict(ys=99), dict(rows=-1),
                                dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(dtype=3), dict(dtype=_lib.DT_F32, X=P + 2),
                                dict(rows=1 << 24, vocab=1 << 20, ys=1 << 20)])
def test_bad_rows_are_refused(kw):
    assert _call(**kw) == 1


@pytest.mark.parametrize("kw", [dict(hist=-1), dict(HIST=P, hist=4, hist_row_stride=-1), dict(HIST=P + 2, hist=4),
                                dict(HIST=P + 4, hist=4, hist_64=1), dict(LEN=P + 1), dict(LEN=P + 4, len_64=1), dict(REP=P + 1),
                                dict(FREQ=P + 2), dict(PRES=P + 3), dict(MASK=P + 2), dict(mask_row_stride=-8),
                                dict(BIAS=P, bias_dtype=_lib.DT_F16), dict(BIAS=P + 2, bias_dtype=_lib.DT_F32),
                                dict(BIAS=P + 1, bias_dtype=_lib.DT_BF16), dict(bias_row_stride=-1)])
def test_bad_parts_are_refused(kw):
    assert _call(_lib.Penalties(**kw)) == 1


def test_no_block_is_refused_and_no_rows_are_taken():
    lib = _lib.load()
    assert lib.ttsp_penalize(None, P, 100, P, 100, 3, 100, 0, None) == 1
    assert _call(rows=0) == 0


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 64, 100])
def test_packed_masks(vocab):
    allowed = torch.rand(3, vocab, generator=torch.Generator().manual_seed(vocab)) < 0.5
    allowed[2] = True
    words = fusedsample.pack_mask(allowed)
    assert words.dtype is torch.int32 and words.shape == (3, -(-vocab // 32))
    for i in range(3):
        for t in range(vocab):
            assert (int(words[i, t // 32]) >> (t % 32)) & 1 == int(allowed[i, t])
    assert torch.equal(fusedsample.pack_mask(allowed[1]), words[1])


def test_a_call_without_a_gpu_is_declined():
    assert fusedsample.penalize(torch.zeros(2, 10)) is None
