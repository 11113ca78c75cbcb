"""Top-k / top-p sampling of one logit row in one HIP launch.

Drop-in for the reference's `app/engine/fusedsample.py` (`MAX_TOP_K`,
`available`, `sample`): the fork's sampler - temperature, top-k, top-p, then a
draw - which the fork runs as a full sort, a softmax, a cumsum, a scatter and
a second softmax. Here one workgroup holds the row in LDS, finds the k-th
largest value by bisection over its 16-bit pattern, gathers the k winners in
index order, ranks them by pairwise counting, and draws
`argmax(v / temperature - log(-log(u)))` over those that survive the top-p
cut, with `u` one uniform number per vocabulary index from `torch.rand`.
That is the Gumbel form of the fork's `argmax(probs / Exp(1))`: exact
sampling from the truncated, tempered distribution (reference:
fusedsample.py:1-19, 225-257). The cumulative mass is summed in fp32 where the
fork's fp16 cumsum rounds, so a draw whose mass lands exactly on the top-p
boundary can differ; the distribution is the same.

`penalize` goes before it: penalties for the tokens that a row's history
holds, biases and a grammar's mask, for the rows of several streams at once
(the reference's sampler has none of them).
"""

from __future__ import annotations

import struct

import torch

from ttspipe_amd import _lib

#: Largest `top_k` the kernel takes; larger requests use the caller's sampler.
MAX_TOP_K = 64

#: Longest row the kernel takes (the row is held in LDS); `sample` returns None
#: for a longer one and the caller's sampler runs.
MAX_VOCAB = 32768


def available() -> bool:
    """True when the HIP library is loadable on a GPU machine."""
    if not _lib.gpu_present():
        return False
    try:
        _lib.lib()
    except Exception:  # noqa: BLE001 - the caller's sampler still works
        return False
    return True


def sample(logits, temperature, top_p, top_k, uniform=None):
    """The fork's `sample(...)[0]`: an int32 tensor of shape (1,) holding the
    drawn index, or None for a row longer than `MAX_VOCAB`. `temperature`/`top_p` are one-element tensors, `top_k` a
    one-element int64 tensor, all on the logits' device (so a captured graph
    can change them in place); `uniform` (optional) supplies the per-index
    uniform numbers (default: `torch.rand`)."""
    row = logits.reshape(-1)
    if row.numel() > MAX_VOCAB:
        return None
    dt = _lib.dtype_code(row.dtype)
    if dt not in (_lib.DT_F16, _lib.DT_BF16):
        row, dt = row.to(torch.float16), _lib.DT_F16
    row = row.contiguous()
    temp = temperature.reshape(-1)[:1].to(row.dtype).contiguous()
    topp = top_p.reshape(-1)[:1].to(row.dtype).contiguous()
    topk = top_k.reshape(-1)[:1].to(torch.int64).contiguous()
    if uniform is None:
        uniform = torch.rand(row.numel(), device=row.device, dtype=torch.float32)
    elif uniform.dtype != torch.float32 or uniform.numel() != row.numel():
        raise ValueError("uniform must hold one float32 per logit")
    out = torch.empty(1, dtype=torch.int32, device=row.device)
    rc = _lib.lib().ttsp_sample_topk(row.data_ptr(), row.numel(), dt, temp.data_ptr(), topp.data_ptr(),
                                     topk.data_ptr(), uniform.contiguous().data_ptr(), out.data_ptr(), _lib.stream())
    _lib.check(rc, "ttsp_sample_topk")
    return out


#: `ttsp_penalties`' fields in order (`_lib.Penalties` names them).
_PENALTIES = struct.Struct("@7P3q7i4x")


def pack_mask(allowed):
    """The words `penalize` takes as `mask` (int32, (..., ceil(V / 32))) from a
    boolean tensor (..., V): bit t % 32 of word t // 32 is allowed[..., t]. Torch
    operations, for programs whose grammar does not write the words itself."""
    v = allowed.shape[-1]
    bits = torch.nn.functional.pad(allowed.to(torch.int64), (0, -v % 32)).unflatten(-1, (-1, 32))
    words = (bits << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _rows_of(t, rows, width, dev, what):
    """(address, row stride) of a tensor (rows, width), (1, width) or (width,) on `dev`. (On every call's host path, as the next.)"""
    shape = t.shape
    if len(shape) == 2:
        n, step = shape[0], t.stride()
        if shape[1] == width and (n == rows or n == 1) and (step[1] == 1 or width < 2) and t.get_device() == dev:
            return t.data_ptr(), step[0] if n > 1 else 0
    elif len(shape) == 1 and shape[0] == width and (width < 2 or t.stride()[0] == 1) and t.get_device() == dev:
        return t.data_ptr(), 0
    raise ValueError(f"{what} must be ({rows}, {width}) or ({width},) with a contiguous last axis, on the logits' device")


def _vector(t, rows, dev, what):
    """(address, 0: one value for all rows) of an fp32 tensor of one value a row, or of one."""
    n = t.numel()
    if t.dtype is torch.float32 and (n == rows or n == 1) and t.dim() < 2 and t.is_contiguous() and t.get_device() == dev:
        return t.data_ptr(), int(n > 1)
    raise ValueError(f"{what} must be a contiguous fp32 tensor of one value a row, or of one, on the logits' device")


def penalize(logits, history=None, *, lengths=None, repetition=None, frequency=None, presence=None, bias=None,
             mask=None, out=None):
    """Logits (rows, V) or (V,) of 16 or 32 bits as the sampler should see them, in
    one launch: with c the number of times token t occurs in its row's history,

        x = logit;  where c > 0:  x = x / repetition if x > 0 else x * repetition,
        x -= frequency * c + presence;  x += bias;  -inf where the mask forbids t

    in fp32 with one rounding to the logits' type at the end. Every part may be
    left out. `history` int32 or int64 (rows, H), or (H,) for all rows: a token
    outside 0 .. V - 1 (-1 for padding) counts for none; `lengths` int32 or int64
    (rows,): only so many of a row's first entries count (values outside
    0 .. H are cut to it). `repetition`, `frequency`, `presence`: fp32, one value a
    row or one in all, on the device, so that a captured graph's can be changed in
    place. `bias` fp32 or of the logits' type, (rows, V) or (V,). `mask` int32
    (rows, ceil(V / 32)) or (ceil(V / 32),): bit t % 32 of word t // 32 set where
    t is allowed (`pack_mask`); a row that allows nothing is -inf throughout, which
    `sample` has no draw for.

    Returns the new logits, in `out` if given: the logits themselves, or a tensor
    of their shape and type that overlaps no input. None where the kernel does not
    take the logits (no GPU, another type, a last axis that is not contiguous);
    ValueError for parts that do not fit them. Work is queued on the current
    stream of the logits' device; with `out` nothing is allocated."""
    dtype, shape, dev = logits.dtype, logits.shape, logits.get_device()
    dt, dims = _lib.dtype_code(dtype), len(shape)
    if not _lib.gpu_present() or dt is None or dims not in (1, 2) or dev < 0:
        return None
    step, vocab = logits.stride(), shape[-1]
    rows, x_row = (shape[0], step[0]) if dims == 2 and shape[0] != 1 else (1, vocab)
    if vocab > 1 << 30 or rows > 1 << 24 or rows * -(-vocab // 2048) > 0x3fffff or (vocab > 1 and step[-1] != 1):
        return None
    hist = hp = hs = h64 = lp = l64 = rp = rr = fp = fr = pp = pr = bp = bs = mp = ms = 0
    bias_dt = dt
    if history is not None:
        h64 = history.dtype is torch.int64
        hist = history.shape[-1] if history.dim() else 0
        if (not h64 and history.dtype is not torch.int32) or not history.dim() or hist >= 1 << 31:
            raise ValueError("history must be an int32 or int64 tensor of at most 2^31 - 1 tokens a row")
        hp, hs = _rows_of(history, rows, hist, dev, "history")
    if lengths is not None:
        l64 = lengths.dtype is torch.int64
        if ((not l64 and lengths.dtype is not torch.int32) or lengths.shape != (rows,) or not lengths.is_contiguous()
                or lengths.get_device() != dev):
            raise ValueError("lengths must be a contiguous int32 or int64 tensor (rows,) on the logits' device")
        lp = lengths.data_ptr()
    if repetition is not None:
        rp, rr = _vector(repetition, rows, dev, "repetition")
    if frequency is not None:
        fp, fr = _vector(frequency, rows, dev, "frequency")
    if presence is not None:
        pp, pr = _vector(presence, rows, dev, "presence")
    if bias is not None:
        if bias.dtype is torch.float32:
            bias_dt = _lib.DT_F32
        elif bias.dtype is not dtype:
            raise ValueError("bias must be fp32 or of the logits' type")
        bp, bs = _rows_of(bias, rows, vocab, dev, "bias")
    if mask is not None:
        if mask.dtype is not torch.int32:
            raise ValueError("mask must hold int32 words")
        mp, ms = _rows_of(mask, rows, -(-vocab // 32), dev, "mask")
    xp = logits.data_ptr()
    if out is None:
        out = logits.new_empty(shape)
        yp, y_row = out.data_ptr(), vocab
    else:
        if out.shape != shape or out.dtype is not dtype or out.get_device() != dev or (vocab > 1 and out.stride()[-1] != 1):
            raise ValueError("out must have the logits' shape, type and device, and a contiguous last axis")
        yp, y_row = out.data_ptr(), out.stride()[0] if rows > 1 else vocab
        if rows > 1 and vocab and y_row < vocab:
            raise ValueError("out's rows must not overlap")
        size = out.element_size()
        if ((xp != yp or x_row != y_row) and rows and vocab and xp < yp + ((rows - 1) * y_row + vocab) * size
                and yp < xp + ((rows - 1) * x_row + vocab) * size):
            raise ValueError("out must be the logits themselves or not overlap them")
    if rows and vocab:
        block = _PENALTIES.pack(hp, lp, rp, fp, pp, bp, mp, hs, bs, ms, hist, h64, l64, rr, fr, pr, bias_dt)
        _lib.launch("ttsp_penalize", dev, block, xp, x_row, yp, y_row, rows, vocab, dt)
    return out
