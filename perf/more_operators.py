"""Attention over a shared prefix, attention through a sliding window with sinks, and
the penalties that logits get before they are sampled, as calls that can be timed
and compared.

Streams that decode together keep their keys and values in pages of one pool,
`[pages, kv heads, page size, head dim]`; a table row per sequence names its
pages (-1: none), slot j of a sequence is row j % page of its page j // page, and
`slots[b]` is its newest slot (-1: it holds nothing).

Operators ("op" of a case):

* "prefix": one new token of each sequence over the rows of the prefix that it
  shares with others (`of[b]`, -1: none) and its own rows 0 .. slots[b]:
  softmax(scale q . k) v over both. A prefix has pages of its own in the same
  pools, `prefix_slots[p]` its newest slot. With a window, own rows j with
  sinks <= j <= slots[b] - window are left out.
* "window": one new token of each sequence over its slots j <= slots[b] with
  j < sinks or j > slots[b] - window. Pages that no row can see any more have
  been given back.
* "prompt": new rows at `positions` over a contiguous cache that holds them
  already: row i sees keys j <= positions[i] with j < sinks or
  j > positions[i] - window.
* "logits": with c the number of times a token occurs in a row's history,
  x = logit; if c > 0: x / r where x > 0, else x r; then
  - (frequency c + presence [c > 0]) + bias, and -inf where the token's bit of
  the mask is 0.

Heads, widths and lengths are those of the repository's model (slow
transformer: 32 query and 8 KV heads of 128, 4096 logits) and generic ones
around them.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # two streams of one short voice prompt, early in their utterances: the smallest call
        dict(name="prefix_pair", op="prefix", seqs=2, prefixes=1, plo=300, phi=300, lo=1, hi=40, nh=32, nkv=8, hd=128, page=64, dtype="bf16", window=0, sinks=0),
        # 32 streams of one voice at different frames
        dict(name="prefix_streams", op="prefix", seqs=32, prefixes=1, plo=2011, phi=2011, lo=20, hi=900, nh=32, nkv=8, hd=128, page=64, dtype="bf16", window=0, sinks=0),
        # a server of several voices; some streams have none
        dict(name="prefix_voices", op="prefix", seqs=24, prefixes=5, plo=500, phi=4000, lo=1, hi=1500, nh=32, nkv=8, hd=128, page=16, dtype="fp16", window=0, sinks=0),
        # a full server over one very long context, each stream's own rows through a window: the largest call
        dict(name="prefix_long", op="prefix", seqs=64, prefixes=1, plo=32763, phi=32763, lo=1, hi=1900, nh=32, nkv=8, hd=128, page=256, dtype="bf16", window=512, sinks=4),
        # one stream that has outgrown its window: the smallest call
        dict(name="window_one", op="window", seqs=1, lo=1500, hi=1500, nh=32, nkv=8, hd=128, page=64, dtype="bf16", window=256, sinks=4),
        # 32 streams, some still shorter than the window
        dict(name="window_streams", op="window", seqs=32, lo=200, hi=8000, nh=32, nkv=8, hd=128, page=16, dtype="fp16", window=1024, sinks=4),
        # a full server of long streams
        dict(name="window_wide", op="window", seqs=64, lo=9000, hi=60000, nh=32, nkv=8, hd=128, page=64, dtype="bf16", window=4093, sinks=64),
        # a span of a prompt over the rows before it
        dict(name="prompt_span", op="prompt", rows=512, start=2000, nh=32, nkv=8, window=1024, sinks=4, dtype="bf16"),
        # a whole long prompt
        dict(name="prompt_long", op="prompt", rows=8111, start=0, nh=32, nkv=8, window=2048, sinks=16, dtype="bf16"),
        # one stream's row against the frames it has just drawn: the smallest call
        dict(name="logits_step", op="logits", rows=1, vocab=4096, history=16, dtype="bf16", repetition=True, additive=False, bias=False, mask=False),
        # 32 streams with everything on
        dict(name="logits_streams", op="logits", rows=32, vocab=32768, history=1023, dtype="fp16", repetition=True, additive=True, bias=True, mask=True),
        # a full server with long histories and a large vocabulary
        dict(name="logits_wide", op="logits", rows=256, vocab=131001, history=4096, dtype="fp32", repetition=True, additive=True, bias=False, mask=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


#: (query heads, KV heads): the repository's models' and other groupings
HEADS = [(32, 8), (32, 8), (8, 2), (16, 8), (4, 2), (7, 7), (20, 4), (32, 2), (24, 1)]
#: groupings of a prompt's attention (at most eight query heads a KV head)
PROMPT_HEADS = [(32, 8), (32, 8), (8, 2), (16, 8), (4, 2), (7, 7), (20, 4), (16, 2), (5, 1)]


def draw(rng):
    op = rng.choice(["prefix", "prefix", "prefix", "window", "window", "prompt", "prompt", "logits", "logits"])
    dtype, page = rng.choice(["bf16", "fp16"]), rng.choice([16, 32, 64, 128, 256])
    hd = rng.choice([128, 128, 64])
    nh, nkv = rng.choice(HEADS)
    if op == "prefix":
        seqs = _log_int(rng, 1, 64)
        prefixes = min(seqs, rng.choice([1, 1, _log_int(rng, 1, 8)]))
        most = min(32768, 64 * 32 * 32768 // (seqs * nh))
        phi = _log_int(rng, 16, min(most, (1 << 22) // (seqs * nkv)) if prefixes > 1 else most)
        hi = _log_int(rng, 1, min(4096, (1 << 20) // (seqs * nkv)))
        window = rng.choice([0, 0, _log_int(rng, 1, 1024)])
        return dict(op=op, seqs=seqs, prefixes=prefixes, plo=rng.choice([max(1, phi // 4), phi]), phi=phi, lo=rng.choice([1, max(1, hi // 2)]),
                    hi=hi, nh=nh, nkv=nkv, hd=hd, page=page, dtype=dtype, window=window, sinks=rng.choice([0, 4, 37]) if window else 0)
    if op == "window":
        seqs = _log_int(rng, 1, 64)
        window = _log_int(rng, 1, max(1, min(16384, 64 * 4096 * 8 // (seqs * max(nkv, nh // 4)))))
        hi = _log_int(rng, max(1, window // 2), 65536)
        return dict(op=op, seqs=seqs, lo=rng.choice([1, max(1, hi // 2), hi]), hi=hi, nh=nh, nkv=nkv, hd=hd, page=page, dtype=dtype,
                    window=window, sinks=rng.choice([0, 1, 4, 16, 64, rng.randint(0, 200)]))
    if op == "prompt":
        nh, nkv = rng.choice(PROMPT_HEADS)
        rows = _log_int(rng, 9, 8000)
        return dict(op=op, rows=rows, start=rng.choice([0, 0, _log_int(rng, 1, 12000 - rows)]), nh=nh, nkv=nkv,
                    window=_log_int(rng, 1, 2000), sinks=rng.choice([0, 4, 16, rng.randint(0, 100)]), dtype=dtype)
    rows = _log_int(rng, 1, 256)
    additive = rng.random() < 0.6
    return dict(op=op, rows=rows, vocab=_log_int(rng, 500, min(160000, 256 * 131001 // rows)), history=_log_int(rng, 1, 4096),
                dtype=rng.choice(["bf16", "fp16", "fp32"]), repetition=not additive or rng.random() < 0.7, additive=additive,
                bias=rng.random() < 0.4, mask=rng.random() < 0.6)


# ------------------------------------------------------------------- inputs


def _randn(g, *shape, dtype, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV).mul_(scale).to(dtype)


def _lengths(g, lo, hi, count):
    n = torch.randint(lo, hi + 1, (count,), generator=g, device=DEV)
    n[-1] = hi
    return n


def _pages(g, used):
    """Tables (a list of them) whose `used` columns name the pages of one pool in random order, -1 elsewhere, and the pool's size."""
    counts = [int(u.sum()) for u in used]
    order, at, tables = torch.randperm(sum(counts), generator=g, device=DEV).to(torch.int32), 0, []
    for u, n in zip(used, counts):
        t = torch.full(u.shape, -1, dtype=torch.int32, device=DEV)
        t[u] = order[at:at + n]
        tables.append(t)
        at += n
    return tables, sum(counts)


def _columns(n, width, page, seen=None):
    """Whether a row of a table has its column's page: for slots below n that `seen` (first, end of what is not seen) does not leave out."""
    col = torch.arange(-(-width // page), device=DEV) * page
    used = col < n[:, None]
    if seen is not None:
        used &= (col < seen[0]) | (col + page > seen[1][:, None])
    return used


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    s = dict(case=dict(case))
    if op == "logits":
        rows, vocab, hist = case["rows"], case["vocab"], case["history"]
        s["logits"] = _randn(g, rows, vocab, dtype=dtype, scale=4.0)
        # tokens drawn so far: a few come often; rows of different lengths, one full
        often = (torch.rand(rows, hist, generator=g, device=DEV).pow_(4) * vocab).long()
        s["history"] = often.clamp_(max=vocab - 1).to(torch.int32)
        s["lengths"] = _lengths(g, max(1, hist // 4), hist, rows).to(torch.int32)
        uniform = lambda lo, hi: torch.rand(rows, generator=g, device=DEV).mul_(hi - lo).add_(lo)  # noqa: E731
        s["repetition"] = uniform(1.0, 1.5) if case["repetition"] else None
        s["frequency"], s["presence"] = (uniform(0.0, 0.5), uniform(0.0, 1.0)) if case["additive"] else (None, None)
        s["bias"] = _randn(g, vocab, dtype=torch.float32) if case["bias"] else None
        s["mask"] = None
        if case["mask"]:
            s["mask"] = torch.randint(-(1 << 31), 1 << 31, (rows, -(-vocab // 32)), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
        return s
    if op == "prompt":
        rows, total = case["rows"], case["start"] + case["rows"]
        s["q"] = _randn(g, rows, case["nh"], 128, dtype=dtype, scale=1.5)[None].transpose(1, 2)
        # the cache of a model that could hold more
        s["k"], s["v"] = (_randn(g, 1, case["nkv"], total + 57, 128, dtype=dtype)[:, :, :total] for _ in "kv")
        s["positions"] = torch.arange(case["start"], total, device=DEV)
        return s
    nkv, hd, page, seqs, nh = case["nkv"], case["hd"], case["page"], case["seqs"], case["nh"]
    n = _lengths(g, case["lo"], case["hi"], seqs)
    s["slots"] = n - 1
    if op == "window":
        used = [_columns(n, case["hi"], page, (case["sinks"], n - case["window"]))]
    else:
        p = _lengths(g, case["plo"], case["phi"], case["prefixes"])
        s["prefix_slots"] = p - 1
        s["of"] = torch.randint(0, case["prefixes"], (seqs,), generator=g, device=DEV, dtype=torch.int32)
        if case["prefixes"] > 1:
            s["of"][torch.rand(seqs, generator=g, device=DEV) < 0.1] = -1
        used = [_columns(n, case["hi"], page), _columns(p, case["phi"], page)]
    tables, pages = _pages(g, used)
    s["block_table"] = tables[0]
    if op == "prefix":
        s["prefix_table"] = tables[1]
    s["k_pages"] = _randn(g, pages, nkv, page, hd, dtype=dtype)
    s["v_pages"] = _randn(g, pages, nkv, page, hd, dtype=dtype)
    s["q"] = _randn(g, seqs, nh, hd, dtype=dtype, scale=1.5)
    return s


# --------------------------------------------------------------- plain forms


def _slots_of(pages, table, slot):
    """[B, kv heads, slots, head dim] in 32 bits: the rows of `slot` [B, slots] through the table (one without a page: row of page 0)."""
    page = pages.shape[2]
    at = table.gather(1, (slot // page).clamp(0, table.shape[1] - 1)).clamp(min=0).long()
    return pages[at, :, slot % page].float().transpose(1, 2)


def _dots(q, k):
    """[B, kv, group, slots]: q [B, nh, hd] with each KV head's rows k [B, kv, slots, hd], scaled."""
    b, nkv, _, hd = k.shape
    return torch.matmul(k, q.float().view(b, nkv, -1, hd).transpose(2, 3).contiguous()).transpose(2, 3) * hd**-0.5


def _visible(s, cap):
    """Slots a sequence's newest token may see, [B, width], and which of them are there."""
    case, last = s["case"], s["slots"][:, None]
    if not case["window"]:
        slot = torch.arange(cap, device=last.device).expand(last.shape[0], cap)
        return slot, slot <= last
    sinks, window = min(case["sinks"], cap), min(case["window"], cap)
    sink = torch.arange(sinks, device=last.device).expand(last.shape[0], sinks)
    near = last - window + 1 + torch.arange(window, device=last.device)
    slot = torch.cat([sink, near], 1)
    there = torch.cat([sink <= last, near >= sinks], 1)
    return slot.clamp(min=0), there


def _one_token(s):
    case, q = s["case"], s["q"]
    slot, there = _visible(s, case["hi"])
    k, v = _slots_of(s["k_pages"], s["block_table"], slot), _slots_of(s["v_pages"], s["block_table"], slot)
    there = there[:, None, None]
    dots = torch.where(there, _dots(q, k), -math.inf)
    top = dots.amax(-1, keepdim=True)
    if case["op"] == "prefix":
        rows = torch.arange(case["phi"], device=q.device).expand(case["prefixes"], case["phi"])
        pk, pv = _slots_of(s["k_pages"], s["prefix_table"], rows), _slots_of(s["v_pages"], s["prefix_table"], rows)
        of = s["of"].clamp(min=0).long()
        seen = ((rows[:1] <= s["prefix_slots"][of][:, None]) & (s["of"] >= 0)[:, None])[:, None, None]
        b, nkv, hd = q.shape[0], case["nkv"], case["hd"]
        if case["prefixes"] == 1:  # one product for all sequences
            qs = q.float().view(b, nkv, -1, hd).transpose(0, 1).reshape(1, nkv, -1, hd)
            far = torch.matmul(pk, qs.transpose(2, 3).contiguous()).transpose(2, 3).reshape(nkv, b, -1, case["phi"])
            far = far.transpose(0, 1) * hd**-0.5
        else:
            far = _dots(q, pk[of])
        far = torch.where(seen, far, -math.inf)
        top = torch.maximum(top, far.amax(-1, keepdim=True))
    e = torch.where(there, torch.exp(dots - top), 0.0)
    total, y = e.sum(-1, keepdim=True), torch.matmul(e, v)
    if case["op"] == "prefix":
        f = torch.where(seen, torch.exp(far - top), 0.0)
        total = total + f.sum(-1, keepdim=True)
        if case["prefixes"] == 1:
            fs = f.transpose(0, 1).reshape(1, nkv, -1, case["phi"])
            y = y + torch.matmul(fs, pv).reshape(nkv, b, -1, hd).transpose(0, 1)
        else:
            y = y + torch.matmul(f, pv[of])
    y = torch.where(total > 0, y / total, 0.0)
    return [y.reshape(q.shape).to(q.dtype)]


def _prompt(s):
    case, pos = s["case"], s["positions"][:, None]
    key = torch.arange(s["k"].shape[2], device=pos.device)
    seen = (key <= pos) & ((key < case["sinks"]) | (key > pos - case["window"]))
    nkv = case["nkv"]
    q = s["q"].float().reshape(nkv, -1, 128)
    k, v = s["k"][0].float(), s["v"][0].float()
    dots = torch.matmul(q, k.transpose(1, 2).contiguous()).view(nkv, -1, *seen.shape).mul_(128**-0.5)
    dots.masked_fill_(~seen, -math.inf)
    e = dots.sub_(dots.amax(-1, keepdim=True)).exp_()
    y = torch.matmul(e.view(nkv, -1, seen.shape[1]), v).view(nkv, -1, case["rows"], 128) / e.sum(-1, keepdim=True)
    return [y.reshape(1, case["nh"], case["rows"], 128).to(s["q"].dtype)]


def _logits(s):
    case, x = s["case"], s["logits"].float()
    vocab, hist = case["vocab"], case["history"]
    there = torch.arange(hist, device=x.device) < s["lengths"][:, None]
    token = torch.where(there, s["history"], vocab).long()
    count = torch.zeros(x.shape[0], vocab + 1, device=x.device).scatter_add_(1, token, torch.ones_like(token, dtype=torch.float32))
    count = count[:, :vocab]
    if s["repetition"] is not None:
        r = s["repetition"][:, None]
        x = torch.where(count > 0, torch.where(x > 0, x / r, x * r), x)
    if s["frequency"] is not None:
        x = x - (s["frequency"][:, None] * count + s["presence"][:, None] * (count > 0))
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["mask"] is not None:
        bit = (s["mask"][:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = torch.where(bit.flatten(1)[:, :vocab] != 0, x, -math.inf)
    return [x.to(s["logits"].dtype)]


# ----------------------------------------------------------------- one pass


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if not own:
        return {"prefix": _one_token, "window": _one_token, "prompt": _prompt, "logits": _logits}[op](s)
    if op == "logits":
        from ttspipe_amd import fusedsample

        return [fusedsample.penalize(s["logits"], s["history"], lengths=s["lengths"], repetition=s["repetition"],
                                     frequency=s["frequency"], presence=s["presence"], bias=s["bias"], mask=s["mask"])]
    if op == "prompt":
        from ttspipe_amd import fastpath

        return [fastpath.prefill_attention(s["q"], s["k"], s["v"], None, case["nh"], case["nkv"], 128, positions=s["positions"],
                                           window=case["window"], sinks=case["sinks"])]
    from ttspipe_amd import pagedcache

    prefix = pagedcache.Prefix(s["prefix_table"], s["prefix_slots"], s["of"]) if op == "prefix" else None
    return [pagedcache.attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["slots"], prefix=prefix,
                                 window=case["window"] or None, sinks=case["sinks"])]


# --------------------------------------------------------------------- work


def _mean_own(case):
    """Mean own rows a sequence's newest token sees (lengths even over lo .. hi)."""
    lo, hi, w = case["lo"], case["hi"], case["window"]
    if not w:
        return (lo + hi) / 2
    top, span = w + case["sinks"], max(1, hi - lo)
    if lo >= top:
        return top
    return (lo + hi) / 2 if hi <= top else ((lo + top) / 2 * (top - lo) + top * (hi - top)) / span


def work(case):
    op = case["op"]
    if op == "logits":
        size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
        n = case["rows"] * case["vocab"]
        read = case["rows"] * (0.625 * case["history"] * 4 + 16) + (4 * case["vocab"] if case["bias"] else 0) + (n / 8 if case["mask"] else 0)
        return dict(bytes=2 * n * size + read, flops=n * (case["repetition"] + 2 * case["additive"] + case["bias"]))
    if op == "prompt":
        rows, start, w, sinks = case["rows"], case["start"], case["window"], case["sinks"]
        total = start + rows
        seen = sum(min(p + 1, w + min(sinks, max(0, p + 1 - w))) for p in range(start, total))
        keys = min(total, rows + w - 1 + sinks)
        return dict(bytes=256 * (2 * rows * case["nh"] + 2 * keys * case["nkv"]) + 8 * rows, flops=4 * 128 * case["nh"] * seen)
    seqs, nh, nkv, hd = (case[x] for x in ("seqs", "nh", "nkv", "hd"))
    own_rows = seqs * _mean_own(case)
    read, pairs = own_rows, own_rows
    if op == "prefix":
        each = (case["plo"] + case["phi"]) / 2 if case["prefixes"] > 1 else case["phi"]
        read, pairs = read + case["prefixes"] * each, pairs + seqs * each
    return dict(bytes=4 * read * nkv * hd + 4 * seqs * nh * hd + 4 * read / case["page"] + 12 * seqs, flops=4 * pairs * nh * hd)


# ---------------------------------------------------- the definition, in 64 bits


def _rows64(pages, row, slots, h):
    page = pages.shape[2]
    return pages[row[slots // page].long(), h, slots % page].double()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "logits":
        x = s["logits"].double()
        for i, n in enumerate(s["lengths"].tolist()):
            token, times = torch.unique(s["history"][i, :n].long(), return_counts=True)
            if s["repetition"] is not None:
                r, y = s["repetition"][i].double(), x[i, token]
                x[i, token] = torch.where(y > 0, y / r, y * r)
            if s["frequency"] is not None:
                x[i, token] -= s["frequency"][i].double() * times + s["presence"][i].double()
        if s["bias"] is not None:
            x += s["bias"].double()
        if s["mask"] is not None:
            words = s["mask"].long()[:, torch.arange(case["vocab"], device=DEV) // 32]
            x[(words >> (torch.arange(case["vocab"], device=DEV) % 32)) % 2 == 0] = -math.inf
        return [x]
    if op == "prompt":
        group = case["nh"] // case["nkv"]
        y = torch.empty(1, case["nh"], case["rows"], 128, dtype=torch.float64, device=DEV)
        key = torch.arange(s["k"].shape[2], device=DEV)
        for h in range(case["nh"]):
            k, v = s["k"][0, h // group].double(), s["v"][0, h // group].double()
            for i in range(0, case["rows"], 1024):
                pos = s["positions"][i:i + 1024, None]
                hidden = (key > pos) | ((key >= case["sinks"]) & (key <= pos - case["window"]))
                w = (s["q"][0, h, i:i + 1024].double() @ k.t() / math.sqrt(128)).masked_fill(hidden, -math.inf)
                y[0, h, i:i + 1024] = torch.softmax(w, 1) @ v
        return [y]
    group = case["nh"] // case["nkv"]
    y = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for h in range(case["nkv"]):
        heads = slice(h * group, (h + 1) * group)
        shared = {}
        for b, last in enumerate(s["slots"].tolist()):
            own_slots = torch.arange(last + 1, device=DEV)
            if case["window"]:
                own_slots = own_slots[(own_slots < case["sinks"]) | (own_slots > last - case["window"])]
            k, v = (_rows64(s[x], s["block_table"][b], own_slots, h) for x in ("k_pages", "v_pages"))
            p = int(s["of"][b]) if op == "prefix" else -1
            q = s["q"][b, heads].double()
            dots = q @ k.t() / math.sqrt(case["hd"])
            if p >= 0:
                if p not in shared:
                    rows = torch.arange(int(s["prefix_slots"][p]) + 1, device=DEV)
                    shared[p] = [_rows64(s[x], s["prefix_table"][p], rows, h) for x in ("k_pages", "v_pages")]
                far = q @ shared[p][0].t() / math.sqrt(case["hd"])
                w = torch.softmax(torch.cat([far, dots], 1), 1)
                y[b, heads] = w[:, : far.shape[1]] @ shared[p][1] + w[:, far.shape[1]:] @ v
            else:
                y[b, heads] = torch.softmax(dots, 1) @ v
    return [y]
