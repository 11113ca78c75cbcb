"""The paged key-value cache's operators, as calls that can be timed and compared.

Streams that decode together keep their keys and values in pages of one pool,
`[pages, kv heads, page size, head dim]`; a table row per sequence names its
pages (-1: none). Slot j of a sequence is row j % page of its page j // page.
`slots[b]` is the newest slot of sequence b (-1: it holds nothing). Beside the
pools a cache may hold, per sequence, KV head and slot, the attention weight
the slot has gathered (`scores`, fp32) and the position its row came from
(`slot_pos`, int32).

Operators ("op" of a case):

* "attend": one new token of each sequence over its slots 0 .. slots[b]:
  softmax(scale q . k) v, zeros for a sequence that holds nothing. With
  "track", each slot's weight, summed over the query heads of its KV head,
  is added to `scores`.
* "rope": the wqkv output's rows: q and k heads normed (x / rms(x) * w) and
  rotated in interleaved pairs at the row's position, k and v written to the
  row's slot, its score set to 0 and its position noted.
* "store": k and v rows written as they are (a prompt's rows from the
  contiguous cache it was prefilled in).
* "evict": sequences of more than `budget` rows keep, in each KV head, the
  first `sinks` positions, the last `recent` ones and otherwise the rows of
  the largest scores, `budget` in all (ties: the lowest slot). Kept rows in
  slots from `budget` on move, in their order, into the free slots below.

Heads, widths and lengths are those of the repository's model (slow
transformer: 32 query and 8 KV heads of 128, cache of 2304; fast transformer:
8 and 2, cache of 16) and generic ones around them.
"""

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
ROPE_BASE = 1e6
TABLE = 8192  # rows of the rotary table
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one stream early in its utterance, the slow transformer's heads: the smallest call
        dict(name="attend_one", op="attend", seqs=1, lo=300, hi=300, nh=32, nkv=8, hd=128, page=64, dtype="bf16", track=False),
        # the fast transformer's codebook steps of 24 streams: caches of at most 16 slots
        dict(name="attend_fast", op="attend", seqs=24, lo=1, hi=16, nh=8, nkv=2, hd=128, page=16, dtype="fp16", track=False),
        # 32 streams at different frames of the model's 2304-position cache
        dict(name="attend_streams", op="attend", seqs=32, lo=200, hi=2304, nh=32, nkv=8, hd=128, page=64, dtype="bf16", track=False),
        # streams whose caches will be evicted from: weights gathered beside the output
        dict(name="attend_track", op="attend", seqs=16, lo=900, hi=6007, nh=32, nkv=8, hd=128, page=16, dtype="fp16", track=True),
        # one very long context
        dict(name="attend_long", op="attend", seqs=1, lo=130995, hi=130995, nh=32, nkv=8, hd=128, page=256, dtype="bf16", track=False),
        # a full server: the largest call
        dict(name="attend_wide", op="attend", seqs=64, lo=2048, hi=5119, nh=32, nkv=8, hd=128, page=16, dtype="bf16", track=False),
        # a decode step's new rows of 32 streams, head norms and tracking on
        dict(name="rope_step", op="rope", rows=32, seqs=32, nh=32, nkv=8, hd=128, page=64, dtype="bf16", norm=True, table="bf16", track=True),
        # ragged prompts of four streams prefilled together
        dict(name="rope_prompts", op="rope", rows=2011, seqs=4, nh=32, nkv=8, hd=128, page=16, dtype="fp16", norm=True, table="fp32", track=False),
        # a prefilled prompt into its pages
        dict(name="store_prompt", op="store", rows=1900, seqs=1, nkv=8, hd=128, page=64, dtype="bf16", track=True),
        # the step that keeps 32 streams at their budget: one row more than it in each
        dict(name="evict_step", op="evict", seqs=32, lo=1025, hi=1025, nkv=8, hd=128, page=64, dtype="bf16", budget=1024, sinks=4, recent=128),
        # long prompts cut down before decoding starts, ragged
        dict(name="evict_prompts", op="evict", seqs=8, lo=1500, hi=8192, nkv=8, hd=128, page=64, dtype="fp16", budget=2048, sinks=4, recent=256),
        # one very long context cut down
        dict(name="evict_long", op="evict", seqs=1, lo=65531, hi=65531, nkv=8, hd=128, page=256, dtype="bf16", budget=8192, sinks=16, recent=1024),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


#: (query heads, KV heads): the repository's models' and other groupings (1 to 24 query heads a KV head)
HEADS = [(32, 8), (32, 8), (8, 2), (16, 8), (4, 2), (7, 7), (20, 4), (32, 2), (24, 1)]


def draw(rng):
    op = rng.choice(["attend"] * 4 + ["rope", "rope", "store", "evict", "evict"])
    dtype, page = rng.choice(["bf16", "fp16"]), rng.choice([16, 32, 64, 128, 256])
    hd = rng.choice([128, 128, 64])
    nh, nkv = rng.choice(HEADS)
    if op == "attend":
        seqs = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, min(131072, max(1, 260000 * 8 // (seqs * nkv))))
        return dict(op=op, seqs=seqs, lo=rng.choice([1, max(1, hi // 2), hi]), hi=hi, nh=nh, nkv=nkv, hd=hd, page=page,
                    dtype=dtype, track=rng.random() < 0.4)
    if op in ("rope", "store"):
        rows = _log_int(rng, 1, 4096)
        seqs = rows if rows <= 64 and rng.random() < 0.6 else _log_int(rng, 1, min(rows, 32))
        case = dict(op=op, rows=rows, seqs=seqs, nkv=nkv, hd=hd, page=page, dtype=dtype, track=rng.random() < 0.5)
        if op == "rope":
            case.update(nh=nh, norm=rng.random() < 0.7, table=rng.choice(["bf16", "fp16", "fp32"]))
        return case
    seqs = _log_int(rng, 1, 32)
    hi = _log_int(rng, 40, 65536 * 8 // (seqs * nkv) if seqs * nkv > 8 else 65536)
    budget = rng.choice([hi - rng.randint(1, 8), max(20, hi // 2), _log_int(rng, 20, hi - 1)])
    sinks, recent = rng.randint(0, min(16, budget // 4)), rng.randint(0, budget // 2)
    return dict(op=op, seqs=seqs, lo=rng.choice([max(1, hi // 4), hi]), hi=hi, nkv=nkv, hd=hd, page=page, dtype=dtype,
                budget=budget, sinks=sinks, recent=recent)


# ------------------------------------------------------------------- inputs


def _randn(g, *shape, dtype, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV).mul_(scale).to(dtype)


def _lengths(case, g):
    n = torch.randint(case["lo"], case["hi"] + 1, (case["seqs"],), generator=g, device=DEV)
    n[-1] = case["hi"]
    return n


def _table(g, n, width, page):
    """Pages of a pool handed out in random order: `ceil(n / page)` to each sequence, -1 beyond."""
    seqs, pages = n.numel(), -(-width // page)
    order = torch.randperm(seqs * pages, generator=g, device=DEV).to(torch.int32).view(seqs, pages)
    used = torch.arange(pages, device=DEV) * page < n[:, None]
    return torch.where(used, order, torch.full_like(order, -1)), seqs * pages


def _rotary(hd, dtype):
    ang = torch.outer(torch.arange(TABLE, device=DEV).double(),
                      1.0 / ROPE_BASE ** (torch.arange(0, hd, 2, device=DEV).double() / hd))
    return torch.stack([ang.cos(), ang.sin()], -1).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op, dtype, nkv, hd, page, seqs = case["op"], DTYPES[case["dtype"]], case["nkv"], case["hd"], case["page"], case["seqs"]
    s = dict(case=dict(case))
    if op in ("attend", "evict"):
        n, width = _lengths(case, g), case["hi"]
    else:  # ragged spans that add up to `rows`, each after some slots that are there already
        rows = case["rows"]
        each = rows / seqs
        ends = torch.rand(seqs, generator=g, device=DEV, dtype=torch.float64) * 0.9 * (each - 1)
        ends = (ends + torch.arange(1, seqs + 1, device=DEV) * each).long()
        ends[-1] = rows
        span = torch.diff(ends, prepend=ends.new_zeros(1))
        start = torch.randint(0, 97, (seqs,), generator=g, device=DEV)
        n, width = start + span, 2 * math.ceil(each) + 97
        s["seqs"] = torch.repeat_interleave(torch.arange(seqs, device=DEV, dtype=torch.int32), span)
        s["slots"] = torch.arange(rows, device=DEV) - (ends - span)[s["seqs"].long()] + start[s["seqs"].long()]
        # a row's position is its slot, or lies further on where the cache was evicted from
        s["positions"] = s["slots"] + torch.randint(0, TABLE - 4352, (seqs,), generator=g, device=DEV)[s["seqs"].long()]
    s["block_table"], pages = _table(g, n, width, page)
    cap = s["block_table"].shape[1] * page
    s["k_pages"] = _randn(g, pages, nkv, page, hd, dtype=dtype)
    s["v_pages"] = _randn(g, pages, nkv, page, hd, dtype=dtype)
    if op == "evict" or case.get("track"):
        # weights that some steps have gathered: a few slots hold most of it, the newest none
        s["scores"] = torch.empty(seqs, nkv, cap, device=DEV).exponential_(generator=g).pow_(3)
        slot = torch.arange(cap, device=DEV)
        s["scores"] *= (slot < n[:, None] - 1)[:, None]
        # eviction has skipped positions and put rows out of order
        s["slot_pos"] = (slot * 3 + slot % 2 * 2).to(torch.int32).expand(seqs, nkv, cap).contiguous()
    if op == "attend":
        s["slots"] = n - 1
        s["q"] = _randn(g, seqs, case["nh"], hd, dtype=dtype, scale=1.5)
    elif op == "rope":
        s["qkv"] = _randn(g, rows, (case["nh"] + 2 * nkv) * hd, dtype=dtype, scale=2.0)
        s["freqs"] = _rotary(hd, DTYPES[case["table"]])
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"], s["k_norm"] = (torch.rand(hd, generator=g, device=DEV).add_(0.5).to(dtype) for _ in "qk")
    elif op == "store":
        # the prompt's rows lie in a contiguous cache [1, kv heads, length, head dim]
        s["k"], s["v"] = (_randn(g, 1, nkv, rows + 5, hd, dtype=dtype)[0, :, :rows].transpose(0, 1) for _ in "kv")
    else:
        s["slots"] = n - 1
        s["positions"] = s["slot_pos"][:, 0].gather(1, s["slots"][:, None])[:, 0].long()
    return s


# --------------------------------------------------------------- plain forms


def _cached(pages, table):
    """[B, kv heads, slots, head dim] in 32 bits: every slot's row through the table (a slot without a page: row of page 0)."""
    t = pages[table.clamp(min=0).long()].float()  # [B, P, kv, page, hd]
    return t.transpose(1, 2).flatten(2, 3)


def _attend(s):
    case = s["case"]
    table, q = s["block_table"], s["q"].float()
    k, v = _cached(s["k_pages"], table), _cached(s["v_pages"], table)
    b, nkv, cap, hd = k.shape
    slot = torch.arange(cap, device=q.device)
    there = (slot <= s["slots"][:, None]) & (table >= 0).repeat_interleave(case["page"], 1)
    there = there[:, None, None]  # [B, 1, 1, cap]
    qt = q.view(b, nkv, -1, hd).transpose(2, 3).contiguous()
    dots = torch.matmul(k, qt).transpose(2, 3) * hd**-0.5  # [B, kv, group, cap]
    dots = torch.where(there, dots, -math.inf)
    e = torch.where(there, torch.exp(dots - dots.amax(-1, keepdim=True)), 0.0)
    p = e / e.sum(-1, keepdim=True)
    p = torch.where(there.any(-1, keepdim=True), p, 0.0)
    y = torch.matmul(p, torch.where(there.transpose(2, 3), v, 0.0))
    out = [y.view(b, -1, hd).to(s["q"].dtype)]
    if case["track"]:
        out.append(s["scores"] + p.sum(2))
    return out


def _norm_rope(x, w, cs):
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    a, b = x[..., 0::2], x[..., 1::2]
    c, d = cs[..., 0], cs[..., 1]
    return torch.stack([a * c - b * d, b * c + a * d], -1).flatten(-2)


def _written(s, k, v):
    """The state's pools with row t in its slot, and its score and position."""
    case, slots, seqs = s["case"], s["slots"], s["seqs"].long()
    page, off = s["block_table"][seqs, slots // case["page"]].long(), slots % case["page"]
    s["k_pages"][page, :, off] = k.to(s["k_pages"].dtype)
    s["v_pages"][page, :, off] = v.to(s["v_pages"].dtype)
    out = [s["k_pages"], s["v_pages"]]
    if case["track"]:
        s["scores"][seqs, :, slots] = 0.0
        s["slot_pos"][seqs, :, slots] = s["positions"][:, None].to(torch.int32)
        out += [s["scores"], s["slot_pos"]]
    return out


def _rope(s):
    case = s["case"]
    x = s["qkv"].view(case["rows"], -1, case["hd"]).float()
    q, k, v = x.split([case["nh"], case["nkv"], case["nkv"]], 1)
    cs = s["freqs"][s["positions"]][:, None].float()
    return [_norm_rope(q, s["q_norm"], cs).to(s["qkv"].dtype)] + _written(s, _norm_rope(k, s["k_norm"], cs), v)


def _moved(pages, table, page, rows, src, dst):
    """pages with, for each (sequence, head) of `rows`, slot src's row in slot dst."""
    b, h = rows
    at = table[b, src // page].long(), h, src % page
    to = table[b, dst // page].long(), h, dst % page
    pages[to] = pages[at]
    return pages


def _evict(s):
    case, scores, pos = s["case"], s["scores"].clone(), s["slot_pos"].clone()
    budget, cap = case["budget"], scores.shape[2]
    slot = torch.arange(cap, device=scores.device).expand_as(pos)
    n = (s["slots"] + 1)[:, None, None]
    safe = (pos < case["sinks"]) | (pos > s["positions"][:, None, None] - case["recent"])
    key = torch.where(torch.isnan(scores), -math.inf, scores)
    key = torch.where(safe, math.inf, key)
    # slots that hold nothing come last: sorted by the key first, then, stably, by whether there is a row
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    order = order.gather(2, torch.sort((order >= n).to(torch.uint8), dim=-1, stable=True).indices)
    kept = torch.zeros_like(pos, dtype=torch.bool).scatter_(2, order[..., :budget], True) & (slot < n)
    hole = ~kept & (slot < budget) & (slot < n)
    mover = kept & (slot >= budget)
    # the j-th mover goes to the j-th hole: both in (sequence, head, slot) order, and equally many in each list
    b, h, src = mover.nonzero(as_tuple=True)
    dst = (hole & mover.any(2, keepdim=True)).nonzero(as_tuple=True)[2]
    scores[b, h, dst] = scores[b, h, src]
    pos[b, h, dst] = pos[b, h, src]
    return [_moved(s[x], s["block_table"], case["page"], (b, h), src, dst) for x in ("k_pages", "v_pages")] + [scores, pos]


# ----------------------------------------------------------------- one pass


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"attend": _attend, "rope": _rope, "store": lambda t: _written(t, t["k"], t["v"]), "evict": _evict}[op](s)
    from ttspipe_amd import pagedcache

    case, pools = s["case"], (s["k_pages"], s["v_pages"])
    if op == "attend":
        # the weights are added in place: to a copy, so that the state can be run again
        scores = s["scores"].clone() if case["track"] else None
        y = pagedcache.attention(s["q"], *pools, s["block_table"], s["slots"], scores=scores)
        return [y, scores] if case["track"] else [y]
    if op == "evict":
        scores, pos = s["scores"].clone(), s["slot_pos"].clone()
        pagedcache.evict(*pools, s["block_table"], s["slots"], scores, pos, s["positions"], case["budget"],
                         sinks=case["sinks"], recent=case["recent"])
        return [*pools, scores, pos]
    tracked = dict(scores=s["scores"], slot_pos=s["slot_pos"]) if case["track"] else {}
    if op == "rope":
        q = pagedcache.qk_rope_kv(s["qkv"], case["nh"], *pools, s["block_table"], s["slots"], s["freqs"], s["positions"],
                                  q_weight=s["q_norm"], k_weight=s["k_norm"], eps=EPS, seqs=s["seqs"], **tracked)
        return [q, *pools, *tracked.values()]
    pagedcache.store(s["k"], s["v"], *pools, s["block_table"], s["slots"], positions=s["positions"], seqs=s["seqs"],
                     **tracked)
    return [*pools, *tracked.values()]


# --------------------------------------------------------------------- work


def work(case):
    op, nkv, hd = case["op"], case["nkv"], case["hd"]
    row = nkv * hd * 2  # bytes of one slot's keys
    if op in ("attend", "evict"):
        n = (case["lo"] + case["hi"]) / 2 * (case["seqs"] - 1) + case["hi"]  # rows in all
    if op == "attend":
        nh = case["nh"]
        small = case["seqs"] * (2 * nh * hd * 2 + 8) + 4 * n / case["page"]
        return dict(bytes=2 * n * row + small + (8 * n * nkv if case["track"] else 0), flops=4 * n * nh * hd)
    if op == "evict":
        # of rows with independent scores, a share budget / n of those past the budget is kept
        seqs = [(case["lo"] + (case["hi"] - case["lo"]) * (i + 0.5) / max(1, case["seqs"] - 1)) if i < case["seqs"] - 1
                else case["hi"] for i in range(case["seqs"])]
        over = [x for x in seqs if x > case["budget"]]
        moved = sum(case["budget"] * (x - case["budget"]) / x for x in over)
        return dict(bytes=sum(over) * nkv * 8 + moved * (4 * row + 16 * nkv), flops=sum(over) * nkv)
    rows = case["rows"]
    tracked = rows * nkv * 8 if case["track"] else 0
    if op == "store":
        return dict(bytes=rows * (4 * row + 20) + tracked, flops=0)
    heads, elem = case["nh"] + 2 * nkv, 4 if case["table"] == "fp32" else 2
    return dict(bytes=rows * (heads * hd * 4 + min(1, 4096 / rows) * hd * elem + 20) + tracked,
                flops=rows * (case["nh"] + nkv) * hd * (7 if case["norm"] else 3))


# ---------------------------------------------------- the definition, in 64 bits


def _rows64(pages, table, b, h, n):
    page = pages.shape[2]
    return pages[table[b, : -(-n // page)].long(), h].reshape(-1, pages.shape[3])[:n].double()


def exact(case, seed):
    s = prepare(case, seed)
    op, page = case["op"], case["page"]
    if op == "attend":
        group = case["nh"] // case["nkv"]
        y = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        scores = s["scores"].double() if case["track"] else None
        for b, n in enumerate((s["slots"] + 1).tolist()):
            for h in range(case["nkv"] if n else 0):
                heads = slice(h * group, (h + 1) * group)
                w = (s["q"][b, heads].double() @ _rows64(s["k_pages"], s["block_table"], b, h, n).t()) / math.sqrt(case["hd"])
                w = torch.softmax(w, 1)
                y[b, heads] = w @ _rows64(s["v_pages"], s["block_table"], b, h, n)
                if scores is not None:
                    scores[b, h, :n] += w.sum(0)
        return [y, scores] if case["track"] else [y]
    if op in ("rope", "store"):
        pools = [s["k_pages"].double(), s["v_pages"].double()]
        if op == "store":
            q, k, v = [], s["k"].double(), s["v"].double()
        else:
            x = s["qkv"].double().view(case["rows"], -1, case["hd"])
            q, k, v = x[:, : case["nh"]], x[:, case["nh"]: -case["nkv"]], x[:, -case["nkv"]:]
            if case["norm"]:
                q, k = (t / (t.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
                        for t, w in ((q, s["q_norm"]), (k, s["k_norm"])))
            turn = torch.view_as_complex(s["freqs"].double()[s["positions"]])[:, None]
            q, k = (torch.view_as_real(torch.view_as_complex(t.reshape(*t.shape[:-1], -1, 2).contiguous()) * turn).flatten(-2)
                    for t in (q, k))
            q = [q]
        for t, (b, j, p) in enumerate(zip(s["seqs"].tolist(), s["slots"].tolist(), s["positions"].tolist())):
            at = s["block_table"][b, j // page]
            pools[0][at, :, j % page], pools[1][at, :, j % page] = k[t], v[t]
            if case["track"]:
                s["scores"][b, :, j], s["slot_pos"][b, :, j] = 0.0, p
        return [*q, *pools] + ([s["scores"].double(), s["slot_pos"]] if case["track"] else [])
    if case["seqs"] * case["nkv"] * case["hi"] > 1 << 22:
        return None
    k, v = s["k_pages"].double(), s["v_pages"].double()
    table, scores, pos = s["block_table"].tolist(), s["scores"].cpu().numpy(), s["slot_pos"].cpu().numpy()
    for b, (last, now) in enumerate(zip(s["slots"].tolist(), s["positions"].tolist())):
        n, budget = last + 1, case["budget"]
        for h in range(case["nkv"] if n > budget else 0):
            safe = lambda j: pos[b, h, j] < case["sinks"] or pos[b, h, j] > now - case["recent"]  # noqa: E731
            rank = sorted(range(n), key=lambda j: (-math.inf if safe(j) else -float(scores[b, h, j]), j))
            kept = set(rank[:budget])
            moves = list(zip((j for j in range(budget, n) if j in kept), (j for j in range(budget) if j not in kept)))
            for src, dst in moves:
                scores[b, h, dst], pos[b, h, dst] = scores[b, h, src], pos[b, h, src]
            if moves:
                src, dst = (torch.tensor(x, device=DEV) for x in zip(*moves))
                _moved(k, s["block_table"], page, (b, h), src, dst)
                _moved(v, s["block_table"], page, (b, h), src, dst)
    return [k, v, torch.from_numpy(scores).double(), torch.from_numpy(pos)]
