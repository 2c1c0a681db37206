"""The attention operators beside the quantized projections: page plan, 8-bit cache write, attention over the cache, attention
over packed prompts.

A case is a dict of plain values; ``kind`` names the operator:

  plan    block table, slot map and page writes of one step, from request lengths (``kv_plan``)
  append  new key / value rows into the paged 8-bit cache (``kv_append``)
  cache   causal grouped attention of the newest tokens over that cache (``kv_attention``)
  prompt  causal grouped attention over packed prompts (``prompt_attention``)

Lengths follow from the case alone, contents and page numbers from the seed. A page of the cache holds int8 codes of ``page``
tokens per head and one power-of-two scale for keys and one for values.
"""
import importlib
import math
import random

import torch

own = False
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _kd():
    return importlib.import_module("dnn-for-kokkos_b200")


def listed():
    return [
        # the bookkeeping in front of every decode step of a busy server
        {"name": "plan_decode_b64", "kind": "plan", "seqs": 64, "page": 64, "ctx": 8192, "fresh": 1, "ended": 4},
        # the same in front of a batch of ragged prompts, some continuing, a large pool
        {"name": "plan_prompts_b200", "kind": "plan", "seqs": 200, "page": 32, "ctx": 3000, "fresh": 1500, "ended": 17},
        # one new token for each sequence of a decode batch
        {"name": "append_decode_b64", "kind": "append", "seqs": 64, "kv_heads": 8, "dim": 128, "page": 64, "fresh": 1, "x": "bf16"},
        # the keys and values of a batch of prompts, in fp32
        {"name": "append_prompts_b9", "kind": "append", "seqs": 9, "kv_heads": 4, "dim": 128, "page": 64, "fresh": 2500, "x": "f32"},
        # one sequence, short context: launch latency decides
        {"name": "cache_b1_1900", "kind": "cache", "seqs": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "ctx": 1900, "fresh": 1,
         "window": 0, "x": "bf16"},
        # a decode batch of ragged contexts
        {"name": "cache_b64_8k", "kind": "cache", "seqs": 64, "heads": 32, "kv_heads": 4, "dim": 128, "page": 64, "ctx": 8192, "fresh": 1,
         "window": 0, "x": "bf16"},
        # a few long documents
        {"name": "cache_b3_130k", "kind": "cache", "seqs": 3, "heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "ctx": 131071, "fresh": 1,
         "window": 0, "x": "bf16"},
        # drafts of up to six tokens verified together, sliding window, small heads, fp32
        {"name": "cache_b20_draft_f32", "kind": "cache", "seqs": 20, "heads": 24, "kv_heads": 8, "dim": 64, "page": 16, "ctx": 5000,
         "fresh": 6, "window": 1024, "x": "f32"},
        # one short prompt: launch latency decides
        {"name": "prompt_77", "kind": "prompt", "seqs": 1, "tokens": 77, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "x": "bf16"},
        # a batch of ragged prompts packed together
        {"name": "prompt_b12_5000", "kind": "prompt", "seqs": 12, "tokens": 5000, "heads": 32, "kv_heads": 4, "dim": 128, "window": 0,
         "x": "bf16"},
        # one long prompt
        {"name": "prompt_8192", "kind": "prompt", "seqs": 1, "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "x": "bf16"},
        # fp32 activations, small heads, sliding window
        {"name": "prompt_b3_f32", "kind": "prompt", "seqs": 3, "tokens": 1500, "heads": 16, "kv_heads": 8, "dim": 64, "window": 512, "x": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "append", "cache", "cache", "cache", "prompt", "prompt", "prompt"])
    if kind == "plan":
        c = {"kind": kind, "seqs": _log(rng, 1, 256), "page": rng.choice([16, 32, 64, 128]), "ctx": _log(rng, 16, 8192),
             "fresh": _log(rng, 1, 1500)}
        c["ended"] = rng.randrange(0, c["seqs"] // 4 + 1)
        return c
    x = rng.choice(["bf16", "bf16", "f32"])
    if kind == "append":
        c = {"kind": kind, "seqs": _log(rng, 1, 128), "kv_heads": rng.choice([1, 2, 4, 5, 8]), "dim": rng.choice([64, 128]),
             "page": rng.choice([16, 32, 64, 128]), "fresh": _log(rng, 1, 2500), "x": x}
        c["fresh"] = max(1, min(c["fresh"], 20000 // c["seqs"]))
        return c
    kv = rng.choice([1, 2, 4, 5, 8])
    c = {"kind": kind, "heads": kv * rng.choice([1, 2, 3, 4, 6, 8]), "kv_heads": kv, "dim": rng.choice([64, 128, 128]), "x": x}
    if kind == "cache":
        c.update(seqs=_log(rng, 1, 64), page=rng.choice([16, 32, 64, 128]), ctx=_log(rng, 64, 131071), fresh=rng.choice([1, 1, 1, 2, 4, 7]))
        c["ctx"] = max(64, min(c["ctx"], 400_000 // c["seqs"]))
        c["window"] = rng.choice([0, 0, 0, 128, 1000])
        return c
    c.update(seqs=_log(rng, 1, 24), tokens=_log(rng, 24, 8192 if x == "bf16" else 1500), window=rng.choice([0, 0, 0, 100, 512]))
    c["tokens"] = min(c["tokens"], int(math.sqrt(8192 * 8192 * 32 / c["heads"])), 12000)
    return c


# ---------------------------------------------------------------------------------------------------
# lengths: from the case alone
def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _lengths(case):
    """(cached, fresh) of every sequence, Python lists; fresh < 0: the sequence has ended."""
    r, b, kind = _rng(case), case["seqs"], case["kind"]
    if kind == "prompt":
        cut = sorted(r.randrange(0, case["tokens"] + 1) for _ in range(b - 1))    # an empty prompt among them by chance
        return [0] * b, [hi - lo for lo, hi in zip([0] + cut, cut + [case["tokens"]])]
    most = case["fresh"]
    fresh = [most if b == 1 else r.randint(1, most) for _ in range(b)]
    if kind == "append":
        return [r.randrange(0, case["page"]) for _ in range(b)], fresh
    cached = [case["ctx"] if b == 1 else r.randint(case["ctx"] // 8, case["ctx"]) for _ in range(b)]
    ended = set(r.sample(range(b), case.get("ended", 0)))
    return cached, [-1 if i in ended else f for i, f in enumerate(fresh)]


def _pages(case):
    """(page, columns of the block table, pages of the pool)."""
    cached, fresh = _lengths(case)
    page = case["page"]
    need = [-(-(c + max(f, 0)) // page) for c, f in zip(cached, fresh)]
    return page, max(need) + 1, sum(need) + (len(need) if case["kind"] == "plan" else 0)


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pool(case, gen):
    """A pool in use: lens, fresh, table with the cached pages, ring of the free ones, state."""
    cached, fresh = _lengths(case)
    page, cols, pages = _pages(case)
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    lens, new = _int(cached), _int(fresh)
    have = (lens + page - 1) // page
    start = torch.cumsum(have, 0) - have
    j = torch.arange(cols, device="cuda")
    held = j[None, :] < have[:, None]
    table = torch.where(held, order[(start[:, None] + j[None, :]).clamp(max=pages - 1)], -1).to(torch.int32).contiguous()
    used = int(have.sum())
    head = (5 * page) % pages                                  # the free pages start somewhere in the ring
    ring = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    at = (head + torch.arange(pages - used, device="cuda")) % pages
    ring[at] = order[used:]
    state = _int([head, pages - used, 0, 0])
    return {"lens0": lens, "fresh": new, "table0": table, "ring0": ring, "state0": state, "page": page, "pages": pages,
            "rows": sum(max(f, 0) for f in fresh)}


def _writes_most(rows, seqs, page):
    return max(1, min(rows, rows // page + 2 * seqs))


def _plan(p):
    """The plan of one step in whole numbers: row_start, first, lens, state, slots, writes, table, ring."""
    page, pages, rows = p["page"], p["pages"], p["rows"]
    table, ring = p["table0"].clone(), p["ring0"].clone()
    b, cols = table.shape
    fresh, lens = p["fresh"].long(), p["lens0"].long().clamp(0, cols * page)
    head, avail = p["state0"][0].long() % pages, p["state0"][1].long().clamp(0, pages)
    n = fresh.clamp(min=0)
    zero = torch.zeros(1, dtype=torch.long, device="cuda")
    row_start = torch.cat([zero, torch.cumsum(n, 0)]).clamp(max=rows)
    m = row_start[1:] - row_start[:-1]
    ended = fresh < 0
    have = (lens + page - 1) // page
    need = torch.where(ended, 0, torch.clamp((lens + m + page - 1) // page, max=cols) - have)
    before = torch.cumsum(need, 0) - need
    got = torch.minimum((avail - before).clamp(min=0), need)
    stored = torch.where(ended, 0, torch.minimum(m, (have + got) * page - lens))
    first = torch.where(ended, 0, lens)
    j = torch.arange(cols, device="cuda")[None, :]
    taken = (j >= have[:, None]) & (j < (have + got)[:, None])
    table = torch.where(taken, ring[(head + before[:, None] + j - have[:, None]) % pages], table)
    back = torch.where(ended, have, 0)
    back0 = torch.cumsum(back, 0) - back
    given = j < back[:, None]
    # every place of the ring once: a place that nothing is given back to keeps what it has
    at = torch.where(given, (head + avail + back0[:, None] + j) % pages, pages)
    ring = torch.cat([ring, ring[:1]]).scatter(0, at.reshape(-1), table.reshape(-1))[:pages]
    # rows
    r = torch.arange(rows, device="cuda")
    s = torch.searchsorted(row_start[1:].contiguous(), r, right=True).clamp(max=b - 1)
    i = r - row_start[s]
    pos = lens[s] + i
    pg = table[s, (pos // page).clamp(max=cols - 1)].long()
    good = (r < row_start[-1]) & (i < stored[s]) & (pg >= 0) & (pg < pages)
    slots = torch.where(good, pg * page + pos % page, -1)
    # touched pages
    most = _writes_most(rows, b, page)
    touched = torch.where(stored > 0, (lens + stored - 1) // page - lens // page + 1, 0)
    upto = torch.cumsum(touched, 0)
    w = torch.arange(most, device="cuda")
    s = torch.searchsorted(upto, w, right=True).clamp(max=b - 1)
    jp = lens[s] // page + w - (upto - touched)[s]
    lo = torch.maximum(jp * page, lens[s])
    hi = torch.minimum((jp + 1) * page, (lens + stored)[s])
    entry = torch.stack([row_start[s] + lo - lens[s], hi - lo, table[s, jp.clamp(0, cols - 1)].long(), lo - jp * page], 1)
    writes = torch.where((w < upto[-1])[:, None], entry, 0)
    state = torch.stack([(head + got.sum()) % pages, avail - got.sum() + back.sum(), n.sum() - stored.sum(), upto[-1]])
    return {"row_start": row_start.int(), "first": first.int(), "lens": (first + stored).int(), "state": state.int(),
            "slots": slots.int(), "writes": writes.int(), "table": table, "ring": ring}


def _heads(n, heads, dim, x, gen, gain=1.0):
    t = torch.randn(n, heads, dim, device="cuda", generator=gen) * gain
    t[..., 5::32] *= 4.0           # a few channels carry more, as keys' channels do
    return t.to(TYPES[x])


def _pow2(e):
    """2^e in fp32 by its bits, for whole e of the normal range."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _scale_of(amax):
    """The smallest power of two s with amax <= 127 s, at least 2^-100; 0 for 0."""
    m, e = torch.frexp(amax)                                  # amax = m 2^e, 1/2 <= m < 1
    e = torch.where(m > 127.0 / 128.0, e - 6, e - 7).clamp(min=-100)
    return torch.where(amax > 0, _pow2(e), torch.zeros_like(amax))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 29)
    kind = case["kind"]
    st = {"case": case, "kind": kind}
    if kind == "prompt":
        _, fresh = _lengths(case)
        n, d = case["tokens"], case["dim"]
        st["row_start"] = _int([sum(fresh[:i]) for i in range(len(fresh) + 1)])
        st["q"] = _heads(n, case["heads"], d, case["x"], gen)
        st["k"] = _heads(n, case["kv_heads"], d, case["x"], gen)
        st["v"] = _heads(n, case["kv_heads"], d, case["x"], gen)
        st["out"] = torch.empty_like(st["q"])
        return st
    st.update(_pool(case, gen))
    b, rows, page = case["seqs"], st["rows"], st["page"]
    if kind == "plan":
        if own:
            kd = _kd()
            st["plan"] = kd.KvPlan.empty(b, rows, page)
            st["table"], st["ring"] = st["table0"].clone(), st["ring0"].clone()
        return st
    p = st["plain"] = _plan(st)
    kv, d, pages = case["kv_heads"], case["dim"], st["pages"]
    codes = [torch.randint(-127, 128, (pages, kv, page, d), dtype=torch.int8, device="cuda", generator=gen) for _ in range(2)]
    scales = [_pow2(torch.randint(-7, -5, (pages, kv), device="cuda", generator=gen)) for _ in range(2)]
    st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"] = *codes, *scales
    if kind == "append":
        st["k"], st["v"] = _heads(rows, kv, d, case["x"], gen), _heads(rows, kv, d, case["x"], gen)
    else:
        st["q"] = _heads(rows, case["heads"], d, case["x"], gen)
        st["out"] = torch.empty_like(st["q"])
    if own:
        kd = _kd()
        st["plan"] = kd.KvPlan(p["row_start"], p["first"], p["lens"], p["state"], p["slots"], p["writes"], page)
        st["cache"] = kd.KvCache(st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"])
        if kind == "cache":
            st["ws"] = torch.empty(kd.kv_attention_workspace_bytes(rows, b, case["heads"], kv, d), dtype=torch.uint8, device="cuda")
    return st


# ---------------------------------------------------------------------------------------------------
# plain forms
def _values(codes, scale):
    """What the cache holds: codes of 7 bits and a sign times powers of two are exact in bf16."""
    return codes * scale[:, :, None, None].to(torch.bfloat16)


def _append(x, codes, scale, p, page):
    """New rows into codes / scale (in place): the page's scale grows to hold them, older codes follow it."""
    w = p["writes"].long()
    row0, count, pg, off = w[:, 0:1], w[:, 1:2], w[:, 2], w[:, 3:4]
    live = (count[:, 0] > 0) & (pg >= 0) & (pg < codes.shape[0])
    t = torch.arange(page, device="cuda")[None, :]
    mine = (t >= off) & (t < off + count)
    x = x[(row0 + t - off).clamp(0, x.shape[0] - 1)].float().transpose(1, 2)           # [writes, heads, page, dim]
    mine = mine[:, None, :, None]
    size = torch.where(mine & torch.isfinite(x), x.abs(), 0.0).amax((2, 3))
    at = pg.clamp(0, codes.shape[0] - 1)
    old = torch.where(off > 0, scale[at], 0.0)
    new = torch.maximum(old, _scale_of(size))
    inv = torch.where(new > 0, 1.0 / new, 0.0)[:, :, None, None]
    was = codes[at]
    kept = torch.round(was.float() * old[:, :, None, None] * inv).to(torch.int8)
    put = torch.nan_to_num(torch.round(x * inv).clamp(-127, 127), nan=0.0).to(torch.int8)
    older = (t < off)[:, None, :, None]
    both = torch.where(mine, put, torch.where(older, kept, was))
    codes[pg[live]] = both[live]
    scale[pg[live]] = new[live]


def _softmax_v(s, v):
    """softmax(s) v over the last axis; a row with nothing left gives 0."""
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
    return (e @ v) / e.sum(-1, keepdim=True).clamp(min=1e-30)


def _cache_attention(st):
    case, p, page = st["case"], st["plain"], st["page"]
    h, kv, d, win = case["heads"], case["kv_heads"], case["dim"], case["window"]
    b, cols = p["table"].shape
    pg = p["table"].long().clamp(min=0)
    k = (st["k_codes"][pg] * st["k_scale"][pg][..., None, None]).transpose(1, 2).reshape(b, kv, cols * page, d)
    v = (st["v_codes"][pg] * st["v_scale"][pg][..., None, None]).transpose(1, 2).reshape(b, kv, cols * page, d)
    start, most = p["row_start"].long(), case["fresh"]
    i = torch.arange(most, device="cuda")[None, :]
    row = start[:-1, None] + i
    real = row < start[1:, None]
    q = st["q"][row.clamp(max=st["rows"] - 1)].float().reshape(b, most, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, d)
    s = (q @ k.transpose(2, 3)).reshape(b, kv, most, h // kv, cols * page) * d ** -0.5
    pos = (p["first"][:, None] + i)[:, None, :, None, None]
    j = torch.arange(cols * page, device="cuda")
    keep = (j <= pos) & (j < p["lens"].long()[:, None, None, None, None])
    if win:
        keep = keep & (j > pos - win)
    s = torch.where(keep, s, -math.inf).reshape(b, kv, -1, cols * page)
    o = _softmax_v(s, v).reshape(b, kv, most, h // kv, d).permute(0, 2, 1, 3, 4).reshape(b, most, h, d)
    return o[real].to(st["q"].dtype)


def _prompt_attention(st):
    case = st["case"]
    n, h, kv, d, win = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["window"]
    q = st["q"].float().reshape(n, kv, h // kv, d).permute(1, 2, 0, 3)
    k, v = (st[x].float().permute(1, 0, 2)[:, None] for x in "kv")
    r = torch.arange(n, device="cuda")
    seq = torch.searchsorted(st["row_start"][1:].long().contiguous(), r, right=True)
    keep = (seq[:, None] == seq[None, :]) & (r[None, :] <= r[:, None])
    if win:
        keep = keep & (r[None, :] > r[:, None] - win)
    s = (q @ k.transpose(2, 3)).mul_(d ** -0.5).masked_fill_(~keep, -math.inf)
    return _softmax_v(s, v).permute(2, 0, 1, 3).reshape(n, h, d).to(st["q"].dtype)


def run(st):
    kind = st["kind"]
    if kind == "plan":
        if own:
            p = st["plan"]
            _kd().kv_plan(st["fresh"], st["lens0"], st["table"], st["ring"], st["state0"], p)
            return {"row_start": p.row_start, "first": p.first, "lens": p.lens, "state": p.state, "slots": p.slots, "writes": p.writes,
                    "table": st["table"], "ring": st["ring"]}
        return _plan(st)
    if kind == "append":
        if own:
            _kd().kv_append(st["k"], st["v"], st["plan"], st["cache"])
        else:
            _append(st["k"], st["k_codes"], st["k_scale"], st["plain"], st["page"])
            _append(st["v"], st["v_codes"], st["v_scale"], st["plain"], st["page"])
        return {"k": _values(st["k_codes"], st["k_scale"]), "v": _values(st["v_codes"], st["v_scale"])}
    if kind == "cache":
        if own:
            _kd().kv_attention(st["q"], st["plan"], st["plain"]["table"], st["cache"], st["out"], st["ws"], window=st["case"]["window"])
            return st["out"]
        return _cache_attention(st)
    if own:
        _kd().prompt_attention(st["q"], st["k"], st["v"], st["row_start"], st["out"], window=st["case"]["window"])
        return st["out"]
    return _prompt_attention(st)


def work(case):
    cached, fresh = _lengths(case)
    kind = case["kind"]
    if kind == "plan":
        page, cols, pages = _pages(case)
        rows = sum(max(f, 0) for f in fresh)
        moved = sum(-(-(c + max(f, 0)) // page) - c // page if f >= 0 else -(-c // page) for c, f in zip(cached, fresh))
        return {"bytes": 20 * len(fresh) + 4 * rows + (8 + 16) * moved, "flops": 0}
    size = {"f32": 4, "bf16": 2}[case["x"]]
    d, kv = case["dim"], case["kv_heads"]
    if kind == "append":
        # the new rows and their codes, the page's scales, and the result read as values
        page, cols, pages = _pages(case)
        return {"bytes": 2 * kv * d * sum(fresh) * (size + 1) + 2 * kv * d * pages * page * 3, "flops": 0}
    h, win = case["heads"], case["window"]
    keys = pairs = 0
    for c, n in zip(cached, fresh):
        if n <= 0:
            continue
        keys += c + n - (max(0, c - win + 1) if win else 0)
        if win:
            pairs += sum(min(c + i + 1, win) for i in range(n))
        else:
            pairs += n * c + n * (n + 1) // 2
    rows = sum(fresh)
    per_key = 2 * kv * d * (1 if kind == "cache" else size)
    scales = 8 * kv * keys // case["page"] if kind == "cache" else 0
    return {"bytes": keys * per_key + scales + 2 * rows * h * d * size, "flops": 4 * d * h * pairs}


# ---------------------------------------------------------------------------------------------------
def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence; whole numbers have no other value than run()'s."""
    kind = case["kind"]
    if kind == "plan":
        return None
    st = prepare(case, seed)
    cached, fresh = _lengths(case)
    d = case["dim"]
    if kind == "append":
        page, out = st["page"], {}
        table = st["plain"]["table"].tolist()
        for name in "kv":
            vals = st[name + "_codes"].double() * st[name + "_scale"].double()[:, :, None, None]
            x, row = st[name].double(), 0
            for b, (c, n) in enumerate(zip(cached, fresh)):
                at, end = c, c + n
                while at < end:
                    pg, off = table[b][at // page], at % page
                    m = min(end - at, page - off)
                    new = x[row:row + m].transpose(0, 1)
                    need = new.abs().amax((1, 2))
                    s = ((torch.ceil(torch.log2(need / 127.0)).long() + 1023) << 52).view(torch.float64)    # 2^e by its bits
                    if off:
                        s = torch.maximum(s, st[name + "_scale"][pg].double())
                        vals[pg, :, :off] = torch.round(vals[pg, :, :off] / s[:, None, None]) * s[:, None, None]
                    vals[pg, :, off:off + m] = torch.round(new / s[:, None, None]) * s[:, None, None]
                    if not off + m == page:      # what lies behind the last token keeps its codes, whose scale is the page's
                        vals[pg, :, off + m:] = st[name + "_codes"][pg, :, off + m:].double() * s[:, None, None]
                    at, row = at + m, row + m
            out[name] = vals
        return out
    h, kv, win = case["heads"], case["kv_heads"], case["window"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (c, n) in enumerate(zip(cached, fresh)):
        if n <= 0:
            continue
        q = st["q"][row:row + n].double()
        if kind == "cache":
            total = c + n
            lo = max(0, c - win + 1) if win else 0
            page = st["page"]
            pg = st["plain"]["table"][b, lo // page:-(-total // page)].long()
            skip = lo % page

            def flat(codes, scale, g):
                t = codes[pg, g].double() * scale[pg, g].double()[:, None, None]
                return t.reshape(-1, d)[skip:skip + total - lo]
        else:
            total, lo = n, 0

            def flat(x, _, g):
                return x[row:row + n, g].double()
        j = torch.arange(lo, total, device="cuda")
        pos = torch.arange(c, c + n, device="cuda")[:, None]
        keep = j[None, :] <= pos
        if win:
            keep &= j[None, :] > pos - win
        names = ("k_codes", "k_scale", "v_codes", "v_scale") if kind == "cache" else ("k", "k", "v", "v")
        for g in range(kv):
            k, v = flat(st[names[0]], st[names[1]], g), flat(st[names[2]], st[names[3]], g)
            for a in range(g * (h // kv), (g + 1) * (h // kv)):
                w = torch.softmax((q[:, a] @ k.T / math.sqrt(d)).masked_fill(~keep, -math.inf), 1)
                out[row:row + n, a] = w @ v
        row += n
    return out
