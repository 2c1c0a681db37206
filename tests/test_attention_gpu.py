"""The attention operators (page plan, 8-bit cache write, attention over the cache and over packed prompts) against plain
implementations in whole numbers and in 64 bits.

Tolerances count roundings. For one output o = sum_j p_j v_j with A = sum_j p_j |v_j| and scores s_j:
  a score is off by at most es = max_j sum_d |q_d k_jd| scale * (rounding of the product's operands + D roundings of its sum),
  plus |s| times a few fp32 roundings (the scale, the base-2 form); a weight then by 2 es relative (its own and the sum's),
  by the rounding of a weight that enters a matrix product, and by (keys) roundings of fp32 sums, which meet A;
  the result by half a step of its type.
bf16 operands are exact in a product; a weight is rounded to bf16 (2^-8) for packed bf16 prompts and to fp16 (2^-11) over the
cache; fp32 operands and weights over the cache are two fp16 parts (2^-22). fp32 prompts take two tf32 parts of each operand, which leaves
out 2^-22 + 2 * 2^-23 = 8 * 2^-24 of a product: the eight roundings that a score and a result have beside those of their sums. Over the cache a weight is also off by half of fp16's
smallest step, 2^-25, where the largest weight of its row is at least 2^6 (it is 2^(7 + s - m), and m, a whole number, is at most one
above the largest score): by 2^-31 of the sum, which meets the sum of |v_j|."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24
OUT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---- page plan ---------------------------------------------------------------------------------------------------------
def plan_plain(fresh, lens, table, ring, state, page, rows, most):
    """kdnn_b200_kv_plan restated on Python lists; table and ring are changed in place."""
    B, cols, pages = len(fresh), len(table[0]), len(ring)
    head, avail = state[0] % pages, max(0, min(pages, state[1]))
    row_start, first, out, slots, writes, missing, taken, back = [0], [], [], [-1] * rows, [], 0, 0, []
    old_ring = list(ring)
    for b in range(B):
        n, length = max(fresh[b], 0), max(0, min(lens[b], cols * page))
        m = min(n, rows - row_start[b])
        row_start.append(row_start[b] + m)
        have = -(-length // page)
        if fresh[b] < 0:
            back += table[b][:have]
            first.append(0)
            out.append(0)
            continue
        need = min(-(-(length + m) // page), cols) - have
        got = max(0, min(need, avail - taken))
        for i in range(got):
            table[b][have + i] = old_ring[(head + taken + i) % pages]
        taken += got
        stored = min(m, (have + got) * page - length)
        missing += n - stored
        first.append(length)
        out.append(length + stored)
        for i in range(stored):
            pos = length + i
            pg = table[b][pos // page]
            if 0 <= pg < pages:
                slots[row_start[b] + i] = pg * page + pos % page
            if i == 0 or pos % page == 0:
                writes.append([row_start[b] + i, 0, pg, pos % page])
            writes[-1][1] += 1
    for i, p in enumerate(back):
        ring[(head + avail + i) % pages] = p
    state_out = [(head + taken) % pages, avail - taken + len(back), missing, len(writes)]
    return dict(row_start=row_start, first=first, lens=out, state=state_out, slots=slots,
                writes=writes + [[0, 0, 0, 0]] * (most - len(writes)))


def make_pool(rng, B, page, ctx, extra, cols=None):
    lens = [rng.choice([0, page, rng.randrange(0, ctx + 1), rng.randrange(0, ctx + 1)]) for _ in range(B)]
    held = [-(-n // page) for n in lens]
    pages = sum(held) + extra
    order = list(range(pages))
    rng.shuffle(order)
    cols = cols or max(held) + 8
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h] + [-7] * (cols - h))
        at += h
    head = rng.randrange(pages)
    ring = [-3] * pages
    for i, p in enumerate(order[at:]):
        ring[(head + i) % pages] = p
    return lens, table, ring, [head, pages - at, 99, 99]


def check_plan(kd, fresh, lens, table, ring, state, page, rows, in_place=False, ldt=None):
    B = len(fresh)
    plan = kd.KvPlan.empty(B, rows, page)
    for t in (plan.row_start, plan.first, plan.slots, plan.writes):
        t.fill_(-55)                                  # every entry is written
    gt = torch.full((B, ldt or len(table[0])), -9, dtype=torch.int32, device="cuda")
    gt[:, :len(table[0])] = i32(table)
    gr, gl, gs = i32(ring), i32(lens), i32(state)
    if in_place:
        plan.lens, plan.state = gl, gs
    kd.kv_plan(i32(fresh), gl, gt[:, :len(table[0])], gr, gs, plan)
    want = plan_plain(fresh, lens, table, ring, state, page, rows, plan.writes.shape[0])
    for name, v in want.items():
        assert getattr(plan, name).tolist() == v, name
    assert gt[:, :len(table[0])].tolist() == table and gr.tolist() == ring
    assert (gt[:, len(table[0]):] == -9).all()
    return plan


@pytest.mark.parametrize("B,page,ctx,fresh", [(1, 16, 0, 1), (1, 64, 1000, 1), (64, 64, 3000, 1), (5, 32, 100, 400), (300, 16, 40, 7),
                                              (37, 128, 5000, 1300), (2000, 64, 300, 2), (8192, 16, 20, 1)])
def test_plan(kd, B, page, ctx, fresh):
    rng = random.Random(B * 1000 + page)
    lens, table, ring, state = make_pool(rng, B, page, ctx, extra=B * (fresh // page + 2))
    new = [rng.choice([fresh, rng.randrange(0, fresh + 1), -1 if rng.random() < 0.3 else fresh]) for _ in range(B)]
    rows = sum(max(n, 0) for n in new)
    check_plan(kd, new, lens, table, ring, state, page, rows + 13, in_place=B % 2 == 0, ldt=len(table[0]) + 3)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,page,ctx,fresh", [(200, 64, 300, 700), (8192, 32, 40, 9)])
def test_plan_of_many_rows(kd, B, page, ctx, fresh, in_place):
    rng = random.Random(B)
    lens, table, ring, state = make_pool(rng, B, page, ctx, extra=B * (fresh // page + 1))
    new = [rng.choice([fresh, 0, -1, rng.randrange(0, fresh + 1)]) for _ in range(B)]
    check_plan(kd, new, lens, table, ring, state, page, sum(max(n, 0) for n in new), in_place=in_place)


def test_plan_when_something_runs_out(kd):
    rng = random.Random(5)
    for extra, cols, cut in ((0, None, 0), (3, None, 0), (100, 4, 0), (100, None, 50), (5, 6, 11)):
        lens, table, ring, state = make_pool(rng, 9, 16, 60, extra=extra, cols=cols)
        new = [0, 40, -1, 1, 17, 80, 16, -5, 33]
        plan = check_plan(kd, new, lens, table, ring, state, 16, max(0, sum(n for n in new if n > 0) - cut))
        assert plan.state[2].item() > 0
    # lengths and states that no plan of this pool leaves
    lens, table, ring, state = make_pool(rng, 4, 32, 200, extra=9)
    lens[1] = -4
    check_plan(kd, [3, 2, -1, 0], lens, table, ring, [state[0] - 3 * len(ring), state[1], 0, 0], 32, 5)


def test_plan_steps_in_place_return_every_page(kd):
    """A pool that is moved from step to step: no page is held twice, and all are free again at the end."""
    B, page, pages, cols = 6, 16, 40, 12
    rng = random.Random(3)
    lens, state, ring = torch.zeros(B, dtype=torch.int32, device="cuda"), i32([0, pages, 0, 0]), torch.arange(pages, dtype=torch.int32, device="cuda")
    table = torch.full((B, cols), -1, dtype=torch.int32, device="cuda")
    for step in range(30):
        fresh = [rng.choice([-1, 0, 1, 1, 5, 30]) for _ in range(B)] if step < 29 else [-1] * B
        plan = kd.KvPlan.empty(B, 200, page)
        plan.lens, plan.state = lens, state
        kd.kv_plan(i32(fresh), lens, table, ring, state, plan)
        t, r, (head, avail, missing, _) = table.tolist(), ring.tolist(), state.tolist()
        held = [p for b, n in enumerate(lens.tolist()) for p in t[b][:-(-n // page)]]
        free = [r[(head + i) % pages] for i in range(avail)]
        assert sorted(held + free) == list(range(pages)), (step, missing)
    assert avail == pages


# ---- cache write -----------------------------------------------------------------------------------------------------------
def scale_for(amax):
    if amax == 0:
        return 0.0
    e = math.ceil(math.log2(amax / 127)) if amax > 2.0 ** -90 else -100
    while 127 * 2.0 ** e < amax:
        e += 1
    while e > -100 and 127 * 2.0 ** (e - 1) >= amax:
        e -= 1
    return 2.0 ** max(e, -100)


def append_plain(x, codes, scale, writes):
    """kdnn_b200_kv_append restated in float64 on the CPU, in place."""
    x = x.double()
    for row0, count, pg, off in writes:
        if count == 0:
            continue
        for h in range(codes.shape[1]):
            new = x[row0:row0 + count, h]
            fin = new[torch.isfinite(new)]
            need = scale_for(fin.abs().max().item() if fin.numel() else 0.0)
            old = scale[pg, h].item() if off else 0.0
            s = max(old, need)
            if off and s != old:
                codes[pg, h, :off] = torch.round(codes[pg, h, :off].double() * (old / s))
            c = torch.round(new / s) if s > 0 else torch.zeros_like(new)
            codes[pg, h, off:off + count] = torch.nan_to_num(c, nan=0.0, posinf=127, neginf=-127).clamp(-127, 127)
            scale[pg, h] = s


def step_of(kd, fresh, lens, page, cols, pages, seed=0, rows=None):
    """A plan whose pages come from a shuffled pool, with the table it filled."""
    B = len(fresh)
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    table, at = torch.full((B, cols), -1, dtype=torch.int32), 0
    for b, n in enumerate(lens):
        h = -(-n // page)
        table[b, :h] = torch.tensor(order[at:at + h], dtype=torch.int32)
        at += h
    ring = i32(order[at:] + [-1] * at)
    table = table.cuda()
    plan = kd.KvPlan.empty(B, sum(max(n, 0) for n in fresh) if rows is None else rows, page)
    kd.kv_plan(i32(fresh), i32(lens), table, ring, i32([0, pages - at, 0, 0]), plan)
    return plan, table


def random_cache(kd, pages, heads, page, dim, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = kd.KvCache.empty(pages, heads, page, dim)
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes.copy_(torch.randint(-127, 128, codes.shape, device="cuda", generator=g))
        scale.copy_(2.0 ** torch.randint(-9, -5, scale.shape, device="cuda", generator=g).float())
    return cache


def rows_of(n, heads, dim, dtype, seed, gain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, heads, dim, device="cuda", generator=g) * gain).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,dim,page,fresh,lens", [
    (1, 16, 16, [1], [0]), (2, 64, 16, [1, 1, 1], [3, 15, 16]), (8, 128, 64, [1] * 9, list(range(0, 180, 20))),
    (3, 80, 32, [70, 0, 33], [5, 9, 0]), (2, 256, 128, [300, 1], [100, 127]), (5, 128, 64, [64, 63, 65, 200], [0, 1, 63, 64]),
])
def test_append(kd, dtype, heads, dim, page, fresh, lens):
    pages = sum(-(-(n + m) // page) for n, m in zip(lens, fresh)) + 2
    plan, _ = step_of(kd, fresh, lens, page, 8, pages, rows=sum(fresh) + 3)
    cache = random_cache(kd, pages, heads, page, dim, 1)
    # rows of a fused projection: keys and values side by side
    kv = rows_of(plan.rows, 2 * heads, dim, dtype, 2, gain=0.7)
    k, v = kv[:, :heads], kv[:, heads:]
    v.mul_(torch.linspace(0.01, 30, plan.rows, device="cuda")[:, None, None].to(dtype))
    want = [t.cpu().clone() for t in (cache.k, cache.k_scale, cache.v, cache.v_scale)]
    append_plain(k.cpu(), want[0], want[1], plan.writes.tolist())
    append_plain(v.cpu(), want[2], want[3], plan.writes.tolist())
    kd.kv_append(k, v, plan, cache)
    for got, w in zip((cache.k, cache.k_scale, cache.v, cache.v_scale), want):
        assert torch.equal(got.cpu(), w)


def test_append_special_values(kd):
    page, dim = 16, 16
    plan, _ = step_of(kd, [5, 20], [0, 10], page, 4, 6)
    k = torch.zeros(25, 1, dim, device="cuda")
    v = rows_of(25, 1, dim, torch.float32, 3)
    k[2, 0, 3], k[7, 0, 1], k[8, 0, 2], k[9, 0, :4] = 1e-42, float("nan"), float("-inf"), torch.tensor([3e38, -127.0, 1e-30, float("inf")])
    v[3, 0, 0], v[4, 0, 1], v[20, 0, 2] = 127.0, 127.5, 254.0
    # another alignment than 16 bytes, and heads that lie apart
    wide = torch.zeros(25 * 40 + 1, device="cuda")[1:].view(25, 40)
    wide[:, 7:7 + dim] = k[:, 0]
    for src in (k, wide[:, 7:7 + dim].unsqueeze(1)):
        cache = random_cache(kd, 6, 1, page, dim, 1)
        want = [t.cpu().clone() for t in (cache.k, cache.k_scale, cache.v, cache.v_scale)]
        append_plain(k.cpu(), want[0], want[1], plan.writes.tolist())
        append_plain(v.cpu(), want[2], want[3], plan.writes.tolist())
        kd.kv_append(src, v, plan, cache)
        for got, w in zip((cache.k, cache.k_scale, cache.v, cache.v_scale), want):
            assert torch.equal(got.cpu(), w)


def test_append_one_at_a_time_stays_within_a_step(kd):
    """Rows written one by one are rounded again when their page's scale grows: off by less than one step of the last
    scale (halves of steps that double), where rows written together are off by half a step."""
    page, dim, n = 32, 64, 75
    x = rows_of(n, 2, dim, torch.float32, 9) * torch.linspace(0.05, 4, n, device="cuda")[:, None, None]
    cache, table = kd.KvCache.empty(4, 2, page, dim), None
    lens, state, ring = i32([0]), i32([0, 4, 0, 0]), i32([2, 0, 3, 1])
    table = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    for i in range(n):
        plan = kd.KvPlan.empty(1, 1, page)
        plan.lens, plan.state = lens, state
        kd.kv_plan(i32([1]), lens, table, ring, state, plan)
        kd.kv_append(x[i:i + 1], x[i:i + 1], plan, cache)
    assert table[0, :3].tolist() == [2, 0, 3]
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        held = (codes.double() * scale.double()[:, :, None, None])[table[0, :3].long()].transpose(1, 2).reshape(-1, 2, dim)[:n]
        step = scale.double()[table[0, :3].long()].repeat_interleave(page, 0)[:n, :, None]
        assert ((held - x.double()).abs() < step).all()


def test_append_leaves_what_no_entry_names(kd):
    page = 16
    plan, _ = step_of(kd, [3], [0], page, 4, 4)
    x = rows_of(3, 2, 64, torch.bfloat16, 4)
    for entry in ([0, 3, 4, 0], [0, 3, -1, 0], [1, 3, 1, 0], [-1, 2, 1, 0], [0, 3, 1, 14], [0, 3, 1, -1], [0, 0, 1, 0], [0, -2, 1, 0]):
        cache = random_cache(kd, 4, 2, page, 64, 5)
        before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
        plan.writes.copy_(i32([entry] * plan.writes.shape[0]))
        kd.kv_append(x, x, plan, cache)
        assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.v, cache.k_scale, cache.v_scale)))


# ---- attention ---------------------------------------------------------------------------------------------------------------
def attend(q, k, v, keep, scale):
    """One sequence in float64: q [n, H, D], k, v [T, KV, D], keep [n, T] -> (o, A, bound of |score|, keys, sum of |v|)."""
    n, H, D = q.shape
    G = H // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    s = torch.einsum("nhd,thd->hnt", q, k) * scale
    big = torch.einsum("nhd,thd->hnt", q.abs(), k.abs()) * abs(scale)
    s = s.masked_fill(~keep, -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e300)
    e = torch.exp(s - top)
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
    big = big.masked_fill(~keep, 0.0).amax(-1) if keep.shape[1] else torch.zeros(H, n, dtype=torch.float64, device=q.device)
    # a masked value does not enter, whatever it is
    v = torch.where((p == 0).all(1).T[..., None], 0.0, v)
    # what weights that vanish may take away: the sum of |v| over the kept keys
    rest = torch.einsum("nt,thd->nhd", keep.double(), v.abs())
    return torch.einsum("hnt,thd->nhd", p, v), torch.einsum("hnt,thd->nhd", p, v.abs()), big.T, keep.sum(-1), rest


def held_to(got, want, A, big, keys, dtype, operand, weight, D, floor=0.0):
    es = big * (2 * operand + D * F32 + 8 * F32)
    bound = A * (2 * es + 2 * weight + (8 + keys[:, None].double().sqrt() * 4) * F32)[..., None] + want.abs() * OUT[dtype] * 1.01 + floor + 1e-30
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), f"{(off / bound).max().item():.3g} of the bound"


def cache_case(kd, dtype, heads, kv, dim, page, fresh, lens, window, seed=0, scale=None, pad=0, strided=False):
    pages = sum(-(-(n + m) // page) for n, m in zip(lens, fresh)) + 3
    cols = max(1, max(-(-(n + m) // page) for n, m in zip(lens, fresh)) + 2)
    plan, table = step_of(kd, fresh, lens, page, cols, pages, seed, rows=sum(max(f, 0) for f in fresh) + pad)
    cache = random_cache(kd, pages, kv, page, dim, seed + 1)
    q = rows_of(plan.rows, heads, dim, dtype, seed + 2)
    out = torch.full_like(q, 777.0)
    if strided:     # a part of a fused projection, unaligned rows of the result
        q = torch.cat([q, q * 0 + 9, q * 0 - 9], 1)[:, :heads] if dtype == torch.float32 else q
        out = torch.full((plan.rows, heads * dim + 3), 777.0, dtype=dtype, device="cuda")[:, 1:1 + heads * dim].view(plan.rows, heads, dim)
    ws = torch.empty(kd.kv_attention_workspace_bytes(plan.rows, len(fresh), heads, kv, dim), dtype=torch.uint8, device="cuda")
    kd.kv_attention(q, plan, table, cache, out, ws, scale=scale, window=window)
    check_cache(plan, table, cache, q, out, lens, fresh, window, dtype, scale)
    return plan, table, cache, q, out, ws


def check_cache(plan, table, cache, q, out, lens, fresh, window, dtype, scale=None):
    page, dim, kv = cache.page, cache.dim, cache.kv_heads
    rs, last = plan.row_start.tolist(), plan.lens.tolist()
    for b in range(len(fresh)):
        n = rs[b + 1] - rs[b]
        if n == 0:
            continue
        T = last[b]
        pg = table[b, :-(-T // page)].long()
        good = (pg >= 0) & (pg < cache.pages)
        at = pg.clamp(0, cache.pages - 1)
        k, v = ((c[at].double() * s[at].double()[..., None, None]).transpose(1, 2).reshape(-1, kv, dim)[:T]
                for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        pos = torch.arange(lens[b], lens[b] + n, device="cuda")[:, None]
        j = torch.arange(T, device="cuda")[None, :]
        keep = (j <= pos) & good.repeat_interleave(page)[None, :T]
        if window:
            keep &= j > pos - window
        o, A, big, keys, rest = attend(q[rs[b]:rs[b + 1]], k, v, keep, dim ** -0.5 if scale is None else scale)
        operand, weight = (0.0, 2.0 ** -11) if dtype == torch.bfloat16 else (2.0 ** -22, 2.0 ** -22)
        held_to(out[rs[b]:rs[b + 1]], o, A, big, keys, dtype, operand, weight, dim, floor=rest * 2.0 ** -31)
    assert (out[rs[-1]:] == 777.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,dim,page,fresh,lens,window", [
    (1, 1, 16, 16, [1], [0], 0),                                     # one token, nothing before it
    (4, 1, 64, 16, [1, 1, 1, 1], [1, 15, 16, 17], 0),                # around a page
    (32, 8, 128, 64, [1] * 5, [63, 64, 100, 1000, 4095], 0),         # a decode batch
    (24, 8, 64, 32, [6, 1, 3, 2], [500, 0, 31, 77], 0),              # drafts
    (8, 8, 128, 128, [5, 0, 9], [300, 200, 129], 0),                 # no grouping, a sequence without rows
    (12, 1, 128, 64, [3, 1], [200, 900], 100),                       # a group of twelve, window
    (40, 2, 96, 32, [2, 17], [65, 40], 16),                          # a group of twenty, odd head size, window within a page
    (6, 2, 256, 16, [1, 4], [333, 50], 0),                           # the largest head
    (3, 3, 80, 64, [70, 130], [0, 61], 0),                           # whole prompts against the cache
    (64, 1, 128, 64, [1, 2], [700, 10], 0),                          # one shared head
    (16, 2, 240, 128, [1, 3], [129, 640], 50),
    (4, 2, 128, 16, [1], [20000], 0),                                # long
    (2, 2, 64, 16, [1], [9000], 3000),
])
def test_cache_attention(kd, dtype, heads, kv, dim, page, fresh, lens, window):
    cache_case(kd, dtype, heads, kv, dim, page, fresh, lens, window, seed=heads + dim)


def test_cache_attention_rows_behind_the_last_sequence_and_strides(kd):
    for dtype in (torch.float32, torch.bfloat16):
        cache_case(kd, dtype, 8, 2, 64, 16, [2, -1, 3, 0], [40, 50, 7, 100], 0, pad=5, strided=True)
        cache_case(kd, dtype, 8, 2, 128, 16, [1, 1], [40, 50], 0, scale=0.0)          # equal weights
        cache_case(kd, dtype, 8, 2, 128, 16, [1, 1], [40, 50], 0, scale=-0.3)
        cache_case(kd, dtype, 8, 2, 128, 16, [1, 1], [40, 50], 10 ** 9)


def test_cache_attention_many_sequences(kd):
    rng = random.Random(8)
    lens = [rng.choice([0, 1, 5, rng.randrange(0, 300)]) for _ in range(400)]
    cache_case(kd, torch.bfloat16, 8, 4, 64, 16, [rng.choice([0, 1, 1, 2]) for _ in lens], lens, 0)


def test_cache_attention_thousands_of_sequences(kd):
    """More than a CTA keeps the lengths of."""
    rng = random.Random(9)
    lens = [rng.randrange(0, 40) for _ in range(3000)]
    cache_case(kd, torch.bfloat16, 2, 1, 64, 16, [rng.choice([0, 1, 1]) for _ in lens], lens, 0)


def test_cache_attention_peaked_and_far_scales(kd):
    """Scores that leave one token, pages whose scales lie far apart, a page of zeros."""
    for dtype in (torch.bfloat16, torch.float32):
        plan, table, cache, q, out, ws = cache_case(kd, dtype, 8, 2, 128, 16, [1, 2], [100, 40], 0)
        cache.k_scale[::2] *= 16
        cache.v_scale[table[0, 1].long()] = 2.0 ** -60
        cache.v_scale[table[0, 2].long()] = 2.0 ** 40
        cache.v_scale[table[0, 3].long()] = 0.0
        cache.v[table[0, 3].long()] = 0
        cache.v_scale[table[1]. long().clamp(min=0)[0]] = 2.0 ** -100
        out.fill_(777.0)
        kd.kv_attention(q, plan, table, cache, out, ws)
        check_cache(plan, table, cache, q, out, [100, 40], [1, 2], 0, dtype)


def test_cache_attention_pages_that_are_not_there(kd):
    for dtype in (torch.bfloat16, torch.float32):
        plan, table, cache, q, out, ws = cache_case(kd, dtype, 4, 2, 64, 16, [1, 3], [100, 40], 0)
        table[0, 2], table[0, 4], table[1, :] = -1, cache.pages, 2 ** 31 - 1
        out.fill_(777.0)
        kd.kv_attention(q, plan, table, cache, out, ws)
        assert (out[1:] == 0).all()                                  # a row that nothing is left for
        check_cache(plan, table, cache, q, out, [100, 40], [1, 3], 0, dtype)
        # a table that ends before the sequence does
        plan, table, cache, q, out, ws = cache_case(kd, dtype, 4, 2, 64, 16, [1], [100], 0)
        short = table[:, :3].contiguous()
        padded = torch.cat([short, torch.full((1, 5), -1, dtype=torch.int32, device="cuda")], 1)
        out.fill_(777.0)
        kd.kv_attention(q, plan, short, cache, out, ws)
        check_cache(plan, padded, cache, q, out, [100], [1], 0, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,dim,page,fresh,lens,window", [
    (32, 8, 128, 64, [1], [1900], 0), (8, 1, 128, 64, [1], [0], 0), (16, 2, 64, 16, [1, 0, 1, 1], [33, 50, 2000, 31], 0),
    (8, 8, 128, 128, [1, 1, 1, 1], [1, 700, 15, 16], 100), (8, 2, 64, 32, [2, 2, 1, 3], [5, 90, 1000, 0], 0), (4, 4, 64, 64, [7], [900], 33),
    (32, 8, 128, 64, [1, 1, 1, 1], [8000, 3, 1023, 1024], 0), (16, 2, 128, 64, [1], [16000], 0),
])
def test_cache_attention_of_short_and_wide_tables(kd, dtype, heads, kv, dim, page, fresh, lens, window):
    """Few sequences: a table with room for short contexts alone, and the same one with room for long ones."""
    plan, table, cache, q, out, ws = cache_case(kd, dtype, heads, kv, dim, page, fresh, lens, window, seed=7, pad=2)
    wide = torch.cat([table, torch.full((len(fresh), 17000 // page), -1, dtype=torch.int32, device="cuda")], 1)
    again = torch.full_like(out, 777.0)
    kd.kv_attention(q, plan, wide, cache, again, ws, window=window)
    check_cache(plan, wide, cache, q, again, lens, fresh, window, dtype)
    third = torch.full_like(out, 777.0)
    kd.kv_attention(q, plan, table, cache, third, ws, window=window)
    assert torch.equal(out, third) and (out[sum(fresh):] == 777.0).all() and (again[sum(fresh):] == 777.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,dim,window", [(8, 1, 128, 0), (4, 1, 64, 0), (16, 2, 96, 0), (8, 1, 256, 0), (6, 6, 128, 30000)])
def test_cache_attention_of_one_long_sequence(kd, dtype, heads, kv, dim, window):
    """A unit of many CTAs' pieces."""
    plan, table, cache, q, out, ws = cache_case(kd, dtype, heads, kv, dim, 64, [1], [40001], window, seed=3)
    again = torch.full_like(out, 777.0)
    kd.kv_attention(q, plan, table, cache, again, ws, window=window)
    assert torch.equal(out, again)


def test_cache_attention_stale_places_do_not_reach_the_result(kd):
    plan, table, cache, q, out, ws = cache_case(kd, torch.bfloat16, 8, 2, 128, 64, [1, 1], [70, 5], 0)
    want = out.clone()
    for b, n in enumerate(plan.lens.tolist()):
        pg = table[b, (n - 1) // 64].long()
        cache.k[pg, :, n % 64:] = 127
        cache.v[pg, :, n % 64:] = -128
    free = torch.ones(cache.pages, dtype=torch.bool)
    for b, n in enumerate(plan.lens.tolist()):
        free[table[b, :-(-n // 64)].long().cpu()] = False
    cache.k_scale[free.cuda()] = float("nan")
    cache.v_scale[free.cuda()] = float("inf")
    kd.kv_attention(q, plan, table, cache, out, ws)
    assert torch.equal(out, want)


def test_cache_attention_in_place_and_twice(kd):
    """out may be q; the same call gives the same bits."""
    plan, table, cache, q, out, ws = cache_case(kd, torch.bfloat16, 32, 8, 128, 64, [1, 4, 2], [3000, 100, 0], 0)
    again = torch.full_like(out, 777.0)
    ws.fill_(0xFF)
    kd.kv_attention(q, plan, table, cache, again, ws)
    assert torch.equal(out, again)
    mine = q.clone()
    kd.kv_attention(mine, plan, table, cache, mine, ws)
    assert torch.equal(mine, out)


def check_prompt(q, k, v, out, starts, window, dtype, scale=None):
    D = q.shape[2]
    for b in range(len(starts) - 1):
        lo, hi = starts[b], starts[b + 1]
        n = hi - lo
        if n <= 0:
            continue
        step = 512 if n > 3000 else n              # rows of a long prompt in parts
        for r0 in range(0, n, step):
            i = torch.arange(r0, min(n, r0 + step), device="cuda")[:, None]
            j = torch.arange(min(n, r0 + step), device="cuda")[None, :]
            keep = j <= i
            if window:
                keep &= j > i - window
            rows = slice(lo + r0, lo + min(n, r0 + step))
            keys = slice(lo, lo + j.shape[1])
            o, A, big, count, _ = attend(q[rows], k[keys], v[keys], keep, D ** -0.5 if scale is None else scale)
            weight = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
            held_to(out[rows], o, A, big, count, dtype, 0.0, weight, D)


def prompt_case(kd, dtype, heads, kv, dim, lens, window, seed=0, lead=0, pad=0, fused=False, scale=None):
    starts = [lead]
    for n in lens:
        starts.append(starts[-1] + n)
    rows = starts[-1] + pad
    if fused:
        qkv = rows_of(rows, heads + 2 * kv, dim, dtype, seed)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    else:
        q, k, v = rows_of(rows, heads, dim, dtype, seed), rows_of(rows, kv, dim, dtype, seed + 1), rows_of(rows, kv, dim, dtype, seed + 2)
    out = torch.full((rows, heads, dim), 777.0, dtype=dtype, device="cuda")
    kd.prompt_attention(q, k, v, i32(starts), out, scale=scale, window=window)
    check_prompt(q, k, v, out, starts, window, dtype, scale)
    assert (out[:lead] == 777.0).all() and (out[starts[-1]:] == 777.0).all()
    return q, k, v, out, starts


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,dim,lens,window", [
    (1, 1, 8, [1], 0), (4, 2, 64, [1, 2, 3], 0), (32, 8, 128, [77], 0), (8, 8, 128, [127, 128, 129], 0),
    (32, 4, 128, [15, 16, 17, 0, 300], 0), (6, 2, 128, [200, 33], 0), (5, 1, 80, [100, 64], 0), (12, 4, 96, [260], 0),
    (4, 1, 256, [150, 3], 0), (2, 1, 200, [90], 20), (24, 8, 64, [700, 1], 100), (8, 2, 128, [600, 257], 1),
    (8, 2, 128, [400], 128), (64, 1, 64, [130], 0), (130, 1, 64, [40], 0), (40, 2, 128, [77, 5], 33), (1, 1, 128, [2500], 0),
    (16, 2, 72, [333], 0),
])
def test_prompt_attention(kd, dtype, heads, kv, dim, lens, window):
    prompt_case(kd, dtype, heads, kv, dim, lens, window, seed=dim + heads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_attention_rows_outside_and_fused_projection(kd, dtype):
    prompt_case(kd, dtype, 8, 2, 128, [50, 0, 140], 0, lead=3, pad=9)
    prompt_case(kd, dtype, 8, 2, 64, [150, 13], 0, fused=True)
    prompt_case(kd, dtype, 8, 2, 128, [150, 13], 70, fused=True, scale=-0.2)
    prompt_case(kd, dtype, 4, 4, 128, [300], 0, scale=0.0)
    # unaligned rows: a pitch that is no multiple of 16 bytes
    n, H, D = 90, 4, 64
    wide = rows_of(n, 1, 3 * H * D + 1, dtype, 4)[:, 0]
    q, k, v = (wide[:, 1 + i * H * D:1 + (i + 1) * H * D].view(n, H, D) for i in range(3))
    out = torch.empty(n, H, D, dtype=dtype, device="cuda")
    kd.prompt_attention(q, k, v, i32([0, 40, n]), out)
    check_prompt(q, k, v, out, [0, 40, n], 0, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,dim,lens,window", [
    (32, 8, 128, [1300, 0, 77], 0), (32, 4, 64, [900, 333], 200), (16, 16, 128, [700, 129, 700], 0), (24, 8, 96, [800, 50], 0),
    (64, 8, 128, [257, 256, 255, 1], 64), (20, 4, 40, [1500], 0),
])
def test_prompt_attention_of_many_rows(kd, dtype, heads, kv, dim, lens, window):
    """Enough work for every SM: two query tiles per CTA."""
    prompt_case(kd, dtype, heads, kv, dim, lens, window, seed=dim + heads, lead=2, pad=3)


@pytest.mark.parametrize("heads,kv,dim,lens,window", [
    (16, 2, 256, [1300, 0, 77], 0), (8, 8, 256, [700, 129], 200), (6, 2, 200, [515], 0), (4, 1, 136, [300, 1, 2], 64),
    (20, 4, 192, [257, 256, 255], 0), (3, 3, 256, [1], 0), (128, 1, 256, [140], 33),
])
def test_prompt_attention_of_wide_heads(kd, heads, kv, dim, lens, window):
    prompt_case(kd, torch.bfloat16, heads, kv, dim, lens, window, seed=dim + heads, lead=1, pad=5)


def test_prompt_attention_of_many_sequences(kd):
    rng = random.Random(4)
    lens = [rng.choice([0, 1, 2, 17, 40]) for _ in range(700)]
    prompt_case(kd, torch.bfloat16, 8, 2, 64, lens, 0)
    prompt_case(kd, torch.float32, 4, 1, 64, lens, 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,heads", [(64, 8), (128, 8), (256, 8), (64, 64), (128, 64)])
def test_prompt_attention_masked_places_hold_anything(kd, dtype, dim, heads):
    """Infinities and NaN in later rows, in other sequences and behind the last one do not reach the rows before them."""
    q, k, v, out, starts = prompt_case(kd, dtype, heads, heads // 4, dim, [100, 150, 40], 0, pad=30)
    want, k0, v0 = out.clone(), k.clone(), v.clone()
    bad = (float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min)
    for i in range(30):
        k[starts[-1] + i], v[starts[-1] + i] = bad[i % 4], bad[(i + 1) % 4]
    k[60, 0], v[60, 1, 5], v[61, 0, 7], k[249], v[249] = bad[0], bad[0], bad[1], bad[0], bad[2]
    kd.prompt_attention(q, k, v, i32(starts), out)
    assert (out[starts[-1]:] == 777.0).all()
    got = out[60:100].float()
    assert torch.isnan(got[:, :4]).all()                              # a NaN key
    assert torch.isnan(got[:, 4:8, 5]).all() and (torch.isinf(got[1:, :4, 7]) | torch.isnan(got[1:, :4, 7])).all()
    # everything else is what it was without them: held to the clean values' result (a row beside such a place may be summed
    # in another order, so by the bound and not by its bits)
    reached = torch.zeros_like(out, dtype=torch.bool)
    reached[60:100, :4] = True
    reached[60:100, 4:8, 5] = True
    reached[249] = True
    check_prompt(q, k0, v0, torch.where(reached, want, out), starts, 0, dtype)


def test_prompt_attention_large_scores(kd):
    for dtype in (torch.bfloat16, torch.float32):
        prompt_case(kd, dtype, 4, 2, 128, [300], 0, scale=8.0)


# ---- together -------------------------------------------------------------------------------------------------------------------
def test_a_prompt_and_its_decode_steps_in_a_graph(kd):
    """Prompts by prompt_attention and into the cache, then decode steps replayed from one graph: every step's result is the
    attention over what the cache holds, and the pool's lengths move on."""
    B, heads, kv, dim, page, pages, cols = 3, 8, 2, 64, 16, 60, 20
    lens, state = torch.zeros(B, dtype=torch.int32, device="cuda"), i32([0, pages, 0, 0])
    ring, table = torch.arange(pages, dtype=torch.int32, device="cuda").flip(0).contiguous(), torch.full((B, cols), -1, dtype=torch.int32, device="cuda")
    cache = kd.KvCache.empty(pages, kv, page, dim)
    prompt = [37, 16, 90]
    n = sum(prompt)
    plan = kd.KvPlan.empty(B, n, page)
    plan.lens, plan.state = lens, state
    q, k, v = (rows_of(n, h, dim, torch.bfloat16, s) for s, h in enumerate((heads, kv, kv)))
    out = torch.empty_like(q)
    kd.kv_plan(i32(prompt), lens, table, ring, state, plan)
    kd.prompt_attention(q, k, v, plan.row_start, out)
    kd.kv_append(k, v, plan, cache)
    check_prompt(q, k, v, out, [0, 37, 53, 143], 0, torch.bfloat16)
    # the same rows over the cache: keys and values within half a step of the page's scale
    over = torch.full_like(q, 777.0)
    ws = torch.empty(kd.kv_attention_workspace_bytes(n, B, heads, kv, dim), dtype=torch.uint8, device="cuda")
    kd.kv_attention(q, plan, table, cache, over, ws)
    check_cache(plan, table, cache, q, over, [0, 0, 0], prompt, 0, torch.bfloat16)
    assert (over.float() - out.float()).abs().max() < 0.25
    # decode
    step = kd.KvPlan.empty(B, B, page)
    step.lens, step.state = lens, state
    fresh, q1, kv1 = i32([1, 1, 1]), torch.empty(B, heads, dim, dtype=torch.bfloat16, device="cuda"), torch.empty(B, 2 * kv, dim, dtype=torch.bfloat16, device="cuda")
    o1 = torch.empty_like(q1)
    stream = torch.cuda.Stream()

    def one():
        kd.kv_plan(fresh, lens, table, ring, state, step)
        kd.kv_append(kv1[:, :kv], kv1[:, kv:], step, cache)
        kd.kv_attention(q1, step, table, cache, o1, ws)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        one()
    assert lens.tolist() == prompt                      # captured, not run
    for i in range(25):
        q1.copy_(rows_of(B, heads, dim, torch.bfloat16, 100 + i))
        kv1.copy_(rows_of(B, 2 * kv, dim, torch.bfloat16, 200 + i, gain=1 + i / 8))
        o1.fill_(777.0)
        graph.replay()
        torch.cuda.synchronize()
        assert lens.tolist() == [p + i + 1 for p in prompt] and state[2].item() == 0
        check_cache(step, table, cache, q1, o1, [p + i for p in prompt], [1] * B, 0, torch.bfloat16)


def test_two_streams_at_once(kd):
    """Two calls on their own streams and workspaces do not meet."""
    cases = [cache_case(kd, torch.bfloat16, 32, 8, 128, 64, [1, 1], [5000, 900], 0, seed=s) for s in (1, 2)]
    want = [c[4].clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (plan, table, cache, q, out, ws) in zip(streams, cases):
            with torch.cuda.stream(s):
                kd.kv_attention(q, plan, table, cache, out, ws)
    torch.cuda.synchronize()
    for w, c in zip(want, cases):
        assert torch.equal(c[4], w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_attention_of_values_that_are_not_finite(kd, dtype):
    """What is not finite and seen stays so, in every later row and no other channel."""
    q, k, v, out, starts = prompt_case(kd, dtype, 32, 8, 128, [700, 60], 0)
    want = out.clone()
    v[3, 2, 9], v[130, 0, 0], k[400, 5, 1] = float("nan"), float("inf"), float("nan")
    kd.prompt_attention(q, k, v, i32(starts), out)
    assert torch.isnan(out[3:700, 8:12, 9]).all() and torch.isnan(out[400:700, 20:24]).all()
    assert not torch.isfinite(out[130:700, 0:4, 0]).any()
    reached = torch.zeros_like(out, dtype=torch.bool)
    reached[3:700, 8:12, 9], reached[400:700, 20:24], reached[130:700, 0:4, 0] = True, True, True
    k[400, 5, 1] = v[3, 2, 9] = v[130, 0, 0] = 0.0
    close = (out.float() - want.float()).abs() <= (2.0 ** -6 if dtype == torch.bfloat16 else 1e-5) * (want.float().abs() + 1)
    assert (close | reached).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,dim", [(150, 64), (90, 128), (70, 256), (2100, 64)])
def test_prompt_attention_at_the_ends_of_the_type(kd, dtype, n, dim):
    """A key whose scores are -inf has no weight; a value near the largest number is met as it is."""
    q, k, v = rows_of(n, 16, dim, dtype, 1), rows_of(n, 8, dim, dtype, 2), rows_of(n, 8, dim, dtype, 3)
    q[:, :, 2] = -q[:, :, 2].abs() - 0.125
    out, far = torch.empty_like(q), torch.empty_like(q)
    v[5, 1, 3], v[9, 2, 7] = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    kd.prompt_attention(q, k, v, i32([0, n]), out)
    check_prompt(q, k, v, out, [0, n], 0, dtype)
    v[5, 1, 3] = 1.0
    k[7, 0, 2] = 1e30                     # q . k is below -1e28
    kd.prompt_attention(q, k, v, i32([0, n]), far)
    k[7, 0, 2] = float("inf")
    kd.prompt_attention(q, k, v, i32([0, n]), out)
    assert torch.isfinite(out).all()
    limit = 2.0 ** -6 if dtype == torch.bfloat16 else 1e-5
    assert ((out.float() - far.float()).abs() <= limit * (far.float().abs() + 1)).all()
    # finite operands whose product is beyond the type, and one whose parts' products would be
    q[:, :, 2] = -1e8
    k[:, :, 2] = 0.0
    k[7, 0, 2] = 1e20
    kd.prompt_attention(q, k, v, i32([0, n]), far)
    k[7, 0, 2] = 1e38
    kd.prompt_attention(q, k, v, i32([0, n]), out)
    assert torch.isfinite(out).all()
    assert ((out.float() - far.float()).abs() <= limit * (far.float().abs() + 1)).all()


def test_calls_on_a_stream_of_their_own(kd):
    """The launch goes to the current stream: work queued there before it is seen, and nothing waits for the default stream."""
    stream = torch.cuda.Stream()
    q, k, v, want, starts = prompt_case(kd, torch.bfloat16, 8, 2, 64, [100, 30], 0)
    rs = i32(starts)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        q2 = torch.zeros_like(q)
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(5):
            big = big @ big * 1e-3
        q2.copy_(q)
        out = torch.empty_like(q)
        kd.prompt_attention(q2, k, v, rs, out)
        got = out.clone()
    stream.synchronize()
    assert torch.equal(got, want)
