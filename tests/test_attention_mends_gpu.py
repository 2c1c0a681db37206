"""The attention operators where calls meet each other and where inputs are far from ordinary; helpers, bounds and their derivation are
those of test_attention_gpu.py."""
import pytest
import torch

from test_attention_gpu import F32, OUT, attend, cache_case, check_prompt, i32, rows_of

pytestmark = pytest.mark.gpu


def test_prompts_behind_one_another(kd):
    """Calls of every kernel form that takes tensor memory, queued without a wait between them, with grids that hold CTAs without work."""
    cases = [(32, 8, 128, [77]), (16, 16, 64, [40, 3, 500]), (8, 4, 256, [300, 129]), (32, 8, 128, [1300, 600]), (8, 8, 64, [10] * 40),
             (12, 4, 200, [90]), (64, 8, 64, [2000])]
    made = []
    for i, (heads, kv, dim, lens) in enumerate(cases):
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        rows = starts[-1] + 700                      # rows behind the last sequence: CTAs that find no part of one
        q, k, v = rows_of(rows, heads, dim, torch.bfloat16, i), rows_of(rows, kv, dim, torch.bfloat16, i + 50), rows_of(rows, kv, dim, torch.bfloat16, i + 90)
        made.append((q, k, v, i32(starts), starts, torch.full_like(q, 777.0)))
    torch.cuda.synchronize()
    for _ in range(30):
        for q, k, v, rs, _, out in made:
            kd.prompt_attention(q, k, v, rs, out)
    torch.cuda.synchronize()
    assert kd.device_status() == 0
    for q, k, v, _, starts, out in made:
        check_prompt(q, k, v, out, starts, 0, torch.bfloat16)
        assert (out[starts[-1]:] == 777.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,dim,lens,window", [
    (32, 8, 128, [77], 0), (8, 2, 64, [300, 5, 130], 0), (4, 4, 128, [700], 0), (8, 8, 64, [600, 333], 100), (1, 1, 72, [129, 128, 127], 1),
    (12, 4, 96, [900], 500), (16, 2, 256, [500, 20], 0), (6, 6, 256, [400], 60), (16, 1, 128, [1500, 300, 800], 0), (64, 1, 64, [100], 7),
    (32, 8, 128, [2000, 900], 0), (20, 4, 40, [1500], 333),
])
def test_prompt_attention_meets_what_is_not_finite_where_it_is_seen_and_nowhere_else(kd, dtype, heads, kv, dim, lens, window):
    """Every result is what the formula gives: infinities of one sign stay, others are NaN, for the rows that see them; all else is the
    attention over the finite values. (Scores are ordinary, so every weight is positive in the kernels too.)"""
    starts = [2]
    for n in lens:
        starts.append(starts[-1] + n)
    rows = starts[-1] + 40
    q, k, v = rows_of(rows, heads, dim, dtype, 1), rows_of(rows, kv, dim, dtype, 2), rows_of(rows, kv, dim, dtype, 3)
    g = torch.Generator(device="cuda").manual_seed(dim + len(lens))
    kind = torch.tensor([float("nan"), float("inf"), float("-inf")], device="cuda", dtype=dtype)
    few = torch.rand(rows, kv, dim, device="cuda", generator=g) < 4.0 / (sum(lens) * dim)       # about four per head
    few[starts[-1]:] = True
    few[:2] = True
    for s in starts[1:-1]:
        few[s - 1, 0, 0] = few[s, -1, 3] = True                                                # at the ends of sequences
    v0 = torch.where(few, 0.0, v)
    v = torch.where(few, kind[torch.randint(0, 3, v.shape, device="cuda", generator=g)], v)
    k0 = k.clone()
    lost = [(b, n - n // 3) for b, n in enumerate(lens) if n > 60]                            # a key that is NaN, of the last head
    for b, i in lost:
        k[starts[b] + i, -1, 1] = float("nan")
    k[starts[-1]:], k[:2], q[starts[-1]:] = float("nan"), float("inf"), float("nan")
    out = torch.full_like(q, 777.0)
    kd.prompt_attention(q, k, v, i32(starts), out, window=window)
    assert (out[:2] == 777.0).all() and (out[starts[-1]:] == 777.0).all()
    G, clean = heads // kv, out.clone()
    for b, n in enumerate(lens):
        part = slice(starts[b], starts[b + 1])
        i = torch.arange(n, device="cuda")
        keep = i[None, :] <= i[:, None]
        if window:
            keep &= i[None, :] > i[:, None] - window
        nan, up, down = (torch.einsum("nt,tgd->ngd", keep.float(), m[part].float()) > 0 for m in (torch.isnan(v), v == float("inf"), v == float("-inf")))
        nan |= up & down
        for c, at in lost:
            if c == b:
                nan[:, -1] |= keep[:, at, None]
        nan, up, down = (m.repeat_interleave(G, 1) for m in (nan, up, down))
        got = out[part]
        assert torch.equal(torch.isnan(got), nan)
        assert (got[up & ~nan] == float("inf")).all() and (got[down & ~nan] == float("-inf")).all()
        lone = nan | up | down
        clean[part] = torch.where(lone, 0.0, got)
        # the finite ones by the ordinary bound
        want = torch.empty_like(out[part])
        kd.prompt_attention(q[part], k0[part], v0[part], i32([0, n]), want, window=window)
        check_prompt(q[part], k0[part], v0[part], torch.where(lone, want, got), [0, n], window, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_attention_takes_no_longer_for_what_is_not_finite(kd, dtype):
    """A row that meets NaN or infinity is not computed on another, slower way."""
    n = 2500
    q, k, v = rows_of(n + 30, 16, 128, dtype, 1), rows_of(n + 30, 4, 128, dtype, 2), rows_of(n + 30, 4, 128, dtype, 3)
    out, starts = torch.empty_like(q), i32([0, n])

    def time_of():
        best = 1e9
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            kd.prompt_attention(q, k, v, starts, out)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    clean = time_of()
    k[n:], v[n:] = float("nan"), float("inf")
    behind = time_of()
    v[n // 2, 1, 7] = float("nan")
    one = time_of()
    v[n // 2:] = float("nan")
    half = time_of()
    limit = 5 * clean + 0.1      # (fp32 tiles that hold one are computed without tensor cores)
    assert max(behind, one, half) < limit, (clean, behind, one, half)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,dim,lens,window", [(8, 2, 128, [20, 300], 0), (8, 8, 64, [2500], 0), (4, 2, 256, [700], 100), (16, 4, 96, [900, 1], 0)])
@pytest.mark.parametrize("size", [3e38, 1e36, 1e20])
def test_prompt_attention_of_values_near_the_largest_number(kd, dtype, heads, kv, dim, lens, window, size):
    """A mean of finite values is finite: of one sign, of both, and of a few large ones among ordinary ones."""
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    rows = starts[-1]
    q, k, v = rows_of(rows, heads, dim, dtype, 1), rows_of(rows, kv, dim, dtype, 2), rows_of(rows, kv, dim, dtype, 3)
    out = torch.empty_like(q)
    for large in (torch.full_like(v, size), torch.where(v > 0, size, -size / 2).to(dtype), torch.where(v > 2.5, size, v).to(dtype)):
        kd.prompt_attention(q, k, large, i32(starts), out, window=window)
        check_prompt(q, k, large, out, starts, window, dtype)


@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("lens", [[700], [720, 20], [850], [60] * 15])
def test_prompt_attention_fp32_around_the_choice_of_groups(kd, dim, lens):
    """Calls of 320 to 480 CTAs, on either side of where one or two groups of warps take a tile."""
    from test_attention_gpu import prompt_case
    prompt_case(kd, torch.float32, 32, 4, dim, lens, 0, seed=dim)
    prompt_case(kd, torch.float32, 32, 4, dim, lens, 50, seed=dim + 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("apart", [4, 20, 28, 40, 90])
@pytest.mark.parametrize("heads,kv,dim,page,fresh,lens", [(8, 2, 128, 16, [1, 2], [100, 40]), (4, 1, 64, 64, [1], [3000]), (6, 2, 256, 32, [5], [200])])
def test_cache_attention_of_scales_that_lie_far_apart(kd, dtype, apart, heads, kv, dim, page, fresh, lens):
    """Every second page's values are 2^-apart of the others', and the others hold codes of 0 in half of the channels: there the small
    pages alone are seen. A weight times scale is off by its rounding (fp16 2^-11, in two parts 2^-22) and by 2^-31 of the row's largest
    one, which meet the codes; a score by the roundings that the ordinary bound counts."""
    plan, table, cache, q, out, ws = cache_case(kd, dtype, heads, kv, dim, page, fresh, lens, 0)
    cache.v_scale.fill_(0.5)
    for row in table.tolist():
        for i, p in enumerate(row):
            if 0 <= p < cache.pages:
                if i % 2:
                    cache.v_scale[p] = 0.5 * 2.0 ** -apart
                else:
                    cache.v[p, :, :, : dim // 2] = 0
    kd.kv_attention(q, plan, table, cache, out, ws)
    rs, G = plan.row_start.tolist(), heads // kv
    for b in range(len(fresh)):
        n, T = rs[b + 1] - rs[b], plan.lens[b].item()
        pg = table[b, :-(-T // page)].long()
        k = (cache.k[pg].double() * cache.k_scale[pg].double()[..., None, None]).transpose(1, 2).reshape(-1, kv, dim)[:T].repeat_interleave(G, 1)
        code = cache.v[pg].double().transpose(1, 2).reshape(-1, kv, dim)[:T].repeat_interleave(G, 1)
        scale = cache.v_scale[pg].double().repeat_interleave(page, 0)[:T].repeat_interleave(G, 1)
        x = q[rs[b]:rs[b + 1]].double()
        keep = torch.arange(T, device="cuda")[None, :] <= torch.arange(lens[b], lens[b] + n, device="cuda")[:, None]
        s = (torch.einsum("nhd,thd->hnt", x, k) * dim ** -0.5).masked_fill(~keep, float("-inf"))
        big = (torch.einsum("nhd,thd->hnt", x.abs(), k.abs()) * dim ** -0.5).masked_fill(~keep, 0.0).amax(-1).T[..., None]
        p = torch.softmax(s, -1)
        pb = p * scale.T[:, None]                                                     # weight times scale
        want, A = torch.einsum("hnt,thd->nhd", pb, code), torch.einsum("hnt,thd->nhd", pb, code.abs())
        floor = pb.amax(-1).T[..., None] * torch.einsum("nt,thd->nhd", keep.double(), code.abs()) * 2.0 ** -31
        operand, weight = (0.0, 2.0 ** -11) if dtype == torch.bfloat16 else (2.0 ** -22, 2.0 ** -22)
        keys = keep.sum(-1).double()[:, None, None]
        bound = A * (2 * big * (2 * operand + (dim + 8) * F32) + 2 * weight + (8 + keys.sqrt() * 4) * F32) + want.abs() * OUT[dtype] * 1.01 + floor + 1e-38
        off = (out[rs[b]:rs[b + 1]].double() - want).abs()
        assert (off <= bound).all(), f"{(off / bound).max().item():.3g} of the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_results_beside_their_inputs_in_one_buffer(kd, dtype):
    """Rows between rows and heads between heads: no element is shared, so the calls are taken, and nothing else is written."""
    n, H, KV, D = 90, 8, 2, 64
    # q, k, v and the result side by side in every row
    buf = rows_of(n, 2 * H + 2 * KV, D, dtype, 1)
    q, k, v, out = buf[:, :H], buf[:, H:H + KV], buf[:, H + KV:H + 2 * KV], buf[:, H + 2 * KV:]
    kept = buf[:, :H + 2 * KV].clone()
    kd.prompt_attention(q, k, v, i32([0, 40, n]), out)
    check_prompt(q, k, v, out, [0, 40, n], 0, dtype)
    assert torch.equal(kept, buf[:, :H + 2 * KV])
    # every second head; and rows of the result behind those of q
    pairs = rows_of(n, 2 * H, D, dtype, 2)
    q, out = pairs[:, ::2], pairs[:, 1::2]
    kept = q.clone()
    k, v = k.contiguous(), v.contiguous()
    kd.prompt_attention(q, k, v, i32([0, 40, n]), out)
    check_prompt(kept, k, v, out, [0, 40, n], 0, dtype)
    assert torch.equal(kept, q)
    both = rows_of(2 * n, H, D, dtype, 3)
    kept = both[:n].clone()
    kd.prompt_attention(both[:n], k, v, i32([0, 40, n]), both[n:])
    check_prompt(kept, k, v, both[n:], [0, 40, n], 0, dtype)
    assert torch.equal(kept, both[:n])
    alternate = rows_of(2 * n, H, D, dtype, 4)
    kept = alternate[::2].clone()
    kd.prompt_attention(alternate[::2], k, v, i32([0, 40, n]), alternate[1::2])
    check_prompt(kept, k, v, alternate[1::2], [0, 40, n], 0, dtype)
    assert torch.equal(kept, alternate[::2])
    plan, table, cache, q, out, ws = cache_case(kd, dtype, H, KV, D, 16, [1, 3], [100, 40], 0)
    want = out.clone()
    wide = torch.cat([q, q], 1)
    kd.kv_attention(wide[:, :H], plan, table, cache, wide[:, H:], ws)
    assert torch.equal(wide[:, H:], want) and torch.equal(wide[:, :H], q)
    same = torch.cat([q, q], 1)
    kd.kv_attention(same[:, :H], plan, table, cache, same[:, :H], ws)
    assert torch.equal(same[:, :H], want) and torch.equal(same[:, H:], q)


# ---- errors as a whole: a bound for each element leaves room for errors that grow with the number of keys, the 2-norm does not. A value
# rounded to bf16 is off by 2^-8 at the most and by 2^-8 (1 / sqrt 3) sqrt(3 / (8 ln 2)) = 1.66e-3 in the mean square (an error uniform within
# half a step, mantissas evenly over their logarithm); random values make the weights' errors and the result's independent, and a result of
# random values is off by the mean square of its weights' errors. A tenth is left for the sample (thousands of elements).
BF16_RMS = 2.0 ** -8 * (1 / 3) ** 0.5 * (3 / (8 * 0.6931471805599453)) ** 0.5


def off_by(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [300, 3000, 20000])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_attention_as_a_whole(kd, dtype, n, dim):
    q, k, v = rows_of(n, 8, dim, dtype, 1), rows_of(n, 2, dim, dtype, 2), rows_of(n, 2, dim, dtype, 3)
    out = torch.empty_like(q)
    kd.prompt_attention(q, k, v, i32([0, n]), out)
    i = torch.arange(n - 24, n, device="cuda")
    want, _, big, _, _ = attend(q[-24:], k, v, torch.arange(n, device="cuda")[None, :] <= i[:, None], dim ** -0.5)
    if dtype == torch.bfloat16:
        limit = 1.1 * BF16_RMS * 2 ** 0.5                                # weights and result
    else:
        limit = 2 * big.mean().item() * 8 * F32 + 8 * F32               # a score's eight roundings, twice (its own and the sum's), and the result's
    assert off_by(out[-24:], want) <= limit


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [300, 3000, 50000])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_cache_attention_as_a_whole(kd, dtype, n, dim):
    plan, table, cache, q, out, ws = cache_case(kd, dtype, 16, 2, dim, 64, [2, 1], [n, n // 2], 0, seed=n)
    gots, wants, bigs = [], [], []
    for b in range(2):
        r0, r1 = plan.row_start.tolist()[b:b + 2]
        T = plan.lens[b].item()
        pg = table[b, :-(-T // 64)].long()
        k, v = ((c[pg].double() * s[pg].double()[..., None, None]).transpose(1, 2).reshape(-1, 2, dim)[:T]
                for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        pos = torch.arange(T - (r1 - r0), T, device="cuda")[:, None]
        want, _, big, _, _ = attend(q[r0:r1], k, v, torch.arange(T, device="cuda")[None, :] <= pos, dim ** -0.5)
        gots.append(out[r0:r1]), wants.append(want), bigs.append(big.mean().item())
    if dtype == torch.bfloat16:
        limit = 1.1 * BF16_RMS * (1 + 2.0 ** -6) ** 0.5                   # fp16 weights have three bits more
    else:
        limit = 2 * max(bigs) * 8 * F32 + 8 * F32
    assert off_by(torch.cat(gots), torch.cat(wants)) <= limit


def test_prompts_and_products_on_two_streams(kd):
    """Kernels that take tensor memory, on two streams at once: prompts of several forms on both, packed products behind them on one."""
    made = []
    for i, (heads, kv, dim, lens) in enumerate([(16, 16, 64, [40, 3, 500]), (32, 8, 128, [700, 600]), (8, 4, 256, [300]), (32, 8, 128, [77])]):
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        q, k, v = (rows_of(starts[-1], h, dim, torch.bfloat16, 10 * i + j) for j, h in enumerate((heads, kv, kv)))
        made.append((q, k, v, i32(starts), torch.empty_like(q)))
    packed = kd.ggml_pack.synth_weight(kd.Q4_K, 1024, 2048, seed=3)
    w = kd.QuantWeight.from_numpy(packed, kd.Q4_K, 1024, 2048, torch.device("cuda"))
    x = rows_of(200, 1, 2048, torch.bfloat16, 77)[:, 0].contiguous()
    ws = torch.empty(kd.quant_gemm_workspace_bytes(200, 2048), dtype=torch.uint8, device="cuda")
    y = torch.empty(200, 1024, dtype=torch.float32, device="cuda")
    torch.cuda.synchronize()
    kd.quant_gemm(x, w, y, ws)
    for q, k, v, rs, out in made:
        kd.prompt_attention(q, k, v, rs, out)
    torch.cuda.synchronize()
    want, product = [m[4].clone() for m in made], y.clone()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[torch.empty_like(m[4]) for m in made] for _ in streams]
    torch.cuda.synchronize()
    for _ in range(25):
        for s, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                for m, out in zip(made, outs[s]):
                    kd.prompt_attention(*m[:4], out)
                    if s == 0:
                        kd.quant_gemm(x, w, y, ws)
    torch.cuda.synchronize()
    assert kd.device_status() == 0 and torch.equal(y, product)
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_captured_prompt_whose_values_change(kd, dtype):
    """Replays of one captured call over values that hold infinities, NaN and numbers near the largest, and over ordinary ones again."""
    n, starts = 500, [0, 300, 500]
    q, k, v = rows_of(n, 8, 128, dtype, 1), rows_of(n, 2, 128, dtype, 2), rows_of(n, 2, 128, dtype, 3)
    out, rs, plain = torch.empty_like(q), i32(starts), v.clone()
    kd.prompt_attention(q, k, v, rs, out)
    torch.cuda.synchronize()
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        kd.prompt_attention(q, k, v, rs, out)
    for kind in ("nan", "plain", "large", "inf", "plain"):
        v.copy_(plain)
        if kind == "large":
            v[::3] = 2e38
        elif kind != "plain":
            v[290, 1, 5] = v[450, 0, 9] = float(kind)
        graph.replay()
        torch.cuda.synchronize()
        if kind == "plain":
            assert torch.equal(out, first)
        elif kind == "large":
            check_prompt(q, k, v, out, starts, 0, dtype)
        else:
            hit = ~torch.isfinite(out)
            assert hit[290:300, 4:, 5].all() and hit[450:, :4, 9].all() and hit.sum() == 10 * 4 + 50 * 4


def test_cache_beyond_two_to_the_31_bytes(kd):
    """Pages whose codes lie behind 2^31 bytes: written, read, and nothing near 2^31 or 2^32 less is."""
    page, kv, dim, pages, heads = 64, 8, 128, 66000, 32
    cache = kd.KvCache(*(torch.zeros((pages, kv, page, dim), dtype=torch.int8, device="cuda") for _ in range(2)),
                       *(torch.zeros((pages, kv), device="cuda") for _ in range(2)))
    assert cache.k.numel() > 2 ** 32
    top = [pages - 1, 32768 + 5, 65536 + 7, 32767, 40000]            # (a page is 2^16 bytes)
    plan = kd.KvPlan.empty(2, 200, page)
    ring = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    ring[:5] = i32(top)
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    kd.kv_plan(i32([130, 70]), i32([0, 0]), table, ring, i32([0, 5, 0, 0]), plan)
    assert table.tolist() == [top[:3] + [-1], top[3:] + [-1, -1]]
    k, v, q = (rows_of(200, h, dim, torch.bfloat16, s) for s, h in enumerate((kv, kv, heads)))
    kd.kv_append(k, v, plan, cache)
    touched = cache.k_scale.amax(1).nonzero()[:, 0].tolist()
    assert touched == sorted(top) and not any(cache.k[p - 32768 if p >= 32768 else p + 32768].any() for p in (32768 + 5, 40000))
    out = torch.full_like(q, 777.0)
    ws = torch.empty(kd.kv_attention_workspace_bytes(200, 2, heads, kv, dim), dtype=torch.uint8, device="cuda")
    kd.kv_attention(q, plan, table, cache, out, ws)
    from test_attention_gpu import check_cache
    check_cache(plan, table, cache, q, out, [0, 0], [130, 70], 0, torch.bfloat16)


@pytest.mark.parametrize("dtype,heads,dim", [(torch.bfloat16, 128, 128), (torch.float32, 64, 256), (torch.bfloat16, 64, 256)])
def test_prompts_beyond_two_to_the_31_elements(kd, dtype, heads, dim):
    n = 2 ** 31 // (heads * dim) + 700
    q, k, v = (torch.zeros((n, h, dim), dtype=dtype, device="cuda") for h in (heads, 2, 2))
    tail = 600
    for i, t in enumerate((q, k, v)):
        t[-tail:] = rows_of(tail, t.shape[1], dim, dtype, i)
    out = torch.full_like(q, 777.0)
    starts = [n - 590, n - 400, n - 13]
    kd.prompt_attention(q, k, v, i32(starts), out)
    part = slice(n - 590, n)
    check_prompt(q[part], k[part], v[part], out[part], [0, 190, 577], 0, dtype)
    assert (out[n - 13:] == 777.0).all() and (out[n - 700:n - 590] == 777.0).all() and (out[:1000] == 777.0).all()
