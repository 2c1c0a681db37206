"""Refusals of the attention operators: every check comes before the first launch, so fake pointers are never touched."""
import ctypes as C

import pytest
import torch

P = 0x10000


def _cache(kd, **kw):
    a = dict(k=P, v=P, k_scale=P, v_scale=P, pages=8, kv_heads=2, page=64, dim=128)
    a.update(kw)
    return kd.KvCacheC(*(a[f[0]] for f in kd.KvCacheC._fields_))


def test_writes_hold_every_plan(kd):
    assert kd.kv_writes(0, 4, 64) == 1
    assert kd.kv_writes(3, 64, 64) == 3                 # no more pages than rows
    assert kd.kv_writes(1000, 2, 16) == 62 + 4
    # a sequence of n rows touches at most n / page + 2 pages
    for page in (16, 32, 64, 128):
        for n in range(1, 300):
            most = max((off + n - 1) // page + 1 for off in range(page))
            assert most <= kd.kv_writes(n, 1, page)


def test_plan_refusals(kd):
    ok = dict(fresh=P, lens=P, seqs=4, page=64, rows=4, table=P, ldt=8, cols=8, ring=P, pages=32, state=P, row_start=P, first=P,
              lens_out=P, state_out=P, slots=P, writes=P, entries=8)

    def call(**kw):
        return kd.lib.kdnn_b200_kv_plan(*dict(ok, **kw).values(), None)

    for kw in (dict(page=48), dict(page=0), dict(seqs=0), dict(seqs=8193), dict(cols=0), dict(ldt=7), dict(pages=0),
               dict(pages=2 ** 31 // 64), dict(cols=2 ** 31 // 64, ldt=2 ** 31), dict(rows=2 ** 31), dict(entries=3), dict(writes=P + 4),
               *({n: None} for n in ("fresh", "lens", "table", "ring", "state", "row_start", "first", "lens_out", "state_out", "slots",
                                     "writes"))):
        assert call(**kw) == kd.KDNN_ERR_INVALID, kw
        assert "kv_plan" in kd.last_error()


def test_append_refusals(kd):
    ok = dict(k=P, ldk=256, hdk=128, v=P, ldv=256, hdv=128, scalar=1, rows=4, writes=P, entries=4, cache=_cache(kd))

    def call(**kw):
        a = dict(ok, **kw)
        a["cache"] = C.byref(a["cache"]) if a["cache"] is not None else None
        return kd.lib.kdnn_b200_kv_append(*a.values(), None)

    for kw in (dict(scalar=2), dict(cache=None), dict(k=None), dict(v=None), dict(writes=None), dict(writes=P + 8), dict(ldk=255),
               dict(hdk=127), dict(hdv=129), dict(rows=2 ** 31), *(dict(cache=_cache(kd, **c)) for c in (
                   dict(k=None), dict(v_scale=None), dict(k=P + 8), dict(page=24), dict(dim=24), dict(dim=272), dict(dim=0),
                   dict(kv_heads=0), dict(pages=0), dict(pages=2 ** 25)))):
        assert call(**kw) == kd.KDNN_ERR_INVALID, kw
        assert "kv_append" in kd.last_error()
    assert call(rows=0) == kd.KDNN_OK and call(entries=0) == kd.KDNN_OK


def test_cache_attention_refusals(kd):
    ok = dict(q=P, ldq=512, hdq=128, scalar=1, rows=4, heads=4, row_start=P, first=P, lens=P, seqs=2, table=P, ldt=8, cols=8,
              cache=_cache(kd), out=P, ldo=512, hdo=128, scale=0.1, window=0, ws=P, ws_bytes=1 << 40)

    def call(**kw):
        a = dict(ok, **kw)
        a["cache"] = C.byref(a["cache"]) if a["cache"] is not None else None
        return kd.lib.kdnn_b200_kv_attention(*a.values(), None)

    for kw in (dict(scalar=7), dict(heads=3), dict(heads=65536 * 2), dict(ldq=511), dict(hdq=100), dict(ldo=400), dict(ldt=4), dict(cols=0),
               dict(seqs=8193), dict(rows=2 ** 30), dict(ws=P + 16), dict(cols=2 ** 31 // 64, ldt=2 ** 31), dict(cache=None),
               dict(cache=_cache(kd, dim=8)), *({n: None} for n in ("q", "row_start", "first", "lens", "table", "out", "ws"))):
        assert call(**kw) == kd.KDNN_ERR_INVALID, kw
        assert "kv_attention" in kd.last_error()
    for kw in (dict(rows=0), dict(seqs=0), dict(heads=0)):
        assert call(**kw) == kd.KDNN_OK, kw


def test_prompt_attention_refusals(kd):
    ok = dict(q=P, ldq=512, hdq=128, k=P, ldk=256, hdk=128, v=P, ldv=256, hdv=128, scalar=1, rows=4, heads=4, kv_heads=2, dim=128,
              row_start=P, seqs=2, out=2 * P, ldo=512, hdo=128, scale=0.1, window=0)

    def call(**kw):
        return kd.lib.kdnn_b200_prompt_attention(*dict(ok, **kw).values(), None)

    for kw in (dict(scalar=-1), dict(dim=0), dict(dim=12), dict(dim=264), dict(kv_heads=0), dict(kv_heads=3), dict(ldq=500), dict(hdk=64),
               dict(ldv=200), dict(hdo=120), dict(seqs=8193), dict(rows=2 ** 30), dict(out=P),
               *({n: None} for n in ("q", "k", "v", "row_start", "out"))):
        assert call(**kw) == kd.KDNN_ERR_INVALID, kw
        assert "prompt_attention" in kd.last_error()
    for kw in (dict(rows=0), dict(seqs=0), dict(heads=0)):
        assert call(**kw) == kd.KDNN_OK, kw


def test_python_checks(kd):
    """Shapes, types and places are checked before the library is called; nothing here has a CUDA device."""
    i32 = dict(dtype=torch.int32)
    plan = kd.KvPlan.empty(2, 5, 16, device="cpu")
    assert plan.seqs == 2 and plan.rows == 5 and tuple(plan.writes.shape) == (4, 4)
    fresh, lens, table, ring, state = (torch.zeros(2, **i32), torch.zeros(2, **i32), torch.zeros(2, 3, **i32), torch.zeros(6, **i32),
                                       torch.zeros(4, **i32))
    for bad in ((fresh[:1], lens, table, ring, state), (fresh, lens.long(), table, ring, state), (fresh, lens, table[0], ring, state),
                (fresh, lens, table, ring, state[:3]), (fresh, lens, table.t().contiguous().t(), ring, state),
                (fresh, lens, table, ring, state)):        # the last one is right but for its place
        with pytest.raises(ValueError):
            kd.kv_plan(*bad, plan)
    with pytest.raises(ValueError):
        kd.KvCache(torch.zeros(2, 1, 16, 64), torch.zeros(2, 1, 16, 64), torch.zeros(2, 1), torch.zeros(2, 1))
    cache = kd.KvCache.empty(4, 2, 16, 64, device="cpu")
    k = torch.zeros(5, 2, 64)
    for a, b in ((k[:4], k), (k, k.double()), (k[:, :1], k), (k[..., :32], k[..., :32]), (k.transpose(1, 2), k), (k, k)):
        with pytest.raises(ValueError):
            kd.kv_append(a, b, plan, cache)
    q = torch.zeros(5, 4, 64)
    ws = torch.zeros(16, dtype=torch.uint8)
    for args, kw in (((q[:3], plan, table, cache, q), {}), ((q, plan, table[:1], cache, q), {}), ((q, plan, table, cache, q.bfloat16()), {}),
                     ((q, plan, table, cache, q), dict(window=-1)), ((q, plan, table, cache, q), {})):
        with pytest.raises(ValueError):
            kd.kv_attention(*args, ws, **kw)
    rs = torch.zeros(3, **i32)
    for args in ((q, k, k[:4], rs, q), (q, k, k, rs.long(), q), (q[0], k, k, rs, q), (q, k, k.bfloat16(), rs, q), (q, k, k, rs, q[:, :2]),
                 (q, k, k, rs, q)):
        with pytest.raises(ValueError):
            kd.prompt_attention(*args)


@pytest.mark.parametrize("name,bad", [
    ("lens", lambda: torch.zeros(1, dtype=torch.int32)), ("lens", lambda: torch.zeros(2)), ("first", lambda: torch.zeros(3, dtype=torch.int32)),
    ("state", lambda: torch.zeros(8, dtype=torch.int32)[::2]), ("slots", lambda: torch.zeros(400, dtype=torch.int32)),
    ("writes", lambda: torch.zeros(3, 4, dtype=torch.int32)), ("row_start", lambda: None), ("page", lambda: 0), ("page", lambda: "16"),
])
def test_a_plan_keeps_its_tensors_when_a_new_one_is_refused(kd, name, bad):
    plan = kd.KvPlan.empty(2, 5, 16, device="cpu")
    before, seqs, rows = getattr(plan, name), plan.seqs, plan.rows
    with pytest.raises((ValueError, AttributeError, TypeError, C.ArgumentError)):
        setattr(plan, name, bad())
    assert getattr(plan, name) is before and (plan.seqs, plan.rows) == (seqs, rows)
    plan._check()


def attention_calls(kd):
    """(name, call(out=..., **pitches)) of both attention calls on fake rows: q at 0x100000 [rows 6, heads 4, dim 64] fp32."""
    def prompt(**kw):
        a = dict(dict(q=0x100000, ldq=256, hdq=64, k=0x200000, ldk=128, hdk=64, v=0x300000, ldv=128, hdv=64, scalar=0, rows=6, heads=4, kv_heads=2,
                      dim=64, row_start=P, seqs=2, out=0x400000, ldo=256, hdo=64, scale=0.1, window=0), **kw)
        return kd.lib.kdnn_b200_prompt_attention(*a.values(), None)

    def cached(**kw):
        a = dict(dict(q=0x100000, ldq=256, hdq=64, scalar=0, rows=6, heads=4, row_start=P, first=P, lens=P, seqs=2, table=P, ldt=8, cols=8,
                      cache=C.byref(_cache(kd, dim=64)), out=0x400000, ldo=256, hdo=64, scale=0.1, window=0, ws=P, ws_bytes=1 << 40), **kw)
        return kd.lib.kdnn_b200_kv_attention(*a.values(), None)
    return prompt, cached


def test_results_that_overlap_their_inputs_are_refused(kd):
    """Every place of the result that shares an element with an input, by brute force, is refused; what is merely beside one is for the GPU
    tests, as it would be launched."""
    q, row, head = 0x100000, 1024, 256
    prompt, cached = attention_calls(kd)
    overlaps = [dict(out=q + 4), dict(out=q + head), dict(out=q - 4 * 1), dict(out=q + 5 * row), dict(out=q - 5 * row), dict(out=q + 5 * row + 3 * head),
                dict(out=q - 3 * row, ldo=512), dict(out=q, ldo=512), dict(out=q - 6 * row + 4), dict(out=q - 8 * 2048 // 2, ldo=2048, hdo=512),
                # heads twice as far apart, the result half a head off
                dict(ldq=512, hdq=128, ldo=512, hdo=128, out=q + 128), dict(ldq=512, hdq=128, ldo=512, hdo=128, out=q + 3 * 512 + 384)]
    for kw in overlaps:
        a = dict(dict(ldq=256, hdq=64, ldo=256, hdo=64), **kw)
        mine = {q + 4 * (r * a["ldq"] + h * a["hdq"] + d) for r in range(6) for h in range(4) for d in range(64)}
        outs = {a["out"] + 4 * (r * a["ldo"] + h * a["hdo"] + d) for r in range(6) for h in range(4) for d in range(64)}
        if not mine & outs:
            continue
        assert prompt(**kw) == kd.KDNN_ERR_INVALID and "overlap" in kd.last_error(), kw
        assert cached(**kw) == kd.KDNN_ERR_INVALID and "overlap" in kd.last_error(), kw
    for kw in (dict(out=0x200000 + 512), dict(out=0x300000 - 1024), dict(out=0x300000, ldo=512)):      # k and v
        assert prompt(**kw) == kd.KDNN_ERR_INVALID and "overlap" in kd.last_error(), kw


def test_plan_arguments_that_overlap_are_refused(kd):
    """What a plan writes on something else that it reads or writes: other CTAs may still have to read it."""
    MB = 1 << 20
    names = ("fresh", "lens", "table", "ring", "state", "row_start", "first", "lens_out", "state_out", "slots", "writes")
    ok = dict(fresh=1 * MB, lens=2 * MB, seqs=300, page=64, rows=5000, table=3 * MB, ldt=100, cols=90, ring=4 * MB, pages=9000, state=5 * MB,
              row_start=6 * MB, first=7 * MB, lens_out=8 * MB, state_out=9 * MB, slots=10 * MB, writes=11 * MB, entries=700)
    size = dict(fresh=300, lens=300, table=299 * 100 + 90, ring=9000, state=4, row_start=301, first=300, lens_out=300, state_out=4, slots=5000,
                writes=2800)

    def call(**kw):
        return kd.lib.kdnn_b200_kv_plan(*dict(ok, **kw).values(), None)

    reads = ("fresh", "lens", "state")
    for a in names:
        for b in names:
            if a == b or (a in reads and b in reads) or {a, b} in ({"lens", "lens_out"}, {"state", "state_out"}):
                continue
            for at in (ok[b], ok[b] + 4 * (size[b] - 1), ok[b] - 4 * (size[a] - 1)):
                if a == "writes":
                    at = at // 16 * 16
                    if not (at < ok[b] + 4 * size[b] and ok[b] < at + 4 * size[a]):
                        continue
                if "table" in (a, b) and at not in (ok[b],) and a != "table":
                    at = ok[b] + 4 * (17 * 100 + 89)              # the last column of a row
                    if a == "writes":
                        at = at // 16 * 16
                assert call(**{a: at}) == kd.KDNN_ERR_INVALID, (a, b, at)
                assert "overlap" in kd.last_error(), (a, b, kd.last_error())


def test_a_workspace_whose_bytes_are_not_there_is_refused(kd, monkeypatch):
    """An expanded tensor has more elements than memory."""
    plan, cache = kd.KvPlan.empty(2, 5, 16, device="cpu"), kd.KvCache.empty(4, 2, 16, 64, device="cpu")
    q, table = torch.zeros(5, 4, 64), torch.zeros(2, 3, dtype=torch.int32)
    calls = []
    monkeypatch.setattr(kd, "_stream_of", lambda *a: 0)
    monkeypatch.setattr(kd.lib, "kdnn_b200_kv_attention", lambda *a: calls.append(a) or 0)
    for ws in (torch.zeros(256, dtype=torch.uint8)[:1].expand(1 << 30), torch.zeros(1 << 12, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError, match="workspace"):
            kd.kv_attention(q, plan, table, cache, torch.zeros_like(q), ws)
    assert not calls
    kd.kv_attention(q, plan, table, cache, torch.zeros_like(q), torch.zeros(64, dtype=torch.float32))
    assert len(calls) == 1 and calls[0][-2] == 256
