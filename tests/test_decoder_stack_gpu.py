"""The decoder stack (dnn-for-kokkos_b200/decoder_stack.py): plan, cache write and both attentions as a model calls them, every
attention call held to a plain implementation in 64 bits, and a captured decode step to the eager one bit for bit."""
import pytest
import torch

from test_attention_gpu import check_cache, check_prompt, i32

pytestmark = pytest.mark.gpu


class Checked:
    """The package, with every attention call checked as it is made."""

    def __init__(self, kd):
        self._kd, self.calls, self.cached, self.fresh = kd, 0, None, None

    def __getattr__(self, name):
        return getattr(self._kd, name)

    def kv_attention(self, q, plan, table, cache, out, workspace, scale=None, window=0):
        out.fill_(777.0)
        self._kd.kv_attention(q, plan, table, cache, out, workspace, scale=scale, window=window)
        check_cache(plan, table, cache, q, out, self.cached, self.fresh, window, q.dtype, scale)
        self.calls += 1

    def prompt_attention(self, q, k, v, row_start, out, scale=None, window=0):
        self._kd.prompt_attention(q, k, v, row_start, out, scale=scale, window=window)
        check_prompt(q, k, v, out, row_start.tolist(), window, q.dtype, scale)
        self.calls += 1


def make(kd, layers=2, window=0, pages=40, seqs=3):
    import importlib
    ds = importlib.import_module(kd.__name__ + ".decoder_stack")
    ms = importlib.import_module(kd.__name__ + ".moe_stack")
    cfg = ms.StackConfig(layers=layers, hidden=512, ffn=256, experts=8, top_k=2, tokens=8)
    return ds, ds.AttentionConfig(heads=8, kv_heads=2, dim=64, window=window, page=16, pages=pages, seqs=seqs, longest=256), cfg


def rows(n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(n, 512, device="cuda", generator=g).to(torch.bfloat16)


@pytest.mark.parametrize("window", [0, 12])
def test_prompts_then_decode_steps(kd, window):
    checked = Checked(kd)
    ds, attn, cfg = make(kd, window=window)
    stack = ds.DecoderStack(checked, torch.device("cuda"), cfg, attn)
    lens = [0, 0, 0]
    for fresh, begin in (([33, 5, 0], True), ([1, 1, 0], False), ([0, 4, 20], False), ([1, -1, 1], False), ([2, 16, 1], False)):
        checked.cached, checked.fresh = [0 if f < 0 else n for n, f in zip(lens, fresh)], [max(f, 0) for f in fresh]
        n = sum(checked.fresh)
        h = stack.step(rows(n, 7 * n), i32(fresh), begin=begin)
        lens = [0 if f < 0 else m + f for m, f in zip(lens, fresh)]
        assert torch.isfinite(h.float()).all()
        assert stack.lens.tolist() == lens and stack.rows_without_place() == 0
    assert checked.calls == 5 * cfg.layers and kd.device_status() == 0
    assert int(stack.state[1]) == attn.pages - sum(-(-m // 16) for m in lens)


def test_decode_steps_from_a_graph_equal_eager_ones(kd):
    ds, attn, cfg = make(kd)
    results = []
    for captured in (False, True):
        stack = ds.DecoderStack(kd, torch.device("cuda"), cfg, attn)
        stack.step(rows(40, 1), i32([20, 3, 17]), begin=True)
        h, fresh, got = rows(3, 2), i32([1, 1, 1]), []
        got.append(stack.step(h, fresh).clone())
        if captured:
            graph, out = ds.decode_graph(stack, h, fresh)
        for i in range(20):
            h.copy_(rows(3, 10 + i))
            if captured:
                graph.replay()
                got.append(out.clone())
            else:
                got.append(stack.step(h, fresh).clone())
        torch.cuda.synchronize()
        assert stack.lens.tolist() == [41, 24, 38] and kd.device_status() == 0
        results.append(torch.stack(got))
    assert torch.equal(*results)


def test_a_pool_that_runs_out_is_counted(kd):
    ds, attn, cfg = make(kd, layers=1, pages=3)
    stack = ds.DecoderStack(kd, torch.device("cuda"), cfg, attn)
    h = stack.step(rows(70, 3), i32([30, 40, 0]), begin=True)
    assert stack.rows_without_place() == 70 - 46 and stack.lens.tolist() == [30, 16, 0] and torch.isfinite(h.float()).all()
    stack.step(rows(0, 4), i32([-1, 0, 0]))
    stack.step(rows(20, 4), i32([0, 0, 20]), begin=True)
    assert stack.rows_without_place() == 0 and stack.lens.tolist() == [0, 16, 20]


def test_heads_that_do_not_fill_a_packed_row_are_refused(kd):
    ds, attn, cfg = make(kd)
    attn.heads, attn.kv_heads = 3, 1
    with pytest.raises(ValueError):
        ds.DecoderStack(kd, torch.device("cuda"), cfg, attn)
