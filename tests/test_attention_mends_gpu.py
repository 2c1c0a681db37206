"""The attention operators where calls meet each other and where inputs are far from ordinary; helpers, bounds and their derivation are
those of test_attention_gpu.py."""
import pytest
import torch

from test_attention_gpu import check_prompt, i32, rows_of

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
