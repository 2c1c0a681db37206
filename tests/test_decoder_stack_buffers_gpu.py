"""The decoder stack's buffers (dnn-for-kokkos_b200/decoder_stack.py) over steps of many sizes, eager and captured."""
import random

import pytest
import torch

from test_attention_gpu import i32
from test_decoder_stack_gpu import make, rows

pytestmark = pytest.mark.gpu


def new_stack(kd, pages=400):
    ds, attn, cfg = make(kd, pages=pages)
    attn.longest = 2048
    return ds, ds.DecoderStack(kd, torch.device("cuda"), cfg, attn)


def test_memory_is_that_of_the_largest_step(kd):
    """Ragged prompts: a new number of rows in every step."""
    ds, stack = new_stack(kd)
    rng = random.Random(1)
    sizes = list(range(20, 600, 13))
    rng.shuffle(sizes)

    def run(n):
        stack.step(rows(n, n), i32([n, 0, 0]), begin=True)
        stack.step(rows(0, 0), i32([-1, 0, 0]))
        torch.cuda.synchronize()
        return torch.cuda.memory_allocated()

    run(max(sizes))
    after = run(max(sizes))
    assert max(run(n) for n in sizes) <= after + 2 ** 20
    assert kd.device_status() == 0


def test_results_do_not_depend_on_the_sizes_of_other_steps(kd):
    """The same steps with and without steps of other sizes, which add no token, between them."""
    results = []
    for between in ((), (9, 64), (130, 1, 500)):
        ds, stack = new_stack(kd)
        got = []
        for i, (fresh, begin) in enumerate((([33, 5, 0], True), ([1, 1, 0], False), ([0, 4, 20], False), ([1, -1, 1], False), ([1, 0, 1], False))):
            n = sum(max(f, 0) for f in fresh)
            got.append(stack.step(rows(n, 100 + i), i32(fresh), begin=begin).clone())
            for m in between:
                stack.step(rows(m, m), i32([0, 0, 0]))
        torch.cuda.synchronize()
        assert stack.lens.tolist() == [36, 0, 22] and kd.device_status() == 0
        results.append(torch.cat(got))
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2])


def test_a_graph_and_eager_steps_of_other_sizes(kd):
    """A captured decode step replayed between eager steps that make the stack's own buffers anew."""
    results = []
    for captured in (False, True):
        ds, stack = new_stack(kd)
        stack.step(rows(40, 1), i32([20, 3, 17]), begin=True)
        h, fresh, got = rows(3, 2), i32([1, 1, 1]), []
        if captured:
            graph, out = ds.decode_graph(stack, h, fresh)
        for i in range(6):
            h.copy_(rows(3, 10 + i))
            if captured:
                graph.replay()
                got.append(out.clone())
            else:
                got.append(stack.step(h, fresh).clone())
            more = [2, 70 * i, 1] if i % 2 else [0, 0, 40]
            got.append(stack.step(rows(sum(more), 50 + i), i32(more)).clone())
            if captured:       # memory that was let go of is used by others
                trash = [torch.full((2 ** 18,), float("nan"), device="cuda") for _ in range(20)]
                del trash
        torch.cuda.synchronize()
        assert kd.device_status() == 0 and stack.rows_without_place() == 0
        results.append(torch.cat(got))
    assert torch.equal(*results)


def test_steps_on_streams_in_turn(kd):
    """Steps that follow one another on different streams, with buffers made anew on the way."""
    results = []
    for streams in (None, [torch.cuda.Stream() for _ in range(3)]):
        ds, stack = new_stack(kd)
        got = []
        torch.cuda.synchronize()
        for i, n in enumerate((5, 80, 3, 200, 7, 700, 1)):
            h, fresh = rows(n, n), i32([n, 0, 0])
            torch.cuda.synchronize()
            with torch.cuda.stream(streams[i % 3] if streams else torch.cuda.current_stream()):
                got.append(stack.step(h, fresh).clone())
                done = torch.cuda.Event()
                done.record()
            if streams:
                streams[(i + 1) % 3].wait_event(done)
        torch.cuda.synchronize()
        results.append(torch.cat(got))
    assert torch.equal(*results) and kd.device_status() == 0


def test_a_step_captured_by_hand(kd):
    ds, stack = new_stack(kd)
    other_ds, other = new_stack(kd)
    for s in (stack, other):
        s.step(rows(40, 1), i32([20, 3, 17]), begin=True)
    h, fresh = rows(3, 2), i32([1, 1, 1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        out = stack.step(h, fresh)
    for i in range(4):
        h.copy_(rows(3, i))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, other.step(h, fresh))
        assert torch.equal(stack.step(rows(9, i), i32([4, 0, 5])), other.step(rows(9, i), i32([4, 0, 5])))
    assert kd.device_status() == 0


def test_rows_behind_the_last_sequence_are_not_what_lay_in_memory(kd):
    """A step with more rows than its sequences have: the rest of the rows meet an attention of 0, whatever steps came before."""
    results = []
    for before in (None, float("nan"), 1e30):
        ds, stack = new_stack(kd)
        stack.step(rows(40, 1), i32([20, 3, 17]), begin=True)
        if before is not None:
            for t in stack._buffers.tensors() if hasattr(stack._buffers, "tensors") else ():
                if t.dtype == torch.bfloat16:
                    t.fill_(before)
        a = stack.step(rows(12, 5), i32([1, 0, 2]))
        b = stack.step(rows(30, 6), i32([-1, 0, 0]))
        c = stack.step(rows(50, 7), i32([33, 0, 0]), begin=True)
        results.append(torch.cat([a, b, c]))
        assert torch.isfinite(results[-1].float()).all()
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2]) and kd.device_status() == 0


def test_a_beginning_step_counts_the_sequences_that_do_not_begin(kd):
    ds, stack = new_stack(kd)
    stack.step(rows(40, 1), i32([20, 3, 17]), begin=True)
    assert stack.prefixes_left_out() == 0
    stack.step(rows(9, 2), i32([4, 0, 5]))
    assert stack.prefixes_left_out() == 0                   # (attended to over the cache)
    stack.step(rows(9, 3), i32([4, -1, 5]), begin=True)
    assert stack.prefixes_left_out() == 2
    stack.step(rows(7, 4), i32([0, 7, 0]), begin=True)
    assert stack.prefixes_left_out() == 0
