"""Decoder layers on one GPU: the MoE stack of moe_stack.py with the attention sub-layer in front of every block, over a paged
8-bit cache that all layers share the bookkeeping of.

One layer, for the rows of a step (new tokens of all sequences, packed):
    q, k, v = x Wqkv^T                                    (quant_gemm, packed Q4_K)
    k, v -> the layer's cache                              (kv_append, places from the step's kv_plan)
    o = attention                                          (prompt_attention for sequences that begin, kv_attention else)
    h' = Scalar(h + o Wo^T),  x' = rmsnorm(h')             (quant_gemm, residual_rmsnorm)
    the MoE block of moe_stack.py                          (moe_block)

Positions enter where the caller's model wants them to (``KvPlan.first`` has every sequence's); none are added here.
The reference's models run the same order of operators (models/lfm2_5/KokkosDNN_LFM25Model.hpp, models/glimmer/KokkosDNN_GlimmerModel.hpp).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from .moe_stack import MoeStack, StackConfig, random_q4k_payload

Q4_K = 12


@dataclass
class AttentionConfig:
    heads: int = 32
    kv_heads: int = 4
    dim: int = 128
    window: int = 0          # tokens a row looks back on; 0: all
    page: int = 64           # tokens of a cache page
    pages: int = 1024        # pages of the pool, shared by all sequences
    seqs: int = 16           # sequences served at once
    longest: int = 8192      # tokens of a sequence at most


class StepBuffers:
    """Plan, activations and workspaces of steps of up to ``capacity`` rows of one stack. A captured step has a set of its own, which lives
    as long as its graph; all others share the stack's. Steps of one stack must not overlap, whatever sets and streams they use: the
    cache and its bookkeeping are one."""

    def __init__(self, stack: "DecoderStack", capacity: int):
        kd, a, c, dev = stack.kd, stack.attn, stack.cfg, stack.dev
        self.kd, self.cfg, self.seqs, self.attn, self.capacity, self.rows = kd, c, a.seqs, stack.attn_workspace, capacity, -1
        self.stream = torch.cuda.current_stream(dev)

        def rows_of(n, dtype=torch.bfloat16):
            return torch.empty((capacity, n), dtype=dtype, device=dev)
        self.plan = kd.KvPlan.empty(a.seqs, capacity, a.page, dev)
        self.plan.lens, self.plan.state = stack.lens, stack.state     # the pool moves from step to step in place
        self.qkv, self.o, self.x = rows_of(stack.width), rows_of(a.heads * a.dim), rows_of(c.hidden)
        self.y, self.zero = rows_of(c.hidden, torch.float32), torch.zeros((capacity, c.hidden), dtype=torch.float32, device=dev)
        self.gemm = torch.empty(max(kd.quant_gemm_workspace_bytes(capacity, n) for n in (c.hidden, a.heads * a.dim)), dtype=torch.uint8, device=dev)
        self.moe = torch.zeros(self._moe_bytes(capacity), dtype=torch.uint8, device=dev)
        self._moe_rows = capacity

    def _moe_bytes(self, rows: int) -> int:
        c = self.cfg
        return self.kd.moe_block_workspace_bytes(rows, 1, c.top_k, c.hidden, c.ffn, c.experts, True)

    def tensors(self):
        p = self.plan
        return (p.row_start, p.first, p.slots, p.writes, self.qkv, self.o, self.x, self.y, self.zero, self.gemm, self.moe)

    def of(self, rows: int) -> dict:
        """Views of ``rows`` rows."""
        if rows > self.capacity:
            raise ValueError(f"StepBuffers: {rows} rows in buffers of {self.capacity}")
        if rows != self.rows:
            p = self.plan
            plan = p if rows == self.capacity else self.kd.KvPlan(p.row_start, p.first, p.lens, p.state, p.slots[:rows],
                                                                  p.writes[:self.kd.kv_writes(rows, self.seqs, p.page)], p.page)
            moe = self.moe[:self._moe_bytes(rows)]
            if rows != self._moe_rows and rows > 0:      # the counters of the block lie elsewhere for another number of rows, and begin at 0
                moe.zero_()
                self._moe_rows = rows
            self.rows, self._views = rows, dict(plan=plan, qkv=self.qkv[:rows], o=self.o[:rows], x=self.x[:rows], y=self.y[:rows],
                                                zero=self.zero[:rows], gemm=self.gemm, attn=self.attn, moe=moe)
        return self._views


class DecoderStack:
    """``step`` runs one step of all sequences: prompts of those that begin, one or several tokens of those that go on. The
    cache's bookkeeping (lengths, block table, free pages) stays on the device. Steps must not overlap."""

    def __init__(self, kd, device, cfg: StackConfig, attn: AttentionConfig):
        if (attn.heads * attn.dim) % 256:
            raise ValueError("DecoderStack: heads * dim must be a multiple of 256 (Q4_K rows)")
        self.kd, self.dev, self.cfg, self.attn = kd, device, cfg, attn
        self.moe = MoeStack(kd, device, cfg)
        a, c = attn, cfg
        self.width = (a.heads + 2 * a.kv_heads) * a.dim
        self.qkv, self.out, self.caches = [], [], []
        for l in range(c.layers):
            g = torch.Generator(device=device).manual_seed(c.seed + 15485863 * l + 5)
            self.qkv.append(kd.QuantWeight(random_q4k_payload(self.width, c.hidden, g, device), Q4_K, self.width, c.hidden))
            self.out.append(kd.QuantWeight(random_q4k_payload(c.hidden, a.heads * a.dim, g, device), Q4_K, c.hidden, a.heads * a.dim))
            self.caches.append(kd.KvCache.empty(a.pages, a.kv_heads, a.page, a.dim, device))
        i32 = dict(dtype=torch.int32, device=device)
        self.lens = torch.zeros(a.seqs, **i32)
        self.table = torch.full((a.seqs, -(-a.longest // a.page)), -1, **i32)
        self.ring = torch.arange(a.pages, **i32)
        self.state = torch.tensor([0, a.pages, 0, 0], **i32)
        self.prefixes = torch.zeros((), **i32)
        # (the same size for every number of rows)
        self.attn_workspace = torch.empty(kd.kv_attention_workspace_bytes(1, a.seqs, a.heads, a.kv_heads, a.dim), dtype=torch.uint8, device=device)
        self._buffers: Optional[StepBuffers] = None
        self._captured = []
        torch.cuda.current_stream(device).synchronize()       # packed weights are complete before the first call

    def buffers(self, rows: int) -> dict:
        """Plan, workspaces and activations of a step of ``rows`` rows: views of one set, as large as the largest step so far."""
        if torch.cuda.is_current_stream_capturing():          # (a set of its own: another step's counters must not lie in it)
            self._captured.append(StepBuffers(self, rows))
            return self._captured[-1].of(rows)
        stream, own = torch.cuda.current_stream(self.dev), self._buffers
        if own is None or rows > own.capacity:
            # a quarter more than before at least, so that slowly growing steps do not make a new set each
            more = max(rows, own.capacity + own.capacity // 4 if own else 0)
            self._buffers = own = None                        # (the old set goes first)
            self._buffers = own = StepBuffers(self, -(-more // 64) * 64)
        if own.stream != stream:
            for t in own.tensors():
                t.record_stream(stream)
        return own.of(rows)

    def step(self, h: torch.Tensor, fresh: torch.Tensor, begin: bool = False, buffers: Optional[StepBuffers] = None) -> torch.Tensor:
        """The residual stream of the step's rows behind the last layer. ``h`` [rows, hidden], packed in the order of the
        sequences; ``fresh`` int32 [seqs] on the device: rows of each sequence, 0 for one that waits, -1 for one that has ended. Rows
        behind the last sequence meet no attention.
        ``begin``: every sequence with rows begins with them (its prompt), so attention is among the step's rows alone; a sequence that
        holds tokens already would lose them, which ``prefixes_left_out`` counts.
        ``buffers``: a set of the caller's own in place of the stack's."""
        kd, a, c = self.kd, self.attn, self.cfg
        rows = h.shape[0]
        b = self.buffers(rows) if buffers is None else buffers.of(rows)
        plan, qkv = b["plan"], b["qkv"].view(rows, a.heads + 2 * a.kv_heads, a.dim)
        q, k, v = qkv[:, :a.heads], qkv[:, a.heads:a.heads + a.kv_heads], qkv[:, a.heads + a.kv_heads:]
        o = b["o"].view(rows, a.heads, a.dim)
        kd.kv_plan(fresh, self.lens, self.table, self.ring, self.state, plan)
        if begin:
            torch.sum((plan.first > 0) & (fresh > 0), 0, dtype=torch.int32, out=self.prefixes)
        x = torch.empty_like(h)
        kd.residual_rmsnorm(h, b["zero"], x)
        b["o"].zero_()      # rows behind the last sequence: attention leaves them as they are, in every layer
        for l in range(c.layers):
            kd.quant_gemm(x, self.qkv[l], b["qkv"], b["gemm"])
            kd.kv_append(k, v, plan, self.caches[l])
            if begin:
                kd.prompt_attention(q, k, v, plan.row_start, o, window=a.window)
            else:
                kd.kv_attention(q, plan, self.table, self.caches[l], o, b["attn"], window=a.window)
            kd.quant_gemm(b["o"], self.out[l], b["y"], b["gemm"])
            kd.residual_rmsnorm(h, b["y"], b["x"])
            h = (h.float() + b["y"]).to(h.dtype)
            gate, up, down = self.moe.layers[l]
            h2, x2 = torch.empty_like(h), torch.empty_like(h)
            kd.moe_block(b["x"], self.moe.routers[l], None, c.top_k, True, 1.0, gate, up, down, b["moe"], resid=h, h_out=h2, xn_out=x2)
            h, x = h2, x2
        return h

    def rows_without_place(self) -> int:
        """Rows of the last step that found no page (synchronises)."""
        return int(self.state[2])

    def prefixes_left_out(self) -> int:
        """Sequences that did not begin with the last ``begin`` step's rows, whose earlier tokens those rows have not met (synchronises)."""
        return int(self.prefixes)


def decode_graph(stack: DecoderStack, h: torch.Tensor, fresh: torch.Tensor, stream: Optional[torch.cuda.Stream] = None):
    """(graph, result): one decode step captured; replay it after writing the next rows into ``h``. The stack must have run a step
    before (kernels are set up by it). The graph has buffers of its own, which it keeps alive."""
    stream = stream or torch.cuda.Stream()
    buffers = StepBuffers(stack, h.shape[0])
    torch.cuda.synchronize(h.device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = stack.step(h, fresh, buffers=buffers)
    graph.buffers, graph.inputs = buffers, (stack, h, fresh)
    return graph, out
