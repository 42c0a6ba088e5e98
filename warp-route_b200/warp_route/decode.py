"""Decode-step driver: a stack of MoE layers replayed from one CUDA graph.

warp-route runs one layer per Python call and synchronises the device after
each (src/bindings.cpp:55,94,140); its README motivates the kernels with
decode-step latency (README.md:17).  `MoEStack` captures the whole stack of
layer calls for a fixed token count once and replays it every step:

    h_0 = x;   h_{l+1} = (h_l + moe_l(h_l)).to(dtype)   (residual, fp32 add, one rounding)

Each layer is ONE kernel launch chain of this package: `moe_decode_layer`
writes both the fp32 sum and the next layer's input from the layer's last
step (the streaming kernel for a token, the grouped tcgen05 path for a
batch), so consecutive layers follow each other with programmatic dependent
launch and no element-wise kernels in between.  Tensor- or expert-parallel
shards pass `comm` (a `PeerComm`): the ranks' partial outputs are summed in
the same kernel before the residual.  An external collective (`all_reduce`,
e.g. torch.distributed.all_reduce on NCCL, captured into the same graph)
still works; the residual is then added after it, as two extra kernels.
Inputs and outputs live in static device buffers; `step(x)` copies x in,
replays, and returns the output buffer.

A layer may carry an attention block (`StackAttention`) before its MoE layer:

    h'_l = (h_l + attn_l(h_l) Wo_l^T).to(dtype);   h_{l+1} = (h'_l + moe_l(h'_l)).to(dtype)

Its keys and values enter a paged cache (`append_paged_kv`, rotated by their
positions), and `shared_prefix_attention` reads that cache.  Where the tokens
of a step go and what they see stands in one `StackContext` for all layers,
static device buffers too, written between steps.  `sample` turns the stack's
output into tokens (`sample_tokens` on the logits of an output head).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Callable, List, Optional

import torch

from .functional import (PeerComm, append_paged_kv, fused_moe_routed, moe_decode_layer,
                         sample_tokens, shared_prefix_attention)


@dataclass
class StackAttention:
    """One layer's attention: wqkv [(num_heads + 2 num_kv_heads) head_dim, H]
    (rows of q, then k, then v), wo [H, num_heads head_dim], its caches
    [num_pages, num_kv_heads, page_size, head_dim], and the frequencies
    inv_freq (float32 [rot_dim / 2], None: no rotation).  With a stack's
    `comm` or `all_reduce` only the MoE layers are sharded: every rank
    computes the whole attention and holds the whole caches."""
    wqkv: torch.Tensor
    wo: torch.Tensor
    num_heads: int
    num_kv_heads: int
    k_cache: torch.Tensor
    v_cache: torch.Tensor
    inv_freq: Optional[torch.Tensor] = None
    interleaved: bool = False
    scale: Optional[float] = None


@dataclass
class StackContext:
    """Where a step's tokens go in the caches and what they see: slots and
    positions int64 [T], context_lens int32 [T] (own keys, this step's token
    among them), block_tables int32 [T, pages]; prefix_pages int32 of the
    prefix_len tokens that all sequences share.  The tensors are read when a
    step runs: write them in place between steps.  prefix_len is a number and
    part of the captured step: a `step` with another one, or with another
    tensor in a field's place, is refused until `close` has released the graph
    (the next step captures anew).  A slot of -1 (and a length of 0) is a
    sequence that does not take part."""
    slots: torch.Tensor
    positions: torch.Tensor
    context_lens: torch.Tensor
    block_tables: torch.Tensor
    prefix_pages: Optional[torch.Tensor] = None
    prefix_len: int = 0

    @staticmethod
    def empty(tokens: int, pages: int, device, prefix_pages: Optional[torch.Tensor] = None,
              prefix_len: int = 0) -> "StackContext":
        """Buffers of a stack in which no sequence takes part yet."""
        return StackContext(
            torch.full((tokens,), -1, dtype=torch.int64, device=device),
            torch.zeros(tokens, dtype=torch.int64, device=device),
            torch.zeros(tokens, dtype=torch.int32, device=device),
            torch.zeros(tokens, pages, dtype=torch.int32, device=device), prefix_pages, prefix_len)


@dataclass
class StackLayer:
    """One layer's (shard of) weights: gate_w [E, H], the packed weight_buf,
    an optional fp32 router bias [E], the expert-parallel shard, and an
    optional attention block in front of it."""
    gate_w: torch.Tensor
    weight_buf: torch.Tensor
    router_bias: Optional[torch.Tensor] = None
    ep_first_expert: int = 0
    ep_num_local: int = 0
    attention: Optional[StackAttention] = None


class MoEStack:
    def __init__(self, layers: List[StackLayer], num_experts: int, hidden_dim: int,
                 intermediate_dim: int, top_k: int, tokens: int,
                 all_reduce: Optional[Callable[[torch.Tensor], None]] = None,
                 comm: Optional[PeerComm] = None, context: Optional[StackContext] = None,
                 head: Optional[torch.Tensor] = None):
        if not layers:
            raise ValueError("MoEStack needs at least one layer")
        if all_reduce is not None and comm is not None:
            raise ValueError("pass either comm (fused sum) or all_reduce (external), not both")
        if context is None and any(L.attention is not None for L in layers):
            raise ValueError("layers with attention need a context")
        if context is not None and context.slots.shape[0] != tokens:
            raise ValueError(f"context is for {context.slots.shape[0]} tokens, the stack for {tokens}")
        self.layers = layers
        self.E, self.H, self.I, self.K = num_experts, hidden_dim, intermediate_dim, top_k
        self.T = tokens
        self.all_reduce = all_reduce
        self.comm = comm
        self.context = context
        self.head = head
        dev = layers[0].gate_w.device
        self.dtype = layers[0].gate_w.dtype
        shape = (hidden_dim,) if tokens == 1 else (tokens, hidden_dim)
        self.x_in = torch.zeros(shape, dtype=self.dtype, device=dev)
        self.h = [torch.zeros(shape, dtype=self.dtype, device=dev) for _ in range(2)]
        self.stream = torch.cuda.Stream(device=dev)
        self.graph: Optional[torch.cuda.CUDAGraph] = None
        self.captured: tuple = ()

    def _fixed(self) -> tuple:
        """What a captured step has by reference or by value besides weights:
        the context's fields and the caches."""
        c = self.context
        if c is None:
            return ()
        caches = [t for L in self.layers if L.attention is not None
                  for t in (L.attention.k_cache, L.attention.v_cache)]
        return (c.prefix_len, c.slots, c.positions, c.context_lens, c.block_tables, c.prefix_pages,
                *caches)

    def layer(self, i: int, h: torch.Tensor, nxt: torch.Tensor) -> torch.Tensor:
        """Layer i on input h: writes the next input into nxt and returns the
        layer's fp32 output (residual included)."""
        L = self.layers[i]
        if self.all_reduce is None:
            return moe_decode_layer(h, L.gate_w, L.weight_buf, self.E, self.H, self.I, self.K,
                                    next_x=nxt, comm=self.comm, router_bias=L.router_bias,
                                    ep_first_expert=L.ep_first_expert,
                                    ep_num_local=L.ep_num_local)
        out, _, _ = fused_moe_routed(h, L.gate_w, L.weight_buf, self.E, self.H, self.I, self.K,
                                     router_bias=L.router_bias,
                                     ep_first_expert=L.ep_first_expert,
                                     ep_num_local=L.ep_num_local)
        self.all_reduce(out)
        torch.add(h.float(), out, out=out)
        nxt.copy_(out)
        return out

    def attention(self, i: int, h: torch.Tensor) -> torch.Tensor:
        """Layer i's attention on input h with the residual: the input of its
        MoE layer (a new tensor)."""
        A, c = self.layers[i].attention, self.context
        d = A.k_cache.shape[3]
        rows = h.view(self.T, self.H)
        heads = torch.nn.functional.linear(rows, A.wqkv).view(self.T, -1, d)
        q, k, v = heads.split([A.num_heads, A.num_kv_heads, A.num_kv_heads], 1)
        q = append_paged_kv(k, v, A.k_cache, A.v_cache, c.slots,
                            positions=None if A.inv_freq is None else c.positions,
                            inv_freq=A.inv_freq, q=q, interleaved=A.interleaved)
        seen = shared_prefix_attention(q, A.k_cache, A.v_cache, c.block_tables, c.context_lens,
                                       prefix_pages=c.prefix_pages, prefix_len=c.prefix_len,
                                       scale=A.scale)
        out = torch.nn.functional.linear(seen.view(self.T, -1), A.wo)
        return (rows.float() + out.float()).to(self.dtype).view(h.shape)

    def _forward(self) -> torch.Tensor:
        h = self.x_in
        for i in range(len(self.layers)):
            nxt = self.h[i & 1]
            if self.layers[i].attention is not None:
                h = self.attention(i, h)
            self.layer(i, h, nxt)
            h = nxt
        return h

    def eager(self, x: torch.Tensor) -> torch.Tensor:
        """The same stack without a graph (for checking and for the first call)."""
        self.x_in.copy_(x)
        return self._forward().clone()

    def capture(self, warmup: int = 2) -> None:
        """Capture the stack into a CUDA graph (warm-up calls run first, on the
        capture stream, so the per-stream workspaces exist before capture).
        The caches stay as they are: the warm-up calls write no slot."""
        slots = None if self.context is None else self.context.slots
        kept = None if slots is None else slots.clone()
        # the capture stream's warm-up writes the same static buffers as any
        # call already queued on the caller's stream: run it after them
        self.stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(self.stream):
            try:
                if slots is not None:
                    slots.fill_(-1)
                for _ in range(warmup):
                    self._forward()
            finally:
                if slots is not None:
                    slots.copy_(kept)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=self.stream):
            self.out = self._forward()
        self.captured = self._fixed()  # and keeps the tensors for as long as the graph reads them
        self.graph = g

    def step(self, x: torch.Tensor) -> torch.Tensor:
        """One decode step: x -> the stack's output (a static buffer that the
        next step overwrites)."""
        if self.graph is None:
            self.capture()
        now, then = self._fixed(), self.captured
        if now[:1] != then[:1] or any(a is not b for a, b in zip(now[1:], then[1:])):
            raise ValueError("prefix_len, the context's tensors and the caches are part of the captured "
                             "step: write the tensors in place, or close() the stack before a change")
        self.x_in.copy_(x)
        self.graph.replay()
        return self.out

    def sample(self, out: torch.Tensor, uniforms: torch.Tensor, **settings) -> torch.Tensor:
        """Tokens (int64 [T]) from the stack's output: logits out head^T in the
        stack's dtype, then `sample_tokens` with its settings (temperature,
        top_k, top_p, min_p)."""
        if self.head is None:
            raise ValueError("sample needs the stack's output head")
        logits = torch.nn.functional.linear(out.view(self.T, self.H), self.head)
        return sample_tokens(logits, uniforms, **settings)

    def close(self) -> None:
        """Release the graph (before destroying a process group it captured
        collectives of)."""
        self.graph = None
        self.captured = ()
