"""Engine-side caller of the hot path: the attention prologue of a Qwen3
decoder layer, as an inference engine runs it around these operators.

Per layer (reference project, README.md:11-12, where the same two operators
are called from a decode engine's Qwen3 layer):

1. ``fused_add_rms_norm_inplace(hidden, residual, input_norm_weight)`` --
   residual += hidden; hidden = RMSNorm(residual) (in place);
2. ``qkv = hidden @ qkv_weight.T`` -- the QKV projection, a plain library
   GEMM (cuBLAS through PyTorch) into a preallocated buffer;
3. ``qk_norm_rope_cache_`` on strided Q / K / V views of ``qkv`` -- per-head
   Q/K RMSNorm + RoPE in place and the paged KV store, with no gather copies
   (the reference's kernel needs contiguous Q / K, so an engine built on it
   copies them out first).

With ``fused_projection=True`` steps 2 and 3 are one kernel: the QKV
projection on the tensor cores with the Q/K norm + RoPE + KV store in its
epilogue (``extensions.qkv_proj_norm_rope_cache_``; bf16, head_dim 128, dense
NHD caches), bit-identical to that kernel's plain GEMM followed by step 3.

:class:`PagedSteps` keeps the block tables of a batch and plans its steps on the
GPU, and :class:`Qwen3Attention` runs a layer's whole attention on such a plan:
the prologue, then the attention of whole prompts or of one token per request
over the paged cache.

:class:`DecodeGraph` captures the prologues of all layers of one decode step
into a single CUDA graph, so the host launches one graph per step; the B200
kernels additionally overlap each launch with the tail of the previous kernel
(programmatic dependent launch).
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import extensions, ops, serving


@dataclass(frozen=True)
class Qwen3AttentionShape:
    hidden: int = 4096
    query_heads: int = 32
    key_heads: int = 8
    head_dim: int = 128
    rope_theta: float = 1e6
    max_positions: int = 32768
    epsilon: float = 1e-6
    # pairs of a head that turn by time, height and width (positions [3, tokens])
    rope_sections: tuple[int, ...] = (16, 24, 24)
    rope_sections_interleaved: bool = False

    @property
    def qkv_width(self) -> int:
        return (self.query_heads + 2 * self.key_heads) * self.head_dim


def rope_cos_sin_cache(shape: Qwen3AttentionShape, device, rotary_dim: int | None = None):
    """fp32 [max_positions, rotary_dim]: cos | sin of position * theta^(-2i/d)."""
    rotary_dim = rotary_dim or shape.head_dim
    inv = 1.0 / (shape.rope_theta ** (torch.arange(0, rotary_dim, 2, dtype=torch.float32,
                                                    device=device) / rotary_dim))
    f = torch.outer(torch.arange(shape.max_positions, dtype=torch.float32, device=device), inv)
    return torch.cat((f.cos(), f.sin()), dim=-1)


class Qwen3AttentionPrologue:
    """Weights and the per-layer call. ``forward`` returns the (strided) Q, K
    and V views into the layer's QKV buffer; K and V are also in the cache."""

    def __init__(self, shape: Qwen3AttentionShape, device, dtype=torch.bfloat16,
                 generator: torch.Generator | None = None):
        self.shape = shape
        g = generator
        std = 1.0 / math.sqrt(shape.hidden)
        self.input_norm_weight = (1 + 0.1 * torch.randn(shape.hidden, device=device,
                                                        generator=g)).to(dtype)
        self.qkv_weight = (std * torch.randn(shape.qkv_width, shape.hidden, device=device,
                                             generator=g)).to(dtype)
        self.query_norm_weight = (1 + 0.1 * torch.randn(shape.head_dim, device=device,
                                                        generator=g)).to(dtype)
        self.key_norm_weight = (1 + 0.1 * torch.randn(shape.head_dim, device=device,
                                                      generator=g)).to(dtype)

    def split(self, qkv: torch.Tensor):
        s = self.shape
        t = qkv.shape[0]
        q_end = s.query_heads * s.head_dim
        k_end = q_end + s.key_heads * s.head_dim
        return (qkv[:, :q_end].view(t, s.query_heads, s.head_dim),
                qkv[:, q_end:k_end].view(t, s.key_heads, s.head_dim),
                qkv[:, k_end:].view(t, s.key_heads, s.head_dim))

    def forward(self, hidden: torch.Tensor, residual: torch.Tensor, positions: torch.Tensor,
                cos_sin_cache: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                slot_mapping: torch.Tensor, qkv_out: torch.Tensor, k_scale=None, v_scale=None,
                kv_cache_layout: str = "NHD", fused_projection: bool = False):
        s = self.shape
        ops.fused_add_rms_norm_inplace(hidden, residual, self.input_norm_weight, s.epsilon)
        if fused_projection:
            extensions.qkv_proj_norm_rope_cache_(
                hidden, self.qkv_weight, qkv_out, s.query_heads, s.key_heads,
                self.query_norm_weight, self.key_norm_weight, positions, cos_sin_cache,
                key_cache, value_cache, slot_mapping, s.epsilon)
            return self.split(qkv_out)
        torch.matmul(hidden, self.qkv_weight.t(), out=qkv_out)
        q, k, v = self.split(qkv_out)
        if positions.dim() == 2:  # [axes, tokens]: time, height, width
            extensions.qk_norm_mrope_cache_(
                q, k, v, self.query_norm_weight, self.key_norm_weight, positions, cos_sin_cache,
                list(s.rope_sections), key_cache, value_cache, slot_mapping, k_scale, v_scale, True,
                s.rope_sections_interleaved, kv_cache_layout, s.epsilon)
            return q, k, v
        extensions.qk_norm_rope_cache_(
            q, k, v, self.query_norm_weight, self.key_norm_weight, positions, cos_sin_cache,
            key_cache, value_cache, slot_mapping, k_scale, v_scale, True, kv_cache_layout,
            s.epsilon)
        return q, k, v


class PagedSteps:
    """Block tables and step plans of up to ``requests`` requests over a cache of
    ``num_blocks`` blocks, all on the GPU: no length has to come back to the host.

    ``context_lens`` is what the cache holds for each request and follows every
    :meth:`plan`; ``query_start``, ``positions`` and ``slot_mapping`` are those of the
    step planned last, packed request after request. ``row_positions``, ``row_slots``
    and ``row_lens`` are the same step as decode runs it, entry r for request r:
    its first token's position and slot and its length with the step, or a position
    and a slot below zero and 0 for a request without a token or without room for it
    (:attr:`unserved`).

    ``prefix_blocks`` blocks, taken off the pool here, are the first of every
    request's row, and every request begins behind them: its ``context_lens``
    starts at their tokens and returns there. :meth:`prefix_writer` plans the
    prompt that fills them. Requests that do not share the prefix stand in a
    second ``PagedSteps`` over the same blocks: ``pool`` is then the first one.
    """

    def __init__(self, requests: int, num_blocks: int, max_blocks: int, max_tokens: int, device,
                 block_size: int = 16, prefix_blocks: int = 0, pool: PagedSteps | None = None):
        def ints(*shape, dtype=torch.int32):
            return torch.zeros(*shape, device=device, dtype=dtype)

        if not 0 <= prefix_blocks <= min(num_blocks, max_blocks):
            raise ValueError("prefix_blocks must be in [0, num_blocks] and fit a row of max_blocks")
        if pool is not None and (prefix_blocks or pool.free_blocks.numel() != num_blocks
                                 or pool.block_size != block_size):
            raise ValueError("a batch over another one's pool has its num_blocks and block_size, "
                             "and no prefix_blocks of its own")
        self.block_size = block_size
        if pool is None:
            self.free_blocks = torch.arange(num_blocks - 1, -1, -1, device=device, dtype=torch.int32)
            self.free_count = torch.full((1,), num_blocks - prefix_blocks, device=device,
                                         dtype=torch.int32)
        else:
            self.free_blocks, self.free_count = pool.free_blocks, pool.free_count
        # the top of the stack, block 0 first
        self.prefix = self.free_blocks[num_blocks - prefix_blocks:].flip(0).clone()
        self.block_table = torch.full((requests, max_blocks), -1, device=device, dtype=torch.int32)
        self.block_table[:, :prefix_blocks] = self.prefix
        self.context_lens = ints(requests).fill_(prefix_blocks * block_size)
        self.query_start = ints(requests + 1)
        self.positions = ints(max_tokens, dtype=torch.int64)
        self.slot_mapping = ints(max_tokens)
        self.row_positions = ints(requests, dtype=torch.int64)
        self.row_slots = ints(requests)
        self.row_lens = ints(requests)

    def prefix_writer(self) -> PagedSteps:
        """A batch of one request whose blocks are those of the prefix: plan it with
        as many tokens as they hold and run :meth:`Qwen3Attention.prompts` on it in
        every layer, before the first request is decoded."""
        blocks = self.prefix.numel()
        writer = PagedSteps(1, self.free_blocks.numel(), blocks, blocks * self.block_size,
                            self.free_blocks.device, self.block_size)
        writer.free_blocks[:blocks] = self.prefix.flip(0)
        writer.free_count.fill_(blocks)
        return writer

    def plan(self, query_lens: torch.Tensor) -> None:
        """The next step, with ``query_lens`` (int32 [requests]) new tokens."""
        serving.plan_step_(self.context_lens, query_lens, self.block_table, self.free_blocks,
                           self.free_count, self.block_size, self.query_start, self.context_lens,
                           self.positions, self.slot_mapping, None, self.row_positions,
                           self.row_slots, self.row_lens)

    @property
    def unserved(self) -> torch.Tensor:
        """Requests (bool [requests], on the GPU) that had tokens in the step planned
        last and got no place for them: their lengths are as before the step."""
        return self.row_slots == -2

    def release(self, finished: torch.Tensor) -> None:
        """Gives the blocks of the requests in ``finished`` (bool [requests]) back,
        all but the shared ones, and sets their lengths to those of the prefix."""
        serving.release_blocks_(self.context_lens, finished, self.block_table, self.free_blocks,
                                self.free_count, self.block_size, self.prefix.numel())
        self.context_lens.masked_fill_(finished, self.prefix.numel() * self.block_size)


class Qwen3Attention:
    """A layer's attention on a planned step: prologue, K and V into the paged
    cache, attention. Returns [tokens, query_heads, head_dim], the input of the
    output projection. ``positions`` default to the plan's; [3, tokens] for
    images and video, packed for prompts and one column per request for decode."""

    def __init__(self, prologue: Qwen3AttentionPrologue, key_cache: torch.Tensor,
                 value_cache: torch.Tensor, cos_sin_cache: torch.Tensor, k_scale=None,
                 v_scale=None, kv_cache_layout: str = "NHD"):
        self.prologue = prologue
        self.key_cache, self.value_cache = key_cache, value_cache
        self.cos_sin_cache = cos_sin_cache
        self.k_scale, self.v_scale = k_scale, v_scale
        self.kv_cache_layout = kv_cache_layout

    def _queries(self, hidden, residual, positions, slots, qkv):
        if qkv is None:
            qkv = torch.empty(hidden.shape[0], self.prologue.shape.qkv_width,
                              device=hidden.device, dtype=hidden.dtype)
        return self.prologue.forward(hidden, residual, positions, self.cos_sin_cache,
                                     self.key_cache, self.value_cache, slots, qkv, self.k_scale,
                                     self.v_scale, self.kv_cache_layout)

    def prompts(self, hidden: torch.Tensor, residual: torch.Tensor, steps: PagedSteps,
                positions: torch.Tensor | None = None, qkv: torch.Tensor | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
        """Whole prompts, packed as ``steps`` planned them from empty contexts: their
        tokens see one another and nothing in the cache. So a batch with a prefix
        has none; its prompts go through :meth:`decode`, a token a step."""
        if steps.prefix.numel():
            raise ValueError("prompts behind a shared prefix do not see it: decode their tokens")
        tokens = hidden.shape[0]
        positions = steps.positions[:tokens] if positions is None else positions
        q, k, v = self._queries(hidden, residual, positions, steps.slot_mapping[:tokens], qkv)
        out = torch.zeros(q.shape, device=q.device, dtype=q.dtype) if out is None else out
        serving.prompt_attention(out, q, k, v, steps.query_start)
        return out

    def decode(self, hidden: torch.Tensor, residual: torch.Tensor, steps: PagedSteps,
               positions: torch.Tensor | None = None, qkv: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """At most one token for every request, as ``steps`` planned them; row r is
        request r's. Requests without a token, and those without room for it
        (``steps.unserved``), store nothing, and their rows come out as zeros."""
        if hidden.shape[0] != steps.row_lens.numel():
            raise ValueError(f"decode takes one row per request ({steps.row_lens.numel()}), with or "
                             f"without a token (got {hidden.shape[0]})")
        positions = steps.row_positions if positions is None else positions
        q, _, _ = self._queries(hidden, residual, positions, steps.row_slots, qkv)
        out = torch.empty(q.shape, device=q.device, dtype=q.dtype) if out is None else out
        serving.paged_decode_attention(out, q, self.key_cache, self.value_cache,
                                       steps.block_table, steps.row_lens, steps.prefix,
                                       self.k_scale, self.v_scale, self.kv_cache_layout)
        return out


class DecodeGraph:
    """The prologues of ``layers`` decoder layers for one decode batch,
    captured once as a CUDA graph over static buffers. Between layers the
    hidden state for the next layer is the previous QKV buffer's first
    ``hidden`` columns (a stand-in for attention + output projection + MLP,
    which are not part of this path), so every layer reads fresh data.

    Fill ``hidden``, ``residual``, ``positions`` and ``slot_mapping`` in
    place, then ``replay()``. ``fused_projection`` None picks the fused
    projection where it measured faster (:meth:`fused_projection_pays`).
    """

    def __init__(self, layers: list[Qwen3AttentionPrologue], batch: int, cos_sin_cache,
                 key_caches: list[torch.Tensor], value_caches: list[torch.Tensor],
                 k_scale=None, v_scale=None, kv_cache_layout: str = "NHD",
                 fused_projection: bool | None = None):
        shape = layers[0].shape
        if shape.qkv_width < shape.hidden:
            raise ValueError("the stand-in between layers needs qkv_width >= hidden")
        dev = cos_sin_cache.device
        dtype = layers[0].qkv_weight.dtype
        if fused_projection is None:
            fused_projection = self.fused_projection_pays(batch, shape, dtype, key_caches,
                                                          k_scale, kv_cache_layout)
        self.fused_projection = fused_projection
        self.layers = layers
        self.hidden = torch.zeros(batch, shape.hidden, device=dev, dtype=dtype)
        self.residual = torch.zeros_like(self.hidden)
        self.positions = torch.zeros(batch, device=dev, dtype=torch.int64)
        self.slot_mapping = torch.full((batch,), -1, device=dev, dtype=torch.int32)
        self.qkv = [torch.empty(batch, shape.qkv_width, device=dev, dtype=dtype) for _ in layers]
        self.layer_hidden = [torch.empty_like(self.hidden) for _ in layers[1:]]
        self._args = (cos_sin_cache, key_caches, value_caches, k_scale, v_scale, kv_cache_layout,
                      fused_projection)
        self._run()  # load kernels and pick cuBLAS algorithms before capture
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self._run()

    @staticmethod
    def fused_projection_pays(batch, shape, dtype, key_caches, k_scale, kv_cache_layout) -> bool:
        """Whether the projection with the fused Q/K epilogue is the faster
        choice: up to four tokens, where it streams the weights on the CUDA
        cores (a Qwen3-8B-shaped batch-1 step: 139.9 us against 166.8 us for
        cuBLAS followed by the Q/K kernel), and only where it applies (bf16,
        head_dim 128, dense bf16 NHD caches). From 16 tokens up cuBLAS followed
        by the Q/K kernel measured faster."""
        return (batch <= 4 and dtype == torch.bfloat16 and shape.head_dim == 128
                and kv_cache_layout == "NHD" and k_scale is None
                and all(c.dtype == torch.bfloat16 and c.is_contiguous() for c in key_caches))

    def _run(self):
        cos_sin, key_caches, value_caches, k_scale, v_scale, layout, fused = self._args
        hidden = self.hidden
        for i, layer in enumerate(self.layers):
            layer.forward(hidden, self.residual, self.positions, cos_sin, key_caches[i],
                          value_caches[i], self.slot_mapping, self.qkv[i], k_scale, v_scale,
                          layout, fused)
            if i + 1 < len(self.layers):
                nxt = self.layer_hidden[i]
                nxt.copy_(self.qkv[i][:, :layer.shape.hidden])
                hidden = nxt

    def replay(self):
        self.graph.replay()
