"""Operators of a serving step around the paged KV cache.

The order in which a step uses them, with the operators there were before:

1. :func:`plan_step_` -- block tables, positions and slot maps from request
   lengths, on the GPU (:func:`release_blocks_` when requests finish);
2. ``extensions.qk_norm_rope_cache_`` or, for positions with several axes,
   ``extensions.qk_norm_mrope_cache_`` -- Q/K norm + rotation, and K and V into
   the cache at ``slot_mapping``;
3. :func:`prompt_attention` for the tokens of whole prompts,
   :func:`paged_decode_attention` for one new token per request.

All are stream-ordered, never synchronise, and can be captured in a CUDA
graph; registered as ``torch.ops.sm120_norm_ext.*``. They run forward only:
none has a gradient. Outputs may not share memory with inputs, but for what is said
to be in place. No fallback when the extension is missing.

The attention kernels bound every wait of theirs. One that runs out (never in
correct operation) is counted in ``serving_capi.device_faults()``; decode rows that
it had a part of are NaN, prompt rows that were not finished are left as they were.
"""
from __future__ import annotations

import functools

import torch

from .ops import _C, _extension


@functools.cache
def _dispatched(name: str):
    return getattr(torch.ops.sm120_norm_ext, name).default


_compiling = torch.compiler.is_compiling


def _call(name: str, *args) -> None:
    """The operator: the extension's function where nothing could look on (small
    steps are bound by the host, and the dispatcher costs as much again), the
    registered operator for tracing, modes, function transforms and tensor
    subclasses among the arguments."""
    extension = _extension()
    if not _compiling() and extension.nothing_looks_on(*args):
        getattr(extension, name)(*args)
    else:
        _dispatched(name)(*args)


def plan_step_(
    context_lens: torch.Tensor,
    query_lens: torch.Tensor,
    block_table: torch.Tensor,
    free_blocks: torch.Tensor,
    free_count: torch.Tensor,
    block_size: int,
    query_start: torch.Tensor,
    seq_lens: torch.Tensor,
    positions: torch.Tensor,
    slot_mapping: torch.Tensor,
    free_count_out: torch.Tensor | None = None,
    row_positions: torch.Tensor | None = None,
    row_slots: torch.Tensor | None = None,
    row_lens: torch.Tensor | None = None,
) -> None:
    """Block tables, positions and slots of the next step, in one launch.

    ``context_lens`` / ``query_lens`` (int32 [R]): tokens of each request in the
    cache and new ones. ``block_table`` (int32 [R, blocks], any row stride) gets
    the blocks that the new tokens need, from the top of the stack
    ``free_blocks[:free_count]`` downwards, in the order of the requests; a
    request gets all it needs or none. ``free_blocks`` (int32 [blocks of the
    cache]) has room for every block; table entries outside [0, its length) are
    no blocks. ``query_start`` (int32 [R + 1]): where
    each request's tokens begin in the step's packed tokens. ``seq_lens`` (int32
    [R], may be ``context_lens`` itself): context + query, or the context alone
    for a request that got no blocks, whose table row is too short or whose
    tokens do not fit. ``positions`` (int64 [T]) and ``slot_mapping`` (int32
    [T]): of every packed token; slot -1 where nothing can be stored, both -1
    behind the last token, which the Q/K norm operators leave untouched.
    ``free_count`` (int32 [1]) is updated in place, or left as it is with the new
    count in ``free_count_out``. ``row_positions`` (int64 [R]), ``row_slots`` and
    ``row_lens`` (int32 [R]; all three or none) are the step with one row per
    request, as :func:`paged_decode_attention` takes it: position and slot of each
    request's first token and its length with the step, or -1, -1, 0 for a request
    without a token and -1, -2, 0 for one whose token got no place."""
    _call("plan_step_", context_lens, query_lens, block_table, free_blocks, free_count, block_size,
          query_start, seq_lens, positions, slot_mapping, free_count_out, row_positions, row_slots,
          row_lens)


def release_blocks_(
    seq_lens: torch.Tensor,
    finished: torch.Tensor,
    block_table: torch.Tensor,
    free_blocks: torch.Tensor,
    free_count: torch.Tensor,
    block_size: int,
    shared_blocks: int = 0,
    free_count_out: torch.Tensor | None = None,
) -> None:
    """Pushes the blocks of the rows with ``finished`` (bool [R]) back on the
    stack ``free_blocks[:free_count]``, row after row; the first
    ``shared_blocks`` of every row (a prefix that others still use) stay out.
    Table entries outside [0, length of ``free_blocks``) are skipped. The table
    and ``seq_lens`` are not written: a row given back must not be given back
    again."""
    _call("release_blocks_", seq_lens, finished, block_table, free_blocks, free_count, block_size,
          shared_blocks, free_count_out)


def prompt_attention(
    out: torch.Tensor,
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    query_start: torch.Tensor,
    scale: float | None = None,
) -> None:
    """Causal attention of packed prompts into ``out`` [T, Hq, D].

    ``query`` [T, Hq, D], ``key`` and ``value`` [T, Hk, D] (bf16 or fp16, D 64, 128
    or 256, Hq a multiple of Hk, heads adjacent, any 16-byte-aligned token
    stride, e.g. views of one projection's output). Sequence s is the tokens
    ``query_start[s] .. query_start[s + 1] - 1`` (int32 [S + 1], on the GPU); its
    lengths need not be known on the host, and no start below the one before it.
    Rows of ``out`` behind the last sequence are left as they were. ``scale`` defaults to 1 / sqrt(D) and must be
    positive."""
    _call("prompt_attention", out, query, key, value, query_start, scale)


def paged_decode_attention(
    out: torch.Tensor,
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    prefix_blocks: torch.Tensor | None = None,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
    kv_cache_layout: str = "NHD",
    scale: float | None = None,
) -> None:
    """Attention of one token per request over a paged cache, into ``out``
    [B, Hq, D].

    ``query`` [B, Hq, D] (bf16 or fp16); caches [blocks, block_size, Hk, D]
    ("NHD") or [blocks, Hk, block_size, D] ("HND"), in query's dtype or fp8 with
    one-element float32 ``k_scale`` / ``v_scale``, as ``qk_norm_rope_cache_``
    fills them. ``seq_lens`` (int32 [B]): tokens of each request, the new one
    among them; a request of length zero gives zeros. ``block_table`` (int32 [B,
    blocks]): entry j holds tokens ``[j * block_size, (j + 1) * block_size)``;
    blocks outside the cache hold no keys.

    ``prefix_blocks`` (int32 [P]): blocks that the requests have in common. A
    request of at least ``P * block_size`` tokens reads its first P blocks from
    there instead of from its row, and they are read once for the whole batch;
    a shorter one is read through its row alone."""
    _call("paged_decode_attention", out, query, key_cache, value_cache, block_table, seq_lens,
          prefix_blocks, k_scale, v_scale, kv_cache_layout, scale)


if _C is not None:
    # Meta implementations: every operator only mutates its arguments.

    @torch.library.register_fake("sm120_norm_ext::plan_step_")
    def _plan_step_meta(context_lens, query_lens, block_table, free_blocks, free_count, block_size,
                        query_start, seq_lens, positions, slot_mapping, free_count_out=None,
                        row_positions=None, row_slots=None, row_lens=None) -> None:
        return None

    @torch.library.register_fake("sm120_norm_ext::release_blocks_")
    def _release_blocks_meta(seq_lens, finished, block_table, free_blocks, free_count, block_size,
                             shared_blocks=0, free_count_out=None) -> None:
        return None

    @torch.library.register_fake("sm120_norm_ext::prompt_attention")
    def _prompt_attention_meta(out, query, key, value, query_start, scale=None) -> None:
        return None

    @torch.library.register_fake("sm120_norm_ext::paged_decode_attention")
    def _paged_decode_attention_meta(out, query, key_cache, value_cache, block_table, seq_lens,
                                     prefix_blocks=None, k_scale=None, v_scale=None,
                                     kv_cache_layout="NHD", scale=None) -> None:
        return None
