"""ctypes binding of the C ABI in ``include/sm120norm_b200_serving.h``.

As ``capi`` for the norm library: integer device addresses, sizes and a
``cudaStream_t`` as an integer; :class:`~sm120_rmsnorm.capi.CApiError` on a
non-zero status.
"""
from __future__ import annotations

import ctypes
import threading
from pathlib import Path

from . import capi
from .capi import BF16, CACHE_AUTO, CACHE_FP8_E4M3, F16, F32, CApiError, QkCacheArgs  # noqa: F401

LIBRARY_NAME = "libsm120norm_b200_serving.so"
LIBRARY_PATH = Path(__file__).resolve().parent / LIBRARY_NAME
MAX_ROPE_AXES = 4

_i64, _i32, _f32, _vp = ctypes.c_int64, ctypes.c_int32, ctypes.c_float, ctypes.c_void_p


class _Sized(ctypes.Structure):
    def __init__(self, **fields):
        super().__init__(struct_size=ctypes.sizeof(type(self)), **fields)


class MropeArgs(_Sized):
    """``sm120s_mrope_args``, field for field."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("axes", _i32), ("sections", _i32 * MAX_ROPE_AXES),
        ("interleaved_sections", _i32), ("position_axis_stride", _i64), ("query_out", _vp),
        ("query_out_token_stride", _i64), ("key_out", _vp), ("key_out_token_stride", _i64),
    ]


class PromptArgs(_Sized):
    """``sm120s_prompt_args``, field for field."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", _i32), ("tokens", _i64), ("sequences", _i64),
        ("query_heads", _i64), ("key_heads", _i64), ("head_dim", _i64), ("query", _vp),
        ("query_token_stride", _i64), ("key", _vp), ("key_token_stride", _i64), ("value", _vp),
        ("value_token_stride", _i64), ("out", _vp), ("out_token_stride", _i64),
        ("query_start", _vp), ("scale", _f32),
    ]


class DecodeArgs(_Sized):
    """``sm120s_decode_args``, field for field."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", _i32), ("cache_dtype", _i32),
        ("reserved", _i32), ("batch", _i64), ("query_heads", _i64), ("key_heads", _i64),
        ("head_dim", _i64), ("query", _vp), ("query_token_stride", _i64), ("out", _vp),
        ("out_token_stride", _i64), ("key_cache", _vp), ("value_cache", _vp),
        ("num_blocks", _i64), ("block_size", _i64), ("cache_block_stride", _i64),
        ("cache_slot_stride", _i64), ("cache_head_stride", _i64), ("k_scale", _vp),
        ("v_scale", _vp), ("block_table", _vp), ("table_width", _i64), ("table_stride", _i64),
        ("seq_lens", _vp), ("prefix_blocks", _vp), ("prefix_blocks_count", _i64),
        ("workspace", _vp), ("workspace_bytes", ctypes.c_size_t), ("scale", _f32),
    ]


# Every symbol include/sm120norm_b200_serving.h declares, with its ctypes signature.
SIGNATURES: dict[str, tuple[list, object]] = {
    "sm120s_abi_version": ([], ctypes.c_int),
    "sm120s_last_error": ([], ctypes.c_char_p),
    "sm120s_get_device_faults": ([ctypes.POINTER(ctypes.c_uint32)], ctypes.c_int),
    "sm120s_reset_device_faults": ([], ctypes.c_int),
    "sm120s_plan_step": ([_vp, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                          _i64, _i64, _i64, _i64, _i64, _vp], ctypes.c_int),
    "sm120s_plan_step_rows": ([_vp, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                               _i64, _i64, _i64, _i64, _i64, _vp], ctypes.c_int),
    "sm120s_release_blocks": ([_vp, _vp, _vp, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _vp],
                              ctypes.c_int),
    "sm120s_qk_norm_mrope_cache": ([ctypes.POINTER(QkCacheArgs), ctypes.POINTER(MropeArgs), _vp],
                                   ctypes.c_int),
    "sm120s_prompt_attention": ([ctypes.POINTER(PromptArgs), _vp], ctypes.c_int),
    "sm120s_paged_decode_workspace": ([ctypes.POINTER(DecodeArgs), ctypes.POINTER(ctypes.c_size_t)],
                                      ctypes.c_int),
    "sm120s_paged_decode_attention": ([ctypes.POINTER(DecodeArgs), _vp], ctypes.c_int),
}

_lock = threading.Lock()
_lib: ctypes.CDLL | None = None


def load() -> ctypes.CDLL:
    """Load (once) and return the shared library with typed signatures."""
    global _lib
    capi.load()
    with _lock:
        if _lib is None:
            lib = ctypes.CDLL(str(LIBRARY_PATH))
            for name, (argtypes, restype) in SIGNATURES.items():
                fn = getattr(lib, name)
                fn.argtypes = argtypes
                fn.restype = restype
            _lib = lib
    return _lib


def _check(status: int) -> None:
    if status != capi.OK:
        raise CApiError(status, load().sm120s_last_error().decode())


def abi_version() -> int:
    return load().sm120s_abi_version()


def device_faults() -> int:
    count = ctypes.c_uint32(0)
    _check(load().sm120s_get_device_faults(ctypes.byref(count)))
    return int(count.value)


def reset_device_faults() -> None:
    _check(load().sm120s_reset_device_faults())


def plan_step(context_lens_ptr, query_lens_ptr, block_table_ptr, table_stride, free_blocks_ptr,
              free_count_ptr, free_count_out_ptr, query_start_ptr, seq_lens_ptr, positions_ptr,
              slot_mapping_ptr, requests, table_width, pool, block_size, tokens, stream=0) -> None:
    _check(load().sm120s_plan_step(
        context_lens_ptr, query_lens_ptr, block_table_ptr, table_stride, free_blocks_ptr,
        free_count_ptr, free_count_out_ptr, query_start_ptr, seq_lens_ptr, positions_ptr,
        slot_mapping_ptr, requests, table_width, pool, block_size, tokens, stream))


def plan_step_rows(context_lens_ptr, query_lens_ptr, block_table_ptr, table_stride, free_blocks_ptr,
                   free_count_ptr, free_count_out_ptr, query_start_ptr, seq_lens_ptr, positions_ptr,
                   slot_mapping_ptr, row_positions_ptr, row_slots_ptr, row_lens_ptr, requests,
                   table_width, pool, block_size, tokens, stream=0) -> None:
    _check(load().sm120s_plan_step_rows(
        context_lens_ptr, query_lens_ptr, block_table_ptr, table_stride, free_blocks_ptr,
        free_count_ptr, free_count_out_ptr, query_start_ptr, seq_lens_ptr, positions_ptr,
        slot_mapping_ptr, row_positions_ptr, row_slots_ptr, row_lens_ptr, requests, table_width,
        pool, block_size, tokens, stream))


def release_blocks(seq_lens_ptr, finished_ptr, block_table_ptr, table_stride, free_blocks_ptr,
                   free_count_ptr, free_count_out_ptr, requests, table_width, pool, block_size,
                   shared_blocks=0, stream=0) -> None:
    _check(load().sm120s_release_blocks(
        seq_lens_ptr, finished_ptr, block_table_ptr, table_stride, free_blocks_ptr, free_count_ptr,
        free_count_out_ptr, requests, table_width, pool, block_size, shared_blocks, stream))


def qk_norm_mrope_cache(args: QkCacheArgs, mrope: MropeArgs, stream=0) -> None:
    _check(load().sm120s_qk_norm_mrope_cache(ctypes.byref(args), ctypes.byref(mrope), stream))


def prompt_attention(args: PromptArgs, stream=0) -> None:
    _check(load().sm120s_prompt_attention(ctypes.byref(args), stream))


def paged_decode_workspace(args: DecodeArgs) -> int:
    """Bytes of workspace that :func:`paged_decode_attention` needs for these sizes."""
    out = ctypes.c_size_t(0)
    _check(load().sm120s_paged_decode_workspace(ctypes.byref(args), ctypes.byref(out)))
    return int(out.value)


def paged_decode_attention(args: DecodeArgs, stream=0) -> None:
    _check(load().sm120s_paged_decode_attention(ctypes.byref(args), stream))
