// cache_args.cu -- checks of sm120n_qk_cache_args (csrc/cache_args.h); linked
// into both libraries.
#include "cache_args.h"

#include <algorithm>

#include "runtime.h"

namespace sm120n {

int check_cache_args(const sm120n_qk_cache_args* a, int* cache_kind) {
  if (a == nullptr) return fail(SM120N_ERR_INVALID_ARGUMENT, "args must be non-null");
  if (a->struct_size != sizeof(sm120n_qk_cache_args)) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "struct_size %u does not match this library's sm120n_qk_cache_args (%zu)",
                a->struct_size, sizeof(sm120n_qk_cache_args));
  }
  if (dtype_size(a->dtype) == 0) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "supported dtypes are float16, bfloat16, and float32");
  }
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) {
    return fail(SM120N_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256 (got %lld)",
                static_cast<long long>(a->head_dim));
  }
  if (a->rotary_dim < 16 || a->rotary_dim > a->head_dim || a->rotary_dim % 16 != 0) {
    return fail(SM120N_ERR_UNSUPPORTED,
                "rotary_dim must be a multiple of 16 in [16, head_dim] (got %lld)",
                static_cast<long long>(a->rotary_dim));
  }
  if (a->rope_style != SM120N_ROPE_NEOX && a->rope_style != SM120N_ROPE_INTERLEAVED) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "unknown rope_style %d", a->rope_style);
  }
  if (a->cache_dtype != SM120N_CACHE_AUTO && a->cache_dtype != SM120N_CACHE_FP8_E4M3) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "unknown cache_dtype %d", a->cache_dtype);
  }
  if (a->tokens < 0 || a->query_heads < 0 || a->key_heads < 0 || a->rope_positions < 0) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "tokens, head counts and rope_positions must be non-negative");
  }
  const int64_t heads = a->query_heads + a->key_heads;
  if (heads > (1 << 20)) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "at most 2^20 heads per token are supported");
  }
  if (a->tokens > (int64_t{1} << 40) / std::max<int64_t>(1, heads)) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "too many tokens");
  }
  const bool store = a->key_cache != nullptr || a->value_cache != nullptr;
  *cache_kind = !store ? kNoCache : a->cache_dtype == SM120N_CACHE_FP8_E4M3 ? kFp8 : kSameType;
  if (a->tokens == 0 || heads == 0) return SM120N_OK;
  if (a->query_token_stride < a->query_heads * a->head_dim ||
      a->key_token_stride < a->key_heads * a->head_dim) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "token strides must cover heads * head_dim elements (rows may not overlap)");
  }
  if ((a->query_heads > 0 && !a->query) || (a->key_heads > 0 && !a->key) || !a->query_weight ||
      !a->key_weight || !a->positions || !a->cos_sin_cache) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "tensor pointers must be non-null");
  }
  if (store) {
    if (!a->key_cache || !a->value_cache) {
      return fail(SM120N_ERR_INVALID_ARGUMENT, "key_cache and value_cache go together");
    }
    if (a->key_heads > 0 && (!a->value || !a->slot_mapping)) {
      return fail(SM120N_ERR_INVALID_ARGUMENT, "a KV store needs value and slot_mapping");
    }
    if (a->value_token_stride < a->key_heads * a->head_dim) {
      return fail(SM120N_ERR_INVALID_ARGUMENT,
                  "token strides must cover heads * head_dim elements (rows may not overlap)");
    }
    if (a->num_blocks < 0 || a->block_size < 1 || a->block_size > INT32_MAX ||
        a->cache_block_stride < 0 || a->cache_slot_stride < 0 || a->cache_head_stride < 0) {
      return fail(SM120N_ERR_INVALID_ARGUMENT,
                  "cache geometry must have num_blocks >= 0, block_size >= 1 and "
                  "non-negative strides");
    }
    if (a->num_blocks > (int64_t{1} << 31) / a->block_size) {
      return fail(SM120N_ERR_INVALID_ARGUMENT, "num_blocks * block_size must be at most 2^31");
    }
    if (*cache_kind == kFp8 && (!a->k_scale || !a->v_scale)) {
      return fail(SM120N_ERR_INVALID_ARGUMENT, "fp8 caches need k_scale and v_scale");
    }
  }
  return SM120N_OK;
}

}  // namespace sm120n
