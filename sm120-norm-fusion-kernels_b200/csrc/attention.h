// attention.h -- arguments shared by the attention kernels' host code.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "runtime.h"
#include "sm120norm_b200_serving.h"

namespace sm120n {

// A paged cache. Strides in elements.
struct KvSource {
  const void* key;
  const void* value;
  int64_t slot_stride;
  int64_t head_stride;
  int64_t block_stride;
  int32_t block_size;
  int32_t num_blocks;
};

struct PromptArgs {
  const void* query;
  void* out;
  const int32_t* query_start;
  const void* key;
  const void* value;
  int64_t query_stride;  // elements between consecutive tokens
  int64_t key_stride;
  int64_t value_stride;
  int64_t out_stride;
  int64_t tokens;
  int32_t sequences;
  int32_t query_heads;
  int32_t key_heads;
  int32_t group;
  float scale_log2;  // scale * log2(e)
  uint32_t wait_polls;  // limit of every wait on an mbarrier
};

// Partial results of a row over a part of its keys: maximum of the scaled
// scores (base 2), sum of exp2, and the weighted values, not yet divided. A part
// whose block gave up a wait has (-inf, NaN), which makes the joined row NaN.
struct DecodeArgs {
  const void* query;
  void* out;
  const int32_t* table;
  const int32_t* seq_lens;
  const int32_t* prefix_blocks;
  const float* k_scale;
  const float* v_scale;
  KvSource kv;
  int64_t query_stride;
  int64_t out_stride;
  int64_t table_stride;
  int32_t batch;
  int32_t table_width;
  int32_t prefix_tokens;
  int32_t query_heads;
  int32_t key_heads;
  int32_t group;
  int32_t row_tiles;      // of 16 query heads of one key head
  int32_t own_grid;       // thread blocks of the pass over each request's own tokens
  int32_t prefix_splits;  // parts of the prefix
  float scale_log2;
  uint32_t wait_polls;  // limit of every wait on an mbarrier
  int64_t* tile_start;  // [batch + 1] key tiles of the requests before, per key head and row tile
  float2* own_state;    // [(batch * key_heads * row_tiles + own_grid) * 16] (maximum, sum)
  float* own_values;    // the same rows x head_dim
  float2* prefix_state;  // [prefix_splits, batch, query_heads]
  float* prefix_values;  // the same rows x head_dim
};

// Blocks of the pass over own tokens that an SM holds.
int own_blocks_per_sm(int cache_dtype, int head_dim, int64_t group);

// One launch each; element types as sm120n_dtype, caches as sm120n_cache_dtype.
int launch_prompt_mma(const PromptArgs& a, int dtype, cudaStream_t stream);  // head size 256
int launch_prefix_mma(const DecodeArgs& a, int dtype, int cache_dtype, int head_dim,
                      cudaStream_t stream);
// Head sizes 64 and 128; the prefix form wants blocks that fill a tile of 128 keys.
int launch_prompt_tc(const PromptArgs& a, int dtype, int head_dim, cudaStream_t stream);
int launch_prefix_tc(const DecodeArgs& a, int dtype, int cache_dtype, int head_dim,
                     cudaStream_t stream);
// Whether TMA boxes of cache blocks, in whole groups of the swizzle's 8 rows,
// make up tiles of `keys` keys.
inline bool block_fills_tiles(int64_t block_size, int keys) {
  return block_size % keys == 0 || (block_size % 8 == 0 && keys % block_size == 0);
}
int launch_own(const DecodeArgs& a, int dtype, int cache_dtype, int head_dim, cudaStream_t stream);
int launch_merge(const DecodeArgs& a, int dtype, int head_dim, cudaStream_t stream);

// Expired-wait counter of the pass over own tokens.
int read_decode_faults(unsigned int* value);
int reset_decode_faults();

}  // namespace sm120n
