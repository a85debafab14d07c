// attention_utils.cuh -- device code that the attention kernels share.
#pragma once

#include <algorithm>

#include "attention.h"
#include "device_utils.cuh"
#include "tensor_map.h"

namespace sm120n {

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Four e4m3 bytes as two words of two fp16 values, exact: one instruction a
// word, which takes either half of a register as it is. (Through the header's
// conversion of a 16-bit pair, taking the pairs apart and putting the halves
// together again cost more than the conversion.)
__device__ __forceinline__ void e4m3_to_half(uint32_t bytes, uint32_t& low, uint32_t& high) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(low), "=r"(high)
      : "r"(bytes));
}

// One row of a prompt by plain arithmetic, one warp, keys one by one: for the
// rows of a block that has an infinite or NaN value among the keys that some
// of its rows must not see (a matrix product would multiply it by zero).
// `token` counts from the sequence's first, `token0`; `head` from the first of all.
template <typename T, int D>
__device__ __noinline__ void plain_prompt_row(const PromptArgs& a, int64_t token0, int64_t token,
                                              int64_t head, int kv_head) {
  constexpr int kPer = D / kWarpSize;
  const int lane = threadIdx.x & (kWarpSize - 1);
  const T* q = static_cast<const T*>(a.query) + (token0 + token) * a.query_stride + head * D;
  float acc[kPer] = {};
  float top = -INFINITY, sum = 0.0f;
  for (int64_t j = 0; j <= token; ++j) {
    const int64_t at = static_cast<int64_t>(kv_head) * D;
    const T* k = static_cast<const T*>(a.key) + (token0 + j) * a.key_stride + at;
    const T* v = static_cast<const T*>(a.value) + (token0 + j) * a.value_stride + at;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      s += static_cast<float>(q[lane + i * kWarpSize]) * static_cast<float>(k[lane + i * kWarpSize]);
    }
#pragma unroll
    for (int d = kWarpSize / 2; d > 0; d /= 2) s += __shfl_xor_sync(kFullMask, s, d);
    s = __fmul_rn(s, a.scale_log2);  // not merged with the difference: both are rounded alike
    const float next = fmaxf(top, s);
    const float base = next == -INFINITY ? 0.0f : next;
    const float keep = exp2_approx(top - base);
    const float e = exp2_approx(s - base);
    top = next;
    sum = sum * keep + e;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      acc[i] = acc[i] * keep + e * static_cast<float>(v[lane + i * kWarpSize]);
    }
  }
  T* out = static_cast<T*>(a.out) + (token0 + token) * a.out_stride + head * D;
#pragma unroll
  for (int i = 0; i < kPer; ++i) out[lane + i * kWarpSize] = static_cast<T>(acc[i] / sum);
}

// The sequence and tile of its rows that entry `index` of the tile list stands
// for: tiles of kRows (token, head) rows, sequence after sequence, the last
// rows of a sequence (they have the most keys) first. Every warp finds it on
// its own, 128 sequences at a step: no barrier, and one round of loads where
// there are few.
struct SequenceTile {
  int64_t first_token;
  int64_t length;
  int64_t tile;  // -1: the list is shorter
};

__device__ __forceinline__ int64_t clamp_start(int32_t v, int64_t tokens) {
  return min(max(static_cast<int64_t>(v), int64_t{0}), tokens);
}

template <int kRows>
__device__ __forceinline__ SequenceTile find_tile(const int32_t* query_start, int sequences,
                                                  int64_t tokens, int group, int64_t index) {
  constexpr int kPer = 4;
  const int lane = threadIdx.x & (kWarpSize - 1);
  int64_t before = 0;
  for (int base = 0; base < sequences; base += kPer * kWarpSize) {
    int64_t start[kPer + 1];
#pragma unroll
    for (int k = 0; k <= kPer; ++k) {
      start[k] = clamp_start(query_start[min(base + lane * kPer + k, sequences)], tokens);
    }
    int64_t tiles[kPer], mine = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      tiles[k] = (max(start[k + 1] - start[k], int64_t{0}) * group + kRows - 1) / kRows;
      mine += tiles[k];
    }
    int64_t upto = mine;
#pragma unroll
    for (int d = 1; d < kWarpSize; d *= 2) {
      const int64_t x = __shfl_up_sync(kFullMask, upto, d);
      if (lane >= d) upto += x;
    }
    const int64_t first = before + upto - mine;
    const unsigned holder = __ballot_sync(kFullMask, index >= first && index < first + mine);
    if (holder) {
      SequenceTile found{0, 0, 0};
      int64_t at = first;
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        if (index >= at && index < at + tiles[k]) {
          found = SequenceTile{start[k], start[k + 1] - start[k], at + tiles[k] - 1 - index};
        }
        at += tiles[k];
      }
      const int source = __ffs(holder) - 1;
      found.first_token = __shfl_sync(kFullMask, found.first_token, source);
      found.length = __shfl_sync(kFullMask, found.length, source);
      found.tile = __shfl_sync(kFullMask, found.tile, source);
      return found;
    }
    before += __shfl_sync(kFullMask, upto, kWarpSize - 1);
  }
  return SequenceTile{0, 0, -1};
}

// ---- host: tensor maps ------------------------------------------------------------
template <typename T>
constexpr CUtensorMapDataType tensor_map_type() {
  return std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// A map whose boxes have rows of `row_bytes` (64 or 128: the swizzle's span; 0: no swizzle).
inline int encode_tensor_map(CUtensorMap* map, const void* base, CUtensorMapDataType type, int rank,
                             const cuuint64_t* dims, const cuuint64_t* byte_strides,
                             const cuuint32_t* box, int row_bytes) {
  int rc = SM120N_OK;
  auto encode = tensor_map_encoder(&rc);
  if (rc != SM120N_OK) return rc;
  const cuuint32_t steps[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, type, static_cast<cuuint32_t>(rank), const_cast<void*>(base), dims,
                            byte_strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            row_bytes == 0    ? CU_TENSOR_MAP_SWIZZLE_NONE
                            : row_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                              : CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    return fail(SM120N_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  }
  return SM120N_OK;
}

// A paged cache as [blocks, heads, slots, head_dim], boxes of one block's slots
// (at most tile_keys) x row_bytes.
inline int encode_cache_map(CUtensorMap* map, const void* base, const KvSource& kv, int head_dim,
                            int heads, CUtensorMapDataType type, int elem, int row_bytes,
                            int tile_keys, bool swizzled) {
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(kv.block_size),
                              static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(kv.num_blocks)};
  // a dimension of one may have no stride of its own
  auto bytes = [elem](int64_t stride) {
    return static_cast<cuuint64_t>(std::max<int64_t>(stride * elem, 16));
  };
  const cuuint64_t strides[3] = {bytes(kv.slot_stride), bytes(kv.head_stride), bytes(kv.block_stride)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(row_bytes / elem),
                             static_cast<cuuint32_t>(std::min(kv.block_size, tile_keys)), 1, 1};
  return encode_tensor_map(map, base, type, 4, dims, strides, box, swizzled ? row_bytes : 0);
}

}  // namespace sm120n
