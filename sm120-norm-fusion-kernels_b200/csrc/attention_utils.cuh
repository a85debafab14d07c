// attention_utils.cuh -- device code that the attention kernels share.
#pragma once

#include "attention.h"
#include "device_utils.cuh"

namespace sm120n {

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One row of a prompt by plain arithmetic, one warp, keys one by one: for the
// rows of a block that has an infinite or NaN value among the keys that some
// of its rows must not see (a matrix product would multiply it by zero). `row`
// counts the (token, head of the group) rows of the sequence at `token0`.
template <typename T, int D>
__device__ __noinline__ void plain_prompt_row(const PromptArgs& a, int64_t token0, int64_t row,
                                              int kv_head) {
  constexpr int kPer = D / kWarpSize;
  const int lane = threadIdx.x & (kWarpSize - 1);
  const int64_t token = row / a.group;
  const int64_t head = static_cast<int64_t>(kv_head) * a.group + (row - token * a.group);
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
    s *= a.scale_log2;
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

// The sequence and tile of its rows that block `index` of the tile list works
// on: tiles of `rows` (token, head) rows, sequence after sequence. Whole block.
struct SequenceTile {
  int64_t first_token;
  int64_t length;
  int64_t tile;  // -1: the list is shorter
  int64_t tiles;
};

__device__ __forceinline__ int64_t clamp_start(int32_t v, int64_t tokens) {
  return min(max(static_cast<int64_t>(v), int64_t{0}), tokens);
}

template <int kBlockThreads>
__device__ __forceinline__ SequenceTile find_tile(const int32_t* query_start, int sequences,
                                                  int64_t tokens, int group, int rows,
                                                  int64_t index) {
  __shared__ int64_t totals[kBlockThreads / kWarpSize];
  __shared__ SequenceTile found;
  const int lane = threadIdx.x & (kWarpSize - 1);
  const int warp = threadIdx.x / kWarpSize;
  if (threadIdx.x == 0) found.tile = -1;
  int64_t before = 0;
  for (int base = 0; base < sequences; base += kBlockThreads) {
    const int i = base + threadIdx.x;
    int64_t first = 0, length = 0;
    if (i < sequences) {
      first = clamp_start(query_start[i], tokens);
      length = max(clamp_start(query_start[i + 1], tokens) - first, int64_t{0});
    }
    const int64_t mine = (length * group + rows - 1) / rows;
    int64_t upto = mine;
#pragma unroll
    for (int d = 1; d < kWarpSize; d *= 2) {
      const int64_t x = __shfl_up_sync(kFullMask, upto, d);
      if (lane >= d) upto += x;
    }
    __syncthreads();
    if (lane == kWarpSize - 1) totals[warp] = upto;
    __syncthreads();
    int64_t all = 0;
    for (int w = 0; w < kBlockThreads / kWarpSize; ++w) {
      if (w < warp) upto += totals[w];
      all += totals[w];
    }
    upto += before;
    if (index < upto && index >= upto - mine) {
      // the last rows of a sequence have the most keys: first
      found = SequenceTile{first, length, upto - 1 - index, mine};
    }
    before += all;
    if (index < before) break;
  }
  __syncthreads();
  return found;
}

}  // namespace sm120n
