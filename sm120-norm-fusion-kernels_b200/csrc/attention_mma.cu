// attention_mma.cu -- attention on warp-level matrix instructions, for what has
// no tensor-memory form: prompts and shared prefixes with heads of 256, and
// prefixes in blocks that do not fill a tile of 128 keys evenly.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j
// with the running maximum m and sum l of a row's exponentials: a tile of keys
// with scores s gives m' = max(m, max s), p = 2^(s - m'), l' = l 2^(m - m') +
// sum p, o' = o 2^(m - m') + p v. Scores, p's sum, o and all states are fp32;
// p is rounded to the 16-bit operand type of the second product only.
//
// The query heads of one key head are rows of one tile, so K and V are read
// once for all of them. A warp owns 16 rows. K and V tiles of 64 keys go
// from global to shared memory by cp.async, kStages tiles deep, 16-byte
// chunks swizzled so that every matrix load is free of bank conflicts. Keys
// behind the end of the sequence, or in a block that does not exist, are
// filled with zeros and masked, so nothing stored there can reach a result.
//
// fp8 caches: e4m3 to fp16 is exact and one instruction for two values, so
// these run the fp16 instruction, with each row of q scaled by a power of two
// into [1, 2) first (exact but for elements 2^14 below the row's largest) and
// the power folded into the row's score scale.
//
// Bound by instructions and their latencies: with heads of 256 a warp's 16 rows of o
// and a tile's scores fill its 255 registers, so that one block of four warps runs on
// an SM, and every tile of 64 keys has two barriers. One prompt of 4096 tokens, 32/8
// heads of 256, takes 1945 us (0.14 PFLOP/s), where products alone would take 166.
#include <algorithm>

#include "attention.h"
#include "attention_utils.cuh"
#include "warp_mma.cuh"

namespace sm120n {
namespace {

constexpr int kTileKeys = 64;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * kWarpSize;

enum Pass : int { kPrompt, kPrefix };

template <typename T, bool kFp8, int D, int kPass>
struct Form {
  static constexpr int kElem = kFp8 ? 1 : 2;
  static constexpr int kRowBytes = D * kElem;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kRows = 16 * kWarps;
  static constexpr int kTileBytes = kTileKeys * kRowBytes;
  static constexpr int kQBytes = kRows * D * 2;
  // tiles of K and V in flight
  static constexpr int kStages = kRowBytes > 256 ? 2 : 3;
  static constexpr size_t kSmem = kQBytes + kStages * 2 * kTileBytes;
};

// A block's piece of work: rows of one key head against keys [key_first, key_last).
struct Piece {
  int64_t first_row;  // kPrompt: packed row (token, head of the group) of the sequence
  int rows;
  int key_first;
  int key_last;
  int kv_head;
  int64_t token0;  // kPrompt: the sequence's first token
};

// Row `row` of a piece: its token and query head, as an offset into q or out.
template <int kPass, typename Args>
__device__ __forceinline__ int64_t row_offset(const Args& a, const Piece& p, int64_t row, int64_t stride,
                                              int d) {
  const int64_t r = p.first_row + row;
  const int64_t token = r / a.group;
  const int64_t head = static_cast<int64_t>(p.kv_head) * a.group + (r - token * a.group);
  return (p.token0 + token) * stride + head * d;
}

template <typename TQ, typename T, bool kFp8, int D, int kPass, typename Args>
struct Worker {
  using F = Form<T, kFp8, D, kPass>;
  const Args& a;
  unsigned char* smem;
  uint32_t* live;     // [kStages + 1][2] which keys of a tile exist, one bit each
  int64_t* offsets;   // [kStages + 1][kTileKeys] elements from the head's first, -1: no such key
  float* row_factor;  // fp8: power of two taken out of q

  int warp, lane;
  float o[D / 8][4];
  float m[2], l[2];

  __device__ __forceinline__ unsigned char* k_tile(int stage) const {
    return smem + F::kQBytes + stage * 2 * F::kTileBytes;
  }

  // Where key `j` is: its token (kPrompt) or its offset within the head, in
  // elements; -1 where there is none.
  __device__ __forceinline__ int64_t key_offset(const Piece& p, int64_t j) const {
    if (j >= p.key_last) return -1;
    if constexpr (kPass == kPrompt) {
      return p.token0 + j;
    } else {
      const int block = static_cast<int>(j / a.kv.block_size);
      const int id = a.prefix_blocks[block];
      if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(a.kv.num_blocks)) return -1;
      return id * a.kv.block_stride + (j - static_cast<int64_t>(block) * a.kv.block_size) * a.kv.slot_stride;
    }
  }

  // Threads 0-63 place a tile's rows; `found` was computed ahead of the wait.
  __device__ __forceinline__ void publish(int slot, int64_t found) {
    if (threadIdx.x < kTileKeys) {
      offsets[slot * kTileKeys + threadIdx.x] = found;
      const uint32_t bits = __ballot_sync(kFullMask, found >= 0);
      if (lane == 0) live[slot * 2 + warp] = bits;
    }
  }

  __device__ __forceinline__ void load_tile(const Piece& p, int stage, int slot) {
    const unsigned char *key, *value;
    int64_t key_step, value_step, head;  // elements
    if constexpr (kPass == kPrompt) {
      key = static_cast<const unsigned char*>(a.key);
      value = static_cast<const unsigned char*>(a.value);
      key_step = a.key_stride;
      value_step = a.value_stride;
      head = static_cast<int64_t>(p.kv_head) * D;
    } else {
      key = static_cast<const unsigned char*>(a.kv.key);
      value = static_cast<const unsigned char*>(a.kv.value);
      key_step = value_step = 1;
      head = p.kv_head * a.kv.head_stride;
    }
    const uint32_t k = shared_address(k_tile(stage));
#pragma unroll 4
    for (int i = threadIdx.x; i < kTileKeys * F::kChunks; i += kThreads) {
      const int row = i / F::kChunks;
      const int c = i % F::kChunks;
      const int64_t at = offsets[slot * kTileKeys + row];
      const int64_t place = max(at, int64_t{0});
      const uint32_t to = k + chunk_at<F::kChunks, kFp8>(row, c) * 16;
      copy16(to, key + (place * key_step + head) * F::kElem + c * 16, at >= 0);
      copy16(to + F::kTileBytes, value + (place * value_step + head) * F::kElem + c * 16, at >= 0);
    }
  }

  // Q of the piece's rows into shared memory, as T; rows that do not exist are zeros.
  __device__ __forceinline__ void load_query(const Piece& p) {
    const TQ* query = static_cast<const TQ*>(a.query);
    constexpr int kQChunks = D / 8;
    const uint32_t base = shared_address(smem);
    if constexpr (!kFp8) {
      for (int i = threadIdx.x; i < F::kRows * kQChunks; i += kThreads) {
        const int row = i / kQChunks, c = i % kQChunks;
        const bool real = row < p.rows;
        const TQ* from = real ? query + row_offset<kPass>(a, p, row, a.query_stride, D) + c * 8 : query;
        copy16(base + (row * kQChunks + (c ^ (row & 7))) * 16, from, real);
      }
    } else {
      // a warp to a row: its largest element, then the scaled row
      for (int row = warp; row < F::kRows; row += kWarps) {
        float v[D / kWarpSize];
        float top = 0.0f;
        const bool real = row < p.rows;
        const TQ* from = query + (real ? row_offset<kPass>(a, p, row, a.query_stride, D) : 0);
#pragma unroll
        for (int i = 0; i < D / kWarpSize; ++i) {
          const int e = lane * (D / kWarpSize) + i;
          v[i] = real ? static_cast<float>(from[e]) : 0.0f;
          top = fmaxf(top, fabsf(v[i]));
        }
#pragma unroll
        for (int d = kWarpSize / 2; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, d));
        // 2^-e and 2^e with e the exponent of the largest element, kept normal
        const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 2), 252);
        const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
        if (lane == 0) row_factor[row] = __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
        for (int i = 0; i < D / kWarpSize; ++i) {
          const int el = lane * (D / kWarpSize) + i;
          T* to = reinterpret_cast<T*>(smem) + row * D + (((el / 8) ^ (row & 7)) * 8 + el % 8);
          *to = static_cast<T>(v[i] * down);
        }
      }
    }
  }

  // Scores of this warp's 16 rows with the keys of the tile in `stage`.
  __device__ __forceinline__ void scores(int stage, float (*s)[4]) {
    constexpr int kNt = kTileKeys / 8;
    const int row0 = warp * 16;
    const uint32_t q = shared_address(smem);
    const uint32_t k = shared_address(k_tile(stage));
#pragma unroll
    for (int n = 0; n < kNt; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
    if constexpr (!kFp8) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t qa[4];
        const int qr = row0 + (lane & 15);
        ldmatrix4(qa, q + (qr * (D / 8) + ((2 * kk + (lane >> 4)) ^ (qr & 7))) * 16);
#pragma unroll
        for (int n = 0; n < kNt; n += 2) {
          uint32_t b[4];
          const int r = n * 8 + (lane & 7) + ((lane >> 4) << 3);
          ldmatrix4(b, k + chunk_at<F::kChunks, false>(r, 2 * kk + ((lane >> 3) & 1)) * 16);
          Mma<T>::mma(s[n], qa, b[0], b[1]);
          Mma<T>::mma(s[n + 1], qa, b[2], b[3]);
        }
      }
    } else {
      // The order of the summed index is free: in each run of 64 elements,
      // step i of four takes elements 16t + 4i .. + 3 of lane t, so that a
      // lane's bytes for four steps are one 16-byte load.
      const int g = lane >> 2, t = lane & 3;
#pragma unroll
      for (int run = 0; run < D / 64; ++run) {
        uint32_t qa[4][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // rows g and g + 8
          const int r = row0 + g + 8 * half;
#pragma unroll
          for (int c = 0; c < 2; ++c) {  // 16 elements = two 16-byte chunks of T
            const int chunk = run * 8 + 2 * t + c;
            const uint4 v = *reinterpret_cast<const uint4*>(smem + (r * (D / 8) + (chunk ^ (r & 7))) * 16);
            qa[2 * c][half] = v.x;
            qa[2 * c][2 + half] = v.y;
            qa[2 * c + 1][half] = v.z;
            qa[2 * c + 1][2 + half] = v.w;
          }
        }
#pragma unroll
        for (int n = 0; n < kNt; ++n) {
          const int r = n * 8 + g;
          const uint4 v = *reinterpret_cast<const uint4*>(
              k_tile(stage) + chunk_at<F::kChunks, true>(r, run * 4 + t) * 16);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t b0, b1;
            e4m3_to_half(w[i], b0, b1);
            Mma<T>::mma(s[n], qa[i], b0, b1);
          }
        }
      }
    }
  }

  // o += p v; p as operand registers, 16 keys each.
  __device__ __forceinline__ void weigh(int stage, const uint32_t (*p)[4]) {
    unsigned char* tile = k_tile(stage) + F::kTileBytes;
    const uint32_t v = shared_address(tile);
#pragma unroll
    for (int kk = 0; kk < kTileKeys / 16; ++kk) {
      if constexpr (!kFp8) {
        const int r = kk * 16 + (lane & 15);
#pragma unroll
        for (int n = 0; n < D / 8; n += 2) {
          uint32_t b[4];
          ldmatrix4_trans(b, v + chunk_at<F::kChunks, false>(r, n + (lane >> 4)) * 16);
          Mma<T>::mma(o[n], p[kk], b[0], b[1]);
          Mma<T>::mma(o[n + 1], p[kk], b[2], b[3]);
        }
      } else {
        // The order of the columns is free: of a run of 32, lane group g
        // holds 4g .. 4g + 3, the i-th of them in product i of four.
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int run = 0; run < D / 32; ++run) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = kk * 16 + 2 * t + (j & 1) + (j >> 1) * 8;
            w[j] = *reinterpret_cast<const uint32_t*>(
                tile + chunk_at<F::kChunks, true>(r, run * 2 + (g >> 2)) * 16 + (g & 3) * 4);
          }
          // pairs of neighbouring keys: columns 0, 1 in one word, 2, 3 in the next
          uint32_t lo[4], hi[4];
          e4m3_to_half(__byte_perm(w[0], w[1], 0x5140), lo[0], lo[1]);
          e4m3_to_half(__byte_perm(w[0], w[1], 0x7362), lo[2], lo[3]);
          e4m3_to_half(__byte_perm(w[2], w[3], 0x5140), hi[0], hi[1]);
          e4m3_to_half(__byte_perm(w[2], w[3], 0x7362), hi[2], hi[3]);
#pragma unroll
          for (int i = 0; i < 4; ++i) Mma<T>::mma(o[run * 4 + i], p[kk], lo[i], hi[i]);
        }
      }
    }
  }

  // Column of o[n][c] (c = 0 or 1 of the row's pair).
  __device__ __forceinline__ int column(int n, int c) const {
    const int t = lane & 3;
    if constexpr (kFp8) return (n / 4) * 32 + 4 * (2 * t + c) + n % 4;
    return n * 8 + 2 * t + c;
  }

  __device__ __forceinline__ uint32_t pack(float x, float y) const {
    return Pack<T>::f32_to_word(x, y);
  }

  // Whether a value of the tile in `stage` is infinite or NaN (16-bit tiles, whole block).
  __device__ __forceinline__ bool unsafe_values(int stage) {
    constexpr uint32_t kExponent = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    const uint4* v = reinterpret_cast<const uint4*>(k_tile(stage) + F::kTileBytes);
    bool bad = false;
    for (int i = threadIdx.x; i < kTileKeys * F::kChunks; i += kThreads) {
      const uint4 x = v[i];
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bad |= (w[j] & kExponent) == kExponent || ((w[j] >> 16) & kExponent) == kExponent;
      }
    }
    return __syncthreads_or(bad);
  }

  // Runs over the piece's keys. kPrompt: true when a value that some rows
  // must not see was infinite or NaN.
  __device__ __forceinline__ bool run(const Piece& p, float scale_log2) {
    constexpr int kNt = kTileKeys / 8;
    constexpr int kRing = F::kStages + 1;
    const int tiles = (p.key_last - p.key_first + kTileKeys - 1) / kTileKeys;
    bool unsafe = false;
    __syncthreads();  // the piece before is done with shared memory
    load_query(p);
#pragma unroll
    for (int t = 0; t < F::kStages; ++t) {
      publish(t, threadIdx.x < kTileKeys ? key_offset(p, p.key_first + int64_t{t} * kTileKeys + threadIdx.x) : -1);
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < F::kStages; ++t) {
      if (t < tiles) load_tile(p, t, t);
      copies_commit();
    }
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.0f;
    const int row0 = warp * 16 + (lane >> 2);
    int64_t limit[2] = {0, 0};  // kPrompt: last key of the row
    if constexpr (kPass == kPrompt) {
      limit[0] = (p.first_row + row0) / a.group;
      limit[1] = (p.first_row + row0 + 8) / a.group;
    }
    for (int t = 0; t < tiles; ++t) {
      const int stage = t % F::kStages;
      const int slot = t % kRing;
      const int64_t ahead =
          threadIdx.x < kTileKeys
              ? key_offset(p, p.key_first + (int64_t{t} + F::kStages) * kTileKeys + threadIdx.x)
              : -1;
      copies_wait<F::kStages - 1>();
      __syncthreads();
      const int64_t key0 = p.key_first + int64_t{t} * kTileKeys;
      if constexpr (kPass == kPrompt) {
        // the last rows see all keys up to key_last; the first stop at theirs
        if (key0 + kTileKeys - 1 > p.first_row / a.group) unsafe = unsafe_values(stage) || unsafe;
      }
      float s[kNt][4];
      scores(stage, s);
      float f0 = scale_log2, f1 = scale_log2;
      if constexpr (kFp8) {
        f0 *= row_factor[row0];
        f1 *= row_factor[row0 + 8];
      }
      const uint32_t live0 = live[slot * 2], live1 = live[slot * 2 + 1];
      const bool whole = (live0 & live1) == kFullMask;
      float top0 = m[0], top1 = m[1];
#pragma unroll
      for (int n = 0; n < kNt; ++n) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int key = n * 8 + 2 * (lane & 3) + c;
          // not merged with the difference to the maximum: both are rounded alike
          s[n][c] = __fmul_rn(s[n][c], f0);
          s[n][2 + c] = __fmul_rn(s[n][2 + c], f1);
          const bool there = whole || (((key < 32 ? live0 : live1) >> (key & 31)) & 1u);
          if (!there || (kPass == kPrompt && key0 + key > limit[0])) s[n][c] = -INFINITY;
          if (!there || (kPass == kPrompt && key0 + key > limit[1])) s[n][2 + c] = -INFINITY;
          top0 = fmaxf(top0, s[n][c]);
          top1 = fmaxf(top1, s[n][2 + c]);
        }
      }
#pragma unroll
      for (int d = 1; d < 4; d *= 2) {
        top0 = fmaxf(top0, __shfl_xor_sync(kFullMask, top0, d));
        top1 = fmaxf(top1, __shfl_xor_sync(kFullMask, top1, d));
      }
      // a row that has seen nothing yet keeps everything at zero
      const float base0 = top0 == -INFINITY ? 0.0f : top0;
      const float base1 = top1 == -INFINITY ? 0.0f : top1;
      const float keep0 = exp2_approx(m[0] - base0);
      const float keep1 = exp2_approx(m[1] - base1);
      m[0] = top0;
      m[1] = top1;
      float sum0 = 0.0f, sum1 = 0.0f;
      uint32_t pr[kNt / 2][4];
#pragma unroll
      for (int n = 0; n < kNt; ++n) {
        const float x0 = exp2_approx(s[n][0] - base0), y0 = exp2_approx(s[n][1] - base0);
        const float x1 = exp2_approx(s[n][2] - base1), y1 = exp2_approx(s[n][3] - base1);
        sum0 += x0 + y0;
        sum1 += x1 + y1;
        pr[n / 2][(n & 1) * 2] = pack(x0, y0);
        pr[n / 2][(n & 1) * 2 + 1] = pack(x1, y1);
      }
      l[0] = l[0] * keep0 + sum0;
      l[1] = l[1] * keep1 + sum1;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        o[n][0] *= keep0;
        o[n][1] *= keep0;
        o[n][2] *= keep1;
        o[n][3] *= keep1;
      }
      weigh(stage, pr);
      publish((t + F::kStages) % kRing, ahead);
      __syncthreads();
      if (t + F::kStages < tiles) load_tile(p, stage, (t + F::kStages) % kRing);
      copies_commit();
    }
    copies_wait<0>();
#pragma unroll
    for (int d = 1; d < 4; d *= 2) {
      l[0] += __shfl_xor_sync(kFullMask, l[0], d);
      l[1] += __shfl_xor_sync(kFullMask, l[1], d);
    }
    return unsafe;
  }
};

#define SM120S_WORKER(FORM)                                                           \
  extern __shared__ __align__(128) unsigned char dynamic_smem[];                      \
  __shared__ uint32_t live[(FORM::kStages + 1) * 2];                                  \
  __shared__ int64_t offsets[(FORM::kStages + 1) * kTileKeys];                        \
  __shared__ float row_factor[FORM::kRows]

// ---- prompts -----------------------------------------------------------------

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) prompt_mma_kernel(PromptArgs a) {
  using F = Form<T, false, D, kPrompt>;
  SM120S_WORKER(F);
  wait_for_upstream_grid();
  release_downstream_grid();
  const SequenceTile tile = find_tile<F::kRows>(a.query_start, a.sequences, a.tokens, a.group,
                                                blockIdx.x / a.key_heads);
  if (tile.tile < 0) return;
  Worker<T, T, false, D, kPrompt, PromptArgs> w{a, dynamic_smem, live, offsets, row_factor};
  w.warp = threadIdx.x / kWarpSize;
  w.lane = threadIdx.x & (kWarpSize - 1);
  Piece p{};
  p.first_row = tile.tile * F::kRows;
  p.rows = static_cast<int>(min(int64_t{F::kRows}, tile.length * a.group - p.first_row));
  p.key_last = static_cast<int>((p.first_row + p.rows - 1) / a.group + 1);
  p.kv_head = static_cast<int>(blockIdx.x % a.key_heads);
  p.token0 = tile.first_token;
  T* out = static_cast<T*>(a.out);
  if (w.run(p, a.scale_log2)) {
    for (int row = w.warp; row < p.rows; row += kWarps) {
      const int64_t token = (p.first_row + row) / a.group;
      const int64_t head = int64_t{p.kv_head} * a.group + (p.first_row + row - token * a.group);
      plain_prompt_row<T, D>(a, p.token0, token, head, p.kv_head);
    }
    return;
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = w.warp * 16 + (w.lane >> 2) + 8 * half;
    if (row >= p.rows) continue;
    const float inv = 1.0f / w.l[half];
    T* to = out + row_offset<kPrompt>(a, p, row, a.out_stride, D);
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      *reinterpret_cast<uint32_t*>(to + n * 8 + 2 * (w.lane & 3)) =
          Pack<T>::f32_to_word(w.o[n][2 * half] * inv, w.o[n][2 * half + 1] * inv);
    }
  }
}

// ---- the shared prefix of a decode batch ----------------------------------------
// Rows: (request, head of the group) of one key head; keys: one part of the prefix.
template <typename TQ, typename T, bool kFp8, int D>
__global__ void __launch_bounds__(kThreads, 1) prefix_mma_kernel(DecodeArgs a) {
  using F = Form<T, kFp8, D, kPrefix>;
  SM120S_WORKER(F);
  wait_for_upstream_grid();
  release_downstream_grid();
  Worker<TQ, T, kFp8, D, kPrefix, DecodeArgs> w{a, dynamic_smem, live, offsets, row_factor};
  w.warp = threadIdx.x / kWarpSize;
  w.lane = threadIdx.x & (kWarpSize - 1);
  Piece p{};
  p.first_row = static_cast<int64_t>(blockIdx.x) * F::kRows;
  p.rows = static_cast<int>(min(int64_t{F::kRows}, int64_t{a.batch} * a.group - p.first_row));
  p.kv_head = blockIdx.y;
  const int64_t tiles = (a.prefix_tokens + kTileKeys - 1) / kTileKeys;
  const int split = blockIdx.z;
  p.key_first = static_cast<int>(tiles * split / a.prefix_splits * kTileKeys);
  p.key_last = static_cast<int>(min(tiles * (split + 1) / a.prefix_splits * kTileKeys,
                                    int64_t{a.prefix_tokens}));
  const float scale = kFp8 ? a.scale_log2 * *a.k_scale : a.scale_log2;
  w.run(p, scale);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = w.warp * 16 + (w.lane >> 2) + 8 * half;
    if (row >= p.rows) continue;
    const int64_t r = p.first_row + row;
    const int64_t request = r / a.group;
    const int64_t at = (static_cast<int64_t>(split) * a.batch + request) * a.query_heads +
                       static_cast<int64_t>(p.kv_head) * a.group + (r - request * a.group);
    if ((w.lane & 3) == 0) a.prefix_state[at] = make_float2(w.m[half], w.l[half]);
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      a.prefix_values[at * D + w.column(n, 0)] = w.o[n][2 * half];
      a.prefix_values[at * D + w.column(n, 1)] = w.o[n][2 * half + 1];
    }
  }
}

template <typename T, int D>
int run_prompt(const PromptArgs& a, cudaStream_t stream) {
  using F = Form<T, false, D, kPrompt>;
  auto kernel = prompt_mma_kernel<T, D>;
  int rc = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), F::kSmem);
  if (rc != SM120N_OK) return rc;
  const int64_t tiles = (a.tokens * a.group + F::kRows - 1) / F::kRows + a.sequences;
  return launch(kernel, dim3(static_cast<unsigned>(tiles * a.key_heads)), dim3(kThreads), F::kSmem,
                stream, a);
}

template <typename TQ, typename T, bool kFp8, int D>
int run_prefix(const DecodeArgs& a, cudaStream_t stream) {
  using F = Form<T, kFp8, D, kPrefix>;
  auto kernel = prefix_mma_kernel<TQ, T, kFp8, D>;
  int rc = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), F::kSmem);
  if (rc != SM120N_OK) return rc;
  const int64_t tiles = (static_cast<int64_t>(a.batch) * a.group + F::kRows - 1) / F::kRows;
  return launch(kernel,
                dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(a.key_heads),
                     static_cast<unsigned>(a.prefix_splits)),
                dim3(kThreads), F::kSmem, stream, a);
}

}  // namespace

#define SM120S_BY_HEAD_DIM(CALL)      \
  switch (head_dim) {                 \
    case 64: return CALL(64);         \
    case 128: return CALL(128);       \
    default: return CALL(256);        \
  }

int launch_prompt_mma(const PromptArgs& a, int dtype, cudaStream_t stream) {
  return dtype == SM120N_F16 ? run_prompt<__half, 256>(a, stream)
                             : run_prompt<__nv_bfloat16, 256>(a, stream);
}

int launch_prefix_mma(const DecodeArgs& a, int dtype, int cache_dtype, int head_dim,
                      cudaStream_t stream) {
  const bool fp8 = cache_dtype == SM120N_CACHE_FP8_E4M3;
#define CALL(D)                                                                          \
  dtype == SM120N_F16 ? (fp8 ? run_prefix<__half, __half, true, D>(a, stream)            \
                             : run_prefix<__half, __half, false, D>(a, stream))          \
                      : (fp8 ? run_prefix<__nv_bfloat16, __half, true, D>(a, stream)     \
                             : run_prefix<__nv_bfloat16, __nv_bfloat16, false, D>(a, stream))
  SM120S_BY_HEAD_DIM(CALL)
#undef CALL
}

}  // namespace sm120n
