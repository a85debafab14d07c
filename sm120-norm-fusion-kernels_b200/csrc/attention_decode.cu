// attention_decode.cu -- a decode step's pass over each request's own cached
// tokens, and the kernel that joins the parts of a row.
//
// Bound by memory: every cached key and value is read once, for all query heads
// of its key head (up to 16 rows of one m16n8k16 tile). The key tiles of all
// (request, key head, row tile) triples stand in one list, cut into
// min(own_grid, tiles) equal runs, none empty: a block's run may end one triple
// and begin others, and every triple it touches gets one partial result, at
// index triple + block, which no other (triple, block) of the list shares. So
// the load is even whatever the lengths are, and nothing depends on the order
// in which blocks run.
//
// A block is four warps that compute and two that load, one K and the queries
// and one V. The loaders walk the run tile by tile across the ends of triples,
// into a ring of stages, with the first tile of a triple also its query rows.
// Cache blocks that fill a tile of 64 keys evenly come by TMA, one box for each
// block and 128 bytes of a row; others row by row with cp.async, which is slower
// to issue (1600 cycles for 32 KB by one warp; 4.4 TB/s). The four warps
// share the rows and split the 64 keys of a tile; each keeps its own maximum,
// sum and values until the triple ends. Keys behind the end, or in a block that
// does not exist, are masked and their values zeroed, so nothing stored there
// can reach a result.
//
// A stage holds K and V as boxes of 64 rows x 128 bytes with the TMA engine's
// swizzle: 16-byte chunk c of row r at c ^ (r & 7), free of bank conflicts for
// the matrix loads. fp8 tiles are read 16 bytes (K) and 4 bytes (V) at a time
// instead; there column c of a group of eight scores stands for key c ^ 4 (c &
// 1), which keeps rows that are read at once apart in both. (Rows of 64 bytes:
// chunk c at c ^ ((r >> 1) & 3).)
//
// fp8 caches: e4m3 to fp16 is exact and one instruction for two values, so
// these run the fp16 instruction, with each row of q scaled by a power of two
// into [1, 2) first (exact but for elements 2^14 below the row's largest) and
// the power folded into the row's score scale.
#include <algorithm>

#include "attention.h"
#include "attention_utils.cuh"
#include "tensor_core.cuh"
#include "tensor_map.h"
#include "warp_mma.cuh"

namespace sm120n {

__device__ unsigned int g_decode_expired_waits = 0;

namespace {

constexpr int kTileKeys = 64;
constexpr int kWarps = 4;  // that compute
constexpr int kLoaders = 2;
constexpr int kThreads = (kWarps + kLoaders) * kWarpSize;
constexpr int kWarpKeys = kTileKeys / kWarps;
constexpr int kMergeColumns = 32;

template <bool kFp8, int D>
struct OwnForm {
  static constexpr int kRowBytes = D * (kFp8 ? 1 : 2);
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kBoxRow = kRowBytes < 128 ? kRowBytes : 128;  // bytes of a row in a box
  static constexpr int kBoxes = kRowBytes / kBoxRow;
  static constexpr int kBoxBytes = kTileKeys * kBoxRow;
  // Byte offset of 16-byte chunk c of row r within a tile.
  __device__ __forceinline__ static int chunk(int r, int c) {
    if constexpr (kBoxRow == 64) return r * 64 + (c ^ ((r >> 1) & 3)) * 16;
    return (c >> 3) * kBoxBytes + r * 128 + ((c & 7) ^ (r & 7)) * 16;
  }
  static constexpr int kTileBytes = kTileKeys * kRowBytes;
  // About 100 KB of tiles to a block and up to two blocks to an SM, or 200 KB and one
  // with heads of 256, whose values and queries fill a thread's registers: well
  // past the 50 KB in flight that latency times bandwidth asks.
  static constexpr int kStages = D == 256 ? (kFp8 ? 5 : 3) : kRowBytes == 256 ? 3 : 5;
  static constexpr int kBlocksPerSm = D == 256 ? 1 : 2;
  static constexpr size_t stage_bytes(int q_rows) { return 2 * kTileBytes + q_rows * D * 2; }
  static constexpr size_t smem(int q_rows) {
    return 1024 + kStages * stage_bytes(q_rows) + static_cast<size_t>(kWarps) * q_rows * kMergeColumns * 4;
  }
  // With the static part and what the system keeps of 228 KB. More than 8 query
  // heads to a key head leave room for one block at D = 128 in 16 bits; a grid of
  // two to an SM then ran in two waves (64/4 heads, 256 requests of 1-1024 tokens,
  // 96.3 us against 88.1; 4 of up to 8192, 27.3 against 18.5).
  static constexpr int blocks_per_sm(int q_rows) {
    return smem(q_rows) + 2048 <= 228 * 1024 / 2 ? kBlocksPerSm : 1;
  }
};

__device__ __forceinline__ int own_tokens(const DecodeArgs& a, int request, int* first_key) {
  const int64_t cap = static_cast<int64_t>(a.table_width) * a.kv.block_size;
  const int64_t n = min(static_cast<int64_t>(max(a.seq_lens[request], 0)), cap);
  const bool shares = n >= a.prefix_tokens;
  *first_key = shares ? a.prefix_tokens : 0;
  return static_cast<int>(n) - *first_key;
}

// A run's walk over the list, the same for the loader and the other warps.
struct Walk {
  int64_t at, end;  // tiles of the list
  int64_t request_start;
  int request;
  // the triple at hand
  int tiles;  // of this request
  int kv_head, first_head;
  int triple;
  int first_key, keys;
  int tile0, tile1;

  __device__ __forceinline__ bool next(const DecodeArgs& a) {
    if (at >= end) return false;
    for (;;) {
      keys = own_tokens(a, request, &first_key);
      tiles = (keys + kTileKeys - 1) / kTileKeys;
      const int64_t all = static_cast<int64_t>(tiles) * a.key_heads * a.row_tiles;
      if (at < request_start + all) break;
      request_start += all;
      ++request;
    }
    triple = static_cast<int>((at - request_start) / tiles);
    kv_head = triple / a.row_tiles;
    first_head = (triple - kv_head * a.row_tiles) * 16;
    const int64_t start = request_start + static_cast<int64_t>(triple) * tiles;
    tile0 = static_cast<int>(at - start);
    tile1 = static_cast<int>(min(end - start, static_cast<int64_t>(tiles)));
    at = start + tile1;
    return true;
  }
};

__device__ __forceinline__ void bar_compute() {  // the four computing warps
  asm volatile("bar.sync 1, 128;" ::: "memory");
}

// One arrival of this thread once its copies so far have landed.
__device__ __forceinline__ void mbarrier_arrive_copies(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(shared_address(bar))
               : "memory");
}

// After an expired wait: a bounded time for the loads of the last uses of the ring
// to land, `uses` of them begun or skipped, before shared memory goes to another block.
template <int kStages>
__device__ __forceinline__ void let_land(uint64_t* full, int uses) {
  for (int u = max(uses - kStages, 0); u < uses; ++u) {
    mbarrier_wait_limited(&full[u % kStages], (u / kStages) & 1, 1u << 16);
  }
}

// Key of column c of a group of eight scores.
template <bool kFp8>
__device__ __forceinline__ int key_of(int c) {
  return kFp8 ? c ^ ((c & 1) << 2) : c;
}

template <typename TQ, typename T, bool kFp8, int D, bool kTma>
__global__ void __launch_bounds__(kThreads, OwnForm<kFp8, D>::kBlocksPerSm)
    own_kernel(const __grid_constant__ CUtensorMap key_map,
               const __grid_constant__ CUtensorMap value_map, const __grid_constant__ DecodeArgs a) {
  using F = OwnForm<kFp8, D>;
  constexpr int kStages = F::kStages;
  extern __shared__ unsigned char dynamic_smem[];
  // the swizzle repeats every 1024 bytes
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(dynamic_smem) + 1023) & ~uintptr_t{1023});
  __shared__ __align__(8) uint64_t full[kStages];
  __shared__ __align__(8) uint64_t empty[kStages];
  __shared__ uint32_t live[kStages][2];  // which keys of a tile exist, one bit each
  __shared__ float2 states[kWarps][16];
  __shared__ int64_t warp_totals[kThreads / kWarpSize];
  __shared__ int64_t found_start;
  __shared__ int found_request;
  const int warp = __shfl_sync(kFullMask, threadIdx.x / kWarpSize, 0);
  const int lane = threadIdx.x & (kWarpSize - 1);
  const int q_rows = a.group <= 8 ? 8 : 16;
  const uint32_t stage_bytes = static_cast<uint32_t>(F::stage_bytes(q_rows));
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      // of each loader: every lane's copies, and the masks or the bytes to come
      mbarrier_init(&full[s], kLoaders * (kWarpSize + 1));
      mbarrier_init(&empty[s], kWarps);
    }
    fence_mbarrier_init();
  }
  // Behind a prefix pass this one reads nothing that pass writes: it starts
  // beside it, and its first block waits for it before it ends, so that this
  // grid's end tells the joining kernel of both. (One block: the others make
  // room for those that have not started.) Whatever came before the prefix pass
  // is complete: that waited for it before it let this kernel start.
  const bool beside_prefix = a.prefix_splits > 0;
  if (!beside_prefix) wait_for_upstream_grid();
  release_downstream_grid();

  const int triples = a.key_heads * a.row_tiles;  // of one request
  // Sums of the requests' tiles, kPer * kThreads requests at a step, kPer
  // neighbours to a thread; f(first request, tiles before it, tiles of each).
  constexpr int kPer = 4;
  auto over_requests = [&](auto f) {
    int64_t before = 0;
    for (int base = 0; base < a.batch; base += kPer * kThreads) {
      const int i = base + kPer * static_cast<int>(threadIdx.x);
      int mine[kPer];
      int64_t all_mine = 0;
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        int first;
        mine[k] = i + k < a.batch ? (own_tokens(a, i + k, &first) + kTileKeys - 1) / kTileKeys : 0;
        all_mine += mine[k];
      }
      int64_t upto = all_mine;
#pragma unroll
      for (int d = 1; d < kWarpSize; d *= 2) {
        const int64_t x = __shfl_up_sync(kFullMask, upto, d);
        if (lane >= d) upto += x;
      }
      __syncthreads();
      if (lane == kWarpSize - 1) warp_totals[warp] = upto;
      __syncthreads();
      int64_t all = 0;
#pragma unroll
      for (int k = 0; k < kThreads / kWarpSize; ++k) {
        if (k < warp) upto += warp_totals[k];
        all += warp_totals[k];
      }
      f(i, before + upto - all_mine, mine);
      before += all;
    }
    return before;
  };
  auto find = [&](int64_t at, int first, int64_t start, const int* n) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (at >= start * triples && at < (start + n[k]) * triples) {
        found_request = first + k;
        found_start = start * triples;
      }
      start += n[k];
    }
  };
  // what the first step of the scan found, for batches that need no other
  int64_t my_start = 0;
  int my_tiles[kPer] = {};
  const int64_t total = over_requests([&](int first, int64_t start, const int* n) {
                          my_start = start;
#pragma unroll
                          for (int k = 0; k < kPer; ++k) {
                            my_tiles[k] = n[k];
                            if (blockIdx.x == 0 && first + k < a.batch) a.tile_start[first + k] = start;
                            start += n[k];
                          }
                        }) * triples;
  if (blockIdx.x == 0 && threadIdx.x == 0) a.tile_start[a.batch] = total / triples;
  const int64_t runs = min(total, int64_t{a.own_grid});
  if (blockIdx.x >= runs) {
    if (beside_prefix && blockIdx.x == 0) wait_for_upstream_grid();
    return;
  }
  Walk walk;
  walk.at = total * blockIdx.x / runs;
  walk.end = total * (blockIdx.x + 1) / runs;
  if (a.batch <= kPer * kThreads) {
    find(walk.at, kPer * static_cast<int>(threadIdx.x), my_start, my_tiles);
  } else {
    over_requests([&](int first, int64_t start, const int* n) { find(walk.at, first, start, n); });
  }
  __syncthreads();
  walk.request = found_request;
  walk.request_start = found_start;

  if (warp >= kWarps) {
    // ---- the loaders: the first brings K and the queries, the second V
    const bool first_loader = warp == kWarps;
    const CUtensorMap* map = first_loader ? &key_map : &value_map;
    const unsigned char* cache =
        static_cast<const unsigned char*>(first_loader ? a.kv.key : a.kv.value);
    const uint32_t part = first_loader ? 0 : F::kTileBytes;
    constexpr int kElem = kFp8 ? 1 : 2;
    // A tile's rows in the cache. kTma: lane b has box b, the slots of one cache
    // block (or 64 of a larger one). Otherwise rows `lane` and `lane + 32`. They
    // are looked up one tile ahead of the wait for its stage.
    constexpr int kMine = kTma ? 1 : 2;
    const int box = kTma ? min(a.kv.block_size, kTileKeys) : 1;
    int block[kMine], slot[kMine], count[kMine];
    auto look_up = [&](int t) {
#pragma unroll
      for (int h = 0; h < kMine; ++h) {
        const int first = (h * kWarpSize + lane) * box;
        const int within = t * kTileKeys + first;
        count[h] = first < kTileKeys ? max(min(box, walk.keys - within), 0) : 0;
        if (count[h] > 0) {
          const uint32_t j = static_cast<uint32_t>(walk.first_key + within);
          const uint32_t b = j / static_cast<uint32_t>(a.kv.block_size);
          slot[h] = static_cast<int>(j - b * a.kv.block_size);
          block[h] = a.table[static_cast<int64_t>(walk.request) * a.table_stride + b];
        }
      }
    };
    int use = 0;
    bool more = walk.next(a);
    int t = walk.tile0;
    if (more) look_up(t);
    while (more) {
      const int stage = use % kStages;
      int now_block[kMine], now_slot[kMine];
      uint32_t bits[2] = {0, 0};  // which keys exist
#pragma unroll
      for (int h = 0; h < kMine; ++h) {
        const bool there = count[h] > 0 &&
                           static_cast<uint32_t>(block[h]) < static_cast<uint32_t>(a.kv.num_blocks);
        // outside the map: arrives as zeros
        now_block[h] = there ? block[h] : kTma ? a.kv.num_blocks : -1;
        now_slot[h] = there ? slot[h] : 0;
        if constexpr (kTma) {
          const uint64_t run =
              !there ? 0 : (count[h] == 64 ? ~uint64_t{0} : (uint64_t{1} << count[h]) - 1) << (lane * box);
          bits[0] = __reduce_or_sync(kFullMask, static_cast<uint32_t>(run));
          bits[1] = __reduce_or_sync(kFullMask, static_cast<uint32_t>(run >> 32));
        } else {
          bits[h] = __ballot_sync(kFullMask, there);
        }
      }
      const bool begins = t == walk.tile0;
      const int kv_head = walk.kv_head;
      const int rows = min(16, a.group - walk.first_head);
      const TQ* query = static_cast<const TQ*>(a.query) +
                        static_cast<int64_t>(walk.request) * a.query_stride +
                        (static_cast<int64_t>(kv_head) * a.group + walk.first_head) * D;
      if (++t >= walk.tile1) {
        more = walk.next(a);
        t = walk.tile0;
      }
      if (more) look_up(t);

      if (use >= kStages &&
          !mbarrier_wait_warp(&empty[stage], (use / kStages - 1) & 1, a.wait_polls)) {
        if (lane == 0) atomicAdd(&g_decode_expired_waits, 1u);
        let_land<kStages>(full, use);
        break;
      }
      unsigned char* tile = smem + stage * stage_bytes;
      const uint32_t to = shared_address(tile);
      if (lane == 0) {
        if (first_loader) {
          live[stage][0] = bits[0];
          live[stage][1] = bits[1];
        }
        if constexpr (kTma) {
          mbarrier_arrive_expect_tx(&full[stage], F::kTileBytes);
        } else {
          mbarrier_arrive(&full[stage]);
        }
      }
      __syncwarp();
      if constexpr (kTma) {
        for (int b = 0; b < kTileKeys / box; ++b) {
          const int from = __shfl_sync(kFullMask, now_block[0], b);
          const int first_slot = __shfl_sync(kFullMask, now_slot[0], b);
          if (elect_lane()) {
#pragma unroll
            for (int h = 0; h < F::kBoxes; ++h) {
              tma_load_4d(tile + part + h * F::kBoxBytes + b * box * F::kBoxRow, map,
                          h * F::kBoxRow / kElem, first_slot, kv_head, from, &full[stage]);
            }
          }
        }
      } else {
#pragma unroll
        for (int h = 0; h < kMine; ++h) {
          const int64_t offset = (now_block[h] * a.kv.block_stride + now_slot[h] * a.kv.slot_stride +
                                  kv_head * a.kv.head_stride) * kElem;
#pragma unroll 8
          for (int i = lane; i < kWarpSize * F::kChunks; i += kWarpSize) {
            const int r = i / F::kChunks;
            const int c = i % F::kChunks;
            const int64_t from = __shfl_sync(kFullMask, offset, r);
            const bool there = (bits[h] >> r) & 1u;
            copy16(to + part + F::chunk(h * kWarpSize + r, c), cache + (there ? from : 0) + c * 16, there);
          }
        }
      }
      if (first_loader && begins) {
        for (int i = lane; i < q_rows * (D / 8); i += kWarpSize) {
          const int row = i / (D / 8), c = i % (D / 8);
          copy16(to + 2 * F::kTileBytes + (row * (D / 8) + (c ^ (row & 7))) * 16,
                 query + (row < rows ? row * D + c * 8 : 0), row < rows);
        }
      }
      mbarrier_arrive_copies(&full[stage]);
      ++use;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }

  // ---- the computing warps
  const float head_scale = kFp8 ? a.scale_log2 * *a.k_scale : a.scale_log2;
  float* merge = reinterpret_cast<float*>(smem + kStages * stage_bytes);  // [kWarps][q_rows][kMergeColumns]
  const int g = lane >> 2, tq = lane & 3;
  const int key0 = warp * kWarpKeys;
  int use = 0;
  bool ok = true;  // false after a wait ran out: keep step with the other warps, mark the rows
  while (walk.next(a)) {
    const int rows = min(16, a.group - walk.first_head);
    uint32_t q[D / 16][4];
    float f0 = head_scale, f1 = head_scale;
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
    for (int t = walk.tile0; t < walk.tile1; ++t, ++use) {
      const int stage = use % kStages;
      if (ok && !mbarrier_wait_warp(&full[stage], (use / kStages) & 1, a.wait_polls)) {
        if (lane == 0) atomicAdd(&g_decode_expired_waits, 1u);
        ok = false;
      }
      if (!ok) continue;
      unsigned char* tile = smem + stage * stage_bytes;
      const uint32_t k = shared_address(tile);
      const uint32_t v = k + F::kTileBytes;
      if (t == walk.tile0) {
        const unsigned char* q_tile = tile + 2 * F::kTileBytes;
        if constexpr (!kFp8) {
          const int r = (lane & 15) & (q_rows - 1);  // rows that do not exist repeat others
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            ldmatrix4(q[kk], shared_address(q_tile) + (r * (D / 8) + ((2 * kk + (lane >> 4)) ^ (r & 7))) * 16);
          }
        } else {
          // in the order of the summed index that scores() below uses, scaled
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int r = (g + 8 * half) & (q_rows - 1);
            uint4 raw[D / 32];
            float most = 0.0f;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              const int chunk = (c / 2) * 8 + 2 * tq + c % 2;
              raw[c] = *reinterpret_cast<const uint4*>(q_tile + (r * (D / 8) + (chunk ^ (r & 7))) * 16);
              float x[8];
              Pack<TQ>::to_f32(raw[c], x);
#pragma unroll
              for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[e]));
            }
            most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 1));
            most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 2));
            // 2^-e and 2^e with e the exponent of the row's largest, kept normal
            const int e = min(max(static_cast<int>(__float_as_uint(most) >> 23), 2), 252);
            const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
            (half ? f1 : f0) *= __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              float x[8];
              Pack<TQ>::to_f32(raw[c], x);
#pragma unroll
              for (int i = 0; i < 8; ++i) x[i] *= down;
              const uint4 y = Pack<T>::from_f32(x);
              // run c / 2 of 64 elements: steps 2 (c % 2) and the next
              const int kk = (c / 2) * 4 + 2 * (c % 2);
              q[kk][half] = y.x;
              q[kk][2 + half] = y.y;
              q[kk + 1][half] = y.z;
              q[kk + 1][2 + half] = y.w;
            }
          }
        }
      }
      // scores of 16 rows x 16 keys
      float s[2][4] = {};
      if constexpr (!kFp8) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t b[4];
          const int r = key0 + (lane & 7) + ((lane >> 4) << 3);
          ldmatrix4(b, k + F::chunk(r, 2 * kk + ((lane >> 3) & 1)));
          Mma<T>::mma(s[0], q[kk], b[0], b[1]);
          Mma<T>::mma(s[1], q[kk], b[2], b[3]);
        }
      } else {
        // The order of the summed index is free: in each run of 64 elements,
        // step i of four takes elements 16t + 4i .. + 3 of lane t, so that a
        // lane's bytes for four steps are one 16-byte load.
#pragma unroll
        for (int run = 0; run < D / 64; ++run) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const uint4 x = *reinterpret_cast<const uint4*>(
                tile + F::chunk(key0 + n * 8 + key_of<true>(g), run * 4 + tq));
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t b0, b1;
              e4m3_to_half(w[i], b0, b1);
              Mma<T>::mma(s[n], q[run * 4 + i], b0, b1);
            }
          }
        }
      }
      const uint32_t there = (live[stage][warp / 2] >> (16 * (warp & 1))) & 0xffffu;  // of its keys
      if (kTma && there != 0xffffu) {
        // whole blocks came, with whatever lies behind the end: no weight, and no value
        for (int i = lane; i < kWarpKeys * F::kChunks; i += kWarpSize) {
          const int r = i / F::kChunks;
          if (!((there >> r) & 1u)) {
            *reinterpret_cast<uint4*>(tile + F::kTileBytes + F::chunk(key0 + r, i % F::kChunks)) =
                make_uint4(0, 0, 0, 0);
          }
        }
        fence_async_shared();  // before TMA fills the stage again
        __syncwarp();
      }
      float top0 = m0, top1 = m1;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const bool real = (there >> (n * 8 + key_of<kFp8>(2 * tq + c))) & 1u;
          // not merged with the difference to the maximum: both are rounded alike
          s[n][c] = real ? __fmul_rn(s[n][c], f0) : -INFINITY;
          s[n][2 + c] = real ? __fmul_rn(s[n][2 + c], f1) : -INFINITY;
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
      if (__any_sync(kFullMask, top0 > m0 || top1 > m1)) {
        const float keep0 = exp2_approx(m0 - base0);
        const float keep1 = exp2_approx(m1 - base1);
        l0 *= keep0;
        l1 *= keep1;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[n][0] *= keep0;
          o[n][1] *= keep0;
          o[n][2] *= keep1;
          o[n][3] *= keep1;
        }
        m0 = top0;
        m1 = top1;
      }
      uint32_t p[4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float x0 = exp2_approx(s[n][0] - base0), y0 = exp2_approx(s[n][1] - base0);
        const float x1 = exp2_approx(s[n][2] - base1), y1 = exp2_approx(s[n][3] - base1);
        l0 += x0 + y0;
        l1 += x1 + y1;
        p[2 * n] = Pack<T>::f32_to_word(x0, y0);
        p[2 * n + 1] = Pack<T>::f32_to_word(x1, y1);
      }
      if constexpr (!kFp8) {
        const int r = key0 + (lane & 15);
#pragma unroll
        for (int n = 0; n < D / 8; n += 2) {
          uint32_t b[4];
          ldmatrix4_trans(b, v + F::chunk(r, n + (lane >> 4)));
          Mma<T>::mma(o[n], p, b[0], b[1]);
          Mma<T>::mma(o[n + 1], p, b[2], b[3]);
        }
      } else {
        // The order of the columns is free: of a run of 32, lane group g
        // holds 4g .. 4g + 3, the i-th of them in product i of four.
#pragma unroll
        for (int run = 0; run < D / 32; ++run) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = key0 + key_of<true>(2 * tq + (j & 1)) + (j >> 1) * 8;
            w[j] = *reinterpret_cast<const uint32_t*>(
                tile + F::kTileBytes + F::chunk(r, run * 2 + (g >> 2)) + (g & 3) * 4);
          }
          // pairs of neighbouring keys: columns 0, 1 in one word, 2, 3 in the next
          uint32_t lo[4], hi[4];
          e4m3_to_half(__byte_perm(w[0], w[1], 0x5140), lo[0], lo[1]);
          e4m3_to_half(__byte_perm(w[0], w[1], 0x7362), lo[2], lo[3]);
          e4m3_to_half(__byte_perm(w[2], w[3], 0x5140), hi[0], hi[1]);
          e4m3_to_half(__byte_perm(w[2], w[3], 0x7362), hi[2], hi[3]);
#pragma unroll
          for (int i = 0; i < 4; ++i) Mma<T>::mma(o[run * 4 + i], p, lo[i], hi[i]);
        }
      }
      __syncwarp();
      if (lane == 0) mbarrier_arrive(&empty[stage]);
    }

    // The four warps' states of the same rows become one partial result, a
    // few columns at a time.
#pragma unroll
    for (int d = 1; d < 4; d *= 2) {
      l0 += __shfl_xor_sync(kFullMask, l0, d);
      l1 += __shfl_xor_sync(kFullMask, l1, d);
    }
    if (tq == 0) {
      states[warp][g] = ok ? make_float2(m0, l0) : make_float2(-INFINITY, NAN);
      states[warp][g + 8] = ok ? make_float2(m1, l1) : make_float2(-INFINITY, NAN);
    }
    bar_compute();
    float weight[2];  // of this warp's values of rows g and g + 8 in the joint result
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, states[w][g + 8 * half].x);
      weight[half] = exp2_approx((half ? m1 : m0) - (top == -INFINITY ? 0.0f : top));
    }
    const int64_t slot = (static_cast<int64_t>(walk.request) * triples + walk.triple + blockIdx.x) * 16;
    if (threadIdx.x < rows) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, states[w][threadIdx.x].x);
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 st = states[w][threadIdx.x];
        sum += st.y * exp2_approx(st.x - (top == -INFINITY ? 0.0f : top));
      }
      a.own_state[slot + threadIdx.x] = make_float2(top, sum);
    }
#pragma unroll
    for (int c0 = 0; c0 < D / kMergeColumns; ++c0) {
#pragma unroll
      for (int i = 0; i < kMergeColumns / 8; ++i) {
        const int n = c0 * (kMergeColumns / 8) + i;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int row = g + 8 * half;
          if (row >= rows) continue;
          float* to = merge + (warp * q_rows + row) * kMergeColumns;
          // columns of o[n]: neighbours, or (fp8) four apart in the run of 32
          const int col = kFp8 ? 8 * tq + i : i * 8 + 2 * tq;
          to[col] = o[n][2 * half] * weight[half];
          to[col + (kFp8 ? 4 : 1)] = o[n][2 * half + 1] * weight[half];
        }
      }
      bar_compute();
      for (int i = threadIdx.x; i < rows * (kMergeColumns / 4); i += kWarps * kWarpSize) {
        const int row = i / (kMergeColumns / 4), c = i % (kMergeColumns / 4);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(merge + (w * q_rows + row) * kMergeColumns + 4 * c);
          sum.x += x.x;
          sum.y += x.y;
          sum.z += x.z;
          sum.w += x.w;
        }
        *reinterpret_cast<float4*>(a.own_values + (slot + row) * D + c0 * kMergeColumns + 4 * c) = sum;
      }
      bar_compute();
    }
  }
  if (!ok) let_land<kStages>(full, use);
  if (beside_prefix && blockIdx.x == 0) wait_for_upstream_grid();
}

// ---- the parts of a row joined ---------------------------------------------------
// One warp to a (request, query head): the parts of the prefix, then the runs
// that touched the row's triple, always in this order. A lane reads the state
// of one part, so that all of them arrive in one latency; then the values.
template <typename TQ, int D>
__global__ void __launch_bounds__(kWarps* kWarpSize) merge_kernel(DecodeArgs a) {
  constexpr int kPer = D / kWarpSize;
  const int lane = threadIdx.x & (kWarpSize - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + threadIdx.x / kWarpSize;
  wait_for_upstream_grid();
  release_downstream_grid();
  if (row >= static_cast<int64_t>(a.batch) * a.query_heads) return;
  const int request = static_cast<int>(row / a.query_heads);
  const int head = static_cast<int>(row - static_cast<int64_t>(request) * a.query_heads);
  const int kv_head = head / a.group;
  const int in_group = head - kv_head * a.group;
  int first_key;
  const int keys = own_tokens(a, request, &first_key);
  const int from_prefix = first_key > 0 ? a.prefix_splits : 0;  // does the request share the prefix?
  int own_runs = 0;
  int64_t own_row = 0;  // of the first run that touched the triple; the others follow 16 rows apart
  if (keys > 0) {
    const int triples = a.key_heads * a.row_tiles;
    const int triple = kv_head * a.row_tiles + in_group / 16;
    const int64_t total = a.tile_start[a.batch] * triples;
    const int64_t n = a.tile_start[request + 1] - a.tile_start[request];
    const int64_t t0 = a.tile_start[request] * triples + triple * n;
    const int64_t runs = min(total, int64_t{a.own_grid});
    // the runs that hold the triple's first and last tile
    const int64_t from = ((t0 + 1) * runs - 1) / total;
    own_runs = static_cast<int>(((t0 + n) * runs - 1) / total - from) + 1;
    own_row = (static_cast<int64_t>(request) * triples + triple + from) * 16 + in_group % 16;
  }
  const int parts = from_prefix + own_runs;
  float top = -INFINITY, sum = 0.0f;
  float acc[kPer] = {};
  for (int first = 0; first < parts; first += kWarpSize) {
    const int part = first + lane;
    float2 state = make_float2(-INFINITY, 0.0f);
    const float* values = nullptr;
    if (part < from_prefix) {
      const int64_t at = static_cast<int64_t>(part) * a.batch * a.query_heads + row;
      state = a.prefix_state[at];
      values = a.prefix_values + at * D;
    } else if (part < parts) {
      const int64_t at = own_row + static_cast<int64_t>(part - from_prefix) * 16;
      state = a.own_state[at];
      values = a.own_values + at * D;
    }
    // nothing seen; a sum that is not zero has seen a NaN and passes it on
    const bool seen = !(state.x == -INFINITY && state.y == 0.0f);
    float next = state.x;
#pragma unroll
    for (int d = kWarpSize / 2; d > 0; d /= 2) next = fmaxf(next, __shfl_xor_sync(kFullMask, next, d));
    next = fmaxf(next, top);
    const float base = next == -INFINITY ? 0.0f : next;
    const float keep = exp2_approx(top - base);
    const float factor = seen ? exp2_approx(state.x - base) : 0.0f;
    float part_sum = seen ? state.y * factor : 0.0f;
#pragma unroll
    for (int d = kWarpSize / 2; d > 0; d /= 2) part_sum += __shfl_xor_sync(kFullMask, part_sum, d);
    top = next;
    sum = sum * keep + part_sum;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] *= keep;
    const unsigned those = __ballot_sync(kFullMask, seen);
    const int count = min(parts - first, kWarpSize);
    constexpr int kAhead = 32 / kPer;  // parts whose values are on their way at once
    for (int k0 = 0; k0 < count; k0 += kAhead) {
      float x[kAhead][kPer];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const float* from = reinterpret_cast<const float*>(
            __shfl_sync(kFullMask, reinterpret_cast<unsigned long long>(values), (k0 + k) & 31));
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[k][i] = 0.0f;
        if (k0 + k < count && ((those >> (k0 + k)) & 1u)) {
          if constexpr (kPer % 4 == 0) {
#pragma unroll
            for (int i = 0; i < kPer; i += 4) {
              *reinterpret_cast<float4*>(x[k] + i) =
                  *reinterpret_cast<const float4*>(from + lane * kPer + i);
            }
          } else {
            *reinterpret_cast<float2*>(x[k]) = *reinterpret_cast<const float2*>(from + lane * kPer);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const float f = __shfl_sync(kFullMask, factor, (k0 + k) & 31);  // 0 for what was not seen
        if (k0 + k < count) {
#pragma unroll
          for (int i = 0; i < kPer; ++i) acc[i] += x[k][i] * f;
        }
      }
    }
  }
  const float v_scale = a.v_scale ? *a.v_scale : 1.0f;
  const float inv = sum == 0.0f ? 0.0f : v_scale / sum;
  TQ* out = static_cast<TQ*>(a.out) + request * a.out_stride + static_cast<int64_t>(head) * D + lane * kPer;
#pragma unroll
  for (int i = 0; i < kPer; i += 2) {
    *reinterpret_cast<uint32_t*>(out + i) = Pack<TQ>::f32_to_word(acc[i] * inv, acc[i + 1] * inv);
  }
}

template <typename TQ, typename T, bool kFp8, int D, bool kTma>
int run_own(const DecodeArgs& a, cudaStream_t stream) {
  using F = OwnForm<kFp8, D>;
  CUtensorMap maps[2] = {};
  for (int i = 0; kTma && i < 2; ++i) {
    const int rc = encode_cache_map(&maps[i], i ? a.kv.value : a.kv.key, a.kv, D, a.key_heads,
                                    kFp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : tensor_map_type<T>(),
                                    kFp8 ? 1 : 2, F::kBoxRow, kTileKeys, true);
    if (rc != SM120N_OK) return rc;
  }
  auto kernel = own_kernel<TQ, T, kFp8, D, kTma>;
  const size_t smem = F::smem(a.group <= 8 ? 8 : 16);
  const int rc = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), F::smem(16));
  if (rc != SM120N_OK) return rc;
  return launch(kernel, dim3(static_cast<unsigned>(a.own_grid)), dim3(kThreads), smem, stream,
                maps[0], maps[1], a);
}

template <typename TQ, typename T, bool kFp8, int D>
int run_own(const DecodeArgs& a, cudaStream_t stream) {
  return block_fills_tiles(a.kv.block_size, kTileKeys) && a.table_width > 0
             ? run_own<TQ, T, kFp8, D, true>(a, stream)
             : run_own<TQ, T, kFp8, D, false>(a, stream);
}

}  // namespace


#define SM120S_BY_HEAD_DIM(CALL)      \
  switch (head_dim) {                 \
    case 64: return CALL(64);         \
    case 128: return CALL(128);       \
    default: return CALL(256);        \
  }

int launch_own(const DecodeArgs& a, int dtype, int cache_dtype, int head_dim, cudaStream_t stream) {
  const bool fp8 = cache_dtype == SM120N_CACHE_FP8_E4M3;
#define CALL(D)                                                                       \
  dtype == SM120N_F16 ? (fp8 ? run_own<__half, __half, true, D>(a, stream)            \
                             : run_own<__half, __half, false, D>(a, stream))          \
                      : (fp8 ? run_own<__nv_bfloat16, __half, true, D>(a, stream)     \
                             : run_own<__nv_bfloat16, __nv_bfloat16, false, D>(a, stream))
  SM120S_BY_HEAD_DIM(CALL)
#undef CALL
}

int own_blocks_per_sm(int cache_dtype, int head_dim, int64_t group) {
  const int q_rows = group <= 8 ? 8 : 16;
#define CALL(D)                                                                              \
  cache_dtype == SM120N_CACHE_FP8_E4M3 ? OwnForm<true, D>::blocks_per_sm(q_rows)             \
                                       : OwnForm<false, D>::blocks_per_sm(q_rows)
  SM120S_BY_HEAD_DIM(CALL)
#undef CALL
}

int launch_merge(const DecodeArgs& a, int dtype, int head_dim, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.batch) * a.query_heads;
  const dim3 grid(static_cast<unsigned>((rows + kWarps - 1) / kWarps));
  const dim3 block(kWarps * kWarpSize);
#define CALL(D)                                                                         \
  dtype == SM120N_F16 ? launch(merge_kernel<__half, D>, grid, block, 0, stream, a)      \
                      : launch(merge_kernel<__nv_bfloat16, D>, grid, block, 0, stream, a)
  SM120S_BY_HEAD_DIM(CALL)
#undef CALL
}

int read_decode_faults(unsigned int* value) {
  const cudaError_t err = cudaMemcpyFromSymbol(value, g_decode_expired_waits, sizeof *value);
  return err == cudaSuccess ? SM120N_OK
                            : fail(SM120N_ERR_CUDA, "reading the fault counter failed: %s",
                                   cudaGetErrorString(err));
}

int reset_decode_faults() {
  const unsigned int zero = 0;
  const cudaError_t err = cudaMemcpyToSymbol(g_decode_expired_waits, &zero, sizeof zero);
  return err == cudaSuccess ? SM120N_OK
                            : fail(SM120N_ERR_CUDA, "resetting the fault counter failed: %s",
                                   cudaGetErrorString(err));
}

}  // namespace sm120n
