// step_plan.cu -- block tables, positions and slot maps of a serving step from
// request lengths, on the GPU; C-ABI entry points sm120s_plan_step and
// sm120s_release_blocks.
//
// The pool of free cache blocks is a stack: free_blocks[0, free_count). With
// c tokens of request r in the cache, q new ones and B slots to a block,
//   held = ceil(c / B), want = ceil((c + q) / B), need = want - held
// and with the running sums over the requests
//   end_r = sum q, upto_r = sum need (of the requests that fit the table),
// request r is served iff it fits (want <= width, end_r <= tokens) and
// need = 0 or upto_r <= free_count. The sums never fall, so the served
// requests with need > 0 are the first ones, and block held + j of request r
// is free_blocks[free_count - 1 - (upto_r - need + j)] whatever the others do:
// every thread can form the new part of a block table from the sums alone, no
// part of the grid waits for another's table entries, and the result does not
// depend on the order in which anything runs.
//
// Both kernels are bound by latency (a 1024-request decode step moves 33 KB).
// One launch of one thread-block cluster: every block repeats the sums over
// the requests (they sit in L2) and takes its share of the tokens. A cluster
// and not a grid because the updates in place (free_count, seq_lens over
// context_lens) must follow every block's reads: that is one cluster barrier,
// with no counter to keep between calls. Replayed from a graph, a step of one
// request takes 2.1 us, one of 1001 decodes 4.5.
#include <cooperative_groups.h>

#include <algorithm>

#include "device_utils.cuh"
#include "runtime.h"
#include "sm120norm_b200_serving.h"

namespace sm120n {
namespace {

namespace cg = cooperative_groups;

constexpr int kPlanThreads = 1024;
constexpr int kPlanCluster = 8;  // the portable cluster size

struct PlanArgs {
  const int32_t* context;
  const int32_t* query;
  int32_t* table;
  const int32_t* free_blocks;
  const int32_t* free_count;
  int32_t* free_count_out;
  int32_t* query_start;
  int32_t* seq_lens;
  int64_t* positions;
  int32_t* slots;
  int64_t table_stride;
  int64_t tokens;
  int requests;
  int width;
  int pool;
  int block_size;
  int64_t* row_positions;  // all three or none
  int32_t* row_slots;
  int32_t* row_lens;
};

// Sums here never fall and matter only up to 2^31 - 2 (tokens, blocks of the
// pool), so they stop at kCap: 32 bits hold them, whatever the lengths are.
constexpr uint32_t kCap = 0x7fffffffu;
__device__ __forceinline__ uint32_t capped(uint32_t a, uint32_t b) { return min(a + b, kCap); }

// Inclusive capped sums of two values over the block, for up to 32 full warps.
__device__ __forceinline__ void block_scan2(uint32_t& a, uint32_t& b, uint32_t (*warp_sums)[2]) {
  const int lane = threadIdx.x & (kWarpSize - 1);
  const int warp = threadIdx.x / kWarpSize;
  const int warps = blockDim.x / kWarpSize;
#pragma unroll
  for (int d = 1; d < kWarpSize; d *= 2) {
    const uint32_t x = __shfl_up_sync(kFullMask, a, d);
    const uint32_t y = __shfl_up_sync(kFullMask, b, d);
    if (lane >= d) {
      a = capped(a, x);
      b = capped(b, y);
    }
  }
  if (lane == kWarpSize - 1) {
    warp_sums[warp][0] = a;
    warp_sums[warp][1] = b;
  }
  __syncthreads();
  // every warp sums the totals of the warps before it
  uint32_t x = lane < warps && lane < warp ? warp_sums[lane][0] : 0;
  uint32_t y = lane < warps && lane < warp ? warp_sums[lane][1] : 0;
#pragma unroll
  for (int d = kWarpSize / 2; d > 0; d /= 2) {
    x = capped(x, __shfl_xor_sync(kFullMask, x, d));
    y = capped(y, __shfl_xor_sync(kFullMask, y, d));
  }
  a = capped(a, x);
  b = capped(b, y);
}

template <int kBlocks>
__device__ __forceinline__ void step_barrier() {
  if constexpr (kBlocks > 1) {
    cg::this_cluster().sync();
  } else {
    __syncthreads();
  }
}

template <int kBlocks>
__device__ __forceinline__ int block_rank() {
  return kBlocks > 1 ? static_cast<int>(blockIdx.x) : 0;  // the grid is one cluster
}

// Division by the block size: a shift where it is a power of two.
struct BlockSize {
  uint32_t size;
  int shift;  // -1: none
  static __device__ __forceinline__ BlockSize of(int n) {
    return BlockSize{static_cast<uint32_t>(n), (n & (n - 1)) == 0 ? __ffs(n) - 1 : -1};
  }
  __device__ __forceinline__ uint32_t blocks(uint32_t tokens) const {  // whole ones
    return shift >= 0 ? tokens >> shift : tokens / size;
  }
  __device__ __forceinline__ uint32_t ceil(uint32_t tokens) const {
    const uint32_t whole = blocks(tokens);
    return whole + (tokens != whole * size);
  }
};

// kRows: also the step with one row per request (one request 2.24 us against 2.03,
// 1001 5.0 against 4.6). At least one block to an SM is asked for: without it the
// compiler kept to 32 registers (a prompt step 8.05 us against 7.75).
template <int kBlocks, int kPer, bool kRows>
__global__ void __cluster_dims__(kBlocks, 1, 1) __launch_bounds__(kPlanThreads, 1)
    plan_step_kernel(PlanArgs a) {
  // the rows of the chunk in work
  __shared__ uint32_t ends[kPlanThreads];   // of their tokens
  __shared__ uint32_t uptos[kPlanThreads];  // new blocks up to and with the row
  __shared__ uint32_t firsts[kPlanThreads];  // position of the first token
  __shared__ int32_t helds[kPlanThreads];   // blocks before the step, -1: not served
  __shared__ uint32_t warp_sums[kPlanThreads / kWarpSize][2];
  __shared__ uint32_t chunk_sums[2];
  __shared__ uint32_t popped;
  const int threads = blockDim.x;
  const int tid = threadIdx.x;
  const int lane = tid & (kWarpSize - 1);
  const int rank = block_rank<kBlocks>();
  if (tid == 0) popped = 0;
  wait_for_upstream_grid();
  release_downstream_grid();
  const uint32_t count = static_cast<uint32_t>(min(max(*a.free_count, 0), a.pool));
  const BlockSize block_size = BlockSize::of(a.block_size);
  const uint32_t tokens = static_cast<uint32_t>(a.tokens);
  uint32_t carry_tokens = 0, carry_need = 0;
  if (rank == 0 && tid == 0) a.query_start[0] = 0;

  // the first row of the chunk whose running sum is above `index`
  auto find = [](const uint32_t* sums, int n, uint32_t index) {
    int low = 0, high = n;
    while (low < high) {
      const int middle = (low + high) / 2;
      if (sums[middle] > index) high = middle; else low = middle + 1;
    }
    return low;
  };

  for (int base = 0; base < a.requests; base += threads) {
    const int r = base + tid;
    const bool live = r < a.requests;
    const uint32_t c = live ? static_cast<uint32_t>(max(a.context[r], 0)) : 0;
    const uint32_t q = live ? static_cast<uint32_t>(max(a.query[r], 0)) : 0;
    const uint32_t held = block_size.ceil(c);
    const uint32_t want = block_size.ceil(c + q);
    bool served = live && want <= static_cast<uint32_t>(a.width) && c + q <= kCap;
    const uint32_t need = served ? want - held : 0;
    uint32_t end = min(q, kCap), upto = need;
    __syncthreads();  // the chunk before is done with the shared arrays
    block_scan2(end, upto, warp_sums);
    if (tid == threads - 1) {
      chunk_sums[0] = end;
      chunk_sums[1] = upto;
    }
    end = capped(end, carry_tokens);
    upto = capped(upto, carry_need);
    // Requests past the end of the token buffer are the last ones, so leaving
    // them in the sums of need changes nothing for those before them.
    served = served && end <= tokens && (need == 0 || upto <= count);
    ends[tid] = end;
    uptos[tid] = upto;
    firsts[tid] = c;
    helds[tid] = served ? static_cast<int32_t>(held) : -1;
    const uint32_t top = __reduce_max_sync(kFullMask, served && need > 0 ? upto : 0);
    if (lane == 0 && top > 0) atomicMax(&popped, top);
    step_barrier<kBlocks>();  // every block has read this chunk and free_count
    const uint32_t first_token = carry_tokens, first_need = carry_need;
    carry_tokens = capped(carry_tokens, chunk_sums[0]);
    carry_need = capped(carry_need, chunk_sums[1]);
    if (rank == 0 && live) {
      a.query_start[r + 1] = static_cast<int32_t>(min(end, tokens));
      a.seq_lens[r] = static_cast<int32_t>(served ? c + q : c);
      if constexpr (kRows) {
        // the request's first token, as the loop over the tokens below finds it
        int slot = q == 0 ? -1 : -2;
        if (served && q > 0) {
          const uint32_t block = block_size.blocks(c);
          const int id = block == held
                             ? a.free_blocks[count - 1 - (upto - need)]
                             : a.table[static_cast<int64_t>(r) * a.table_stride + block];
          if (id >= 0 && id < a.pool) {
            slot = static_cast<int>(id * block_size.size + (c - block * block_size.size));
          }
        }
        a.row_slots[r] = slot;
        a.row_lens[r] = slot >= 0 ? static_cast<int32_t>(c + q) : 0;
        a.row_positions[r] = slot >= 0 ? int64_t{c} : -1;
      }
    }
    const int in_chunk = min(threads, a.requests - base);

    // New table entries: the e-th block taken is the e-th from the top, whoever
    // takes it; those taken end at `popped`.
    const uint32_t last_need = min(carry_need, popped);
    for (uint32_t e = first_need + static_cast<uint32_t>(rank * threads + tid); e < last_need;
         e += static_cast<uint32_t>(kBlocks * threads)) {
      const int i = find(uptos, in_chunk, e);
      const uint32_t before = i == 0 ? first_need : uptos[i - 1];
      a.table[static_cast<int64_t>(base + i) * a.table_stride + helds[i] + (e - before)] =
          a.free_blocks[count - 1 - e];
    }

    // Tokens of the chunk, kPer neighbours to a thread: one search for the first
    // of them, one block id for each block they touch.
    const uint32_t last_token = min(carry_tokens, tokens);
    for (uint32_t g = first_token / kPer + static_cast<uint32_t>(rank * threads + tid);
         kPer * g < last_token; g += static_cast<uint32_t>(kBlocks * threads)) {
      const uint32_t from = max(kPer * g, first_token);
      const uint32_t to = min(kPer * g + kPer, last_token);
      int i = find(ends, in_chunk, from);
      uint32_t begin = i == 0 ? first_token : ends[i - 1];
      uint32_t taken = i == 0 ? first_need : uptos[i - 1];  // blocks before the row's new ones
      int known_row = -1, id = -1;
      uint32_t known_block = 0;
      int64_t p[kPer];
      int32_t s[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const uint32_t t = kPer * g + j;
        if (t < from || t >= to) continue;
        while (ends[i] <= t) {
          begin = ends[i];
          taken = uptos[i++];
        }
        const uint32_t position = firsts[i] + (t - begin);  // below 2^32
        p[j] = position;
        s[j] = -1;
        const int held_blocks = helds[i];
        if (held_blocks < 0) continue;
        const uint32_t block = block_size.blocks(position);
        if (i != known_row || block != known_block) {
          known_row = i;
          known_block = block;
          const int fresh = static_cast<int>(block) - held_blocks;
          id = fresh < 0 ? a.table[static_cast<int64_t>(base + i) * a.table_stride + block]
                         : a.free_blocks[count - 1 - (taken + fresh)];
        }
        if (id >= 0 && id < a.pool) {
          s[j] = static_cast<int32_t>(id * block_size.size + (position - block * block_size.size));
        }
      }
      if (kPer == 4 && to == from + kPer &&
          ((reinterpret_cast<uintptr_t>(a.positions) | reinterpret_cast<uintptr_t>(a.slots)) & 15) == 0) {
        *reinterpret_cast<longlong2*>(a.positions + from) = make_longlong2(p[0], p[1 % kPer]);
        *reinterpret_cast<longlong2*>(a.positions + from + 2) = make_longlong2(p[kPer / 2], p[kPer - 1]);
        *reinterpret_cast<int4*>(a.slots + from) = make_int4(s[0], s[1 % kPer], s[kPer / 2], s[kPer - 1]);
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const uint32_t t = kPer * g + j;
          if (t < from || t >= to) continue;
          a.positions[t] = p[j];
          a.slots[t] = s[j];
        }
      }
    }
  }
  if (a.requests == 0) step_barrier<kBlocks>();
  if (rank == 0 && tid == 0) *a.free_count_out = static_cast<int32_t>(count - popped);
  for (int64_t t = int64_t{carry_tokens} + static_cast<int64_t>(rank) * threads + tid; t < a.tokens;
       t += static_cast<int64_t>(kBlocks) * threads) {
    a.positions[t] = -1;
    a.slots[t] = -1;
  }
}

struct ReleaseArgs {
  const int32_t* seq_lens;
  const uint8_t* finished;
  const int32_t* table;
  int32_t* free_blocks;
  const int32_t* free_count;
  int32_t* free_count_out;
  int64_t table_stride;
  int requests;
  int width;
  int pool;
  int block_size;
  int shared_blocks;
};

constexpr int kReleaseRows = 128;  // of a block in one round
constexpr int kAhead = 8;          // groups of 32 entries of a row in flight

// Rounds of kReleaseRows rows to a block, the blocks' rows in order. The rows
// that give something back are listed; a warp counts the ids of a row that go
// back; sums over the list and over the blocks before it give every row its
// place; the warp then writes them.
template <int kBlocks>
__global__ void __cluster_dims__(kBlocks, 1, 1) __launch_bounds__(kPlanThreads)
    release_blocks_kernel(ReleaseArgs a) {
  __shared__ int listed[kReleaseRows];  // rows of the block, in order
  __shared__ int ends[kReleaseRows];    // entries of a listed row that may go back: up to here
  __shared__ int place[kReleaseRows];   // counts, then exclusive sums
  __shared__ int warp_rows[kReleaseRows / kWarpSize];
  __shared__ int block_total[2];  // by the parity of the round
  const int tid = threadIdx.x;
  const int lane = tid & (kWarpSize - 1);
  const int warp = tid / kWarpSize;
  const int warps = blockDim.x / kWarpSize;
  const int rank = block_rank<kBlocks>();
  const BlockSize block_size = BlockSize::of(a.block_size);
  wait_for_upstream_grid();
  release_downstream_grid();
  const int64_t count = min(max(*a.free_count, 0), a.pool);
  int64_t carry = count;
  int round = 0;
  for (int base = 0; base < a.requests; base += kBlocks * kReleaseRows, round ^= 1) {
    const int first = base + rank * kReleaseRows;
    int n = 0;
    if (tid < kReleaseRows) {
      const int r = first + tid;
      const bool there = r < a.requests;
      const bool done = there && a.finished[r];
      const int tokens = there ? a.seq_lens[r] : 0;  // beside `finished`, not behind it
      if (done) {
        n = static_cast<int>(min(block_size.ceil(static_cast<uint32_t>(max(tokens, 0))),
                                 static_cast<uint32_t>(a.width)));
      }
      place[tid] = 0;
    }
    const unsigned gives = __ballot_sync(kFullMask, n > a.shared_blocks);
    if (tid < kReleaseRows && lane == 0) warp_rows[warp] = __popc(gives);
    __syncthreads();
    int rows = 0;
    {
      int before = 0;
#pragma unroll
      for (int w = 0; w < kReleaseRows / kWarpSize; ++w) {
        if (w < warp) before += warp_rows[w];
        rows += warp_rows[w];
      }
      if (n > a.shared_blocks) {
        const int at = before + __popc(gives & ((1u << lane) - 1));
        listed[at] = first + tid;
        ends[at] = n;
      }
    }
    __syncthreads();
    // f(entry is in the pool, id) over a listed row, 32 entries at a time in order
    auto over_entries = [&](int i, auto f) {
      const int end = ends[i];
      const int32_t* ids = a.table + static_cast<int64_t>(listed[i]) * a.table_stride;
      for (int j0 = a.shared_blocks; j0 < end; j0 += kAhead * kWarpSize) {
        int id[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int j = j0 + k * kWarpSize + lane;
          id[k] = j < end ? ids[j] : -1;
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          if (j0 + k * kWarpSize < end) {
            f(static_cast<uint32_t>(id[k]) < static_cast<uint32_t>(a.pool), id[k]);
          }
        }
      }
    };
    for (int i = warp; i < rows; i += warps) {
      int found = 0;
      over_entries(i, [&](bool back, int) { found += back; });
      found = __reduce_add_sync(kFullMask, found);
      if (lane == 0) place[i] = found;
    }
    __syncthreads();
    if (warp == 0) {
      static_assert(kReleaseRows == 4 * kWarpSize, "four rows to a lane");
      int v[4], sum = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = sum;
        sum += place[4 * lane + k];
      }
      int upto = sum;
#pragma unroll
      for (int d = 1; d < kWarpSize; d *= 2) {
        const int x = __shfl_up_sync(kFullMask, upto, d);
        if (lane >= d) upto += x;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) place[4 * lane + k] = upto - sum + v[k];
      if (lane == kWarpSize - 1) block_total[round] = upto;
    }
    step_barrier<kBlocks>();
    // a lane reads one block's total
    int64_t total = 0;
    if (lane < kBlocks) {
      if constexpr (kBlocks > 1) {
        total = *cg::this_cluster().map_shared_rank(&block_total[round], lane);
      } else {
        total = block_total[round];
      }
    }
    int64_t before = lane < rank ? total : 0;
#pragma unroll
    for (int d = kWarpSize / 2; d > 0; d /= 2) {
      before += __shfl_xor_sync(kFullMask, before, d);
      total += __shfl_xor_sync(kFullMask, total, d);
    }
    for (int i = warp; i < rows; i += warps) {
      int64_t at = carry + before + place[i];
      over_entries(i, [&](bool back, int id) {
        const unsigned set = __ballot_sync(kFullMask, back);
        const int64_t mine = at + __popc(set & ((1u << lane) - 1));
        if (back && mine < a.pool) a.free_blocks[mine] = id;
        at += __popc(set);
      });
    }
    carry += total;
    __syncthreads();  // the next round's lists and counts follow these reads
  }
  // no block leaves while another may still read its total
  step_barrier<kBlocks>();
  if (rank == 0 && tid == 0) {
    *a.free_count_out = static_cast<int32_t>(min(carry, static_cast<int64_t>(a.pool)));
  }
}

int check_pool(const void* free_blocks, int64_t pool, const void* free_count, const void* count_out,
               int64_t requests, int64_t width, int64_t table_stride, int64_t block_size) {
  // row and entry indices are 32-bit and run up to a round past the end
  if (requests < 0 || width < 0 || pool < 0 || requests > (1 << 30) || width > (1 << 30) ||
      pool >= INT32_MAX) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "requests and table width must be in [0, 2^30], the pool size in [0, 2^31 - 1)");
  }
  if (block_size < 1 || block_size > INT32_MAX || pool > (int64_t{1} << 31) / block_size) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "block_size must be positive and pool * block_size at most 2^31");
  }
  if (table_stride < width) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "block table rows may not overlap");
  }
  if (!free_count || !count_out || (pool > 0 && !free_blocks)) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "tensor pointers must be non-null");
  }
  return SM120N_OK;
}

unsigned plan_threads(int64_t work) {
  int64_t threads = 64;
  while (threads < work && threads < kPlanThreads) threads *= 2;
  return static_cast<unsigned>(threads);
}

}  // namespace
}  // namespace sm120n

using namespace sm120n;

extern "C" int sm120s_plan_step(const int32_t* context_lens, const int32_t* query_lens,
                                int32_t* block_table, int64_t table_stride,
                                const int32_t* free_blocks, const int32_t* free_count,
                                int32_t* free_count_out, int32_t* query_start, int32_t* seq_lens,
                                int64_t* positions, int32_t* slot_mapping, int64_t requests,
                                int64_t table_width, int64_t pool, int64_t block_size,
                                int64_t tokens, void* stream) {
  return sm120s_plan_step_rows(context_lens, query_lens, block_table, table_stride, free_blocks,
                               free_count, free_count_out, query_start, seq_lens, positions,
                               slot_mapping, nullptr, nullptr, nullptr, requests, table_width, pool,
                               block_size, tokens, stream);
}

extern "C" int sm120s_plan_step_rows(const int32_t* context_lens, const int32_t* query_lens,
                                     int32_t* block_table, int64_t table_stride,
                                     const int32_t* free_blocks, const int32_t* free_count,
                                     int32_t* free_count_out, int32_t* query_start,
                                     int32_t* seq_lens, int64_t* positions, int32_t* slot_mapping,
                                     int64_t* row_positions, int32_t* row_slots, int32_t* row_lens,
                                     int64_t requests, int64_t table_width, int64_t pool,
                                     int64_t block_size, int64_t tokens, void* stream) {
  clear_error();
  int rc = check_pool(free_blocks, pool, free_count, free_count_out, requests, table_width,
                      table_stride, block_size);
  if (rc != SM120N_OK) return rc;
  if (tokens < 0 || tokens >= INT32_MAX) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "tokens must be in [0, 2^31 - 1)");
  }
  if (!query_start || (requests > 0 && (!context_lens || !query_lens || !seq_lens)) ||
      (requests > 0 && table_width > 0 && !block_table) ||
      (tokens > 0 && (!positions || !slot_mapping))) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "tensor pointers must be non-null");
  }
  if (requests > 0 && (!row_positions || !row_slots || !row_lens) &&
      (row_positions || row_slots || row_lens)) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "row_positions, row_slots and row_lens go together");
  }
  const PlanArgs a{context_lens, query_lens, block_table, free_blocks, free_count, free_count_out,
                   query_start, seq_lens, positions, slot_mapping, table_stride, tokens,
                   static_cast<int>(requests), static_cast<int>(table_width),
                   static_cast<int>(pool), static_cast<int>(block_size), row_positions, row_slots,
                   row_lens};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  // A token to a thread of one block, then four, then four to a thread of a
  // cluster: 1001 decodes take 4.5 us with one token to a thread, 5.4 with four
  // and 5.8 on a cluster, a prompt step of a few thousand tokens 7.75 us with
  // four and 7.9 on a cluster, which is there for those that are longer.
  const bool rows = row_slots != nullptr;
  if (tokens <= kPlanThreads) {
    return launch(rows ? plan_step_kernel<1, 1, true> : plan_step_kernel<1, 1, false>, dim3(1),
                  dim3(plan_threads(std::max(requests, tokens))), 0, s, a);
  }
  if (tokens <= 4 * kPlanThreads) {
    return launch(rows ? plan_step_kernel<1, 4, true> : plan_step_kernel<1, 4, false>, dim3(1),
                  dim3(kPlanThreads), 0, s, a);
  }
  return launch(rows ? plan_step_kernel<kPlanCluster, 4, true> : plan_step_kernel<kPlanCluster, 4, false>,
                dim3(kPlanCluster), dim3(kPlanThreads), 0, s, a);
}

extern "C" int sm120s_release_blocks(const int32_t* seq_lens, const uint8_t* finished,
                                     const int32_t* block_table, int64_t table_stride,
                                     int32_t* free_blocks, const int32_t* free_count,
                                     int32_t* free_count_out, int64_t requests,
                                     int64_t table_width, int64_t pool, int64_t block_size,
                                     int64_t shared_blocks, void* stream) {
  clear_error();
  int rc = check_pool(free_blocks, pool, free_count, free_count_out, requests, table_width,
                      table_stride, block_size);
  if (rc != SM120N_OK) return rc;
  if (shared_blocks < 0) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "shared_blocks must be non-negative");
  }
  if (requests > 0 && (!seq_lens || !finished || (table_width > 0 && !block_table))) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "tensor pointers must be non-null");
  }
  const ReleaseArgs a{seq_lens, finished, block_table, free_blocks, free_count, free_count_out,
                      table_stride, static_cast<int>(requests), static_cast<int>(table_width),
                      static_cast<int>(pool), static_cast<int>(block_size),
                      static_cast<int>(std::min(shared_blocks, table_width))};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (requests <= kReleaseRows) {
    return launch(release_blocks_kernel<1>, dim3(1), dim3(kPlanThreads), 0, s, a);
  }
  return launch(release_blocks_kernel<kPlanCluster>, dim3(kPlanCluster), dim3(kPlanThreads), 0, s, a);
}
