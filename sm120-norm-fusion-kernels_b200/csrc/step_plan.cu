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
// with no counter to keep between calls. Eight blocks of 1024 threads write
// the 12 bytes of 65536 tokens in about a microsecond.
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
};

// Inclusive sums of two values over the block, for up to 32 full warps.
__device__ __forceinline__ void block_scan2(int64_t& a, int64_t& b, int64_t (*warp_sums)[2]) {
  const int lane = threadIdx.x & (kWarpSize - 1);
  const int warp = threadIdx.x / kWarpSize;
#pragma unroll
  for (int d = 1; d < kWarpSize; d *= 2) {
    const int64_t x = __shfl_up_sync(kFullMask, a, d);
    const int64_t y = __shfl_up_sync(kFullMask, b, d);
    if (lane >= d) {
      a += x;
      b += y;
    }
  }
  if (lane == kWarpSize - 1) {
    warp_sums[warp][0] = a;
    warp_sums[warp][1] = b;
  }
  __syncthreads();
  const int warps = blockDim.x / kWarpSize;
  // every warp sums the totals of the warps before it
  int64_t x = lane < warps && lane < warp ? warp_sums[lane][0] : 0;
  int64_t y = lane < warps && lane < warp ? warp_sums[lane][1] : 0;
#pragma unroll
  for (int d = kWarpSize / 2; d > 0; d /= 2) {
    x += __shfl_xor_sync(kFullMask, x, d);
    y += __shfl_xor_sync(kFullMask, y, d);
  }
  a += x;
  b += y;
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

// A row of the chunk in work, as the tokens need it.
struct PlanRow {
  int64_t end;   // of its tokens
  int32_t first;  // position of its first token
  int32_t held;
  int32_t pop;  // index into free_blocks of its first new block; blocks go down from there
  int32_t served;
};

template <int kBlocks, int kPer>
__global__ void __cluster_dims__(kBlocks, 1, 1) __launch_bounds__(kPlanThreads)
    plan_step_kernel(PlanArgs a) {
  __shared__ PlanRow rows[kPlanThreads];
  __shared__ int64_t warp_sums[kPlanThreads / kWarpSize][2];
  __shared__ int64_t chunk_sums[2];
  __shared__ int popped;
  const int threads = blockDim.x;
  const int tid = threadIdx.x;
  const int lane = tid & (kWarpSize - 1);
  const int rank = block_rank<kBlocks>();
  if (tid == 0) popped = 0;
  wait_for_upstream_grid();
  release_downstream_grid();
  const int count = min(max(*a.free_count, 0), a.pool);
  const uint32_t block_size = static_cast<uint32_t>(a.block_size);
  int64_t carry_tokens = 0, carry_need = 0;
  if (rank == 0 && tid == 0) a.query_start[0] = 0;

  for (int base = 0; base < a.requests; base += threads) {
    const int r = base + tid;
    const bool live = r < a.requests;
    const int64_t c = live ? max(a.context[r], 0) : 0;
    const int64_t q = live ? max(a.query[r], 0) : 0;
    const uint32_t c_blocks = static_cast<uint32_t>(c) / block_size;
    const int64_t held = c_blocks + (static_cast<uint32_t>(c) - c_blocks * block_size != 0);
    const uint32_t both = static_cast<uint32_t>(c + q);  // below 2^32
    const uint32_t both_blocks = both / block_size;
    const int64_t want = int64_t{both_blocks} + (both - both_blocks * block_size != 0);
    bool served = live && want <= a.width && c + q <= INT32_MAX;
    const int64_t need = served ? want - held : 0;
    int64_t end = q, upto = need;
    __syncthreads();  // the chunk before is done with the shared arrays
    block_scan2(end, upto, warp_sums);
    if (tid == threads - 1) {
      chunk_sums[0] = end;
      chunk_sums[1] = upto;
    }
    end += carry_tokens;
    upto += carry_need;
    // Requests past the end of the token buffer are the last ones, so leaving
    // them in the sums of need changes nothing for those before them.
    served = served && end <= a.tokens && (need == 0 || upto <= count);
    PlanRow row;
    row.end = end;
    row.first = static_cast<int32_t>(c);
    row.held = static_cast<int32_t>(held);
    row.pop = static_cast<int32_t>(count - 1 - (upto - need));  // not read unless served
    row.served = served;
    rows[tid] = row;
    const int top = __reduce_max_sync(kFullMask, served && need > 0 ? static_cast<int>(upto) : 0);
    if (lane == 0 && top > 0) atomicMax(&popped, top);
    step_barrier<kBlocks>();  // every block has read this chunk and free_count
    const int64_t first_token = carry_tokens;
    carry_tokens += chunk_sums[0];
    carry_need += chunk_sums[1];
    if (rank == 0 && live) {
      a.query_start[r + 1] = static_cast<int32_t>(min(end, a.tokens));
      a.seq_lens[r] = static_cast<int32_t>(served ? c + q : c);
    }

    // New table entries: the rows of a warp go round the blocks; few entries
    // are written by the row's own thread, many by the whole warp.
    const int mine = served && r % kBlocks == rank ? static_cast<int>(need) : 0;
    if (mine > 0 && mine <= 2) {
      for (int j = 0; j < mine; ++j) {
        a.table[r * a.table_stride + row.held + j] = a.free_blocks[row.pop - j];
      }
    }
    for (unsigned many = __ballot_sync(kFullMask, mine > 2); many; many &= many - 1) {
      const int source = __ffs(many) - 1;
      const int n = __shfl_sync(kFullMask, mine, source);
      const int pop = __shfl_sync(kFullMask, row.pop, source);
      const int at = __shfl_sync(kFullMask, row.held, source);
      int32_t* entry = a.table + static_cast<int64_t>(r - lane + source) * a.table_stride + at;
      for (int j = lane; j < n; j += kWarpSize) entry[j] = a.free_blocks[pop - j];
    }

    // Tokens of the chunk, kPer neighbours to a thread: one search for the first
    // of them, one block id for each block they touch.
    const int64_t last_token = min(carry_tokens, a.tokens);
    const int in_chunk = min(threads, a.requests - base);
    for (int64_t g = first_token / kPer + static_cast<int64_t>(rank) * threads + tid;
         kPer * g < last_token; g += static_cast<int64_t>(kBlocks) * threads) {
      const int64_t from = max(kPer * g, first_token);
      const int64_t to = min(kPer * g + kPer, last_token);
      int low = 0, high = in_chunk;  // the first row whose end is behind `from`
      while (low < high) {
        const int middle = (low + high) / 2;
        if (rows[middle].end > from) high = middle; else low = middle + 1;
      }
      int i = low;
      int64_t begin = i == 0 ? first_token : rows[i - 1].end;
      int known_row = -1, id = -1;
      uint32_t known_block = 0;
      int64_t p[kPer];
      int32_t s[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int64_t t = kPer * g + j;
        if (t < from || t >= to) continue;
        while (rows[i].end <= t) begin = rows[i++].end;
        p[j] = rows[i].first + (t - begin);
        s[j] = -1;
        if (!rows[i].served) continue;
        const uint32_t position = static_cast<uint32_t>(p[j]);  // below 2^31 for a served request
        const uint32_t block = position / block_size;
        if (i != known_row || block != known_block) {
          known_row = i;
          known_block = block;
          const int fresh = static_cast<int>(block) - rows[i].held;
          id = fresh < 0 ? a.table[static_cast<int64_t>(base + i) * a.table_stride + block]
                         : a.free_blocks[rows[i].pop - fresh];
        }
        if (id >= 0 && id < a.pool) {
          s[j] = static_cast<int32_t>(id * block_size + (position - block * block_size));
        }
      }
      if (kPer == 4 && from == kPer * g && to == from + kPer &&
          ((reinterpret_cast<uintptr_t>(a.positions) | reinterpret_cast<uintptr_t>(a.slots)) & 15) == 0) {
        *reinterpret_cast<longlong2*>(a.positions + from) = make_longlong2(p[0], p[1 % kPer]);
        *reinterpret_cast<longlong2*>(a.positions + from + 2) = make_longlong2(p[kPer / 2], p[kPer - 1]);
        *reinterpret_cast<int4*>(a.slots + from) = make_int4(s[0], s[1 % kPer], s[kPer / 2], s[kPer - 1]);
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int64_t t = kPer * g + j;
          if (t < from || t >= to) continue;
          a.positions[t] = p[j];
          a.slots[t] = s[j];
        }
      }
    }
  }
  if (a.requests == 0) step_barrier<kBlocks>();
  if (rank == 0 && tid == 0) *a.free_count_out = count - popped;
  for (int64_t t = carry_tokens + static_cast<int64_t>(rank) * threads + tid; t < a.tokens;
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
constexpr int kRowsOfWarp = kReleaseRows / (kPlanThreads / kWarpSize);
constexpr int kAhead = 4;  // groups of 32 entries of each row in flight

// Rounds of kReleaseRows rows to a block, the blocks' rows in order. A warp
// counts the ids of its rows that go back; sums over the block's rows and over
// the blocks before it give every row its place; the warp then writes them. A
// warp's rows are read side by side, several groups of entries ahead: one row
// after the other the loads' latencies add up (19 us against 8 for 1000 rows).
template <int kBlocks>
__global__ void __cluster_dims__(kBlocks, 1, 1) __launch_bounds__(kPlanThreads)
    release_blocks_kernel(ReleaseArgs a) {
  __shared__ int ends[kReleaseRows];   // entries of a row that may go back: up to here
  __shared__ int place[kReleaseRows];  // counts, then exclusive sums
  __shared__ int block_total[2];       // by the parity of the round
  const int tid = threadIdx.x;
  const int lane = tid & (kWarpSize - 1);
  const int warp = tid / kWarpSize;
  const int rank = block_rank<kBlocks>();
  wait_for_upstream_grid();
  release_downstream_grid();
  const int64_t count = min(max(*a.free_count, 0), a.pool);
  int64_t carry = count;
  int round = 0;
  for (int base = 0; base < a.requests; base += kBlocks * kReleaseRows, round ^= 1) {
    const int first = base + rank * kReleaseRows;
    if (tid < kReleaseRows) {
      const int r = first + tid;
      uint32_t n = 0;
      if (r < a.requests && a.finished[r]) {
        const uint32_t tokens = static_cast<uint32_t>(max(a.seq_lens[r], 0));
        n = tokens / static_cast<uint32_t>(a.block_size);
        n += tokens - n * static_cast<uint32_t>(a.block_size) != 0;
      }
      ends[tid] = static_cast<int>(min(n, static_cast<uint32_t>(a.width)));
    }
    __syncthreads();
    // f(row of the warp, entry there and in the pool, id) for the warp's rows
    // side by side, in the order of the entries for each
    auto over_entries = [&](auto f) {
      int most = 0;
#pragma unroll
      for (int i = 0; i < kRowsOfWarp; ++i) most = max(most, ends[warp * kRowsOfWarp + i]);
      for (int j0 = a.shared_blocks; j0 < most; j0 += kAhead * kWarpSize) {
        int id[kRowsOfWarp][kAhead];
#pragma unroll
        for (int i = 0; i < kRowsOfWarp; ++i) {
          const int n = ends[warp * kRowsOfWarp + i];
          const int32_t* ids = a.table + static_cast<int64_t>(first + warp * kRowsOfWarp + i) * a.table_stride;
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            const int j = j0 + k * kWarpSize + lane;
            id[i][k] = j < n ? ids[j] : -1;
          }
        }
#pragma unroll
        for (int i = 0; i < kRowsOfWarp; ++i) {
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            f(i, static_cast<uint32_t>(id[i][k]) < static_cast<uint32_t>(a.pool), id[i][k]);
          }
        }
      }
    };
    int found[kRowsOfWarp] = {};
    over_entries([&](int i, bool back, int) { found[i] += back; });
#pragma unroll
    for (int i = 0; i < kRowsOfWarp; ++i) {
      const int all = __reduce_add_sync(kFullMask, found[i]);
      if (lane == 0) place[warp * kRowsOfWarp + i] = all;
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
    int64_t before = carry;
#pragma unroll
    for (int k = 0; k < kBlocks; ++k) {
      int total;
      if constexpr (kBlocks > 1) {
        total = *cg::this_cluster().map_shared_rank(&block_total[round], k);
      } else {
        total = block_total[round];
      }
      if (k < rank) before += total;
      carry += total;
    }
    int64_t at[kRowsOfWarp];
#pragma unroll
    for (int i = 0; i < kRowsOfWarp; ++i) at[i] = before + place[warp * kRowsOfWarp + i];
    over_entries([&](int i, bool back, int id) {
      const unsigned set = __ballot_sync(kFullMask, back);
      const int64_t mine = at[i] + __popc(set & ((1u << lane) - 1));
      if (back && mine < a.pool) a.free_blocks[mine] = id;
      at[i] += __popc(set);
    });
    __syncthreads();  // the next round's lengths and counts follow these reads
  }
  // no block leaves while another may still read its total
  step_barrier<kBlocks>();
  if (rank == 0 && tid == 0) {
    *a.free_count_out = static_cast<int32_t>(min(carry, static_cast<int64_t>(a.pool)));
  }
}

int check_pool(const void* free_blocks, int64_t pool, const void* free_count, const void* count_out,
               int64_t requests, int64_t width, int64_t table_stride, int64_t block_size) {
  if (requests < 0 || width < 0 || pool < 0 || requests > INT32_MAX || width > INT32_MAX) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "requests, table width and pool size must be in [0, 2^31)");
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
  clear_error();
  int rc = check_pool(free_blocks, pool, free_count, free_count_out, requests, table_width,
                      table_stride, block_size);
  if (rc != SM120N_OK) return rc;
  if (tokens < 0 || tokens > INT32_MAX) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "tokens must be in [0, 2^31)");
  }
  if (!query_start || (requests > 0 && (!context_lens || !query_lens || !seq_lens)) ||
      (requests > 0 && table_width > 0 && !block_table) ||
      (tokens > 0 && (!positions || !slot_mapping))) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "tensor pointers must be non-null");
  }
  const PlanArgs a{context_lens, query_lens, block_table, free_blocks, free_count, free_count_out,
                   query_start, seq_lens, positions, slot_mapping, table_stride, tokens,
                   static_cast<int>(requests), static_cast<int>(table_width),
                   static_cast<int>(pool), static_cast<int>(block_size)};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  // A token to a thread of one block, then four, then four to a thread of a
  // cluster: 1024 decodes 4.6 us with one token to a thread, 5.6 with four.
  if (tokens <= kPlanThreads) {
    return launch(plan_step_kernel<1, 1>, dim3(1), dim3(plan_threads(std::max(requests, tokens))), 0,
                  s, a);
  }
  if (tokens <= 4 * kPlanThreads) {
    return launch(plan_step_kernel<1, 4>, dim3(1), dim3(kPlanThreads), 0, s, a);
  }
  return launch(plan_step_kernel<kPlanCluster, 4>, dim3(kPlanCluster), dim3(kPlanThreads), 0, s, a);
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
