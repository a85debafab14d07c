// attention_tc.cu -- attention on the fifth-generation tensor cores, for head
// sizes 64 and 128: causal attention of packed prompts, and the shared prefix
// of a decode batch.
//
// A block works on 256 rows of one key head -- (token, head of the group) of a
// prompt, or (request, head of the group) of a decode batch -- as two tiles of
// 128, against tiles of 128 keys:
//   S_i = Q_i K^T      tcgen05.mma, both operands in shared memory -> TMEM
//   P_i = 2^(scale S_i - m_i)   one thread per row; TMEM -> registers -> TMEM
//   O_i += P_i V       tcgen05.mma, P from TMEM, V in shared memory -> TMEM
// S_i takes 128 columns of tensor memory and O_i takes D. At D = 128 that is all
// 512, so P_i lies in the first half of S_i and S_i of the next key tile follows
// the product with P_i; while the 128 threads of one tile exponentiate, the
// tensor cores work on the other tile. At D = 64 P_i has columns of its own, and
// the next S_i is formed as soon as this one has been read. Both products of a
// tile pair take 2048 cycles at D = 128, and so do the pair's 32768
// exponentials on the special-function units (16 a cycle).
//
// Warps 0-3 and 4-7: softmax and epilogue of tile 0 and 1, a thread to a row, so
// that no reduction crosses threads (two threads to a row, sharing the maximum
// through shared memory, measured slower: 1898 us against 1782 for 16384
// tokens). Warp 8: issues the matrix instructions; at D = 64 only tile 0's, and
// warp 9 tile 1's, since there the waits for one tile would hold up the other
// (4096 tokens: 110 us with two issuers, 116 with one; at D = 128, where the
// tiles take turns, 158 with two and four more warps, 146 with one). The next
// warp loads K and V tiles by TMA into kStages shared-memory stages. The rest of
// the warps (prompts) look for infinite or NaN values in the V tiles that
// some rows must not see, where a product would multiply them by zero; a block
// that meets one does its rows by plain arithmetic instead. Q and O go through
// shared memory so that global accesses are whole rows: a thread reading or
// writing its own row touches 32 lines in every instruction of its warp (4000
// cycles for a block's rows).
//
// Prefixes in fp8 caches run as fp16: TMA brings raw tiles to a ring of their
// own, and six warps (five at D = 64) convert them into the stages, exactly (two
// warps took 3.5 us to a pair of tiles, where the products and exponentials
// take 2). Each row of q is scaled by a power of two into [1, 2) first (exact but
// for elements 2^14 below the row's largest) and the power goes into the row's
// score scale.
//
// The running maximum of a row follows the true one only when that has grown
// by more than 2^8 (kSlack): p then stays below 256, exact enough in 16 bits
// at any scale, and O is hardly ever rescaled; the softmax threads do it
// themselves, between S_j (whose completion implies that of the product
// before it) and the release of P_j.
//
// scale * s - m is one fused operation: the product is not rounded, m is. Past
// kFar that difference is no longer small against the exponent (2^27: p past fp16,
// 2^31: infinite); there products are rounded as m was, a step of their own.
//
// Every wait on an mbarrier is bounded; one that runs out is counted
// (sm120s_get_device_faults) and ends the block: a prompt's rows that are not
// finished then are left as they were, a prefix's are marked for the kernel that
// joins them.
#include <algorithm>
#include <cfloat>

#include "attention.h"
#include "attention_utils.cuh"
#include "tensor_core.cuh"
#include "tensor_map.h"

namespace sm120n {

__device__ unsigned int g_attention_expired_waits = 0;

namespace {

constexpr int kTileRows = 128;
constexpr int kTileKeys = 128;
constexpr uint32_t kBoxBytes = kTileKeys * 128;  // 64 elements of 128 rows
constexpr float kSlack = 8.0f;                   // log2 of how far a maximum may lag
constexpr float kFar = 1u << 22;                 // scaled scores whose last place is 1/2

enum Pass : int { kPrompt, kPrefix };

// A block of one or two row tiles. Two share K and V and fill the SM. One
// leaves room for a second block: half the rows to a block and twice as many
// blocks, which spread more evenly over the SMs.
template <int D, int kTiles, bool kFp8 = false>
struct TcShape {
  static constexpr int kStages =  // K and V tiles alternate: even
      kTiles == 2 ? (D == 64 ? 8 : 4) : (D == 64 ? 4 : 2);
  static constexpr uint32_t kTileBytes = kTileKeys * D * 2;
  static constexpr uint32_t kQBytes = kTileRows * D * 2;
  static constexpr int kRawTiles = D == 64 ? 4 : 2;  // fp8 tiles on their way to be converted
  static constexpr uint32_t kRawBytes = kTileKeys * D;
  static constexpr size_t kSmem =
      kTiles * kQBytes + kStages * kTileBytes + (kFp8 ? kRawTiles * kRawBytes : 0) + 1024;
  static constexpr uint32_t kOutColumn = kTiles * kTileKeys;  // of tile 0; tile 1 is D further
  static constexpr bool kOwnP = D == 64;  // P beside S, 64 columns for each tile
  static constexpr uint32_t kPColumn = kOwnP ? kOutColumn + kTiles * D : 0;
  static constexpr uint32_t kPStep = kOwnP ? kTileKeys / 2 : kTileKeys;
  static constexpr uint32_t kTmemColumns = kTiles * 256;
  static constexpr int kSoftmaxWarps = 4 * kTiles;
  static constexpr int kIssuers = D == 64 ? kTiles : 1;
  static constexpr int kLoadWarp = kSoftmaxWarps + kIssuers;
  static constexpr int kWarps = kSoftmaxWarps + (kFp8 ? 8 : 4);
  static constexpr int kThreads = kWarps * kWarpSize;
  static constexpr int kGuardWarps = kWarps - kLoadWarp - 1;  // look on, or convert
  // Registers at launch: 168 for 384 threads, 128 for 512 and for each of two
  // blocks of 256; 2 x 208 + 88 = 3 x 168, 2 x 208 + 2 x 48 = 4 x 128 and
  // 208 + 48 = 2 x 128.
  static constexpr int kSoftmaxRegisters = 208;
  static constexpr int kOtherRegisters = kTiles == 2 && !kFp8 ? 88 : 48;
};

// Instruction descriptor of tcgen05.mma.kind::f16: fp32 accumulator (bit 4), the
// operands' type (bits 7 and 10: 0 fp16, 1 bf16), B with its outer dimension
// contiguous (bit 16), N >> 3 at bit 17, M >> 4 at bit 24.
template <typename T>
__device__ __forceinline__ constexpr uint32_t instruction(int n, bool outer_b) {
  const uint32_t type = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (type << 7) | (type << 10) | (outer_b ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kTileRows >> 4) << 24);
}

// Descriptor of a V tile as B of the second product: d contiguous (64 of them
// in a 128-byte swizzled row, the next 64 a box further: leading offset), keys
// in groups of 8 rows, 1024 bytes apart (stride offset).
__device__ __forceinline__ uint64_t value_descriptor(const void* tile) {
  const uint64_t address = shared_address(tile);
  return ((address & 0x3FFFFull) >> 4) | (uint64_t{kBoxBytes >> 4} << 16) |
         (uint64_t{1024 >> 4} << 32) | (uint64_t{1} << 46) | (uint64_t{2} << 61);
}

__device__ __forceinline__ void mma_from_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc,
                                              uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 columns of this thread's TMEM lane; the values may be used after tmem_wait_load.
__device__ __forceinline__ void tmem_load32_async(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]),
        "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]),
        "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}

// Waits for this thread's TMEM loads; the empty statements keep every use of
// the loaded values behind the wait.
template <int N>
__device__ __forceinline__ void tmem_wait_load(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));
}

__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
      "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
      "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_store() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

template <int kRegisters>
__device__ __forceinline__ void grow_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegisters));
}
template <int kRegisters>
__device__ __forceinline__ void shrink_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegisters));
}
// What a block works on. Row r is head (first_head + r) % group of the group and
// token (or request) first_token + (first_head + r) / group.
struct Work {
  int64_t first_token;  // within the sequence
  int64_t token0;       // kPrompt: the sequence's first token
  int first_head;
  int rows;       // up to 128 for each row tile
  int key_first;  // kPrefix: first key of its part of the prefix
  int key_last;
  int kv_head;
  int split;  // kPrefix
};

template <int kTiles>
__device__ __forceinline__ void place_rows(Work& w, int64_t first_row, int64_t all_rows, int group) {
  w.first_token = first_row / group;
  w.first_head = static_cast<int>(first_row - w.first_token * group);
  w.rows = static_cast<int>(min(int64_t{kTiles * kTileRows}, all_rows - first_row));
}

struct Barriers {
  uint64_t full[8];
  uint64_t empty[8];
  uint64_t raw_full[4];
  uint64_t raw_empty[4];
  uint64_t q_full;
  uint64_t s_full[2];
  uint64_t p_ready[2];
  uint64_t o_full[2];
  uint64_t s_free[2];   // kOwnP: S has been read
  uint64_t p_free[2];   // kOwnP: the product with P is complete
  uint64_t guarded;
  uint64_t done;
};

struct Control {
  Barriers bar;
  uint32_t tmem;
  int aborted;
  int unsafe;  // a value that some rows must not see is infinite or NaN
  int holes;   // kPrefix: a block of the prefix does not exist
  int loads;   // tiles that the loader has asked for
};

// By a whole warp.
__device__ __forceinline__ bool wait_in(Control& c, uint64_t* bar, uint32_t parity, uint32_t polls) {
  if (mbarrier_wait_warp(bar, parity, polls)) return true;
  if ((threadIdx.x & (kWarpSize - 1)) == 0) {
    atomicAdd(&g_attention_expired_waits, 1u);
    atomicExch(&c.aborted, 1);
  }
  __syncwarp();
  return false;
}

// Token (or request) and head of a row, the head among all query heads.
struct RowPlace {
  int64_t token;  // within the sequence
  int64_t head;
};
template <typename Args>
__device__ __forceinline__ RowPlace row_place(const Args& a, const Work& w, int row) {
  const uint32_t r = static_cast<uint32_t>(w.first_head + row);
  const uint32_t step = r / static_cast<uint32_t>(a.group);
  return RowPlace{w.first_token + step,
                  static_cast<int64_t>(w.kv_head) * a.group + (r - step * a.group)};
}

// fp8: raw tiles, which TMA has brought, into the swizzled fp16 stages. A thread
// has 16 bytes of a row at a time, 32 in the stage.
template <typename S, int D>
__device__ __forceinline__ void convert_tiles(Control& c, unsigned char* stages,
                                              const unsigned char* raw_tiles, int tiles, int thread,
                                              uint32_t polls) {
  constexpr int kRowChunks = D / 16;
  constexpr int kAll = kTileKeys * kRowChunks;
  for (int t = 0; t < 2 * tiles; ++t) {
    const int stage = t % S::kStages;
    const int slot = t % S::kRawTiles;
    if (!wait_in(c, &c.bar.raw_full[slot], (t / S::kRawTiles) & 1, polls)) return;
    if (t >= S::kStages && !wait_in(c, &c.bar.empty[stage], (t / S::kStages - 1) & 1, polls)) return;
    const unsigned char* raw = raw_tiles + slot * S::kRawBytes;
    unsigned char* to = stages + stage * S::kTileBytes;
#pragma unroll 4
    for (int at = thread; at < kAll; at += S::kGuardWarps * kWarpSize) {
      const uint4 v = load16_shared(raw + at * 16);
      const int row = at / kRowChunks;
      const int chunk = 2 * (at % kRowChunks);  // of 16 bytes in the stage
      const uint32_t words[4] = {v.x, v.y, v.z, v.w};
      uint32_t h[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) e4m3_to_half(words[e], h[2 * e], h[2 * e + 1]);
      unsigned char* box = to + (chunk / 8) * kBoxBytes + row * 128;
      *reinterpret_cast<uint4*>(box + ((chunk % 8) ^ (row & 7)) * 16) =
          make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint4*>(box + (((chunk + 1) % 8) ^ (row & 7)) * 16) =
          make_uint4(h[4], h[5], h[6], h[7]);
    }
    fence_async_shared();
    __syncwarp();
    if ((threadIdx.x & (kWarpSize - 1)) == 0) {
      mbarrier_arrive(&c.bar.full[stage]);
      mbarrier_arrive(&c.bar.raw_empty[slot]);
    }
  }
}

// TQ: type of q and out; T: operand type of the products.
template <typename TQ, typename T, bool kFp8, int D, int kTiles, int kPass, typename Args>
__device__ __forceinline__ void attend(const Args& a, const Work& w, const CUtensorMap* key_map,
                                       const CUtensorMap* value_map, Control& c, unsigned char* smem) {
  using S = TcShape<D, kTiles, kFp8>;
  constexpr int kStages = S::kStages;
  const int warp = __shfl_sync(kFullMask, threadIdx.x / kWarpSize, 0);  // known to be uniform
  const int lane = threadIdx.x & (kWarpSize - 1);
  unsigned char* stages = smem + kTiles * S::kQBytes;
  unsigned char* raw_tiles = stages + kStages * S::kTileBytes;

  // key tiles of each row tile
  int n[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    const int rows = min(w.rows - i * kTileRows, kTileRows);
    if (rows <= 0) {
      n[i] = 0;
    } else if constexpr (kPass == kPrompt) {
      n[i] = static_cast<int>(row_place(a, w, i * kTileRows + rows - 1).token / kTileKeys + 1);
    } else {
      n[i] = (w.key_last - w.key_first + kTileKeys - 1) / kTileKeys;
    }
  }
  const int tiles = max(n[0], n[1]);

  if (warp < S::kSoftmaxWarps) {
    grow_registers<S::kSoftmaxRegisters>();
    const int i = warp / 4;
    const int warp_row = (warp % 4) * kWarpSize;  // of the tile
    const int row = i * kTileRows + warp_row + lane;
    const RowPlace place = row_place(a, w, row);
    const int live_rows = min(max(w.rows - (row - lane), 0), kWarpSize);  // of the warp
    unsigned char* rows_smem = smem + i * S::kQBytes + warp_row * 128;  // of the warp, in each box
    float scale = a.scale_log2;
    float sign = 1.0f;  // of the keys' scale: goes into Q, so that larger products are larger scores
    if constexpr (kFp8) {
      const float k_scale = *a.k_scale;
      sign = copysignf(1.0f, k_scale);
      scale *= fabsf(k_scale);
    }
    // Q of the warp's rows into the swizzled operand layout, whole rows at a time
    {
      constexpr int kChunks = D / 8;
      constexpr int kRowsAtOnce = kWarpSize / kChunks;
      constexpr int kBatch = 16;  // all loads of a 128-wide head in flight
      const TQ* query = static_cast<const TQ*>(a.query) + (lane % kChunks) * 8;
      const int64_t offset = (w.token0 + place.token) * a.query_stride + place.head * D;
      constexpr int kLoads = kWarpSize / kRowsAtOnce < kBatch ? kWarpSize / kRowsAtOnce : kBatch;
#pragma unroll 1
      for (int r0 = 0; r0 < kWarpSize; r0 += kLoads * kRowsAtOnce) {
        uint4 v[kLoads];
#pragma unroll
        for (int t = 0; t < kLoads; ++t) {
          const int r = r0 + t * kRowsAtOnce + lane / kChunks;
          const int64_t at = __shfl_sync(kFullMask, offset, r);
          v[t] = r < live_rows ? load16(query + at) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < kLoads; ++t) {
          const int r = r0 + t * kRowsAtOnce + lane / kChunks;
          if constexpr (kFp8) {
            float f[8];
            Pack<TQ>::to_f32(v[t], f);
            float most = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(f[e]));
#pragma unroll
            for (int d = 1; d < kChunks; d *= 2) most = fmaxf(most, __shfl_xor_sync(kFullMask, most, d));
            // 2^-e and 2^e with e the exponent of the row's largest, kept normal
            const int e = min(max(static_cast<int>(__float_as_uint(most) >> 23), 2), 252);
            const float down = sign * __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] *= down;
            v[t] = Pack<T>::from_f32(f);
            const float up = __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
            for (int k = 0; k < kRowsAtOnce; ++k) {
              const float mine = __shfl_sync(kFullMask, up, k * kChunks);
              if (lane == r0 + t * kRowsAtOnce + k) scale *= mine;
            }
          }
          const int chunk = lane % kChunks;
          *reinterpret_cast<uint4*>(rows_smem + (chunk / 8) * kBoxBytes + r * 128 +
                                    ((chunk % 8) ^ (r & 7)) * 16) = v[t];
        }
      }
      // The scores are then zero to every bit, but the first maximum still counts
      // as larger than none: infinity times zero would not.
      if (kFp8 && scale < FLT_MIN) scale = FLT_MIN;
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbarrier_arrive(&c.bar.q_full);
    }
    const uint32_t lane_base = c.tmem + (static_cast<uint32_t>(warp_row) << 16);
    const uint32_t s_at = lane_base + i * kTileKeys;
    const uint32_t p_at = lane_base + S::kPColumn + i * S::kPStep;
    const uint32_t o_at = lane_base + S::kOutColumn + i * D;
    float top = -INFINITY;  // raw maximum that `base` follows
    float base = 0.0f;      // scale * the maximum in use
    float sum = 0.0f;
    float step = scale;     // 1 where some row of the warp has |base| > kFar
    // last key of the row, counted from the first key tile's first
    const int64_t limit = kPass == kPrompt ? place.token : int64_t{w.key_last} - w.key_first - 1;
    const int64_t first_limit =  // smallest of the tile: tiles behind it need no mask
        kPass == kPrompt ? row_place(a, w, i * kTileRows).token : limit;
    bool ok = true;
    for (int j = 0; j < n[i]; ++j) {
      if (!wait_in(c, &c.bar.s_full[i], j & 1, a.wait_polls)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t raw[kTileKeys];
#pragma unroll
      for (int q = 0; q < kTileKeys / 32; ++q) tmem_load32_async(s_at + 32 * q, raw + 32 * q);
      tmem_wait_load<kTileKeys>(raw);
      if constexpr (S::kOwnP) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbarrier_arrive(&c.bar.s_free[i]);
      }
      float* s = reinterpret_cast<float*>(raw);
      const int64_t key0 = int64_t{j} * kTileKeys;
      // Tiles that some row must not see whole: `last` is the row's last key of
      // the tile. It does not fall from lane to lane, so lane 0 tells which runs
      // of 32 keys need no mask.
      if (key0 + kTileKeys - 1 > first_limit) {
        const int last = static_cast<int>(max(min(limit - key0, int64_t{kTileKeys}), int64_t{-1}));
        const int all_see = __shfl_sync(kFullMask, last, 0) + 1;
#pragma unroll
        for (int q = 0; q < kTileKeys / 32; ++q) {
          if (32 * q + 32 > all_see) {
#pragma unroll
            for (int k = 32 * q; k < 32 * q + 32; ++k) {
              if (k > last) s[k] = -INFINITY;
            }
          }
        }
      }
      if constexpr (kPass == kPrefix) {
        if (*reinterpret_cast<volatile int*>(&c.holes)) {
#pragma unroll
          for (int k = 0; k < kTileKeys; ++k) {
            const int64_t key = min(w.key_first + key0 + k, int64_t{a.prefix_tokens} - 1);
            const int id = a.prefix_blocks[key / a.kv.block_size];
            if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(a.kv.num_blocks)) s[k] = -INFINITY;
          }
        }
      }
      float m0 = s[0], m1 = s[1], m2 = s[2], m3 = s[3];
#pragma unroll
      for (int k = 4; k < kTileKeys; k += 4) {
        m0 = fmaxf(m0, s[k]);
        m1 = fmaxf(m1, s[k + 1]);
        m2 = fmaxf(m2, s[k + 2]);
        m3 = fmaxf(m3, s[k + 3]);
      }
      const float next = fmaxf(fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)), top);
      if constexpr (S::kOwnP) {
        // P and O are free for this tile once the last product is complete
        if (j > 0 && !wait_in(c, &c.bar.p_free[i], (j - 1) & 1, a.wait_polls)) {
          ok = false;
          break;
        }
        tc_fence_after();
      }
      const bool lags = (next - top) * scale > kSlack;  // also where top is still -inf
      if (__any_sync(kFullMask, lags)) {
        const float moved = lags ? next * scale : base;
        const float keep = lags ? exp2_approx(top == -INFINITY ? -INFINITY : base - moved) : 1.0f;
        if (j > 0) {
#pragma unroll 1
          for (int q = 0; q < D / 32; ++q) {
            uint32_t o[32];
            tmem_load32_async(o_at + 32 * q, o);
            tmem_wait_load<32>(o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
            tmem_store32(o_at + 32 * q, o);
          }
        }
        sum *= keep;
        base = moved;
        if (lags) top = next;
        step = __any_sync(kFullMask, fabsf(base) > kFar) ? 1.0f : scale;
      }
      if (__builtin_expect(step != scale, 0)) {
#pragma unroll
        for (int k = 0; k < kTileKeys; ++k) s[k] = __fmul_rn(s[k], scale);
      }
      const float2 factor = make_float2(step, step);
      const float2 shift = make_float2(-base, -base);
      float2 sum_a = make_float2(0.f, 0.f), sum_b = make_float2(0.f, 0.f);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t p[32];
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const int at = 64 * q + 2 * k;
          float2 x = __ffma2_rn(make_float2(s[at], s[at + 1]), factor, shift);
          float2 y = __ffma2_rn(make_float2(s[at + 2], s[at + 3]), factor, shift);
          x = make_float2(exp2_approx(x.x), exp2_approx(x.y));
          y = make_float2(exp2_approx(y.x), exp2_approx(y.y));
          sum_a = __fadd2_rn(sum_a, x);
          sum_b = __fadd2_rn(sum_b, y);
          p[k] = Pack<T>::f32_to_word(x.x, x.y);
          p[k + 1] = Pack<T>::f32_to_word(y.x, y.y);
        }
        tmem_store32(p_at + 32 * q, p);
      }
      sum_a = __fadd2_rn(sum_a, sum_b);
      sum += sum_a.x + sum_a.y;
      tmem_wait_store();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbarrier_arrive(&c.bar.p_ready[i]);
    }
    if (ok && n[i] > 0) ok = wait_in(c, &c.bar.o_full[i], 0, a.wait_polls);
    if constexpr (kPass == kPrompt) {
      if (ok) ok = wait_in(c, &c.bar.guarded, 0, a.wait_polls);
    }
    ok = ok && !*reinterpret_cast<volatile int*>(&c.aborted);
    ok = __all_sync(kFullMask, ok);
    tc_fence_after();
    if constexpr (kPass == kPrefix) {
      if (!ok && lane < live_rows) {
        a.prefix_state[(static_cast<int64_t>(w.split) * a.batch + place.token) * a.query_heads +
                       place.head] = make_float2(-INFINITY, NAN);
      }
    }
    if (ok && live_rows > 0) {
      if (kPass == kPrompt && *reinterpret_cast<volatile int*>(&c.unsafe)) {
        if constexpr (kPass == kPrompt) {
          for (int r = 0; r < live_rows; ++r) {
            const RowPlace to = row_place(a, w, row - lane + r);
            plain_prompt_row<T, D>(a, w.token0, to.token, to.head, w.kv_head);
          }
        }
      } else {
        // O through the warp's rows of the Q tile (its products are complete),
        // kColumns at a time: 64 of fp32 partials, 128 bytes a row and box
        constexpr int kElem = kPass == kPrompt ? 2 : 4;
        constexpr int kColumns = kPass == kPrompt ? D : D / 2;
        constexpr int kChunks = kColumns * kElem / 16;
        constexpr int kRowsAtOnce = kWarpSize / kChunks;
        const float inv = kPass == kPrompt ? 1.0f / sum : 1.0f;
        unsigned char* out;
        int64_t offset;  // bytes, of this lane's row
        if constexpr (kPass == kPrompt) {
          out = static_cast<unsigned char*>(a.out);
          offset = ((w.token0 + place.token) * a.out_stride + place.head * D) * kElem;
        } else {
          const int64_t at = (static_cast<int64_t>(w.split) * a.batch + place.token) * a.query_heads +
                             place.head;
          if (lane < live_rows) {
            a.prefix_state[at] = make_float2(top == -INFINITY ? -INFINITY : base, sum);
          }
          out = reinterpret_cast<unsigned char*>(a.prefix_values);
          offset = at * D * kElem;
        }
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += kColumns) {
#pragma unroll
          for (int q = 0; q < kColumns / 32; ++q) {
            uint32_t o[32];
            tmem_load32_async(o_at + c0 + 32 * q, o);
            tmem_wait_load<32>(o);
            float* f = reinterpret_cast<float*>(o);
            constexpr int kPerChunk = 16 / kElem;
#pragma unroll
            for (int k = 0; k < 32 / kPerChunk; ++k) {
              const int chunk = q * (32 / kPerChunk) + k;
              uint4 v;
              if constexpr (kPass == kPrompt) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[8 * k + e] *= inv;
                v = Pack<TQ>::from_f32(f + 8 * k);
              } else {
                v = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
              }
              *reinterpret_cast<uint4*>(rows_smem + (chunk / 8) * kBoxBytes + lane * 128 +
                                        ((chunk % 8) ^ (lane & 7)) * 16) = v;
            }
          }
          __syncwarp();
#pragma unroll 4
          for (int r0 = 0; r0 < kWarpSize; r0 += kRowsAtOnce) {
            const int r = r0 + lane / kChunks;
            const int chunk = lane % kChunks;
            const int64_t at = __shfl_sync(kFullMask, offset, r);
            if (r < live_rows) {
              store16(out + at + c0 * kElem + chunk * 16,
                      load16_shared(rows_smem + (chunk / 8) * kBoxBytes + r * 128 +
                                    ((chunk % 8) ^ (r & 7)) * 16));
            }
          }
          __syncwarp();
        }
      }
    }
  } else {
    shrink_registers<S::kOtherRegisters>();
    if (warp < S::kLoadWarp) {
      // The whole warp keeps step; the instructions are one lane's.
      constexpr uint32_t kScore = instruction<T>(kTileKeys, false);
      constexpr uint32_t kValue = instruction<T>(D, true);
      const int issuer = warp - S::kSoftmaxWarps;
      const uint32_t tmem = c.tmem;
      const uint64_t first_key = smem_descriptor(stages);
      const uint64_t first_value = value_descriptor(stages);
      auto full = [&](int t) { return wait_in(c, &c.bar.full[t % kStages], (t / kStages) & 1, a.wait_polls); };
      auto score = [&](int i, int t) {  // with the key tile of stage use t
        const uint64_t q = smem_descriptor(smem + i * S::kQBytes);
        const uint64_t k = first_key + (t % kStages) * (S::kTileBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          // 16 elements along d: 32 bytes inside a box, then the next box
          const uint32_t step = (kk / 4) * (kBoxBytes >> 4) + 2 * (kk % 4);
          mma_bf16(tmem + i * kTileKeys, q + step, k + step, kScore, kk != 0);
        }
        mma_commit(&c.bar.s_full[i]);
      };
      auto weigh = [&](int i, int t) {  // with the value tile of stage use t
        const uint64_t v = first_value + (t % kStages) * (S::kTileBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < kTileKeys / 16; ++kk) {
          mma_from_tmem(tmem + S::kOutColumn + i * D, tmem + S::kPColumn + i * S::kPStep + 8 * kk,
                        v + kk * (2048 >> 4), kValue, t > 1 || kk != 0);
        }
        if (t / 2 == n[i] - 1) {
          mma_commit(&c.bar.o_full[i]);
        } else if (S::kOwnP) {
          mma_commit(&c.bar.p_free[i]);
        }
      };
      auto mine = [&](int i) { return S::kIssuers == 1 || i == issuer; };
      // A stage is free once every issuer has committed behind its products with it.
      bool ok = wait_in(c, &c.bar.q_full, 0, a.wait_polls) && full(0);
      tc_fence_after();
      if (ok && elect_lane()) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          if (mine(i) && n[i] > 0) score(i, 0);
        }
        mma_commit(&c.bar.empty[0]);
      }
      for (int j = 0; ok && j < tiles; ++j) {
        const bool more = j + 1 < tiles;
        if (S::kOwnP && more) {
          ok = full(2 * j + 2);
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            if (!ok || !mine(i) || j + 1 >= n[i]) continue;
            ok = wait_in(c, &c.bar.s_free[i], j & 1, a.wait_polls);
            tc_fence_after();
            if (ok && elect_lane()) score(i, 2 * j + 2);
          }
          if (ok && elect_lane()) mma_commit(&c.bar.empty[(2 * j + 2) % kStages]);
        }
        ok = ok && full(2 * j + 1) && (S::kOwnP || !more || full(2 * j + 2));
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          if (!ok || !mine(i) || j >= n[i]) continue;
          ok = wait_in(c, &c.bar.p_ready[i], j & 1, a.wait_polls);
          tc_fence_after();
          if (ok && elect_lane()) {
            weigh(i, 2 * j + 1);
            if (!S::kOwnP && j + 1 < n[i]) score(i, 2 * j + 2);
          }
        }
        if (ok && elect_lane()) {
          mma_commit(&c.bar.empty[(2 * j + 1) % kStages]);
          if (!S::kOwnP && more) mma_commit(&c.bar.empty[(2 * j + 2) % kStages]);
        }
      }
      if (elect_lane()) mma_commit(&c.bar.done);
    } else if (warp == S::kLoadWarp) {
      int t = 0;
      for (; t < 2 * tiles; ++t) {
        const int ring = kFp8 ? S::kRawTiles : kStages;
        const int slot = t % ring;
        uint64_t* loaded = kFp8 ? &c.bar.raw_full[slot] : &c.bar.full[slot];
        uint64_t* emptied = kFp8 ? &c.bar.raw_empty[slot] : &c.bar.empty[slot];
        if (*reinterpret_cast<volatile int*>(&c.aborted)) break;
        if (t >= ring && !wait_in(c, emptied, (t / ring - 1) & 1, a.wait_polls)) break;
        const CUtensorMap* map = t & 1 ? value_map : key_map;
        const int key0 = (t / 2) * kTileKeys;
        if constexpr (kPass == kPrompt) {
          unsigned char* to = stages + slot * S::kTileBytes;
          if (elect_lane()) {
            mbarrier_arrive_expect_tx(loaded, S::kTileBytes);
#pragma unroll
            for (int h = 0; h < D / 64; ++h) {
              tma_load_2d(to + h * kBoxBytes, map, w.kv_head * D + 64 * h,
                          static_cast<int>(w.token0) + key0, loaded);
            }
          }
        } else {
          // One box to a block of the cache (or 128 slots of a larger one) and
          // 128 bytes of a row. Lane b finds box b; one lane asks for all of
          // them. Blocks that do not exist, and what is behind the end, lie
          // outside the map and arrive as zeros.
          constexpr int kBoxes = kFp8 ? 1 : D / 64;
          const int row_bytes = kFp8 ? D : 128;
          unsigned char* to = kFp8 ? raw_tiles + slot * S::kRawBytes : stages + slot * S::kTileBytes;
          const int box = min(a.kv.block_size, kTileKeys);
          const int64_t key = int64_t{w.key_first} + key0 + lane * box;
          int id = a.kv.num_blocks, first_slot = 0;
          if (lane * box < kTileKeys && key < w.key_last) {
            const uint32_t block = static_cast<uint32_t>(key) / static_cast<uint32_t>(a.kv.block_size);
            const int found = a.prefix_blocks[block];
            if (static_cast<uint32_t>(found) < static_cast<uint32_t>(a.kv.num_blocks)) {
              id = found;
              first_slot = static_cast<int>(key - static_cast<int64_t>(block) * a.kv.block_size);
            } else {
              *reinterpret_cast<volatile int*>(&c.holes) = 1;  // before the tile can arrive
            }
          }
          __syncwarp();
          if (elect_lane()) mbarrier_arrive_expect_tx(loaded, kFp8 ? S::kRawBytes : S::kTileBytes);
          for (int b = 0; b < kTileKeys / box; ++b) {
            const int block = __shfl_sync(kFullMask, id, b);
            const int at = __shfl_sync(kFullMask, first_slot, b);
            if (elect_lane()) {
#pragma unroll
              for (int h = 0; h < kBoxes; ++h) {
                tma_load_4d(to + h * kBoxBytes + b * box * row_bytes, map, 64 * h, at, w.kv_head,
                            block, loaded);
              }
            }
          }
        }
      }
      if (lane == 0) c.loads = t;
    } else if (kFp8) {
      if constexpr (kFp8) {
        convert_tiles<S, D>(c, stages, raw_tiles, tiles,
                            (warp - S::kLoadWarp - 1) * kWarpSize + lane, a.wait_polls);
      }
    } else if (kPass == kPrompt) {
      // V tiles that reach past the block's first row's last key
      constexpr uint32_t kExponent = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
      const int64_t first_limit = w.first_token;
      bool bad = false;
      for (int j = 0; j < tiles; ++j) {
        const int stage = (2 * j + 1) % kStages;
        if (!wait_in(c, &c.bar.full[stage], ((2 * j + 1) / kStages) & 1, a.wait_polls)) break;
        if (int64_t{j + 1} * kTileKeys - 1 > first_limit) {
          const uint4* v = reinterpret_cast<const uint4*>(stages + stage * S::kTileBytes);
#pragma unroll 4
          for (int t = (warp - S::kLoadWarp - 1) * kWarpSize + lane;
               t < static_cast<int>(S::kTileBytes / 16); t += S::kGuardWarps * kWarpSize) {
            const uint4 x = v[t];
            const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              bad |= (words[k] & kExponent) == kExponent || ((words[k] >> 16) & kExponent) == kExponent;
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbarrier_arrive(&c.bar.empty[stage]);
      }
      if (bad) *reinterpret_cast<volatile int*>(&c.unsafe) = 1;
      __threadfence_block();
      __syncwarp();
      if (lane == 0) mbarrier_arrive(&c.bar.guarded);
    }
  }
  __syncwarp();
}

// Set-up and release around attend(): barriers, tensor memory.
template <typename S>
__device__ __forceinline__ void open_block(Control& c, bool guarded, bool converted) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbarrier_init(&c.bar.full[s], converted ? S::kGuardWarps : 1);
      mbarrier_init(&c.bar.empty[s], S::kIssuers + (guarded && (s & 1) ? S::kGuardWarps : 0));
    }
    for (int s = 0; converted && s < S::kRawTiles; ++s) {
      mbarrier_init(&c.bar.raw_full[s], 1);
      mbarrier_init(&c.bar.raw_empty[s], S::kGuardWarps);
    }
    mbarrier_init(&c.bar.q_full, S::kSoftmaxWarps);
    for (int i = 0; i < 2; ++i) {
      mbarrier_init(&c.bar.s_full[i], 1);
      mbarrier_init(&c.bar.p_ready[i], 4);
      mbarrier_init(&c.bar.s_free[i], 4);
      mbarrier_init(&c.bar.p_free[i], 1);
      mbarrier_init(&c.bar.o_full[i], 1);
    }
    mbarrier_init(&c.bar.guarded, S::kGuardWarps);
    mbarrier_init(&c.bar.done, S::kIssuers);
    c.aborted = 0;
    c.unsafe = 0;
    c.holes = 0;
    c.loads = 0;
    fence_mbarrier_init();
  }
  if (threadIdx.x / kWarpSize == S::kSoftmaxWarps) tmem_alloc(&c.tmem, S::kTmemColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
}

template <typename S, bool kFp8 = false>
__device__ __forceinline__ void close_block(Control& c) {
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x / kWarpSize == S::kSoftmaxWarps) {
    // the issuer's last commit: no matrix instruction is still at work
    if ((threadIdx.x & (kWarpSize - 1)) == 0) {
      mbarrier_wait_bounded(&c.bar.done, 0);
    }
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(c.tmem, S::kTmemColumns);
  }
  if (c.aborted && threadIdx.x == S::kLoadWarp * kWarpSize) {
    // an expired wait: the loads that are still on their way land first
    constexpr int kRing = kFp8 ? S::kRawTiles : S::kStages;
    uint64_t* landed = kFp8 ? c.bar.raw_full : c.bar.full;
    for (int t = max(c.loads - kRing, 0); t < c.loads; ++t) {
      mbarrier_wait_bounded(&landed[t % kRing], (t / kRing) & 1);
    }
  }
}

__device__ __forceinline__ unsigned char* aligned_tiles(unsigned char* p) {
  return reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~uintptr_t{1023});
}

template <typename T, int D, int kTiles>
__global__ void __launch_bounds__(TcShape<D, kTiles>::kThreads, 3 - kTiles)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap key_map,
                     const __grid_constant__ CUtensorMap value_map,
                     const __grid_constant__ PromptArgs a) {
  using S = TcShape<D, kTiles>;
  extern __shared__ unsigned char dynamic_smem[];
  __shared__ Control control;
  wait_for_upstream_grid();
  const SequenceTile tile = find_tile<kTiles * kTileRows>(a.query_start, a.sequences, a.tokens,
                                                          a.group, blockIdx.x / a.key_heads);
  if (tile.tile < 0) return;
  open_block<S>(control, true, false);
  // Not before this block has its tensor memory: blocks of the next kernel may take
  // theirs before they wait for this one, and would then hold what it waits for.
  release_downstream_grid();
  Work w{};
  place_rows<kTiles>(w, tile.tile * kTiles * kTileRows, tile.length * a.group, a.group);
  w.token0 = tile.first_token;
  w.kv_head = static_cast<int>(blockIdx.x % a.key_heads);
  attend<T, T, false, D, kTiles, kPrompt>(a, w, &key_map, &value_map, control,
                                          aligned_tiles(dynamic_smem));
  close_block<S>(control);
}

template <typename TQ, typename T, bool kFp8, int D>
__global__ void __launch_bounds__(TcShape<D, 2, kFp8>::kThreads, 1)
    prefix_tc_kernel(const __grid_constant__ CUtensorMap key_map,
                     const __grid_constant__ CUtensorMap value_map,
                     const __grid_constant__ DecodeArgs a) {
  using S = TcShape<D, 2, kFp8>;
  extern __shared__ unsigned char dynamic_smem[];
  __shared__ Control control;
  open_block<S>(control, false, kFp8);
  wait_for_upstream_grid();
  release_downstream_grid();
  Work w{};
  place_rows<2>(w, static_cast<int64_t>(blockIdx.x) * 2 * kTileRows,
                static_cast<int64_t>(a.batch) * a.group, a.group);
  w.kv_head = blockIdx.y;
  w.split = blockIdx.z;
  const int64_t tiles = (a.prefix_tokens + kTileKeys - 1) / kTileKeys;
  w.key_first = static_cast<int>(tiles * w.split / a.prefix_splits * kTileKeys);
  w.key_last = static_cast<int>(min(tiles * (w.split + 1) / a.prefix_splits * kTileKeys,
                                    int64_t{a.prefix_tokens}));
  attend<TQ, T, kFp8, D, 2, kPrefix>(a, w, &key_map, &value_map, control,
                                     aligned_tiles(dynamic_smem));
  close_block<S, kFp8>(control);
}

// ---- host ----------------------------------------------------------------------
// Blocks of one row tile spread evenly over the SMs and waste less where sequences
// end; blocks of two load K and V once for both. Two are taken behind
// kTwoTileHalfWaves two-tile blocks per SM, in halves, and at D = 128 for sequences
// of kTwoTiles of them on average. Measured (graph, 32/8 heads unless stated;
// one tile against two, two-tile blocks per SM in brackets):
// D = 128: 512 tokens 12.9 us against 14.8, 1024 (0.9) 19.5 against 22.1, 2500 (2.1)
// 60.8 against 61.9, but 2048 (1.7) 43.5 against 41.2; 4096 (3.5) 139.5 against 134.6,
// 64/8 heads 4096 (6.9) 288 against 278, 8192 (6.9) 507 against 491, 16384 (13.8) 1932
// against 1870. 64 prompts of 1-200 tokens (5.4; 1.6 tiles each) 70 against 78, 30 of
// 1-500 (6.3; 3.9) 85 against 89, 19 of 1-1500 (12; 12) even, 8 of 1-2000 (6.8; 16) 128
// against 126.
// D = 64: 1024 tokens 16.1 against 20.4, 4096 (3.5) even, 64 of 1-200 52 against 63, 19
// of 1-1500 (12) 145 against 161, 8192 (6.9) even; 16384 (13.8) 1383 against 1316.
template <int D>
constexpr int kTwoTileHalfWaves = D == 64 ? 24 : 5;
template <int D>
constexpr int kTwoTiles = D == 64 ? 0 : 10;

template <typename T, int D, int kTiles>
int run_prompt(const PromptArgs& a, const CUtensorMap* maps, cudaStream_t stream) {
  using S = TcShape<D, kTiles>;
  auto kernel = prompt_tc_kernel<T, D, kTiles>;
  const int rc = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), S::kSmem);
  if (rc != SM120N_OK) return rc;
  constexpr int64_t kRows = kTiles * kTileRows;
  const int64_t tiles = (a.tokens * a.group + kRows - 1) / kRows + a.sequences;
  return launch(kernel, dim3(static_cast<unsigned>(tiles * a.key_heads)), dim3(S::kThreads),
                S::kSmem, stream, maps[0], maps[1], a);
}

template <typename T, int D>
int run_prompt_tiles(const PromptArgs& a, cudaStream_t stream) {
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.key_heads) * D,
                                static_cast<cuuint64_t>(a.tokens)};
    // one token has no stride of its own
    const int64_t row = a.tokens > 1 ? (i ? a.value_stride : a.key_stride) : int64_t{a.key_heads} * D;
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row) * 2};
    const cuuint32_t box[2] = {64, kTileKeys};
    const int rc = encode_tensor_map(&maps[i], i ? a.value : a.key, tensor_map_type<T>(), 2, dims,
                                     strides, box, 128);
    if (rc != SM120N_OK) return rc;
  }
  DeviceInfo dev;
  const int rc = current_device_info(&dev);
  if (rc != SM120N_OK) return rc;
  const int64_t pairs = (a.tokens * a.group + 2 * kTileRows - 1) / (2 * kTileRows) * a.key_heads;
  const bool two = 2 * pairs > kTwoTileHalfWaves<D> * int64_t{dev.sm_count} &&
                   a.tokens * a.group >= int64_t{kTwoTiles<D>} * 2 * kTileRows * a.sequences;
  return two ? run_prompt<T, D, 2>(a, maps, stream) : run_prompt<T, D, 1>(a, maps, stream);
}

template <typename TQ, typename T, bool kFp8, int D>
int run_prefix(const DecodeArgs& a, cudaStream_t stream) {
  using S = TcShape<D, 2, kFp8>;
  CUtensorMap maps[2] = {};
  for (int i = 0; i < 2; ++i) {
    const int rc = encode_cache_map(&maps[i], i ? a.kv.value : a.kv.key, a.kv, D, a.key_heads,
                                    kFp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : tensor_map_type<T>(),
                                    kFp8 ? 1 : 2, kFp8 ? D : 128, kTileKeys, !kFp8);
    if (rc != SM120N_OK) return rc;
  }
  auto kernel = prefix_tc_kernel<TQ, T, kFp8, D>;
  const int rc = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), S::kSmem);
  if (rc != SM120N_OK) return rc;
  const int64_t tiles = (static_cast<int64_t>(a.batch) * a.group + 2 * kTileRows - 1) / (2 * kTileRows);
  return launch(kernel,
                dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(a.key_heads),
                     static_cast<unsigned>(a.prefix_splits)),
                dim3(S::kThreads), S::kSmem, stream, maps[0], maps[1], a);
}

template <int D>
int run_prefix_typed(const DecodeArgs& a, int dtype, bool fp8, cudaStream_t stream) {
  if (dtype == SM120N_F16) {
    return fp8 ? run_prefix<__half, __half, true, D>(a, stream)
               : run_prefix<__half, __half, false, D>(a, stream);
  }
  return fp8 ? run_prefix<__nv_bfloat16, __half, true, D>(a, stream)
             : run_prefix<__nv_bfloat16, __nv_bfloat16, false, D>(a, stream);
}

}  // namespace

int launch_prompt_tc(const PromptArgs& a, int dtype, int head_dim, cudaStream_t stream) {
  if (head_dim == 64) {
    return dtype == SM120N_F16 ? run_prompt_tiles<__half, 64>(a, stream)
                               : run_prompt_tiles<__nv_bfloat16, 64>(a, stream);
  }
  return dtype == SM120N_F16 ? run_prompt_tiles<__half, 128>(a, stream)
                             : run_prompt_tiles<__nv_bfloat16, 128>(a, stream);
}

int launch_prefix_tc(const DecodeArgs& a, int dtype, int cache_dtype, int head_dim,
                     cudaStream_t stream) {
  const bool fp8 = cache_dtype == SM120N_CACHE_FP8_E4M3;
  return head_dim == 64 ? run_prefix_typed<64>(a, dtype, fp8, stream)
                        : run_prefix_typed<128>(a, dtype, fp8, stream);
}

}  // namespace sm120n

using namespace sm120n;

extern "C" int sm120s_get_device_faults(uint32_t* out_count) {
  clear_error();
  if (!out_count) return fail(SM120N_ERR_INVALID_ARGUMENT, "out_count must be non-null");
  int rc = wait_for_device();
  if (rc != SM120N_OK) return rc;
  unsigned int mine = 0, decode = 0;
  const cudaError_t err = cudaMemcpyFromSymbol(&mine, g_attention_expired_waits, sizeof mine);
  if (err != cudaSuccess) {
    return fail(SM120N_ERR_CUDA, "reading the fault counter failed: %s", cudaGetErrorString(err));
  }
  rc = read_decode_faults(&decode);
  if (rc == SM120N_OK) *out_count = mine + decode;
  return rc;
}

extern "C" int sm120s_reset_device_faults(void) {
  clear_error();
  const int rc = wait_for_device();
  if (rc != SM120N_OK) return rc;
  const unsigned int zero = 0;
  const cudaError_t err = cudaMemcpyToSymbol(g_attention_expired_waits, &zero, sizeof zero);
  if (err != cudaSuccess) {
    return fail(SM120N_ERR_CUDA, "resetting the fault counter failed: %s", cudaGetErrorString(err));
  }
  return reset_decode_faults();
}
