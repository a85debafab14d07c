// head_mrope.cu -- per-head Q/K RMSNorm + rotation by positions with several
// axes + paged KV store; C-ABI entry point sm120s_qk_norm_mrope_cache.
//
// Tokens of images and video have a place in time, height and width, and each
// pair of a head turns by the position along one of them:
//   n = x * (1 / sqrt(mean(x^2) + eps)) * w
//   y_i = n_i cos - n_j sin,  y_j = n_j cos + n_i sin
//   cos / sin = cos_sin_cache[positions[axis(i)][token]] at index i
// for the pairs (i, j) of the half split or of neighbours, the rest of the
// head passed through as n. Everything is fp32 and rounded once, to the
// output's type and on its own to the cache's: there is no other
// implementation whose roundings would have to be matched here, and one
// rounding is the more accurate choice.
//
// Bound by memory. Lane layout and loads are those of head_cache_kernel: a head
// on D/16 lanes, 16-byte accesses, rotation partners in one lane, so only the
// sum of squares crosses lanes. A unit of work is a run of heads of one token
// on one warp: positions, slot and table entries are read once for the run (a
// head's table row is twice the bytes of the head). A lane holds 8 neighbouring
// trigonometric entries [8p, 8p + 8); the axis of each is fixed for the whole
// call and kept as 2 bits in a register. Lanes whose entries lie in one section,
// and all lanes of a token whose positions agree (text), read one table row
// with 16-byte loads; the others pick each entry from its axis's row (8191
// tokens, 64/8 heads: 65.0 us against 64.5).
#include <cuda_fp8.h>

#include <algorithm>

#include "cache_args.h"
#include "head_utils.cuh"
#include "row_overlap.h"
#include "runtime.h"
#include "sm120norm_b200_serving.h"

namespace sm120n {
namespace {

constexpr int kMaxAxes = SM120S_MAX_ROPE_AXES;

template <typename T>
struct MropeArgs {
  const T* query;
  const T* key;
  const T* value;
  T* query_out;
  T* key_out;
  int64_t query_stride;  // elements between consecutive tokens
  int64_t key_stride;
  int64_t value_stride;
  int64_t query_out_stride;
  int64_t key_out_stride;
  const T* query_weight;
  const T* key_weight;
  const int64_t* positions;  // axis a of token t at positions[a * axis_stride + t]
  int64_t axis_stride;
  const float* cos_sin;  // [rope_positions, rotary_dim]
  int64_t rope_positions;
  void* key_cache;
  void* value_cache;
  const int32_t* slots;
  int64_t block_stride;  // cache elements
  int64_t slot_stride;
  int64_t head_stride;
  int64_t cache_slots;
  const float* k_scale;
  const float* v_scale;
  int64_t tokens;
  uint32_t block_size;
  int query_heads;
  int key_heads;
  int rotary_dim;
  int axes;
  int section_end[kMaxAxes];  // sections one after another: where each ends
  int section[kMaxAxes];
  bool in_turns;
  bool interleaved;
  float epsilon;
  uint32_t parts;   // units of a token
  int part_heads;   // heads of a unit
  HeadDivisor parts_div;
};

// Axis whose position turns pair i.
template <typename T>
__device__ __forceinline__ uint32_t axis_of_pair(const MropeArgs<T>& a, int i) {
  if (a.in_turns) {
    const int axis = i % a.axes;
    return axis > 0 && i < a.axes * a.section[axis] ? axis : 0;
  }
  uint32_t axis = 0;
#pragma unroll
  for (int k = 0; k < kMaxAxes - 1; ++k) axis += k < a.axes - 1 && i >= a.section_end[k];
  return axis;
}

template <typename T, bool kVector>
__device__ __forceinline__ void store_fp8_half(uint8_t* p, const float2* f, float scale) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 q = make_float2(__fdiv_rn(f[i].x, scale), __fdiv_rn(f[i].y, scale));
    b[i] = static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(q, __NV_SATFINITE, __NV_E4M3));
  }
  store_fp8_chunk<kVector>(p, make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16)));
}

// Three blocks to an SM: with four the loads ahead spill (8191 tokens, 64/8
// heads: 65.5 us against 70.2), with two too few bytes are in flight (90.7).
template <typename T, int D, int kCache, bool kVector>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2) head_mrope_kernel(MropeArgs<T> a) {
  constexpr int kLanes = D / (2 * kChunkElems);
  constexpr int kHeadsPerWarp = kWarpSize / kLanes;
  const int rotary = a.rotary_dim;
  const int lane = threadIdx.x & (kWarpSize - 1);
  const int part = lane % kLanes;
  const int head_in_warp = lane / kLanes;
  const bool rotates = part < rotary / (2 * kChunkElems);
  const bool split = rotates && !a.interleaved;
  const int off_a = split ? part * kChunkElems : part * 2 * kChunkElems;
  const int off_b = split ? rotary / 2 + part * kChunkElems : off_a + kChunkElems;
  const int trig = part * kChunkElems;  // cos at [trig, trig + 8), sin R/2 further
  uint32_t axes = 0;                    // 2 bits for each of the lane's entries
  if (rotates) {
#pragma unroll
    for (int i = 0; i < kChunkElems; ++i) axes |= axis_of_pair(a, trig + i) << (2 * i);
  }
  const bool one_axis = axes == (axes & 3u) * 0x5555u;

  const int heads = a.query_heads + a.key_heads;
  const uint32_t units = static_cast<uint32_t>(a.tokens) * a.parts;
  const uint32_t warp = (blockIdx.x * blockDim.x + threadIdx.x) / kWarpSize;
  const uint32_t warps = (gridDim.x * blockDim.x) / kWarpSize;
  wait_for_upstream_grid();
  release_downstream_grid();

  float k_scale = 1.0f, v_scale = 1.0f;
  if constexpr (kCache == kFp8) {
    k_scale = *a.k_scale;
    v_scale = *a.v_scale;
  }

  for (uint32_t unit = warp; unit < units; unit += warps) {
    const uint32_t token = divide(a.parts_div, unit);
    const int first_head = static_cast<int>(unit - token * a.parts) * a.part_heads;
    const int last_head = min(first_head + a.part_heads, heads);
    // the token's rotation, for all heads of the unit
    const int64_t* places = a.positions + token;
    const int64_t place = places[static_cast<int64_t>(axes & 3u) * a.axis_stride];
    int64_t low = place, high = place;
    for (int k = 0; k < a.axes; ++k) {
      const int64_t p = places[k * a.axis_stride];
      low = min(low, p);
      high = max(high, p);
    }
    int64_t slot = -1;
    if (kCache != kNoCache && last_head > a.query_heads) slot = a.slots[token];
    if (low < 0 || high >= a.rope_positions) continue;
    float2 c[4], s[4];
    if (rotates) {
      if (one_axis || low == high) {
        const float* row = a.cos_sin + place * rotary;
        load8_pairs<kVector>(row + trig, c);
        load8_pairs<kVector>(row + rotary / 2 + trig, s);
      } else {
#pragma unroll
        for (int i = 0; i < kChunkElems; ++i) {
          const int64_t p = places[static_cast<int64_t>((axes >> (2 * i)) & 3u) * a.axis_stride];
          const float* entry = a.cos_sin + p * rotary + trig + i;
          (i & 1 ? c[i / 2].y : c[i / 2].x) = entry[0];
          (i & 1 ? s[i / 2].y : s[i / 2].x) = entry[rotary / 2];
        }
      }
    }
    const T* query = a.query + static_cast<int64_t>(token) * a.query_stride;
    const T* key = a.key + static_cast<int64_t>(token) * a.key_stride;
    int64_t cache_at = 0;
    if (kCache != kNoCache && slot >= 0 && slot < a.cache_slots) {
      const uint32_t block = static_cast<uint32_t>(slot) / a.block_size;
      cache_at = static_cast<int64_t>(block) * a.block_stride +
                 static_cast<int64_t>(static_cast<uint32_t>(slot) - block * a.block_size) * a.slot_stride;
    } else {
      slot = -1;
    }
    // kHeadsPerWarp heads at a time, the next ones loaded ahead
    Half8<T> next_a{}, next_b{};
    auto load_head = [&](int h) {
      if (h >= last_head) return;
      const T* head = h < a.query_heads ? query + static_cast<int64_t>(h) * D
                                        : key + static_cast<int64_t>(h - a.query_heads) * D;
      next_a = load_half<T, kVector>(head + off_a);
      next_b = load_half<T, kVector>(head + off_b);
    };
    load_head(first_head + head_in_warp);
    for (int h0 = first_head; h0 < last_head; h0 += kHeadsPerWarp) {
      const int h = h0 + head_in_warp;
      const bool active = h < last_head;
      const bool is_query = h < a.query_heads;
      const int kv_head = h - a.query_heads;
      const Half8<T> x_a = next_a, x_b = next_b;
      load_head(h + kHeadsPerWarp);
      Half8<T> v_a{}, v_b{};
      const bool store = kCache != kNoCache && active && !is_query && slot >= 0;
      if (store) {
        const T* vh = a.value + static_cast<int64_t>(token) * a.value_stride +
                      static_cast<int64_t>(kv_head) * D;
        v_a = load_half<T, kVector>(vh + off_a);
        v_b = load_half<T, kVector>(vh + off_b);
      }
      const float2 acc = half_sum_squares<T>(x_b, half_sum_squares<T>(x_a, make_float2(0.f, 0.f)));
      const float total = group_allreduce_sum<kLanes>(__fadd_rn(acc.x, acc.y));  // before any exit
      if (!active) continue;
      const float inv = head_inverse_rms<D>(make_float2(total, 0.0f), a.epsilon);
      const T* weight = is_query ? a.query_weight : a.key_weight;
      float2 n_a[4], n_b[4];
      {
        float2 w[4];
        unpack_pairs<T>(x_a, n_a);
        unpack_pairs<T>(load_half<T, kVector>(weight + off_a), w);
#pragma unroll
        for (int i = 0; i < 4; ++i) n_a[i] = make_float2(n_a[i].x * inv * w[i].x, n_a[i].y * inv * w[i].y);
        unpack_pairs<T>(x_b, n_b);
        unpack_pairs<T>(load_half<T, kVector>(weight + off_b), w);
#pragma unroll
        for (int i = 0; i < 4; ++i) n_b[i] = make_float2(n_b[i].x * inv * w[i].x, n_b[i].y * inv * w[i].y);
      }
      if (rotates) {
        if (a.interleaved) {  // (x, y) of a float2 are partners, entries 0-3 in n_a and 4-7 in n_b
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float ca = i & 1 ? c[i / 2].y : c[i / 2].x;
            const float sa = i & 1 ? s[i / 2].y : s[i / 2].x;
            const float cb = i & 1 ? c[2 + i / 2].y : c[2 + i / 2].x;
            const float sb = i & 1 ? s[2 + i / 2].y : s[2 + i / 2].x;
            n_a[i] = make_float2(n_a[i].x * ca - n_a[i].y * sa, n_a[i].y * ca + n_a[i].x * sa);
            n_b[i] = make_float2(n_b[i].x * cb - n_b[i].y * sb, n_b[i].y * cb + n_b[i].x * sb);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 u = n_a[i], v = n_b[i];
            n_a[i] = make_float2(u.x * c[i].x - v.x * s[i].x, u.y * c[i].y - v.y * s[i].y);
            n_b[i] = make_float2(v.x * c[i].x + u.x * s[i].x, v.y * c[i].y + u.y * s[i].y);
          }
        }
      }
      T* out = is_query ? a.query_out + static_cast<int64_t>(token) * a.query_out_stride +
                              static_cast<int64_t>(h) * D
                        : a.key_out + static_cast<int64_t>(token) * a.key_out_stride +
                              static_cast<int64_t>(kv_head) * D;
      const Half8<T> y_a = pack_pairs<T>(n_a);
      const Half8<T> y_b = pack_pairs<T>(n_b);
      store_half<T, kVector>(out + off_a, y_a);
      store_half<T, kVector>(out + off_b, y_b);
      if (store) {
        const int64_t base = cache_at + static_cast<int64_t>(kv_head) * a.head_stride;
        if constexpr (kCache == kSameType) {
          T* kc = static_cast<T*>(a.key_cache) + base;
          T* vc = static_cast<T*>(a.value_cache) + base;
          store_half<T, kVector>(kc + off_a, y_a);
          store_half<T, kVector>(kc + off_b, y_b);
          store_half<T, kVector>(vc + off_a, v_a);
          store_half<T, kVector>(vc + off_b, v_b);
        } else {
          uint8_t* kc = static_cast<uint8_t*>(a.key_cache) + base;
          uint8_t* vc = static_cast<uint8_t*>(a.value_cache) + base;
          store_fp8_half<T, kVector>(kc + off_a, n_a, k_scale);
          store_fp8_half<T, kVector>(kc + off_b, n_b, k_scale);
          unpack_pairs<T>(v_a, n_a);
          unpack_pairs<T>(v_b, n_b);
          store_fp8_half<T, kVector>(vc + off_a, n_a, v_scale);
          store_fp8_half<T, kVector>(vc + off_b, n_b, v_scale);
        }
      }
    }
  }
}

template <typename T, int D, int kCache>
int run_mrope(MropeArgs<T> a, cudaStream_t stream) {
  constexpr bool kFp8Cache = kCache == kFp8;
  constexpr int64_t kCacheElem = kFp8Cache ? 1 : sizeof(T);
  constexpr uintptr_t kCacheAlign = kFp8Cache ? 8 : 16;
  auto rows16 = [](int64_t stride) { return (stride * static_cast<int64_t>(sizeof(T))) % 16 == 0; };
  auto cache_rows = [](int64_t stride) {
    return (stride * kCacheElem) % static_cast<int64_t>(kCacheAlign) == 0;
  };
  const bool vector =
      aligned16(a.query) && aligned16(a.key) && aligned16(a.query_out) && aligned16(a.key_out) &&
      aligned16(a.query_weight) && aligned16(a.key_weight) && aligned16(a.cos_sin) &&
      rows16(a.query_stride) && rows16(a.key_stride) && rows16(a.query_out_stride) &&
      rows16(a.key_out_stride) &&
      (kCache == kNoCache ||
       (aligned16(a.value) && rows16(a.value_stride) && aligned_to(a.key_cache, kCacheAlign) &&
        aligned_to(a.value_cache, kCacheAlign) && cache_rows(a.block_stride) &&
        cache_rows(a.slot_stride) && cache_rows(a.head_stride)));
  auto kernel = vector ? head_mrope_kernel<T, D, kCache, true> : head_mrope_kernel<T, D, kCache, false>;
  constexpr int64_t kHeadsPerWarp = kWarpSize / (D / (2 * kChunkElems));
  DeviceInfo dev;
  int rc = current_device_info(&dev);
  if (rc != SM120N_OK) return rc;
  const int64_t heads = a.query_heads + a.key_heads;
  const int threads = 256;
  int resident = 1;
  rc = max_resident_ctas(reinterpret_cast<const void*>(kernel), threads, 0, &resident);
  if (rc != SM120N_OK) return rc;
  const int64_t most_warps = int64_t{dev.sm_count} * resident * (threads / kWarpSize);
  // Units of `per` groups of heads: the warps run over them in rounds, and a
  // unit's start (positions, table entries) costs about as much as 1.5 groups.
  // The fewest parts of a token with the least of rounds x (per + 1.5).
  const int64_t groups = (heads + kHeadsPerWarp - 1) / kHeadsPerWarp;
  int64_t least = INT64_MAX;
  for (int64_t parts = 1; parts <= std::min<int64_t>(groups, 64); ++parts) {
    const int64_t per = (groups + parts - 1) / parts;
    const int64_t rounds = (a.tokens * parts + most_warps - 1) / most_warps;
    if (rounds * (2 * per + 3) < least) {
      least = rounds * (2 * per + 3);
      a.parts = static_cast<uint32_t>((groups + per - 1) / per);
      a.part_heads = static_cast<int>(per * kHeadsPerWarp);
    }
  }
  a.parts_div = make_head_divisor(a.parts);
  // tokens * parts < 2^31 per launch (32-bit unit indices)
  const int64_t max_tokens = ((int64_t{1} << 31) - 1) / a.parts;
  const int64_t all_tokens = a.tokens;
  for (int64_t done = 0; done < all_tokens; done += max_tokens) {
    MropeArgs<T> c = a;
    c.tokens = std::min(max_tokens, all_tokens - done);
    c.query = a.query + done * a.query_stride;
    c.key = a.key + done * a.key_stride;
    c.query_out = a.query_out + done * a.query_out_stride;
    c.key_out = a.key_out + done * a.key_out_stride;
    c.positions = a.positions + done;
    if (kCache != kNoCache && a.key_heads > 0) {
      c.value = a.value + done * a.value_stride;
      c.slots = a.slots + done;
    }
    // few units: small blocks, so that they spread over the SMs
    const int64_t warps_needed = c.tokens * a.parts;
    const int64_t block_warps = std::max<int64_t>(
        1, std::min<int64_t>(threads / kWarpSize, warps_needed / dev.sm_count));
    const int64_t blocks = std::min<int64_t>((warps_needed + block_warps - 1) / block_warps,
                                             most_warps / block_warps);
    rc = launch(kernel, dim3(static_cast<unsigned>(blocks)),
                dim3(static_cast<unsigned>(block_warps * kWarpSize)), 0, stream, c);
    if (rc != SM120N_OK) return rc;
  }
  return SM120N_OK;
}

template <typename T, int D>
int run_mrope_kind(const MropeArgs<T>& a, int cache_kind, cudaStream_t stream) {
  switch (cache_kind) {
    case kNoCache: return run_mrope<T, D, kNoCache>(a, stream);
    case kSameType: return run_mrope<T, D, kSameType>(a, stream);
    default: return run_mrope<T, D, kFp8>(a, stream);
  }
}

template <typename T>
int run_mrope_typed(const sm120n_qk_cache_args& in, const sm120s_mrope_args& m, int cache_kind,
                    cudaStream_t stream) {
  MropeArgs<T> a{};
  a.query = static_cast<const T*>(in.query);
  a.key = static_cast<const T*>(in.key);
  a.value = static_cast<const T*>(in.value);
  a.query_stride = in.query_token_stride;
  a.key_stride = in.key_token_stride;
  a.value_stride = in.value_token_stride;
  a.query_out = static_cast<T*>(m.query_out ? m.query_out : in.query);
  a.key_out = static_cast<T*>(m.key_out ? m.key_out : in.key);
  a.query_out_stride = m.query_out ? m.query_out_token_stride : in.query_token_stride;
  a.key_out_stride = m.key_out ? m.key_out_token_stride : in.key_token_stride;
  a.query_weight = static_cast<const T*>(in.query_weight);
  a.key_weight = static_cast<const T*>(in.key_weight);
  a.positions = in.positions;
  a.axis_stride = m.position_axis_stride;
  a.cos_sin = in.cos_sin_cache;
  a.rope_positions = in.rope_positions;
  a.key_cache = in.key_cache;
  a.value_cache = in.value_cache;
  a.slots = in.slot_mapping;
  a.block_stride = in.cache_block_stride;
  a.slot_stride = in.cache_slot_stride;
  a.head_stride = in.cache_head_stride;
  a.block_size = static_cast<uint32_t>(std::max<int64_t>(in.block_size, 1));
  a.cache_slots = cache_kind == kNoCache ? 0 : in.num_blocks * in.block_size;
  a.k_scale = in.k_scale;
  a.v_scale = in.v_scale;
  a.tokens = in.tokens;
  a.query_heads = static_cast<int>(in.query_heads);
  a.key_heads = static_cast<int>(in.key_heads);
  a.rotary_dim = static_cast<int>(in.rotary_dim);
  a.axes = m.axes;
  int end = 0;
  for (int k = 0; k < m.axes; ++k) {
    a.section[k] = m.sections[k];
    a.section_end[k] = end += m.sections[k];
  }
  a.in_turns = m.interleaved_sections != 0;
  a.interleaved = in.rope_style == SM120N_ROPE_INTERLEAVED;
  a.epsilon = in.epsilon;
  switch (in.head_dim) {
    case 64: return run_mrope_kind<T, 64>(a, cache_kind, stream);
    case 128: return run_mrope_kind<T, 128>(a, cache_kind, stream);
    default: return run_mrope_kind<T, 256>(a, cache_kind, stream);
  }
}

int check_mrope_args(const sm120n_qk_cache_args& in, const sm120s_mrope_args* m) {
  if (m == nullptr) return fail(SM120N_ERR_INVALID_ARGUMENT, "mrope args must be non-null");
  if (m->struct_size != sizeof(sm120s_mrope_args)) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "struct_size %u does not match this library's sm120s_mrope_args (%zu)",
                m->struct_size, sizeof(sm120s_mrope_args));
  }
  if (m->axes < 1 || m->axes > kMaxAxes) {
    return fail(SM120N_ERR_UNSUPPORTED, "positions must have 1 to %d axes (got %d)", kMaxAxes, m->axes);
  }
  int64_t sum = 0;
  for (int k = 0; k < m->axes; ++k) {
    if (m->sections[k] < 0) {
      return fail(SM120N_ERR_INVALID_ARGUMENT, "sections must be non-negative");
    }
    sum += m->sections[k];
  }
  if (sum != in.rotary_dim / 2) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "sections must add up to half the rotary width (%lld, got %lld)",
                static_cast<long long>(in.rotary_dim / 2), static_cast<long long>(sum));
  }
  if (m->interleaved_sections) {
    // axis k > 0 takes pairs k, k + axes, ...: section[k] of them have to exist
    for (int k = 1; k < m->axes; ++k) {
      if (m->sections[k] > 0 && k + (m->sections[k] - 1) * int64_t{m->axes} >= in.rotary_dim / 2) {
        return fail(SM120N_ERR_INVALID_ARGUMENT,
                    "interleaved section %d has more pairs than its turns", k);
      }
    }
  }
  if (m->position_axis_stride < 0) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "position_axis_stride must be non-negative");
  }
  if (in.tokens > 0 && ((m->query_out && m->query_out_token_stride < in.query_heads * in.head_dim) ||
                        (m->key_out && m->key_out_token_stride < in.key_heads * in.head_dim))) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "token strides must cover heads * head_dim elements (rows may not overlap)");
  }
  return SM120N_OK;
}

// What is written may overlap nothing that another head reads or writes: its own
// input only as the same rows (in place).
int check_mrope_overlaps(const sm120n_qk_cache_args& in, const sm120s_mrope_args& m, int cache_kind) {
  const int64_t elem = dtype_size(in.dtype);
  auto rows = [&](const void* p, int64_t stride, int64_t heads) {
    return row_set(p, in.tokens, stride, heads * in.head_dim, elem);
  };
  const bool stores = cache_kind != kNoCache && in.key_heads > 0;
  const RowSet query = rows(in.query, in.query_token_stride, in.query_heads);
  const RowSet key = rows(in.key, in.key_token_stride, in.key_heads);
  const RowSet value = rows(stores ? in.value : nullptr, in.value_token_stride, in.key_heads);
  const RowSet query_out =
      m.query_out ? rows(m.query_out, m.query_out_token_stride, in.query_heads) : query;
  const RowSet key_out = m.key_out ? rows(m.key_out, m.key_out_token_stride, in.key_heads) : key;
  auto same = [](const RowSet& a, const RowSet& b) {
    return a.data == b.data && (a.count <= 1 || a.stride == b.stride);
  };
  auto refuse = [](const char* out, const char* other) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "%s may not overlap %s", out, other);
  };
  if (!same(query_out, query) && rows_overlap(query_out, query)) return refuse("query_out", "its input");
  if (!same(key_out, key) && rows_overlap(key_out, key)) return refuse("key_out", "its input");
  if (rows_overlap(query_out, key)) return refuse(m.query_out ? "query_out" : "query", "key");
  if (rows_overlap(key_out, query)) return refuse(m.key_out ? "key_out" : "key", "query");
  if (rows_overlap(query_out, key_out)) return refuse("query_out", "key_out");
  if (rows_overlap(query_out, value)) return refuse(m.query_out ? "query_out" : "query", "value");
  // a head's value is read by the threads that write its key, before they do
  if (!same(key_out, value) && rows_overlap(key_out, value)) {
    return refuse(m.key_out ? "key_out" : "key", "value");
  }
  if (!stores || in.num_blocks < 1) return SM120N_OK;
  // a cache from its first to its last element
  const int64_t elems = (in.num_blocks - 1) * in.cache_block_stride +
                        (in.block_size - 1) * in.cache_slot_stride +
                        (in.key_heads - 1) * in.cache_head_stride + in.head_dim;
  for (const void* cache : {in.key_cache, in.value_cache}) {
    const RowSet all = row_set(cache, 1, elems, elems, cache_kind == kFp8 ? 1 : elem);
    if (rows_overlap(query_out, all)) return refuse(m.query_out ? "query_out" : "query", "the caches");
    if (rows_overlap(key_out, all)) return refuse(m.key_out ? "key_out" : "key", "the caches");
  }
  return SM120N_OK;
}

}  // namespace
}  // namespace sm120n

using namespace sm120n;

extern "C" int sm120s_qk_norm_mrope_cache(const sm120n_qk_cache_args* args,
                                          const sm120s_mrope_args* mrope, void* stream) {
  clear_error();
  int cache_kind = kNoCache;
  int rc = check_cache_args(args, &cache_kind);
  if (rc != SM120N_OK) return rc;
  rc = check_mrope_args(*args, mrope);
  if (rc != SM120N_OK) return rc;
  if (args->tokens == 0 || args->query_heads + args->key_heads == 0) return SM120N_OK;
  rc = check_mrope_overlaps(*args, *mrope, cache_kind);
  if (rc != SM120N_OK) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (args->dtype) {
    case SM120N_F32: return run_mrope_typed<float>(*args, *mrope, cache_kind, s);
    case SM120N_F16: return run_mrope_typed<__half>(*args, *mrope, cache_kind, s);
    default: return run_mrope_typed<__nv_bfloat16>(*args, *mrope, cache_kind, s);
  }
}
