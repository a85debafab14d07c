// attention.cu -- C-ABI entry points sm120s_prompt_attention and
// sm120s_paged_decode_attention: argument checks, the choice of the kernels
// and the layout of the workspace.
#include "attention.h"

#include <algorithm>
#include <cmath>

#include "row_overlap.h"

namespace sm120n {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

int check_heads(int dtype, int64_t query_heads, int64_t key_heads, int64_t head_dim, float scale) {
  if (dtype != SM120N_F16 && dtype != SM120N_BF16) {
    return fail(SM120N_ERR_UNSUPPORTED, "attention supports float16 and bfloat16");
  }
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    return fail(SM120N_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256 (got %lld)",
                static_cast<long long>(head_dim));
  }
  if (key_heads < 1 || query_heads < 1 || query_heads % key_heads != 0 || query_heads >= (1 << 16)) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "query_heads must be a positive multiple of key_heads, below 2^16");
  }
  if (!(scale > 0.0f) || !std::isfinite(scale * kLog2e)) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "scale must be positive and finite");
  }
  return SM120N_OK;
}

// A row of `heads` heads at every token: 16-byte aligned, not overlapping.
int check_rows(const void* p, int64_t stride, int64_t tokens, int64_t heads, int64_t head_dim,
               const char* name) {
  if (!p) return fail(SM120N_ERR_INVALID_ARGUMENT, "tensor pointers must be non-null");
  if (stride < heads * head_dim) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "token strides must cover heads * head_dim elements (rows may not overlap)");
  }
  if (!aligned16(p) || (tokens > 1 && stride % 8 != 0)) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "%s rows must be 16-byte aligned", name);
  }
  return SM120N_OK;
}

// Rows of `heads` heads at every token, in 16-bit elements.
RowSet head_rows(const void* p, int64_t stride, int64_t tokens, int64_t heads, int64_t head_dim) {
  return row_set(p, tokens, stride, heads * head_dim, 2);
}

int check_apart(const RowSet& out, const RowSet& in, const char* name) {
  return rows_overlap(out, in)
             ? fail(SM120N_ERR_INVALID_ARGUMENT, "out may not overlap %s", name)
             : SM120N_OK;
}

// Whether the prefix runs on tensor memory: 256 rows and 128 keys to a tile
// there, 64 and 64 otherwise.
bool prefix_on_tensor_memory(const sm120s_decode_args& a) {
  return a.head_dim <= 128 && block_fills_tiles(a.block_size, 128);
}

struct Plan {
  int row_tiles;
  int own_grid;
  int prefix_splits;
  size_t own_state, own_values, prefix_state, prefix_values;  // offsets into the workspace
  size_t bytes;
};

int check_decode_sizes(const sm120s_decode_args* a) {
  if (a == nullptr) return fail(SM120N_ERR_INVALID_ARGUMENT, "args must be non-null");
  if (a->struct_size != sizeof(sm120s_decode_args)) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "struct_size %u does not match this library's sm120s_decode_args (%zu)",
                a->struct_size, sizeof(sm120s_decode_args));
  }
  int rc = check_heads(a->dtype, a->query_heads, a->key_heads, a->head_dim, a->scale);
  if (rc != SM120N_OK) return rc;
  if (a->cache_dtype != SM120N_CACHE_AUTO && a->cache_dtype != SM120N_CACHE_FP8_E4M3) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "unknown cache_dtype %d", a->cache_dtype);
  }
  if (a->batch < 0 || a->batch > (1 << 20) || a->table_width < 0 || a->prefix_blocks_count < 0 ||
      a->num_blocks < 0) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "batch must be in [0, 2^20], table and prefix lengths non-negative");
  }
  if (a->batch * a->query_heads > INT32_MAX) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "batch * query_heads must be below 2^31");
  }
  if (a->block_size < 1 || a->block_size > INT32_MAX ||
      a->num_blocks > (int64_t{1} << 31) / a->block_size) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "block_size must be positive and num_blocks * block_size at most 2^31");
  }
  // key indices are 32-bit, and so is the sum of the requests' key tiles
  if (a->table_width > ((int64_t{1} << 31) - 64) / a->block_size) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "table_width * block_size must be below 2^31 - 64");
  }
  if (a->prefix_blocks_count > 0 && a->prefix_blocks_count > a->table_width) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "block_table rows must reach past the prefix (width %lld, prefix %lld blocks)",
                static_cast<long long>(a->table_width),
                static_cast<long long>(a->prefix_blocks_count));
  }
  return SM120N_OK;
}

// Parts of a prefix on tensor memory, at most `most` (a block to an SM). More of
// them are shorter, but each takes SMs from the own tokens' pass for its start,
// and is read again when the parts are joined: step * tiles / parts + cost *
// parts is least at the root below. A few parts fewer are taken where that
// leaves half of the SMs to the own tokens, whose blocks, two to an SM, then run
// in two waves beside the prefix. Measured (graph, 61 requests of 1-600 own
// tokens, 32/8 heads, D = 128, bf16), `most` against this: prefixes of 2048
// tokens 43.5 us (16 parts) against 36.5 (4), 8192 52 (18) against 42 (8),
// 16384 61 (18) against 50 (9); with 1-32 own tokens and 8192 33.6 against 30.7.
// Where a part has many blocks, there are few parts, and all of them won: 300
// requests, 1024 tokens, 82 us with 3 parts against 87.6 with 2; 128 requests, D =
// 64, 4096 tokens, 62.7 with 9 against 67.5 with 4.
// Held against each number of parts from 1 to `most` on 100 batches (8 to 256 requests,
// prefixes of 1024 to 32768 tokens, own tokens up to 64, 600 and 2048, groups of 2, 4
// and 8, D = 64 and 128, fp8): in the median it took 1.03 times the best one's time, 23
// batches lay above 1.1 and the worst at 1.33 (100 requests with prefixes of 1024
// tokens, 32/4 heads, 38.5 us against 29 in one part). What it lacks is the lengths,
// which are not on the host.
int prefix_parts(const sm120s_decode_args& a, int most, int64_t blocks, int64_t tiles,
                 int64_t triples, int sm_count) {
  if (12 * blocks > sm_count) return most;
  const double step = (a.cache_dtype == SM120N_CACHE_FP8_E4M3 ? 2.2 : 1.8) *  // us, 128 keys
                      (a.head_dim == 64 ? 0.72 : 1.0);
  const double start = 16.0, join_bytes = 1.5e6;  // us of an SM; bytes in a us
  const int own_room =
      own_blocks_per_sm(a.cache_dtype, static_cast<int>(a.head_dim), a.query_heads / a.key_heads) * sm_count;
  const double wanted =  // of the SMs
      std::min(1.0, static_cast<double>(std::max<int64_t>(triples, 1)) / own_room);
  const double cost = start * blocks / sm_count * wanted +
                      static_cast<double>(a.batch) * a.query_heads * a.head_dim * 4 / join_bytes;
  int64_t parts = std::min<int64_t>(most, std::llround(std::sqrt(step * tiles / cost)));
  const int64_t beside = sm_count / 2 / blocks;
  if (triples >= own_room && parts > beside && 10 * beside >= 7 * parts) parts = beside;
  parts = std::max<int64_t>(parts, 1);
  const int64_t steps = (tiles + parts - 1) / parts;
  return static_cast<int>((tiles + steps - 1) / steps);  // no more than take as many steps
}

int plan_decode(const sm120s_decode_args& a, Plan* plan) {
  DeviceInfo dev;
  const int rc = current_device_info(&dev);
  if (rc != SM120N_OK) return rc;
  const int64_t group = a.query_heads / a.key_heads;
  plan->row_tiles = static_cast<int>((group + 15) / 16);
  const int64_t triples = a.batch * a.key_heads * plan->row_tiles;
  const int64_t most_tiles = (a.table_width * a.block_size + 63) / 64;
  plan->own_grid = static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>(
             own_blocks_per_sm(a.cache_dtype, static_cast<int>(a.head_dim), group) * dev.sm_count,
             triples * most_tiles)));
  plan->prefix_splits = 0;
  if (a.prefix_blocks_count > 0 && a.num_blocks > 0) {
    const bool tc = prefix_on_tensor_memory(a);
    const int64_t tile_rows = tc ? 256 : 64, tile_keys = tc ? 128 : 64;
    const int64_t row_tiles = (a.batch * group + tile_rows - 1) / tile_rows;
    const int64_t tiles = (a.prefix_blocks_count * a.block_size + tile_keys - 1) / tile_keys;
    const int64_t blocks = std::max<int64_t>(1, row_tiles * a.key_heads);
    const int most = static_cast<int>(std::max<int64_t>(
        1, std::min<int64_t>(tiles, (tc ? 1 : 2) * dev.sm_count / blocks)));
    plan->prefix_splits = tc ? prefix_parts(a, most, blocks, tiles, triples, dev.sm_count) : most;
  }
  size_t at = (static_cast<size_t>(a.batch + 1) * sizeof(int64_t) + 15) / 16 * 16;
  const size_t own_rows = static_cast<size_t>(triples + plan->own_grid) * 16;
  const size_t prefix_rows = static_cast<size_t>(plan->prefix_splits) * a.batch * a.query_heads;
  plan->own_state = at;
  at += own_rows * sizeof(float2);
  plan->own_values = at;
  at += own_rows * a.head_dim * sizeof(float);
  plan->prefix_state = at;
  at += (prefix_rows * sizeof(float2) + 15) / 16 * 16;
  plan->prefix_values = at;
  at += prefix_rows * a.head_dim * sizeof(float);
  plan->bytes = at;
  return SM120N_OK;
}

}  // namespace
}  // namespace sm120n

using namespace sm120n;

extern "C" int sm120s_prompt_attention(const sm120s_prompt_args* args, void* stream) {
  clear_error();
  if (args == nullptr) return fail(SM120N_ERR_INVALID_ARGUMENT, "args must be non-null");
  const sm120s_prompt_args& in = *args;
  if (in.struct_size != sizeof(sm120s_prompt_args)) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "struct_size %u does not match this library's sm120s_prompt_args (%zu)",
                in.struct_size, sizeof(sm120s_prompt_args));
  }
  int rc = check_heads(in.dtype, in.query_heads, in.key_heads, in.head_dim, in.scale);
  if (rc != SM120N_OK) return rc;
  const int64_t group = in.query_heads / in.key_heads;
  // 32-bit indices that run up to a step of the search past the end
  if (in.tokens < 0 || in.sequences < 0 || in.sequences > INT32_MAX - 256 ||
      in.tokens > INT32_MAX - 256) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "tokens and sequences must be in [0, 2^31 - 256)");
  }
  if (in.tokens == 0 || in.sequences == 0) return SM120N_OK;
  // one thread block to a tile of 64 rows or more of one key head
  if ((in.tokens * group / 64 + 1 + in.sequences) * in.key_heads > INT32_MAX) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "too many tokens for one call");
  }
  if (!in.query_start) return fail(SM120N_ERR_INVALID_ARGUMENT, "tensor pointers must be non-null");
  rc = check_rows(in.query, in.query_token_stride, in.tokens, in.query_heads, in.head_dim, "query");
  if (rc == SM120N_OK) rc = check_rows(in.key, in.key_token_stride, in.tokens, in.key_heads, in.head_dim, "key");
  if (rc == SM120N_OK) rc = check_rows(in.value, in.value_token_stride, in.tokens, in.key_heads, in.head_dim, "value");
  if (rc == SM120N_OK) rc = check_rows(in.out, in.out_token_stride, in.tokens, in.query_heads, in.head_dim, "out");
  if (rc != SM120N_OK) return rc;
  const RowSet out = head_rows(in.out, in.out_token_stride, in.tokens, in.query_heads, in.head_dim);
  rc = check_apart(out, head_rows(in.query, in.query_token_stride, in.tokens, in.query_heads, in.head_dim), "query");
  if (rc == SM120N_OK) rc = check_apart(out, head_rows(in.key, in.key_token_stride, in.tokens, in.key_heads, in.head_dim), "key");
  if (rc == SM120N_OK) rc = check_apart(out, head_rows(in.value, in.value_token_stride, in.tokens, in.key_heads, in.head_dim), "value");
  if (rc != SM120N_OK) return rc;
  PromptArgs a{};
  a.query = in.query;
  a.out = in.out;
  a.query_start = in.query_start;
  a.key = in.key;
  a.value = in.value;
  a.key_stride = in.key_token_stride;
  a.value_stride = in.value_token_stride;
  a.query_stride = in.query_token_stride;
  a.out_stride = in.out_token_stride;
  a.tokens = in.tokens;
  a.sequences = static_cast<int32_t>(in.sequences);
  a.query_heads = static_cast<int32_t>(in.query_heads);
  a.key_heads = static_cast<int32_t>(in.key_heads);
  a.group = static_cast<int32_t>(group);
  a.scale_log2 = in.scale * kLog2e;
  a.wait_polls = wait_poll_limit();
  const int head_dim = static_cast<int>(in.head_dim);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return head_dim <= 128 ? launch_prompt_tc(a, in.dtype, head_dim, s)
                         : launch_prompt_mma(a, in.dtype, s);
}

extern "C" int sm120s_paged_decode_workspace(const sm120s_decode_args* args, size_t* bytes) {
  clear_error();
  int rc = check_decode_sizes(args);
  if (rc != SM120N_OK) return rc;
  if (!bytes) return fail(SM120N_ERR_INVALID_ARGUMENT, "bytes must be non-null");
  Plan plan;
  rc = plan_decode(*args, &plan);
  if (rc == SM120N_OK) *bytes = plan.bytes;
  return rc;
}

extern "C" int sm120s_paged_decode_attention(const sm120s_decode_args* args, void* stream) {
  clear_error();
  int rc = check_decode_sizes(args);
  if (rc != SM120N_OK) return rc;
  const sm120s_decode_args& in = *args;
  if (in.batch == 0) return SM120N_OK;
  rc = check_rows(in.query, in.query_token_stride, in.batch, in.query_heads, in.head_dim, "query");
  if (rc == SM120N_OK) rc = check_rows(in.out, in.out_token_stride, in.batch, in.query_heads, in.head_dim, "out");
  if (rc != SM120N_OK) return rc;
  const bool fp8 = in.cache_dtype == SM120N_CACHE_FP8_E4M3;
  if (!in.seq_lens || (in.table_width > 0 && !in.block_table) ||
      (in.prefix_blocks_count > 0 && !in.prefix_blocks) ||
      (in.num_blocks > 0 && (!in.key_cache || !in.value_cache))) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "tensor pointers must be non-null");
  }
  if (fp8 && (!in.k_scale || !in.v_scale)) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "fp8 caches need k_scale and v_scale");
  }
  if (in.table_stride < in.table_width) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "block table rows may not overlap");
  }
  const int64_t pack = fp8 ? 16 : 8;
  if (in.cache_block_stride < 0 || in.cache_slot_stride < 0 || in.cache_head_stride < 0) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "cache strides must be non-negative");
  }
  if (!aligned16(in.key_cache) || !aligned16(in.value_cache) || in.cache_block_stride % pack != 0 ||
      in.cache_slot_stride % pack != 0 || in.cache_head_stride % pack != 0) {
    return fail(SM120N_ERR_INVALID_ARGUMENT, "cache rows must be 16-byte aligned");
  }
  if ((in.num_blocks > 1 && in.cache_block_stride < in.head_dim) ||
      (in.block_size > 1 && in.cache_slot_stride < in.head_dim) ||
      (in.key_heads > 1 && in.cache_head_stride < in.head_dim)) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "cache strides must cover head_dim elements (rows may not overlap)");
  }
  const RowSet out = head_rows(in.out, in.out_token_stride, in.batch, in.query_heads, in.head_dim);
  rc = check_apart(out, head_rows(in.query, in.query_token_stride, in.batch, in.query_heads, in.head_dim), "query");
  // a cache from its first to its last element
  const int64_t elems = in.num_blocks < 1 ? 0 : (in.num_blocks - 1) * in.cache_block_stride +
                                                    (in.block_size - 1) * in.cache_slot_stride +
                                                    (in.key_heads - 1) * in.cache_head_stride + in.head_dim;
  if (rc == SM120N_OK) rc = check_apart(out, row_set(in.key_cache, 1, elems, elems, fp8 ? 1 : 2), "key_cache");
  if (rc == SM120N_OK) rc = check_apart(out, row_set(in.value_cache, 1, elems, elems, fp8 ? 1 : 2), "value_cache");
  if (rc != SM120N_OK) return rc;
  Plan plan;
  rc = plan_decode(in, &plan);
  if (rc != SM120N_OK) return rc;
  if (!in.workspace || !aligned16(in.workspace) || in.workspace_bytes < plan.bytes) {
    return fail(SM120N_ERR_INVALID_ARGUMENT,
                "workspace must be 16-byte aligned and hold %zu bytes (sm120s_paged_decode_workspace)",
                plan.bytes);
  }
  unsigned char* space = static_cast<unsigned char*>(in.workspace);
  DecodeArgs a{};
  a.query = in.query;
  a.out = in.out;
  a.table = in.block_table;
  a.seq_lens = in.seq_lens;
  a.prefix_blocks = in.prefix_blocks;
  a.k_scale = fp8 ? in.k_scale : nullptr;
  a.v_scale = fp8 ? in.v_scale : nullptr;
  a.kv.key = in.key_cache;
  a.kv.value = in.value_cache;
  a.kv.slot_stride = in.cache_slot_stride;
  a.kv.head_stride = in.cache_head_stride;
  a.kv.block_stride = in.cache_block_stride;
  a.kv.block_size = static_cast<int32_t>(in.block_size);
  a.kv.num_blocks = static_cast<int32_t>(std::min<int64_t>(in.num_blocks, INT32_MAX));
  a.query_stride = in.query_token_stride;
  a.out_stride = in.out_token_stride;
  a.table_stride = in.table_stride;
  a.batch = static_cast<int32_t>(in.batch);
  // a cache without blocks holds no keys, whatever the tables say
  a.table_width = in.num_blocks > 0 ? static_cast<int32_t>(in.table_width) : 0;
  a.prefix_tokens = in.num_blocks > 0 ? static_cast<int32_t>(in.prefix_blocks_count * in.block_size) : 0;
  a.query_heads = static_cast<int32_t>(in.query_heads);
  a.key_heads = static_cast<int32_t>(in.key_heads);
  a.group = static_cast<int32_t>(in.query_heads / in.key_heads);
  a.row_tiles = plan.row_tiles;
  a.own_grid = plan.own_grid;
  a.prefix_splits = plan.prefix_splits;
  a.scale_log2 = in.scale * kLog2e;
  a.wait_polls = wait_poll_limit();
  a.tile_start = reinterpret_cast<int64_t*>(space);
  a.own_state = reinterpret_cast<float2*>(space + plan.own_state);
  a.own_values = reinterpret_cast<float*>(space + plan.own_values);
  a.prefix_state = reinterpret_cast<float2*>(space + plan.prefix_state);
  a.prefix_values = reinterpret_cast<float*>(space + plan.prefix_values);
  const int head_dim = static_cast<int>(in.head_dim);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.prefix_splits > 0) {
    rc = prefix_on_tensor_memory(in) ? launch_prefix_tc(a, in.dtype, in.cache_dtype, head_dim, s)
                                     : launch_prefix_mma(a, in.dtype, in.cache_dtype, head_dim, s);
    if (rc != SM120N_OK) return rc;
  }
  rc = launch_own(a, in.dtype, in.cache_dtype, head_dim, s);
  if (rc != SM120N_OK) return rc;
  return launch_merge(a, in.dtype, head_dim, s);
}
