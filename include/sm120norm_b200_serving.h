/*
 * sm120norm_b200_serving.h -- C ABI of the B200 (sm_100a) serving operators
 * around the paged KV cache: step planning, Q/K norm + rotation by positions
 * with several axes, prompt attention and paged decode attention.
 *
 * The library (libsm120norm_b200_serving.so) stands beside
 * libsm120norm_b200.so and follows its conventions: plain pointers, sizes and
 * an opaque CUDA stream; every entry point validates its scalar arguments,
 * launches on the CURRENT CUDA device on the given stream, never synchronises,
 * never allocates, and returns an sm120n_status. On failure a message for the
 * calling thread is available from sm120s_last_error(). The process-wide
 * switch sm120n_set_programmatic_launch applies to these kernels too.
 *
 * Cache layout, slots and fp8 storage are those of sm120n_qk_norm_rope_cache:
 * what that operator stores, these read.
 */
#ifndef SM120NORM_B200_SERVING_H_
#define SM120NORM_B200_SERVING_H_

#include <stddef.h>
#include <stdint.h>

#include "sm120norm_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SM120S_ABI_VERSION 1

SM120N_API int sm120s_abi_version(void);

/* Message describing the last failing call made by this thread ("" if none). */
SM120N_API const char* sm120s_last_error(void);

/*
 * Number of bounded waits that expired in these kernels on the current device
 * since the last reset. Zero in correct operation. A block of prompt attention
 * that gave up left the rows that it had not finished unwritten; in decode
 * attention the rows that the block had a part of are NaN. The limit is
 * sm120n_set_wait_limit's, here of every wait on an mbarrier. Both synchronise the
 * current device.
 */
SM120N_API int sm120s_get_device_faults(uint32_t* out_count);
SM120N_API int sm120s_reset_device_faults(void);

/*
 * Plans one serving step. With c = max(context_lens[r], 0) tokens of request r
 * in the cache, q = max(query_lens[r], 0) new ones and B = block_size:
 *   held = ceil(c / B), want = ceil((c + q) / B), end_r = q_0 + ... + q_r
 *   request r fits iff want <= table_width and end_r <= tokens; its need is
 *   want - held if want <= table_width, else 0; upto_r = need_0 + ... + need_r
 *   r is served iff it fits and (its need is 0 or upto_r <= free_count)
 * and writes
 *   block_table[r, held + j] = free_blocks[free_count - 1 - (upto_r - need + j)]
 *                              for j < need of a served request
 *   query_start[0] = 0, query_start[r + 1] = min(end_r, tokens)
 *   seq_lens[r]    = c + q, or c for a request that is not served
 *   positions[t]   = c + (t - (end_r - q)) for the tokens t of request r
 *   slot_mapping[t] = block_table[r, positions[t] / B] * B + positions[t] % B,
 *                    -1 for a request that is not served and for a table entry
 *                    outside [0, pool)
 *   positions = slot_mapping = -1 behind the last token (the Q/K norm
 *                    operators leave such tokens untouched)
 *   free_count_out = free_count - the blocks handed out.
 * A request gets all blocks it needs or none, in the order of the requests:
 * after the first one whose blocks are not there, none that needs blocks is
 * served. block_table [requests, table_width] int32, rows table_stride apart;
 * free_blocks [pool] is a stack whose top is free_blocks[free_count - 1]; it is
 * not written. free_count_out may be free_count and seq_lens may be
 * context_lens; other buffers may not overlap. tokens is the length of
 * positions (int64) and slot_mapping (int32). A request of 2^31 tokens or more is
 * not served. requests and table_width up to 2^30.
 */
SM120N_API int sm120s_plan_step(const int32_t* context_lens, const int32_t* query_lens,
                     int32_t* block_table, int64_t table_stride, const int32_t* free_blocks,
                     const int32_t* free_count, int32_t* free_count_out, int32_t* query_start,
                     int32_t* seq_lens, int64_t* positions, int32_t* slot_mapping,
                     int64_t requests, int64_t table_width, int64_t pool, int64_t block_size,
                     int64_t tokens, void* stream);

/*
 * The same, and the step with one row per request, as decode attention takes it
 * whoever has a token. For r with q > 0 whose first token got a place:
 *   row_positions[r] = c, row_slots[r] = its slot, row_lens[r] = c + q
 * and otherwise row_positions[r] = -1, row_lens[r] = 0 and row_slots[r] = -1 for a
 * request without a token, -2 for one whose token got no place. Each [requests],
 * all three or none (NULL).
 */
SM120N_API int sm120s_plan_step_rows(const int32_t* context_lens, const int32_t* query_lens,
                     int32_t* block_table, int64_t table_stride, const int32_t* free_blocks,
                     const int32_t* free_count, int32_t* free_count_out, int32_t* query_start,
                     int32_t* seq_lens, int64_t* positions, int32_t* slot_mapping,
                     int64_t* row_positions, int32_t* row_slots, int32_t* row_lens,
                     int64_t requests, int64_t table_width, int64_t pool, int64_t block_size,
                     int64_t tokens, void* stream);

/*
 * Gives the blocks of finished requests back: the entries
 * block_table[r, shared_blocks .. ceil(seq_lens[r] / block_size)) of every row
 * with finished[r] != 0, row after row, go to free_blocks[free_count ...];
 * free_count_out = free_count + their number. Entries outside [0, pool), and
 * what no longer fits free_blocks, are left out. The table and seq_lens are not
 * written. free_count_out may be free_count.
 */
SM120N_API int sm120s_release_blocks(const int32_t* seq_lens, const uint8_t* finished,
                          const int32_t* block_table, int64_t table_stride,
                          int32_t* free_blocks, const int32_t* free_count,
                          int32_t* free_count_out, int64_t requests, int64_t table_width,
                          int64_t pool, int64_t block_size, int64_t shared_blocks, void* stream);

#define SM120S_MAX_ROPE_AXES 4

/*
 * What sm120s_qk_norm_mrope_cache takes beyond sm120n_qk_cache_args, whose
 * `positions` then points to axis 0 of axis 0's tokens: axis a of token t is
 * positions[a * position_axis_stride + t] (stride 0: one row for all axes).
 * sections add up to rotary_dim / 2. One after another: the first sections[0]
 * pairs turn by axis 0, the next sections[1] by axis 1, and so on. Interleaved:
 * pair i turns by axis k = i mod axes if k > 0 and i < axes * sections[k], else
 * by axis 0. query_out / key_out: NULL for in place, or adjacent heads at these
 * token strides (elements): the input's own rows, or rows that share nothing with
 * query, key, value, the caches and one another. (value may be key's own rows.)
 */
typedef struct sm120s_mrope_args {
  uint32_t struct_size; /* sizeof(sm120s_mrope_args) */
  int32_t axes;         /* 1 to SM120S_MAX_ROPE_AXES */
  int32_t sections[SM120S_MAX_ROPE_AXES];
  int32_t interleaved_sections;
  int64_t position_axis_stride;
  void* query_out;
  int64_t query_out_token_stride;
  void* key_out;
  int64_t key_out_token_stride;
} sm120s_mrope_args;

/*
 * Per-head Q/K RMSNorm + rotation by positions with several axes + KV store:
 *   n = x * (1 / sqrt(mean(x^2) + eps)) * w
 *   pairs of n rotated as in sm120n_qk_norm_rope_cache (rope_style), each by
 *   the cos_sin_cache row of its axis's position; the rest of the head is n
 * in fp32 throughout, rounded once to the activation dtype and, on its own
 * from the same fp32 value, to an fp8 cache (sat(y / scale), nearest even).
 * (sm120n_qk_norm_rope_cache rounds after the norm and after the weight too,
 * so with all axes alike the two may differ in a last place.) A token with a
 * position outside [0, rope_positions) on any axis is left untouched and
 * stores nothing; slots outside the cache store nothing.
 */
SM120N_API int sm120s_qk_norm_mrope_cache(const sm120n_qk_cache_args* args,
                               const sm120s_mrope_args* mrope, void* stream);

/*
 * Causal attention of packed prompts. Sequence s is the tokens
 * [query_start[s], query_start[s + 1]) (clamped to [0, tokens]; one that ends
 * before it begins is empty); its token i gives, for query head h with key
 * head h / (query_heads / key_heads),
 *   out[i, h] = sum_{j <= i} p_j v_j / sum_j p_j,  p_j = exp(scale * q_i . k_j)
 * with fp32 scores and sums, p rounded to the activation dtype for the second
 * product, and the result rounded once. Keys behind token i take no part,
 * whatever they hold. Rows behind the last sequence are left as they were.
 * Sequences may not overlap: after a start that falls, rows of several sequences
 * may come from any of them, and where the sequences have more than `tokens`
 * tokens in all, rows of the last ones may be left as they were.
 * query, out [tokens, query_heads, head_dim], key, value [tokens, key_heads,
 * head_dim]: heads adjacent, token strides in elements, rows 16-byte aligned.
 * out may not overlap the inputs. dtype f16 or bf16; head_dim 64, 128 or 256;
 * scale finite and positive.
 */
typedef struct sm120s_prompt_args {
  uint32_t struct_size; /* sizeof(sm120s_prompt_args) */
  int32_t dtype;
  int64_t tokens;
  int64_t sequences;
  int64_t query_heads; /* a multiple of key_heads */
  int64_t key_heads;
  int64_t head_dim;
  const void* query;
  int64_t query_token_stride;
  const void* key;
  int64_t key_token_stride;
  const void* value;
  int64_t value_token_stride;
  void* out;
  int64_t out_token_stride;
  const int32_t* query_start; /* [sequences + 1] */
  float scale;
} sm120s_prompt_args;

SM120N_API int sm120s_prompt_attention(const sm120s_prompt_args* args, void* stream);

/*
 * Attention of one token per request over a paged cache, for a batch whose
 * requests may begin with the same blocks. With P = prefix_blocks_count *
 * block_size and n = min(max(seq_lens[b], 0), table_width * block_size), the
 * keys of request b are
 *   n >= P: the P tokens of prefix_blocks, then tokens P .. n - 1 of row b of
 *           block_table (entry j is the block of tokens [j * block_size, ...),
 *           the entries before P / block_size are not read)
 *   n < P:  tokens 0 .. n - 1 of row b alone
 *   out[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q_b . k_j)
 * fp32 scores, sums and values, p rounded to 16 bits for the second product;
 * zeros where there is no key. Blocks outside [0, num_blocks) hold no keys. The
 * prefix is read once for all requests. out may not overlap query or a cache.
 * query, out [batch, query_heads, head_dim], heads adjacent; caches as
 * sm120n_qk_cache_args (one shape and stride for both), rows 16-byte aligned and
 * at least head_dim elements apart in every dimension;
 * fp8 caches stand for code * k_scale[0] / code * v_scale[0]. dtype f16 or bf16.
 * workspace: sm120s_paged_decode_workspace bytes, 16-byte aligned, written and
 * read by this call alone: calls that may run at the same time, or graphs that
 * may be replayed at the same time, need one each.
 */
typedef struct sm120s_decode_args {
  uint32_t struct_size; /* sizeof(sm120s_decode_args) */
  int32_t dtype;
  int32_t cache_dtype; /* sm120n_cache_dtype */
  int32_t reserved;
  int64_t batch;
  int64_t query_heads; /* a multiple of key_heads */
  int64_t key_heads;
  int64_t head_dim; /* 64, 128 or 256 */
  const void* query;
  int64_t query_token_stride;
  void* out;
  int64_t out_token_stride;
  const void* key_cache;
  const void* value_cache;
  int64_t num_blocks;
  int64_t block_size;
  int64_t cache_block_stride;
  int64_t cache_slot_stride;
  int64_t cache_head_stride;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_table; /* [batch, table_width] */
  int64_t table_width;
  int64_t table_stride;
  const int32_t* seq_lens;
  const int32_t* prefix_blocks;
  int64_t prefix_blocks_count;
  void* workspace;
  size_t workspace_bytes;
  float scale;
} sm120s_decode_args;

/* Bytes of workspace for a call with these sizes on the current device (the
 * pointers, strides and workspace fields are not looked at). */
SM120N_API int sm120s_paged_decode_workspace(const sm120s_decode_args* args, size_t* bytes);

SM120N_API int sm120s_paged_decode_attention(const sm120s_decode_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SM120NORM_B200_SERVING_H_ */
