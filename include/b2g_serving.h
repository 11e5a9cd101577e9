/*
 * b2g_serving.h — C ABI of the operators that serve a model from a paged,
 * 8-bit key/value cache: block tables and slot map, the cache write, the
 * attention of one token per request over the cache, and the causal
 * attention of whole prompts.
 *
 * Conventions as in b2g_gemm.h: plain pointers and sizes, b2g_status return
 * codes, asynchronous launches on the caller's stream, nothing allocated and
 * nothing synchronised, bounded device-side waits (b2g_read_device_error).
 * The values that live on the device (lengths, tables, slots) are not read by
 * the host; the kernels check each index that they form from them against the
 * buffers' sizes, so a wrong value gives a wrong or missing result and no
 * access out of bounds.  The reference has no counterpart to these operators.
 *
 * The cache.  k_cache, v_cache: (num_blocks, kv_heads, block_size, dim) codes
 * of 8 bits, dense, 16-byte aligned; k_scale, v_scale: (num_blocks, kv_heads)
 * fp32.  A code c of a block and head stands for c * scale.  block_size: a
 * power of two from 16 to 256; dim: a multiple of 16, at most 128.
 */
#ifndef B2G_SERVING_H
#define B2G_SERVING_H

#include "b2g_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum b2g_dtype { B2G_F16 = 0, B2G_BF16 = 1 } b2g_dtype;
typedef enum b2g_codes { B2G_I8 = 0, B2G_E4M3 = 1 } b2g_codes;

/*
 * Block tables, slot map and row offsets of one serving step.
 *
 * Request r holds context_lens[r] tokens and gains new_lens[r] (negative
 * counts as 0).  Its table row has ceil(context / block_size) entries
 * already; the blocks that its new tokens need beyond those are taken from
 * the top of the stack free_blocks[0 .. *free_count), the requests in order
 * and each request's blocks in order, and written into its row of
 * block_table (row r at block_table + r * table_ld, table_width entries).
 *   slots[t]      = block * block_size + place of the t-th new token (the
 *                   requests one after another); -1 where there is no block
 *                   and for t past the last new token
 *   cu_seqlens[r] = new tokens before request r (requests + 1 values)
 *   seq_lens[r]   = context_lens[r] + new_lens[r]
 *   *free_count_out = *free_count - blocks needed; below 0: that many blocks
 *                   were missing, and their entries are -1
 * A table row that is too short takes no block for what lies beyond it.
 * free_count is not written: pass *free_count_out to the next step.
 * The sum of new_lens is below 2^31.  requests <= B2G_MAX_TABLE_REQUESTS.
 */
#define B2G_MAX_TABLE_REQUESTS 16384
B2G_API int b2g_block_tables(const int32_t* context_lens, const int32_t* new_lens,
                             int64_t requests, int32_t* block_table, int64_t table_width,
                             int64_t table_ld, const int32_t* free_blocks, int64_t free_capacity,
                             const int32_t* free_count, int64_t total_tokens, int block_size,
                             int64_t* slots, int32_t* cu_seqlens, int32_t* seq_lens,
                             int32_t* free_count_out, b2g_stream_t stream);

/*
 * The cache write: token t's key and value of each head go to slot slots[t].
 * Tokens in consecutive slots of one block form a group.  With fill = the
 * group's first place in its block, for each head, and for keys and values:
 *   scale' = max(fill > 0 ? scale : 0, max |x| over the group / qmax)
 *   the fill codes that the block held: round(code * (scale / scale'))
 *   the new codes: round(x * (1 / scale'))
 * with qmax 127 (int8) or 448 (e4m3) and rounding to nearest even, in fp32.
 * Infinities and NaN do not count for the scale; an infinity is stored as the
 * largest code, NaN as 0 (int8) or NaN (e4m3).  A slot outside the cache
 * (-1) is skipped.  The tokens of one block are one group: no block is met
 * twice in a call.
 * k, v: element (t, h, i) at t * token_stride + h * head_stride + i, strides
 * multiples of 8 elements, 16-byte aligned.
 */
typedef struct b2g_cache_append_desc {
  int32_t dtype;                /* b2g_dtype of k and v                    */
  int32_t codes;                /* b2g_codes of the cache                  */
  int64_t tokens, kv_heads, dim;
  int64_t num_blocks, block_size;
  const void* k; int64_t k_token_stride, k_head_stride;
  const void* v; int64_t v_token_stride, v_head_stride;
  const int64_t* slots;
  void* k_cache; void* v_cache;
  float* k_scale; float* v_scale;
} b2g_cache_append_desc;
B2G_API int b2g_cache_append(const b2g_cache_append_desc* desc, b2g_stream_t stream);

/*
 * One query token per request over the cache, query head j reading kv head
 * j / (heads / kv_heads) (the cache is read once for every 16 of them):
 *   out[r][j] = sum_n softmax_n(scale * q[r][j] . K[r][n]) V[r][n],
 *   n < seq_lens[r], token n in block block_table[r][n / block_size]
 * Lengths are cut to table_width * block_size; a block number outside the
 * cache leaves its tokens out.  num_blocks * kv_heads * block_size, the rows
 * that the kernel counts, stays below 2^31; so do table_width * block_size and
 * requests * table_width * block_size / 64.  A request without tokens gives
 * zeros, and -infinity for its log sum.  scale 0 selects 1/sqrt(dim), below 0 or not
 * finite is an error.
 * q: (requests, heads, dim), element (r, j, i) at r * q_row_stride +
 * j * q_head_stride + i (multiples of 8, 16-byte aligned); out: dense
 * (requests, heads, dim); lse: null, or (requests, heads) fp32 natural
 * logarithms of the softmax's sums.  (Over int8 codes a score is the difference
 * of two sums in fp32, an error of up to 2^-13 * scale * k_scale * sum |q|.)
 */
typedef struct b2g_cache_attention_desc {
  int32_t dtype;                /* b2g_dtype of q and out                  */
  int32_t codes;                /* b2g_codes of the cache                  */
  int64_t requests, heads, kv_heads, dim;
  int64_t num_blocks, block_size;
  const void* q; int64_t q_row_stride, q_head_stride;
  const void* k_cache; const void* v_cache;
  const float* k_scale; const float* v_scale;
  const int32_t* block_table; int64_t table_width, table_ld;
  const int32_t* seq_lens;
  float scale;
  void* out;
  float* lse;
  void* workspace;              /* device memory, >= ..._workspace_bytes() */
  int64_t workspace_bytes;
} b2g_cache_attention_desc;
B2G_API int64_t b2g_cache_attention_workspace_bytes(const b2g_cache_attention_desc* desc);
B2G_API int b2g_cache_attention(const b2g_cache_attention_desc* desc, b2g_stream_t stream);

/*
 * Attention of whole prompts, packed one after another: sequence s has the
 * query rows cu_q[s] .. cu_q[s+1] and the key rows cu_k[s] .. cu_k[s+1]
 * (cu_k null: the same rows).  causal != 0: query i of n sees key j of m
 * where j <= i + m - n (the last query sees the last key).  A row that sees
 * nothing gives zeros, and -infinity for its log sum; so does a query row that
 * belongs to no sequence.
 * What stands in another sequence never reaches a row.  Within its own, a
 * weight of 0 is still multiplied by the value: an infinity or NaN in v also
 * reaches earlier rows that share its tile of 128 keys.
 * q, k, v, out: element (t, h, i) at t * token_stride + h * head_stride + i,
 * strides multiples of 8 elements, 16-byte aligned; heads a multiple of
 * kv_heads, heads / kv_heads <= 128; dim a multiple of 16, at most 128.
 * scale 0 selects 1/sqrt(dim), below 0 or not finite is an error.  lse: null,
 * or (tokens, heads) fp32, the natural logarithms of the sums; a part of the
 * exponentials is a polynomial whose relative error, and so the lse's absolute
 * one, reaches 7.5e-5 for bf16 and 2.7e-6 for fp16.
 */
typedef struct b2g_prompt_attention_desc {
  int32_t dtype;                /* b2g_dtype of q, k, v and out            */
  int32_t causal;
  int64_t tokens, tokens_k, sequences, heads, kv_heads, dim;
  const void* q; int64_t q_token_stride, q_head_stride;
  const void* k; int64_t k_token_stride, k_head_stride;
  const void* v; int64_t v_token_stride, v_head_stride;
  void* out; int64_t out_token_stride, out_head_stride;
  const int32_t* cu_q;
  const int32_t* cu_k;
  float scale;
  float* lse;
} b2g_prompt_attention_desc;
B2G_API int b2g_prompt_attention(const b2g_prompt_attention_desc* desc, b2g_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* B2G_SERVING_H */
