/*
 * mpx_cache8.h — C ABI of the 8-bit paged KV cache (libmpx_attn.so): the append
 * of keys and values, their read-back, and the attention over such pages.
 * Conventions (errors, streams, pointers, strides) are those of mpx_attn.h.
 *
 * Pools k_pool, v_pool: (num_blocks, block_size, H_kv, D) codes, contiguous,
 * 16-byte aligned, D a multiple of 16 up to 256, block_size at most
 * MPX8_MAX_BLOCK_SIZE. Scales k_scales, v_scales: float32 (num_blocks, H_kv),
 * contiguous. A code c of page p and head h stands for value(c) * scales[p, h];
 * value(c) is the signed integer (MPX8_INT8) or the OCP e4m3 number
 * (MPX8_E4M3, largest 448).
 */
#ifndef MPX_CACHE8_H
#define MPX_CACHE8_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MPX8_E4M3 0
#define MPX8_INT8 1
#define MPX8_MAX_BLOCK_SIZE 32768

/*
 * Write new tokens into their pages: token t of sequence b goes to position
 * start_pos[b] + t, as mpx_kv_append (and, with cos_cache and sin_cache, K
 * rotated to it, as mpx_kv_append_rope; NULL: as given), quantised.
 *
 * Each page and head has one scale for K and one for V, a power of two. With a
 * the largest finite |value| that the call brings to the page and head (K after
 * rotation, which is exact: codes are rounded once) and M = 448 (e4m3) or 127 (int8):
 *   need = 2^e, e the least integer with a <= M * 2^e, kept in -100 .. 113;
 *   a call that writes slot 0 of a page starts it anew: scale = need;
 *   else scale = max(old scale, need), and where it grew the codes of the slots
 *   before the first one written are brought to it (round(code * old / new)).
 * New codes are round(value / scale), ties to even; values past the largest
 * code saturate; NaN stays NaN in e4m3 and becomes 0 in int8. Slots behind the
 * last one written keep their bytes, which then stand for nothing: a sequence
 * ends where it was last written. One call writes a page for one sequence.
 *
 *   k, v       (B, T, H, D) of `dtype` through {batch, token, head} strides
 *   n_tokens   int32 (B,): tokens of each sequence, the rest of T is not read; NULL: T
 *   errors     int32[3], [4] with tables: the words of mpx_kv_append(_rope), each written
 *              0 or 1 (calls with no row write nothing)
 */
int mpx_kv_append8(const void* k, const void* v, void* k_pool, void* v_pool, float* k_scales,
                   float* v_scales, const int32_t* block_tables, const int32_t* start_pos,
                   const int32_t* n_tokens, const int64_t* k_strides, const int64_t* v_strides,
                   int B, int T, int H, int D, int num_blocks, int block_size, int max_blocks,
                   int dtype, int code, const void* cos_cache, const void* sin_cache, int n_pos,
                   int cache_dtype, int32_t* errors, void* stream);

/*
 * The same for pages that hold more than a sequence's end: every slot that the call
 * does not write keeps its value, before and behind the written ones. Only a call that
 * writes all slots of a page starts it anew; any other has scale = max(old scale, need),
 * and where it grew all other slots' codes are brought to it (once each, to the nearest).
 * A page that holds nothing yet has the scale 0.
 */
int mpx_kv_write8(const void* k, const void* v, void* k_pool, void* v_pool, float* k_scales,
                  float* v_scales, const int32_t* block_tables, const int32_t* start_pos,
                  const int32_t* n_tokens, const int64_t* k_strides, const int64_t* v_strides,
                  int B, int T, int H, int D, int num_blocks, int block_size, int max_blocks,
                  int dtype, int code, const void* cos_cache, const void* sin_cache, int n_pos,
                  int cache_dtype, int32_t* errors, void* stream);

/*
 * Values of cached tokens: k_out, v_out (B, T, H, D) of `dtype`, contiguous,
 * 16-byte aligned. Row t of sequence b is position start_pos[b] + t; rows t >=
 * n_tokens[b], and rows without a page in the table, are zeros.
 */
int mpx_kv_load8(const void* k_pool, const void* v_pool, const float* k_scales,
                 const float* v_scales, const int32_t* block_tables, const int32_t* start_pos,
                 const int32_t* n_tokens, void* k_out, void* v_out, int B, int T, int H, int D,
                 int num_blocks, int block_size, int max_blocks, int dtype, int code,
                 void* stream);

/*
 * Attention of Sq queries a sequence over its cached tokens:
 *   o_i = sum_t softmax_t(scale * q_i . k_t + slope_h * (t - pos_i)) v_t
 * over t < context_lens[b] with a page id in [0, num_blocks) and, where causal,
 * t <= pos_i. pos_i = query_start[b] + i, with query_start NULL: i, and for
 * Sq == 1 context_lens[b] (and no causal mask), as in mpx_paged_decode and
 * mpx_paged_prefill. Rows that see no token are NaN. Scales must be positive, but
 * those of pages that no visible token is in; they and all slots that no sequence
 * reaches may hold anything. Scales may be any factor apart, but that float16 queries in more
 * than 32 rows (Sq H / H_kv; 16 above head dim 128) want K and V in float16's range: what is
 * under 2^-31 of a scale near it counts as nothing there. An e4m3 NaN in V may also reach rows
 * that share a tile with its token and do not see it (their weight of 0 times NaN).
 *
 *   q, o       (B, Sq, H, D) of `dtype` through {batch, head, seq} strides, q
 *              16-byte aligned in base and strides; H a multiple of H_kv
 *   workspace  mpx_paged_attend8_call_workspace_bytes(...) bytes (positions: whether
 *              query_start is given), 16-byte aligned; at most 256 MiB, whatever the
 *              tables' width, or none. mpx_paged_attend8_workspace_bytes(...): enough for
 *              any causal and query_start
 */
int mpx_paged_attend8(const void* q, const void* k_pool, const void* v_pool,
                      const float* k_scales, const float* v_scales, const int32_t* block_tables,
                      const int32_t* context_lens, const int32_t* query_start,
                      const float* alibi_slopes, void* o, const int64_t* q_strides,
                      const int64_t* o_strides, int B, int Sq, int H, int H_kv, int D,
                      int num_blocks, int block_size, int max_blocks, float scale, int causal,
                      int dtype, int code, void* workspace, size_t workspace_bytes, void* stream);
size_t mpx_paged_attend8_workspace_bytes(int B, int Sq, int H, int H_kv, int D, int block_size,
                                         int max_blocks, int dtype);
size_t mpx_paged_attend8_call_workspace_bytes(int B, int Sq, int H, int H_kv, int D,
                                              int block_size, int max_blocks, int dtype,
                                              int causal, int positions);

#ifdef __cplusplus
}
#endif
#endif
