/* fagq_cache.h - C ABI of the quantised paged key/value cache: writing it,
 * reading it back, and attention over it (libfagq.so, gfx950).  No counterpart
 * in the reference repository; its page tables are those that the DSA transform
 * reads (src/task02_dsa_topk_page_table_transform.py:1666-1726).
 *
 * Layout, contiguous:
 *   codes  [num_pages, H, page_size, D]       fp8 e4m3fn or int8
 *   scales [num_pages, H, D / G, page_size]   fp32 or UE8M0 (column-major in a page)
 * page_size is a power of two, 16 to 65536.  A slot is page * page_size + offset.
 * A value is code * scale.  Keys and values have one such pair each; a cache of
 * latents passes null for everything that is named v.
 *
 * Same conventions as fagq.h: device pointers, stream-ordered, no allocation,
 * no synchronization; returns 0, a FAGQ_E_* code or -hipError_t.  Indexes that
 * are read on the device (slots, page tables, lengths) never lead outside the
 * tensors: what is out of range is left out, as each function says.
 */
#ifndef FAGQ_CACHE_H_
#define FAGQ_CACHE_H_

#include <stdint.h>

#include "fagq.h"
#include "fagq_rope.h"   /* enum fagq_index */

#ifdef __cplusplus
extern "C" {
#endif

#define FAGQ_CACHE_MIN_PAGE 16
#define FAGQ_CACHE_MAX_PAGE 65536
#define FAGQ_CACHE_MAX_D 1024

/* k, v [T, H, D] (dtype: FAGQ_DT_*), D contiguous, any token and head strides;
 * strides (host memory, in elements): {token, head} of k, v.  Token t goes to
 * slots[t]; one whose slot lies outside [0, num_pages * page_size) is not
 * written.  Two tokens may not name one slot (its content is then undefined;
 * no other slot is touched).  Each group of G values:
 *   s = max(max|x| * fp32(1 / QMAX), 1e-12),   code = encode(x * (1 / s))
 * UE8M0: s = 2^ceil(log2 s), code = encode(x / s).  fp8 (QMAX 448) and int8
 * (QMAX 127) round to nearest even.  Values are finite.
 * G in {64, 128, 256}, D % G == 0, D <= FAGQ_CACHE_MAX_D; T <= 2^24.
 * k, v 16-byte aligned, strides multiples of 16 bytes. */
FAGQ_API int fagq_kv_cache_write_launch(const void* k, const void* v, const void* slots,
                                        void* k_cache, void* v_cache, void* k_scale,
                                        void* v_scale, const int64_t* strides, int64_t T,
                                        int64_t H, int64_t D, int64_t G, int64_t num_pages,
                                        int64_t page_size, int dtype, int q_format,
                                        int scale_format, int index_dtype, void* stream);

/* Gathers the tokens of B sequences: token j of sequence b, at slot
 * page_table[b, j / page_size] * page_size + j % page_size, goes to row
 * cu_seqlens[b] + j of k_out, v_out [rows, H, D] (dtype, contiguous), as
 * code * scale in fp32, rounded once.  page_table int32 [B, table_width],
 * cu_seqlens int32 [B + 1], ascending from 0.  Tokens whose page lies outside the
 * table or the cache (-1: none) become zeros.  Rows behind cu_seqlens[B] are left
 * as they were.  The cache may be null where num_pages is 0, page_table where the
 * width is 0: all tokens are zeros then.  rows <= 2^31 - 1, and FAGQ_E_TOO_LARGE
 * where 2^24 workgroups do not cover them. */
FAGQ_API int fagq_kv_cache_read_launch(const void* k_cache, const void* v_cache,
                                       const void* k_scale, const void* v_scale,
                                       const int32_t* page_table, const int32_t* cu_seqlens,
                                       void* k_out, void* v_out, int64_t B, int64_t rows,
                                       int64_t H, int64_t D, int64_t G, int64_t num_pages,
                                       int64_t page_size, int64_t table_width, int dtype,
                                       int q_format, int scale_format, void* stream);

/* Attention of the newest S tokens of each of B sequences over the cache.
 *
 *   q, out [B, S, Hq, D] bf16 or fp16 (dtype); Hq % H == 0, query head h reads
 *   cache head h / (Hq / H).  Keys of query (b, s): the prefix_len tokens of
 *   prefix_pages, which all sequences share, then tokens
 *   j < min(kv_lens[b], table_width * page_size) - S + s + 1 of the pages of
 *   page_table[b] (kv_lens[b] counts own tokens, the newest S among them).
 *   out = softmax(q . key * sm_scale) value; a query without keys gets zeros.
 *   Tokens on pages outside [0, num_pages) are left out.
 *
 * One scale for each token and head (G == D), D in {64, 128, 256}.  strides
 * (host memory, in elements): {sequence, token, head} of q, multiples of 8, below
 * 2^31; out is contiguous.  page_table int32 [B, table_width], null if the
 * width is 0; kv_lens [B] (index_dtype); prefix_pages int32
 * [ceil(prefix_len / page_size)], null without.
 * max_kv_len: no kv_lens[b] is larger; longer ones are cut to it.  It, and not the
 * lengths, decides how the work is split and whether codes are read past the caches.
 * Sums and softmax are in fp32; the probabilities, times their value scales, are
 * rounded to fp16 (relative to the row's largest) for the product with the codes.
 * Codes and scales of the tokens that a sequence reads are finite, value scales 0 to
 * 2^64 (below 2^-64 what a key adds is exact to 2^-88 of its codes only; UE8M0 0
 * counts as 0); what lies in other slots does not matter.
 * The workspace (16-byte aligned) belongs to this call until it has run: calls that
 * may overlap need one each.  Its size is that of exactly these B ... max_kv_len:
 * fewer sequences or a smaller bound are cut into more parts and may need more (1024
 * keys, 64 + 8 heads of 128: B 16 2.1 MB, B 64 none), so one that serves several
 * calls is as large as the largest of theirs.
 * FAGQ_E_TOO_LARGE (workspace: -1) for 2^24 rows or workgroups and more. */
FAGQ_API int64_t fagq_paged_attention_workspace_bytes(int64_t B, int64_t S, int64_t Hq, int64_t H,
                                                      int64_t D, int64_t prefix_len,
                                                      int64_t max_kv_len);
FAGQ_API int fagq_paged_attention_launch(const void* q, const void* k_cache, const void* v_cache,
                                         const void* k_scale, const void* v_scale,
                                         const int32_t* page_table, const void* kv_lens,
                                         const int32_t* prefix_pages, void* out, void* workspace,
                                         int64_t workspace_bytes, const int64_t* strides,
                                         int64_t B, int64_t S, int64_t Hq, int64_t H, int64_t D,
                                         int64_t num_pages, int64_t page_size, int64_t table_width,
                                         int64_t prefix_len, int64_t max_kv_len, float sm_scale,
                                         int dtype, int q_format, int scale_format,
                                         int index_dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FAGQ_CACHE_H_ */
