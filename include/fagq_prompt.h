/* fagq_prompt.h - C ABI of the causal attention of whole prompts, packed one
 * behind the other, and its gradients (libfagq.so, gfx950).  No counterpart in
 * the reference repository, whose MLA backward (src/task03_mla_bwd_nope_dkdv.py)
 * is of one shared latent and not of grouped heads.
 *
 * B sequences: the queries of sequence b are rows cu_seqlens[b] to
 * cu_seqlens[b + 1] - 1 of q [T, Hq, D], its keys and values those rows of k and
 * v [Tk, H, D] that cu_seqlens_k names (null: the same as cu_seqlens).  With n
 * queries and m keys, query i sees the keys j <= i + m - n: the newest query sees
 * all, as in a prefill that continues a context.  Query head h reads head
 * h / (Hq / H).
 *
 *   x_ij = sm_scale q_i . k_j,   lse_i = ln sum_j e^x_ij,   out_i = sum_j e^(x_ij - lse_i) v_j
 *
 * and 0 and -inf for a query that sees no key.  The gradients, with dout:
 *
 *   P = e^(x - lse),  delta_i = dout_i . out_i,  dS_ij = P_ij (dout_i . v_j - delta_i)
 *   dq_i = sm_scale sum_j dS_ij k_j
 *   dk_j = sm_scale sum dS_ij q_i,  dv_j = sum P_ij dout_i   (over i and the heads of the group)
 *
 * Sums, maxima and exponentials are in fp32; P and dS are rounded to the element
 * type for the products that they enter, in fp16 times powers of two that keep dS
 * in its range whatever dout's size: gradients that fp16 holds are right.
 *
 * Same conventions as fagq.h: device pointers, stream-ordered, no allocation, no
 * synchronization; returns 0, a FAGQ_E_* code or -hipError_t.  cu_seqlens and
 * cu_seqlens_k are int32 [B + 1], ascending from 0; whatever they hold, nothing is
 * read or written outside the tensors.  The rows that they name are finite; rows
 * behind the last sequence are not read.
 */
#ifndef FAGQ_PROMPT_H_
#define FAGQ_PROMPT_H_

#include <stdint.h>

#include "fagq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Which outputs' rows behind the last sequence are filled, with 0, lse with -inf;
 * those of the others are left as they were. */
enum fagq_prompt_fill { FAGQ_FILL_OUT = 1, FAGQ_FILL_LSE = 2 };
enum fagq_prompt_bwd_fill { FAGQ_FILL_DQ = 1, FAGQ_FILL_DK = 2, FAGQ_FILL_DV = 4 };

/* q, k, v: dtype (FAGQ_DT_BF16, FAGQ_DT_F16), D contiguous, D in {64, 128, 256},
 * Hq % H == 0.  strides (host memory, in elements): {token, head} of q, k, v,
 * multiples of 8; token strides below 2^24, head strides below 2^31.  out
 * [T, Hq, D] contiguous; lse fp32 [Hq, T], or null.  k and v may be null where Tk
 * is 0.  16-byte aligned, but lse and the lengths 4.  Workspace: 16-byte aligned,
 * of fagq_prompt_attention_workspace_bytes (0: may be null); calls that may overlap
 * need one each.  FAGQ_E_TOO_LARGE (workspace: -1) for more than 2^31 - 1024 tokens,
 * and for 2^24 workgroups and more: (T / 128 + B) Hq of them at least. */
FAGQ_API int64_t fagq_prompt_attention_workspace_bytes(int64_t B, int64_t T, int64_t Tk,
                                                       int64_t Hq, int64_t H, int64_t D);
FAGQ_API int fagq_prompt_attention_launch(const void* q, const void* k, const void* v,
                                          const int32_t* cu_seqlens, const int32_t* cu_seqlens_k,
                                          void* out, float* lse, void* workspace,
                                          int64_t workspace_bytes, const int64_t* strides,
                                          int64_t B, int64_t T, int64_t Tk, int64_t Hq, int64_t H,
                                          int64_t D, float sm_scale, int dtype, int fill,
                                          void* stream);

/* out, lse: of the call above.  dout [T, Hq, D], dq, dk, dv: dtype.  strides:
 * {token, head} of dout, q, k, v, dq, dk, dv, as above; out and lse are contiguous.
 * Gradients are written, not added to.  The sums are added in an order that depends
 * on the sizes alone: equal calls give equal bits.  FAGQ_E_TOO_LARGE where the forward
 * has it, and for 2^24 tiles of keys and more, (Tk / 128 + B) H, which Tk above T only
 * can have. */
FAGQ_API int64_t fagq_prompt_attention_bwd_workspace_bytes(int64_t B, int64_t T, int64_t Tk,
                                                           int64_t Hq, int64_t H, int64_t D);
FAGQ_API int fagq_prompt_attention_bwd_launch(const void* dout, const void* q, const void* k,
                                              const void* v, const void* out, const float* lse,
                                              const int32_t* cu_seqlens,
                                              const int32_t* cu_seqlens_k, void* dq, void* dk,
                                              void* dv, void* workspace, int64_t workspace_bytes,
                                              const int64_t* strides, int64_t B, int64_t T,
                                              int64_t Tk, int64_t Hq, int64_t H, int64_t D,
                                              float sm_scale, int dtype, int fill, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FAGQ_PROMPT_H_ */
