/* fagq_rope.h - C ABI of the norms of queries and keys for each head with the
 * rotation by position in the same pass, and their gradients (libfagq.so,
 * gfx950).  No counterpart in the reference repository: its RMSNorm
 * (src/task01_fused_add_rmsnorm_group_quant.py:88-100) is over hidden rows.
 *
 * For each row x (one head of one token, D wide) of q and of k:
 *
 *   rstd = 1 / sqrt(mean(x^2) + eps),   n = x * rstd * weight
 *   y    = n with its first R dims rotated by the token's position p:
 *          (a, b) -> (a cos[p, i] - b sin[p, i], b cos[p, i] + a sin[p, i]),
 *          pair i of R / 2: (n[i], n[i + R / 2]), or (n[2 i], n[2 i + 1]) if interleaved
 *
 * all in fp32 (squares too: values lie below 2^59), rounded once to the element type.  A token whose position lies
 * outside [0, table_rows) is padding: its rows of y are zeros, and so are its
 * gradients.  The backward takes the same inputs and dy:
 *
 *   dn = dy rotated back,  a = dn * weight
 *   dx = rstd * (a - x rstd^2 mean(a x)),  dweight = sum over rows of dn x rstd
 *
 * Same conventions as fagq.h: device pointers, stream-ordered, no allocation,
 * no synchronization; returns 0, a FAGQ_E_* code or -hipError_t.
 */
#ifndef FAGQ_ROPE_H_
#define FAGQ_ROPE_H_

#include <stdint.h>

#include "fagq.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FAGQ_ROPE_MAX_D 512

enum fagq_index { FAGQ_IDX_I32 = 0, FAGQ_IDX_I64 = 1 };

/* q [T, Hq, D], k [T, Hk, D], q_out, k_out of the same shapes: dtype (FAGQ_DT_*),
 * D contiguous, any token and head strides.  strides (host memory, in elements):
 * {token, head} of q, k, q_out, k_out.  q_weight, k_weight [D]: dtype.  cos, sin
 * [table_rows, R / 2] fp32, contiguous.  positions [T] (index_dtype).
 * All pointers but positions 16-byte aligned, strides multiples of 16 bytes and
 * below 2^31 elements.  16 <= R <= D <= FAGQ_ROPE_MAX_D, D % 16 == 0, R % 16 == 0.
 * q_out may be q itself, and k_out k (same pointer and strides); outputs overlap
 * nothing else.  FAGQ_E_TOO_LARGE where 2^24 workgroups do not cover the heads. */
FAGQ_API int fagq_qk_norm_rope_launch(const void* q, const void* k, const void* q_weight,
                                      const void* k_weight, const float* cos, const float* sin,
                                      const void* positions, void* q_out, void* k_out,
                                      const int64_t* strides, int64_t T, int64_t Hq, int64_t Hk,
                                      int64_t D, int64_t R, int64_t table_rows, float eps,
                                      int interleaved, int dtype, int index_dtype, void* stream);

/* Workspace bytes of fagq_qk_norm_rope_bwd_launch: each workgroup's sums of both
 * weight gradients.  -1 for sizes that the launch refuses. */
FAGQ_API int64_t fagq_qk_norm_rope_bwd_workspace_bytes(int64_t T, int64_t Hq, int64_t Hk,
                                                       int64_t D);

/* dq_out, dk_out: gradients of q_out and k_out.  Writes dq, dk (dtype) and
 * dq_weight, dk_weight [D] (fp32).  strides: {token, head} of dq_out, dk_out, q,
 * k, dq, dk.  workspace: 16-byte aligned, overwritten; calls that may overlap need
 * one each.  Outputs overlap nothing.
 * The sums are added in an order that depends on the sizes alone. */
FAGQ_API int fagq_qk_norm_rope_bwd_launch(const void* dq_out, const void* dk_out, const void* q,
                                          const void* k, const void* q_weight,
                                          const void* k_weight, const float* cos, const float* sin,
                                          const void* positions, void* dq, void* dk,
                                          float* dq_weight, float* dk_weight, void* workspace,
                                          int64_t workspace_bytes, const int64_t* strides,
                                          int64_t T, int64_t Hq, int64_t Hk, int64_t D, int64_t R,
                                          int64_t table_rows, float eps, int interleaved,
                                          int dtype, int index_dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FAGQ_ROPE_H_ */
