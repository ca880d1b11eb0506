// paged_attn_inst.hip - instantiations of the paged attention for one element type, code
// format and scale format (FAGQ_ATTN_E, FAGQ_ATTN_QF, FAGQ_ATTN_SF).
#include "paged_attn_kernels.hpp"

namespace fagq {
namespace attn {
namespace {

template <int D, int R, int RP>
const void* kernel() {
  return reinterpret_cast<const void*>(
      &paged_attention<FAGQ_ATTN_E, FAGQ_ATTN_QF, FAGQ_ATTN_SF, D, R, RP>);
}

// The pairs (R, RP) that plan_for makes: 16 rows of a sequence go with a prefix of any unit, more
// rows with units of their own size; R D <= 256.
template <int D>
const void* lookup(int R, int RP) {
  if (R == 1 && RP == 0) return kernel<D, 1, 0>();
  if (R == 1 && RP == 1) return kernel<D, 1, 1>();
  if constexpr (D <= 128) {
    if (R == 1 && RP == 2) return kernel<D, 1, 2>();
    if (R == 2) return RP == 0 ? kernel<D, 2, 0>() : kernel<D, 2, 2>();
  }
  if constexpr (D == 64) {
    if (R == 1 && RP == 4) return kernel<D, 1, 4>();
    if (R == 4) return RP == 0 ? kernel<D, 4, 0>() : kernel<D, 4, 4>();
  }
  return nullptr;
}

}  // namespace

#define FAGQ_ATTN_NAME2(e, q, s) lookup_e##e##_q##q##_s##s
#define FAGQ_ATTN_NAME(e, q, s) FAGQ_ATTN_NAME2(e, q, s)

const void* FAGQ_ATTN_NAME(FAGQ_ATTN_E, FAGQ_ATTN_QF, FAGQ_ATTN_SF)(int D, int R, int RP) {
  return D == 64 ? lookup<64>(R, RP) : D == 128 ? lookup<128>(R, RP) : lookup<256>(R, RP);
}

}  // namespace attn
}  // namespace fagq
