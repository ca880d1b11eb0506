// paged_attn_inst.hip - instantiations of the paged attention for one element type, code
// format and scale format (FAGQ_ATTN_E, FAGQ_ATTN_QF, FAGQ_ATTN_SF).
#include "paged_attn_kernels.hpp"

namespace fagq {
namespace attn {
namespace {

template <int D, int R, int RP, int FORM, bool TREE = false>
const void* kernel() {
  return reinterpret_cast<const void*>(
      &paged_attention<FAGQ_ATTN_E, FAGQ_ATTN_QF, FAGQ_ATTN_SF, D, R, RP, FORM, TREE>);
}

// What plan_for makes, R D <= 256 or, for heads of 128 and 256, tall units: without a prefix, units
// of any height; with one, 16 rows go with a prefix of units of any height, more rows with units of
// their own height or tall ones, tall ones with tall ones.  Units of 16 rows may be scheduled,
// but not those of trees.
template <int D, int R, int RP>
const void* lookup(int form, bool tree) {
  if (tree) return kernel<D, R, RP, kStatic, true>();
  if constexpr (R == 1) {
    if constexpr (RP == 0)
      if (form == kScheduledOnce) return kernel<D, R, RP, kScheduledOnce>();
    if (form != kStatic) return kernel<D, R, RP, kScheduled>();
  }
  return kernel<D, R, RP, kStatic>();
}
template <int D, int R>
const void* lookup(int RP, int form, bool tree) {
  if constexpr (R == kTall ? D >= 128 : R * D <= 256) {
    if (RP == 0) return lookup<D, R, 0>(form, tree);
    if constexpr (D >= 128)
      if (RP == kTall) return lookup<D, R, kTall>(form, tree);
    if constexpr (R != kTall)
      if (RP == R) return lookup<D, R, R>(form, tree);
    if constexpr (R == 1 && 2 * D <= 256)
      if (RP == 2) return lookup<D, R, 2>(form, tree);
    if constexpr (R == 1 && 4 * D <= 256)
      if (RP == 4) return lookup<D, R, 4>(form, tree);
  }
  return nullptr;
}
template <int D>
const void* lookup(int R, int RP, int form, bool tree) {
  return R == 1   ? lookup<D, 1>(RP, form, tree)
         : R == 2 ? lookup<D, 2>(RP, form, tree)
         : R == 4 ? lookup<D, 4>(RP, form, tree)
                  : lookup<D, kTall>(RP, form, tree);
}

}  // namespace

#define FAGQ_ATTN_NAME2(e, q, s) lookup_e##e##_q##q##_s##s
#define FAGQ_ATTN_NAME(e, q, s) FAGQ_ATTN_NAME2(e, q, s)

const void* FAGQ_ATTN_NAME(FAGQ_ATTN_E, FAGQ_ATTN_QF, FAGQ_ATTN_SF)(int D, int R, int RP, int form,
                                                                    bool tree) {
  return D == 64    ? lookup<64>(R, RP, form, tree)
         : D == 128 ? lookup<128>(R, RP, form, tree)
                    : lookup<256>(R, RP, form, tree);
}

}  // namespace attn
}  // namespace fagq
