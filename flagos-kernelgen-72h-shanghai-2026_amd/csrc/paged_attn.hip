// paged_attn.hip - attention of the newest tokens of each sequence over the quantised paged
// cache (include/fagq_cache.h).
//
// One pass with a running maximum m and sum l of the softmax: for key j with
// x = q . (code_k s_k) sm_scale,  m' = max(m, x),  l = l e^(m - m') + e^(x - m'),
// o = o e^(m - m') + e^(x - m') code_v s_v.  Parts of a row's keys have m, l and o of their
// own and are joined by the same rule.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "fagq.h"
#include "fagq_cache.h"
#include "fagq_cache_index.hpp"
#include "fagq_dispatch.hpp"

namespace fagq {
namespace attn {
namespace {

constexpr int kWaves = 4;

struct Args {
  const uint16_t* q;
  const uint8_t* kc;
  const uint8_t* vc;
  const void* ks;
  const void* vs;
  const int32_t* table;
  const void* lens;
  const int32_t* prefix;
  uint16_t* out;
  int64_t num_pages;
  int32_t qs[3];             // {sequence, token, head} strides, elements
  int32_t S, Hq, H, group;
  int32_t page_shift;
  int32_t width;
  int32_t prefix_len;
  int32_t most;              // tokens of a sequence that are read at most
  int32_t idx64, sf, qf;
  float scale2;              // sm_scale * log2(e)
};

__device__ __forceinline__ float code_value(int qf, uint8_t c) {
  return qf == QF_FP8 ? __builtin_amdgcn_cvt_f32_fp8((int)c, 0) : (float)(int8_t)c;
}
__device__ __forceinline__ float scale_value(int sf, const void* p, int64_t at) {
  return sf == SF_F32 ? static_cast<const float*>(p)[at]
                      : __builtin_ldexpf(1.0f, (int)static_cast<const uint8_t*>(p)[at] - 127);
}

// One workgroup for each query row; its waves take every fourth key, a lane D / 64 dims.
template <int E, int D>
__global__ __launch_bounds__(64 * kWaves) void paged_attention_rows(Args a) {
  constexpr int N = D / 64;
  __shared__ float part[kWaves][D + 2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = blockIdx.x;                   // (b, s, hq)
  const int hq = row % a.Hq, s = row / a.Hq % a.S, b = row / a.Hq / a.S;
  const int h = hq / a.group;
  const int64_t len = a.idx64 ? static_cast<const int64_t*>(a.lens)[b]
                              : (int64_t) static_cast<const int32_t*>(a.lens)[b];
  const int64_t keys = a.prefix_len + cache::seen_tokens(len, a.most, a.S, s);
  float q[N], o[N] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i)
    q[i] = lo16<E>(a.q[(int64_t)b * a.qs[0] + (int64_t)s * a.qs[1] + (int64_t)hq * a.qs[2] +
                       lane * N + i]) * a.scale2;
  for (int64_t j = wave; j < keys; j += kWaves) {
    const bool front = j < a.prefix_len;
    const int64_t t = front ? j : j - a.prefix_len;
    const int64_t slot =
        front ? cache::slot_of(a.prefix, ((int64_t)a.prefix_len - 1 >> a.page_shift) + 1,
                               a.num_pages, a.page_shift, t)
              : cache::slot_of(a.table + (int64_t)b * a.width, a.width, a.num_pages, a.page_shift, t);
    if (slot < 0) continue;
    const int64_t at = (((slot >> a.page_shift) * a.H + h) << a.page_shift) +
                       (slot & ((1 << a.page_shift) - 1));
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) x += q[i] * code_value(a.qf, a.kc[at * D + lane * N + i]);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d);
    x *= scale_value(a.sf, a.ks, at);
    const float top = x > m ? x : m;
    const float keep = __builtin_amdgcn_exp2f(m - top), w = __builtin_amdgcn_exp2f(x - top);
    const float wv = w * scale_value(a.sf, a.vs, at);
    l = l * keep + w;
    m = top;
#pragma unroll
    for (int i = 0; i < N; ++i)
      o[i] = o[i] * keep + wv * code_value(a.qf, a.vc[at * D + lane * N + i]);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) part[wave][lane * N + i] = o[i];
  if (lane == 0) {
    part[wave][D] = m;
    part[wave][D + 1] = l;
  }
  __syncthreads();
  float top = -INFINITY, total = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = part[w][D] > top ? part[w][D] : top;
  float f[kWaves];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    f[w] = part[w][D] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(part[w][D] - top);
    total += f[w] * part[w][D + 1];
  }
  const float inv = total > 0.0f ? 1.0f / total : 0.0f;
  for (int d = threadIdx.x; d < D; d += 64 * kWaves) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += f[w] * part[w][d];
    a.out[(int64_t)row * D + d] = (uint16_t)pack16<E>(v * inv, 0.0f);
  }
}

// ---------------------------------------------------------------------------------- host

bool aligned(const void* p, uintptr_t a) {
  return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na > 0 && nb > 0 && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

int log2_of(int64_t v) {
  int s = 0;
  while ((1ll << s) < v) ++s;
  return s;
}

int check_sizes(int64_t B, int64_t S, int64_t Hq, int64_t H, int64_t D, int64_t prefix_len,
                int64_t max_kv_len) {
  if (B < 0 || S < 1 || H < 1 || Hq < H || Hq % H != 0 || (D != 64 && D != 128 && D != 256) ||
      prefix_len < 0 || max_kv_len < 0)
    return FAGQ_E_SHAPE;
  if (B > 65535 || S > 65535 || Hq > 4096 || B * S * Hq > (1ll << 24) ||
      prefix_len > (1ll << 30) || max_kv_len > (1ll << 30))
    return FAGQ_E_TOO_LARGE;
  return FAGQ_OK;
}

template <int E>
const void* kernel_for(int64_t D) {
  return D == 64    ? reinterpret_cast<const void*>(&paged_attention_rows<E, 64>)
         : D == 128 ? reinterpret_cast<const void*>(&paged_attention_rows<E, 128>)
                    : reinterpret_cast<const void*>(&paged_attention_rows<E, 256>);
}

}  // namespace
}  // namespace attn
}  // namespace fagq

extern "C" {

FAGQ_API int64_t fagq_paged_attention_workspace_bytes(int64_t B, int64_t S, int64_t Hq, int64_t H,
                                                      int64_t D, int64_t prefix_len,
                                                      int64_t max_kv_len) {
  using namespace fagq::attn;
  if (check_sizes(B, S, Hq, H, D, prefix_len, max_kv_len) != FAGQ_OK) return -1;
  return 0;
}

FAGQ_API int fagq_paged_attention_launch(const void* q, const void* k_cache, const void* v_cache,
                                         const void* k_scale, const void* v_scale,
                                         const int32_t* page_table, const void* kv_lens,
                                         const int32_t* prefix_pages, void* out, void* workspace,
                                         int64_t workspace_bytes, const int64_t* strides,
                                         int64_t B, int64_t S, int64_t Hq, int64_t H, int64_t D,
                                         int64_t num_pages, int64_t page_size, int64_t table_width,
                                         int64_t prefix_len, int64_t max_kv_len, float sm_scale,
                                         int dtype, int q_format, int scale_format,
                                         int index_dtype, void* stream) {
  using namespace fagq;
  using namespace fagq::attn;
  if (!q || !k_cache || !v_cache || !k_scale || !v_scale || !kv_lens || !out || !strides ||
      (table_width > 0 && !page_table) || (prefix_len > 0 && !prefix_pages))
    return FAGQ_E_NULL;
  if (dtype != FAGQ_DT_BF16 && dtype != FAGQ_DT_F16) return FAGQ_E_FORMAT;
  if (q_format != FAGQ_Q_FP8_E4M3FN && q_format != FAGQ_Q_INT8) return FAGQ_E_FORMAT;
  if (scale_format != FAGQ_SCALE_F32 && scale_format != FAGQ_SCALE_UE8M0) return FAGQ_E_FORMAT;
  if (index_dtype != FAGQ_IDX_I32 && index_dtype != FAGQ_IDX_I64) return FAGQ_E_FORMAT;
  if (!std::isfinite(sm_scale)) return FAGQ_E_SHAPE;
  const int sizes = check_sizes(B, S, Hq, H, D, prefix_len, max_kv_len);
  if (sizes != FAGQ_OK) return sizes;
  if (num_pages < 0 || table_width < 0 || page_size < FAGQ_CACHE_MIN_PAGE ||
      (page_size & (page_size - 1)) != 0)
    return FAGQ_E_SHAPE;
  if (page_size > FAGQ_CACHE_MAX_PAGE || num_pages > (1ll << 31) - 1 ||
      table_width > (1ll << 31) - 1)
    return FAGQ_E_TOO_LARGE;
  for (int i = 0; i < 3; ++i) {
    if (strides[i] < 0) return FAGQ_E_SHAPE;
    if (strides[i] >= (1ll << 31)) return FAGQ_E_TOO_LARGE;
    if (strides[i] % 8 != 0) return FAGQ_E_ALIGN;
  }
  const int64_t ss = scale_format == FAGQ_SCALE_F32 ? 4 : 1;
  const int64_t is = index_dtype == FAGQ_IDX_I64 ? 8 : 4;
  if (!aligned(q, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) ||
      !aligned(k_scale, 4) || !aligned(v_scale, 4) || !aligned(page_table, 4) ||
      !aligned(kv_lens, is) || !aligned(prefix_pages, 4) || !aligned(out, 16))
    return FAGQ_E_ALIGN;
  const int64_t need = fagq_paged_attention_workspace_bytes(B, S, Hq, H, D, prefix_len, max_kv_len);
  if (need > 0 && !workspace) return FAGQ_E_NULL;
  if (workspace_bytes < need) return FAGQ_E_SHAPE;
  if (!aligned(workspace, 16)) return FAGQ_E_ALIGN;
  if (B == 0) return FAGQ_OK;
  const int64_t ncodes = num_pages * page_size * H * D, nscales = num_pages * page_size * H * ss;
  const void* ins[8] = {q, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, prefix_pages};
  const int64_t nin[8] = {((B - 1) * strides[0] + (S - 1) * strides[1] + (Hq - 1) * strides[2] + D) * 2,
                          ncodes, ncodes, nscales, nscales, B * table_width * 4, B * is,
                          (prefix_len + page_size - 1) / page_size * 4};
  const int64_t nout = B * S * Hq * D * 2;
  for (int i = 0; i < 8; ++i)
    if (overlap(out, nout, ins[i], nin[i]) || overlap(workspace, need, ins[i], nin[i]))
      return FAGQ_E_ALIAS;
  if (overlap(out, nout, workspace, need)) return FAGQ_E_ALIAS;
  const int dcheck = device_check();
  if (dcheck != FAGQ_OK) return dcheck;
  Args a = {};
  a.q = static_cast<const uint16_t*>(q);
  a.kc = static_cast<const uint8_t*>(k_cache), a.vc = static_cast<const uint8_t*>(v_cache);
  a.ks = k_scale, a.vs = v_scale, a.table = page_table, a.lens = kv_lens, a.prefix = prefix_pages;
  a.out = static_cast<uint16_t*>(out);
  a.num_pages = num_pages;
  for (int i = 0; i < 3; ++i) a.qs[i] = (int32_t)strides[i];
  a.S = (int32_t)S, a.Hq = (int32_t)Hq, a.H = (int32_t)H, a.group = (int32_t)(Hq / H);
  a.page_shift = log2_of(page_size), a.width = (int32_t)table_width;
  a.prefix_len = (int32_t)prefix_len;
  const int64_t room = table_width > (max_kv_len >> a.page_shift) ? max_kv_len
                                                                  : table_width << a.page_shift;
  a.most = (int32_t)(room < max_kv_len ? room : max_kv_len);
  a.idx64 = index_dtype == FAGQ_IDX_I64;
  a.sf = scale_format == FAGQ_SCALE_F32 ? SF_F32 : SF_UE8M0;
  a.qf = q_format == FAGQ_Q_FP8_E4M3FN ? QF_FP8 : QF_I8_RNE;
  a.scale2 = sm_scale * 1.44269504088896340736f;
  void* args[] = {&a};
  return launch_kernel(dtype == FAGQ_DT_BF16 ? kernel_for<ET_BF16>(D) : kernel_for<ET_F16>(D),
                       dim3((unsigned)(B * S * Hq)), dim3(64 * kWaves), args, 0,
                       static_cast<hipStream_t>(stream));
}

}  // extern "C"
