// kv_cache.hip - the quantised paged key/value cache: values quantised as they are
// written, and gathered back (include/fagq_cache.h).
//
// Both directions are bound by HBM and hold no state: a lane has 8 consecutive values
// (16 bytes of a 16-bit type, 8 bytes of codes), a group of G values is G / 8 consecutive
// lanes, and its largest magnitude a DPP reduction among them, as in the row quantizer.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "fagq.h"
#include "fagq_cache.h"
#include "fagq_cache_index.hpp"
#include "fagq_diag.h"
#include "fagq_dispatch.hpp"

namespace fagq {
namespace cache {
namespace {

constexpr int kThreads = 256;

template <int E> struct Elem { using type = uint16_t; };
template <> struct Elem<ET_F32> { using type = float; };

template <int E>
__device__ __forceinline__ void load8(const typename Elem<E>::type* p, float (&f)[8]) {
  if constexpr (E == ET_F32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(p + 4 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[4 * h + i] = __uint_as_float(v[i]);
    }
  } else {
    const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = lo16<E>(v[i]);
      f[2 * i + 1] = hi16<E>(v[i]);
    }
  }
}
template <int E>
__device__ __forceinline__ void store8(typename Elem<E>::type* p, const float (&f)[8]) {
  if constexpr (E == ET_F32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(f[4 * h + i]);
      *reinterpret_cast<u32x4*>(p + 4 * h) = v;
    }
  } else {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pack16<E>(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<u32x4*>(p) = v;
  }
}

struct WriteArgs {
  const void* x[2];          // k, v
  void* codes[2];
  void* scales[2];
  const void* slots;
  int64_t num_slots;
  int32_t st[2], sh[2];      // strides in elements
  int32_t chunks;            // T * H * D / 8
  int32_t H, D, groups;      // groups of a head row
  int32_t page_shift;
  int32_t idx64;
};

// One thread: 8 values of one token's head row.  blockIdx.y: k or v.
template <int E, int QF, int SF, int LPG>
__global__ __launch_bounds__(kThreads) void kv_cache_write(WriteArgs a) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  const int o = blockIdx.y;
  const int per_row = a.D / 8, per_token = a.H * per_row;
  const bool in = i < a.chunks;
  const int t = in ? i / per_token : 0;
  const int c = in ? i - t * per_token : 0;
  const int h = c / per_row, d = (c - h * per_row) * 8;
  int64_t slot = a.idx64 ? static_cast<const int64_t*>(a.slots)[t]
                         : (int64_t) static_cast<const int32_t*>(a.slots)[t];
  const bool ok = in && slot >= 0 && slot < a.num_slots;
  float f[8];
  load8<E>(static_cast<const typename Elem<E>::type*>(a.x[o]) +
               ((int64_t)t * a.st[o] + (int64_t)h * a.sh[o] + d), f);
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t b = __float_as_uint(f[j]) & 0x7fffffffu;
    m = m > b ? m : b;
  }
  m = group_max_bits<LPG>(m);
  constexpr float inv_qmax = QF == QF_FP8 ? 1.0f / 448.0f : 1.0f / 127.0f;
  float s = __uint_as_float(m) * inv_qmax;
  s = s > 1e-12f ? s : 1e-12f;
  int e = 0;
  if constexpr (SF == SF_UE8M0) {
    e = ceil_log2_bits(s);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = __builtin_ldexpf(f[j], -e);
  } else {
    const float r = 1.0f / s;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= r;
  }
  if (!ok) return;
  const int64_t page = slot >> a.page_shift;
  const int64_t off = slot & ((1 << a.page_shift) - 1);
  const int64_t row = (((page * a.H + h) << a.page_shift) + off) * a.D + d;
  *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(a.codes[o]) + row) = encode8<QF>(f);
  if ((threadIdx.x & (LPG - 1)) == 0) {
    const int g = d / (LPG * 8);
    const int64_t at = (((page * a.H + h) * a.groups + g) << a.page_shift) + off;
    if constexpr (SF == SF_UE8M0)
      static_cast<uint8_t*>(a.scales[o])[at] = (uint8_t)(e + 127);
    else
      static_cast<float*>(a.scales[o])[at] = s;
  }
}

struct ReadArgs {
  const void* codes[2];
  const void* scales[2];
  void* out[2];
  const int32_t* table;
  const int32_t* cu;
  int64_t num_pages;
  int64_t rows;
  int32_t B, width;
  int32_t H, D, groups, g_shift;
  int32_t page_shift;
  int32_t per_wg;            // rows of a workgroup
};

constexpr int kMaxRowsPerWg = 64;

// Eight codes as fp32.
template <int QF>
__device__ __forceinline__ void decode8(u32x2 v, float (&f)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (QF == QF_FP8) {
      typedef float f32x2 __attribute__((ext_vector_type(2)));
      const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)v[h], false);
      const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)v[h], true);
      f[4 * h + 0] = lo[0], f[4 * h + 1] = lo[1], f[4 * h + 2] = hi[0], f[4 * h + 3] = hi[1];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[4 * h + j] = (float)((int)(v[h] << (24 - 8 * j)) >> 24);
    }
  }
}

// A workgroup takes per_wg consecutive output rows: each row's page is looked up once, by one
// thread, into LDS (a binary search over cu_seqlens and a read of the page table), then all
// threads gather.  blockIdx.y: k or v.
template <int E, int QF, int SF>
__global__ __launch_bounds__(kThreads) void kv_cache_read(ReadArgs a) {
  __shared__ int64_t where[kMaxRowsPerWg];      // each row's slot, kNoPage or kNoRow
  const int64_t row0 = (int64_t)blockIdx.x * a.per_wg;
  if ((int)threadIdx.x < a.per_wg) {
    const int64_t r = row0 + threadIdx.x;
    int64_t at = kNoRow;
    if (r < a.rows)
      at = gathered_slot(a.cu, a.table, a.B, a.width, a.num_pages, a.page_shift, r);
    where[threadIdx.x] = at;
  }
  __syncthreads();
  const int o = blockIdx.y;
  const int per_row = a.D / 8, per_token = a.H * per_row;
  for (int i = threadIdx.x; i < a.per_wg * per_token; i += kThreads) {
    const int t = i / per_token, c = i - t * per_token;
    const int h = c / per_row, d = (c - h * per_row) * 8;
    const int64_t at = where[t];
    if (at == kNoRow) continue;
    float f[8];
    if (at == kNoPage) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.0f;
    } else {
      const int64_t page = at >> a.page_shift, off = at & ((1 << a.page_shift) - 1);
      const int64_t ph = page * a.H + h;
      const u32x2 v = *reinterpret_cast<const u32x2*>(
          static_cast<const uint8_t*>(a.codes[o]) + (((ph << a.page_shift) + off) * a.D + d));
      const int64_t sat = ((ph * a.groups + (d >> a.g_shift)) << a.page_shift) + off;
      float s;
      if constexpr (SF == SF_UE8M0)
        s = __builtin_ldexpf(1.0f, (int)static_cast<const uint8_t*>(a.scales[o])[sat] - 127);
      else
        s = static_cast<const float*>(a.scales[o])[sat];
      decode8<QF>(v, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= s;
    }
    store8<E>(static_cast<typename Elem<E>::type*>(a.out[o]) +
                  ((row0 + t) * per_token + c) * 8, f);
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

int check_layout(int64_t H, int64_t D, int64_t G, int64_t num_pages, int64_t page_size, int dtype,
                 int q_format, int scale_format) {
  if (dtype != FAGQ_DT_BF16 && dtype != FAGQ_DT_F16 && dtype != FAGQ_DT_F32) return FAGQ_E_FORMAT;
  if (q_format != FAGQ_Q_FP8_E4M3FN && q_format != FAGQ_Q_INT8) return FAGQ_E_FORMAT;
  if (scale_format != FAGQ_SCALE_F32 && scale_format != FAGQ_SCALE_UE8M0) return FAGQ_E_FORMAT;
  if (G != 64 && G != 128 && G != 256) return FAGQ_E_GROUP;
  if (H < 1 || D < 1 || D % G != 0 || num_pages < 0 || page_size < FAGQ_CACHE_MIN_PAGE ||
      (page_size & (page_size - 1)) != 0)
    return FAGQ_E_SHAPE;
  if (D > FAGQ_CACHE_MAX_D || H > 4096 || page_size > FAGQ_CACHE_MAX_PAGE ||
      num_pages > (1ll << 31) - 1)
    return FAGQ_E_TOO_LARGE;
  return FAGQ_OK;
}

template <int E, int QF, int SF>
const void* write_kernel(int64_t G) {
  return G == 64    ? reinterpret_cast<const void*>(&kv_cache_write<E, QF, SF, 8>)
         : G == 128 ? reinterpret_cast<const void*>(&kv_cache_write<E, QF, SF, 16>)
                    : reinterpret_cast<const void*>(&kv_cache_write<E, QF, SF, 32>);
}
template <int E>
const void* write_kernel(int64_t G, int qf, int sf) {
  if (qf == FAGQ_Q_FP8_E4M3FN)
    return sf == FAGQ_SCALE_F32 ? write_kernel<E, QF_FP8, SF_F32>(G)
                                : write_kernel<E, QF_FP8, SF_UE8M0>(G);
  return sf == FAGQ_SCALE_F32 ? write_kernel<E, QF_I8_RNE, SF_F32>(G)
                              : write_kernel<E, QF_I8_RNE, SF_UE8M0>(G);
}
template <int E>
const void* read_kernel(int qf, int sf) {
  if (qf == FAGQ_Q_FP8_E4M3FN)
    return sf == FAGQ_SCALE_F32 ? reinterpret_cast<const void*>(&kv_cache_read<E, QF_FP8, SF_F32>)
                                : reinterpret_cast<const void*>(&kv_cache_read<E, QF_FP8, SF_UE8M0>);
  return sf == FAGQ_SCALE_F32 ? reinterpret_cast<const void*>(&kv_cache_read<E, QF_I8_RNE, SF_F32>)
                              : reinterpret_cast<const void*>(&kv_cache_read<E, QF_I8_RNE, SF_UE8M0>);
}

}  // namespace
}  // namespace cache
}  // namespace fagq

extern "C" {

FAGQ_API int fagq_kv_cache_write_launch(const void* k, const void* v, const void* slots,
                                        void* k_cache, void* v_cache, void* k_scale,
                                        void* v_scale, const int64_t* strides, int64_t T,
                                        int64_t H, int64_t D, int64_t G, int64_t num_pages,
                                        int64_t page_size, int dtype, int q_format,
                                        int scale_format, int index_dtype, void* stream) {
  using namespace fagq;
  using namespace fagq::cache;
  if (!k || !slots || !k_cache || !k_scale || !strides) return FAGQ_E_NULL;
  const int n = v ? 2 : 1;
  if ((v == nullptr) != (v_cache == nullptr) || (v == nullptr) != (v_scale == nullptr))
    return FAGQ_E_NULL;
  if (index_dtype != FAGQ_IDX_I32 && index_dtype != FAGQ_IDX_I64) return FAGQ_E_FORMAT;
  const int layout = check_layout(H, D, G, num_pages, page_size, dtype, q_format, scale_format);
  if (layout != FAGQ_OK) return layout;
  if (T < 0) return FAGQ_E_SHAPE;
  if (T > (1ll << 31) - 1 || T * H * D >= (1ll << 34) - 8 * kThreads) return FAGQ_E_TOO_LARGE;
  const int64_t es = dtype == FAGQ_DT_F32 ? 4 : 2;
  const int64_t ss = scale_format == FAGQ_SCALE_F32 ? 4 : 1;
  const int64_t ncodes = num_pages * page_size * H * D, nscales = ncodes / G * ss;
  const void* x[2] = {k, v};
  void* codes[2] = {k_cache, v_cache};
  void* scales[2] = {k_scale, v_scale};
  if (!aligned(slots, index_dtype == FAGQ_IDX_I64 ? 8 : 4)) return FAGQ_E_ALIGN;
  for (int i = 0; i < n; ++i) {
    for (int j = 0; j < 2; ++j) {
      const int64_t s = strides[2 * i + j];
      if (s < 0) return FAGQ_E_SHAPE;
      if (s >= (1ll << 31)) return FAGQ_E_TOO_LARGE;
      if (s % (16 / es) != 0) return FAGQ_E_ALIGN;
    }
    if (!aligned(x[i], 16) || !aligned(codes[i], 16) || !aligned(scales[i], ss))
      return FAGQ_E_ALIGN;
  }
  if (T == 0 || num_pages == 0) return FAGQ_OK;
  for (int i = 0; i < n; ++i) {
    const void* outs[4] = {codes[0], scales[0], codes[1], scales[1]};
    const int64_t nouts[4] = {ncodes, nscales, ncodes, nscales};
    const int64_t nx = ((T - 1) * strides[2 * i] + (H - 1) * strides[2 * i + 1] + D) * es;
    for (int j = 0; j < 2 * n; ++j) {
      if (overlap(x[i], nx, outs[j], nouts[j])) return FAGQ_E_ALIAS;
      if (overlap(slots, T * (index_dtype == FAGQ_IDX_I64 ? 8 : 4), outs[j], nouts[j]))
        return FAGQ_E_ALIAS;
      for (int l = j + 1; l < 2 * n; ++l)
        if (overlap(outs[j], nouts[j], outs[l], nouts[l])) return FAGQ_E_ALIAS;
    }
  }
  const int dcheck = device_check();
  if (dcheck != FAGQ_OK) return dcheck;
  WriteArgs a = {};
  for (int i = 0; i < n; ++i) {
    a.x[i] = x[i], a.codes[i] = codes[i], a.scales[i] = scales[i];
    a.st[i] = (int32_t)strides[2 * i], a.sh[i] = (int32_t)strides[2 * i + 1];
  }
  a.slots = slots, a.num_slots = num_pages * page_size;
  a.chunks = (int32_t)(T * H * D / 8);
  a.H = (int32_t)H, a.D = (int32_t)D, a.groups = (int32_t)(D / G);
  a.page_shift = log2_of(page_size), a.idx64 = index_dtype == FAGQ_IDX_I64;
  const void* fn = dtype == FAGQ_DT_BF16  ? write_kernel<ET_BF16>(G, q_format, scale_format)
                   : dtype == FAGQ_DT_F16 ? write_kernel<ET_F16>(G, q_format, scale_format)
                                          : write_kernel<ET_F32>(G, q_format, scale_format);
  void* args[] = {&a};
  return launch_kernel(fn, dim3((unsigned)((a.chunks + (int64_t)kThreads - 1) / kThreads), (unsigned)n),
                       dim3(kThreads), args, 0, static_cast<hipStream_t>(stream));
}

FAGQ_API int fagq_kv_cache_read_launch(const void* k_cache, const void* v_cache,
                                       const void* k_scale, const void* v_scale,
                                       const int32_t* page_table, const int32_t* cu_seqlens,
                                       void* k_out, void* v_out, int64_t B, int64_t rows,
                                       int64_t H, int64_t D, int64_t G, int64_t num_pages,
                                       int64_t page_size, int64_t table_width, int dtype,
                                       int q_format, int scale_format, void* stream) {
  using namespace fagq;
  using namespace fagq::cache;
  if (!k_cache || !k_scale || !page_table || !cu_seqlens || !k_out) return FAGQ_E_NULL;
  const int n = v_cache ? 2 : 1;
  if ((v_cache == nullptr) != (v_scale == nullptr) || (v_cache == nullptr) != (v_out == nullptr))
    return FAGQ_E_NULL;
  const int layout = check_layout(H, D, G, num_pages, page_size, dtype, q_format, scale_format);
  if (layout != FAGQ_OK) return layout;
  if (B < 0 || rows < 0 || table_width < 0) return FAGQ_E_SHAPE;
  if (B > (1 << 24) || rows > (1ll << 31) - 1 || table_width > (1ll << 31) - 1)
    return FAGQ_E_TOO_LARGE;
  const int64_t es = dtype == FAGQ_DT_F32 ? 4 : 2;
  const int64_t ss = scale_format == FAGQ_SCALE_F32 ? 4 : 1;
  const int64_t ncodes = num_pages * page_size * H * D, nscales = ncodes / G * ss;
  const int64_t nout = rows * H * D * es;
  const void* codes[2] = {k_cache, v_cache};
  const void* scales[2] = {k_scale, v_scale};
  void* outs[2] = {k_out, v_out};
  if (!aligned(page_table, 4) || !aligned(cu_seqlens, 4)) return FAGQ_E_ALIGN;
  for (int i = 0; i < n; ++i)
    if (!aligned(codes[i], 16) || !aligned(scales[i], ss) || !aligned(outs[i], 16))
      return FAGQ_E_ALIGN;
  if (B == 0 || rows == 0) return FAGQ_OK;
  if (n == 2 && overlap(k_out, nout, v_out, nout)) return FAGQ_E_ALIAS;
  for (int i = 0; i < n; ++i) {
    if (overlap(outs[i], nout, page_table, B * table_width * 4) ||
        overlap(outs[i], nout, cu_seqlens, (B + 1) * 4))
      return FAGQ_E_ALIAS;
    for (int j = 0; j < n; ++j)
      if (overlap(outs[i], nout, codes[j], ncodes) || overlap(outs[i], nout, scales[j], nscales))
        return FAGQ_E_ALIAS;
  }
  const int dcheck = device_check();
  if (dcheck != FAGQ_OK) return dcheck;
  ReadArgs a = {};
  for (int i = 0; i < n; ++i) a.codes[i] = codes[i], a.scales[i] = scales[i], a.out[i] = outs[i];
  a.table = page_table, a.cu = cu_seqlens, a.num_pages = num_pages, a.rows = rows;
  a.B = (int32_t)B, a.width = (int32_t)table_width;
  a.H = (int32_t)H, a.D = (int32_t)D, a.groups = (int32_t)(D / G), a.g_shift = log2_of(G);
  a.page_shift = log2_of(page_size);
  // 16 chunks of 8 values for each thread where there are rows enough, one row at least.
  int64_t per = 16 * kThreads / (H * D / 8);
  const int64_t fill = rows / 1024;
  per = per > fill ? fill : per;
  a.per_wg = (int32_t)(per < 1 ? 1 : per > kMaxRowsPerWg ? kMaxRowsPerWg : per);
  const void* fn = dtype == FAGQ_DT_BF16  ? read_kernel<ET_BF16>(q_format, scale_format)
                   : dtype == FAGQ_DT_F16 ? read_kernel<ET_F16>(q_format, scale_format)
                                          : read_kernel<ET_F32>(q_format, scale_format);
  void* args[] = {&a};
  return launch_kernel(fn, dim3((unsigned)((rows + a.per_wg - 1) / a.per_wg), (unsigned)n),
                       dim3(kThreads), args, 0, static_cast<hipStream_t>(stream));
}

FAGQ_API int fagq_diag_cache_slots(const int32_t* page_table, const int32_t* cu_seqlens, int64_t B,
                                   int64_t table_width, int64_t num_pages, int64_t page_size,
                                   int64_t* out, int64_t rows) {
  using namespace fagq::cache;
  if (!page_table || !cu_seqlens || !out) return FAGQ_E_NULL;
  if (B < 0 || B > (1 << 24) || table_width < 0 || num_pages < 0 ||
      page_size < FAGQ_CACHE_MIN_PAGE || page_size > FAGQ_CACHE_MAX_PAGE ||
      (page_size & (page_size - 1)) != 0 || rows < 0)
    return FAGQ_E_SHAPE;
  for (int64_t r = 0; r < rows; ++r)
    out[r] = gathered_slot(cu_seqlens, page_table, (int)B, table_width, num_pages,
                           log2_of(page_size), r);
  return FAGQ_OK;
}

}  // extern "C"
