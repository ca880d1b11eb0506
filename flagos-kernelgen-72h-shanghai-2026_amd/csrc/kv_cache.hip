// kv_cache.hip - the quantised paged key/value cache: values quantised as they are
// written, and gathered back (include/fagq_cache.h).
//
// Both directions are bound by HBM and hold no state (8 x 16384 tokens, 8 heads of 128, fp8 read
// back to bf16: 137 us, 5.9 TB/s; 16384 latents of 512 written: 7.2 us, of which the 25 MB are
// 3.8 and the rest is the start and drain of one round of workgroups): a lane has 8 consecutive values
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
// Chunks of a thread that are under way at once: with one, the threads that fit the GPU have too
// few bytes in flight to reach HBM's rate.
constexpr int kInFlight = 4;

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
// Streamed past the caches: what is gathered is not read again by this call, and the codes'
// lines stay (143.6 against 155.3 us for 8 x 16384 tokens, 8 heads of 128).
template <int E>
__device__ __forceinline__ void store8(typename Elem<E>::type* p, const float (&f)[8]) {
  if constexpr (E == ET_F32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(f[4 * h + i]);
      __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p + 4 * h));
    }
  } else {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pack16<E>(f[2 * i], f[2 * i + 1]);
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p));
  }
}

// How a workgroup's threads stand over tokens and their H D / 8 chunks of 8 values: a thread keeps
// its chunk (blockIdx.z: which 256 of them) and steps over tokens, so that no index is divided in
// the loops.  `side` tokens stand side by side where a token has fewer chunks than threads.
struct Stand {
  int token, side, chunk, h, d;
  bool on;
};
__device__ __forceinline__ Stand stand(int H, int D) {
  const int per_row = D / 8, chunks = H * per_row;
  Stand s;
  s.side = chunks < kThreads ? kThreads / chunks : 1;
  s.token = chunks < kThreads ? (int)threadIdx.x / chunks : 0;
  s.chunk = (int)threadIdx.x - s.token * chunks + (int)blockIdx.z * kThreads;
  s.on = s.token < s.side && s.chunk < chunks;
  s.h = s.chunk / per_row;
  s.d = (s.chunk - s.h * per_row) * 8;
  return s;
}

struct WriteArgs {
  const void* x[2];          // k, v
  void* codes[2];
  void* scales[2];
  const void* slots;
  int64_t num_slots;
  int32_t st[2], sh[2];      // strides in elements
  int32_t T, H, D, groups;   // groups of a head row
  int32_t page_shift;
  int32_t idx64;
};

// blockIdx.y: k or v.  A thread has U tokens' chunks under way at once.
template <int E, int QF, int SF, int LPG, int U>
__global__ __launch_bounds__(kThreads) void kv_cache_write(WriteArgs a) {
  const Stand w = stand(a.H, a.D);
  const int o = blockIdx.y;
  const int t0 = (int)blockIdx.x * w.side * U + w.token;
  const auto* x = static_cast<const typename Elem<E>::type*>(a.x[o]) + (int64_t)w.h * a.sh[o] + w.d;
  float f[U][8];
  int64_t slot[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int t = t0 + u * w.side;
    slot[u] = -1;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[u][j] = 0.0f;
    if (!w.on || t >= a.T) continue;
    slot[u] = a.idx64 ? static_cast<const int64_t*>(a.slots)[t]
                      : (int64_t) static_cast<const int32_t*>(a.slots)[t];
    load8<E>(x + (int64_t)t * a.st[o], f[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = __float_as_uint(f[u][j]) & 0x7fffffffu;
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
      for (int j = 0; j < 8; ++j) f[u][j] = __builtin_ldexpf(f[u][j], -e);
    } else {
      const float r = 1.0f / s;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[u][j] *= r;
    }
    if (slot[u] < 0 || slot[u] >= a.num_slots) continue;
    const int64_t ph = (slot[u] >> a.page_shift) * a.H + w.h;
    const int64_t off = slot[u] & ((1 << a.page_shift) - 1);
    *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(a.codes[o]) +
                              ((ph << a.page_shift) + off) * a.D + w.d) = encode8<QF>(f[u]);
    if ((threadIdx.x & (LPG - 1)) == 0) {
      const int64_t at = ((ph * a.groups + w.d / (LPG * 8)) << a.page_shift) + off;
      if constexpr (SF == SF_UE8M0)
        static_cast<uint8_t*>(a.scales[o])[at] = (uint8_t)(e + 127);
      else
        static_cast<float*>(a.scales[o])[at] = s;
    }
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

template <int SF> struct ScaleWord { using type = float; };
template <> struct ScaleWord<SF_UE8M0> { using type = uint8_t; };

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
// threads gather, kInFlight rows at once.  blockIdx.y: k or v.
template <int E, int QF, int SF>
__global__ __launch_bounds__(kThreads) void kv_cache_read(ReadArgs a) {
  __shared__ int64_t code_at[kMaxRowsPerWg];    // of head 0, dim 0; kNoPage, kNoRow
  __shared__ int64_t scale_at[kMaxRowsPerWg];
  const int64_t row0 = (int64_t)blockIdx.x * a.per_wg;
  if ((int)threadIdx.x < a.per_wg) {
    const int64_t r = row0 + threadIdx.x;
    int64_t at = kNoRow;
    if (r < a.rows)
      at = cache::gathered_slot(a.cu, a.table, a.B, a.width, a.num_pages, a.page_shift, r);
    if (at >= 0) {
      const int64_t ph = (at >> a.page_shift) * a.H, off = at & ((1 << a.page_shift) - 1);
      at = ((ph << a.page_shift) + off) * a.D;
      scale_at[threadIdx.x] = ((ph * a.groups) << a.page_shift) + off;
    }
    code_at[threadIdx.x] = at;
  }
  __syncthreads();
  const Stand w = stand(a.H, a.D);
  if (!w.on) return;
  const int o = blockIdx.y;
  using Word = typename ScaleWord<SF>::type;
  const uint8_t* codes =
      static_cast<const uint8_t*>(a.codes[o]) + (((int64_t)w.h << a.page_shift) * a.D + w.d);
  const Word* scales = static_cast<const Word*>(a.scales[o]) +
                       ((int64_t)(w.h * a.groups + (w.d >> a.g_shift)) << a.page_shift);
  auto* out = static_cast<typename Elem<E>::type*>(a.out[o]) + (row0 * a.H * a.D + w.chunk * 8);
  for (int t0 = w.token; t0 < a.per_wg; t0 += kInFlight * w.side) {
    u32x2 code[kInFlight];
    Word scale[kInFlight];
    int64_t at[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int t = t0 + u * w.side;
      at[u] = t < a.per_wg ? code_at[t] : kNoRow;
      code[u] = u32x2{0, 0};
      scale[u] = 0;
      if (at[u] < 0) continue;
      code[u] = *reinterpret_cast<const u32x2*>(codes + at[u]);
      scale[u] = scales[scale_at[t]];
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (at[u] == kNoRow) continue;
      float f[8], s;
      if constexpr (SF == SF_UE8M0) s = __builtin_ldexpf(1.0f, (int)scale[u] - 127);
      else s = scale[u];
      decode8<QF>(code[u], f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = at[u] == kNoPage ? 0.0f : f[j] * s;
      store8<E>(out + (int64_t)(t0 + u * w.side) * a.H * a.D, f);
    }
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

template <int E, int QF, int SF, int U>
const void* write_kernel(int64_t G) {
  return G == 64    ? reinterpret_cast<const void*>(&kv_cache_write<E, QF, SF, 8, U>)
         : G == 128 ? reinterpret_cast<const void*>(&kv_cache_write<E, QF, SF, 16, U>)
                    : reinterpret_cast<const void*>(&kv_cache_write<E, QF, SF, 32, U>);
}
template <int E, int U>
const void* write_kernel(int64_t G, int qf, int sf) {
  if (qf == FAGQ_Q_FP8_E4M3FN)
    return sf == FAGQ_SCALE_F32 ? write_kernel<E, QF_FP8, SF_F32, U>(G)
                                : write_kernel<E, QF_FP8, SF_UE8M0, U>(G);
  return sf == FAGQ_SCALE_F32 ? write_kernel<E, QF_I8_RNE, SF_F32, U>(G)
                              : write_kernel<E, QF_I8_RNE, SF_UE8M0, U>(G);
}
template <int E>
const void* write_kernel(int64_t G, int qf, int sf, int in_flight) {
  return in_flight == 1 ? write_kernel<E, 1>(G, qf, sf) : write_kernel<E, kInFlight>(G, qf, sf);
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
  if (T > (1ll << 24)) return FAGQ_E_TOO_LARGE;
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
  a.T = (int32_t)T, a.H = (int32_t)H, a.D = (int32_t)D, a.groups = (int32_t)(D / G);
  a.page_shift = log2_of(page_size), a.idx64 = index_dtype == FAGQ_IDX_I64;
  const int64_t chunks = H * D / 8, side = chunks < kThreads ? kThreads / chunks : 1;
  const int64_t wide = (chunks + kThreads - 1) / kThreads;
  // One chunk for each thread while that leaves less than four workgroups for a CU.
  const int u = (T + side - 1) / side * wide * n < 4 * 256 ? 1 : kInFlight;
  const void* fn = dtype == FAGQ_DT_BF16  ? write_kernel<ET_BF16>(G, q_format, scale_format, u)
                   : dtype == FAGQ_DT_F16 ? write_kernel<ET_F16>(G, q_format, scale_format, u)
                                          : write_kernel<ET_F32>(G, q_format, scale_format, u);
  void* args[] = {&a};
  const int64_t per_wg = side * u;
  return launch_kernel(fn, dim3((unsigned)((T + per_wg - 1) / per_wg), (unsigned)n, (unsigned)wide),
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
  // A cache of no pages and a table of no width have nothing to point to, and are never read.
  if ((num_pages > 0 && (!k_cache || !k_scale)) || (table_width > 0 && !page_table) || !cu_seqlens ||
      !k_out)
    return FAGQ_E_NULL;
  const int n = v_out ? 2 : 1;
  if (num_pages > 0 &&
      ((v_cache == nullptr) != (v_out == nullptr) || (v_scale == nullptr) != (v_out == nullptr)))
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
  const int64_t chunks = H * D / 8, side = chunks < kThreads ? kThreads / chunks : 1;
  const int64_t wide = (chunks + kThreads - 1) / kThreads;
  // kInFlight rows for each thread where that leaves 4 workgroups for each CU, one row at least.
  // More rows spread the loads under way over more of HBM's pages (8 x 16384 tokens: 137.6 us,
  // with twice as many rows 143.6, with four times 163).
  int64_t per = kInFlight * side;
  const int64_t fill = rows * n * wide / (4 * 256);
  per = per > fill ? fill : per;
  a.per_wg = (int32_t)(per < 1 ? 1 : per > kMaxRowsPerWg ? kMaxRowsPerWg : per);
  const void* fn = dtype == FAGQ_DT_BF16  ? read_kernel<ET_BF16>(q_format, scale_format)
                   : dtype == FAGQ_DT_F16 ? read_kernel<ET_F16>(q_format, scale_format)
                                          : read_kernel<ET_F32>(q_format, scale_format);
  void* args[] = {&a};
  const int64_t groups = (rows + a.per_wg - 1) / a.per_wg;
  if (groups >= (1ll << 32) / kThreads) return FAGQ_E_TOO_LARGE;
  return launch_kernel(fn, dim3((unsigned)groups, (unsigned)n, (unsigned)wide),
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
