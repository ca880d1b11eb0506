// qk_rope.hip - RMS norm of each query and key head with the rotation by position in
// the same pass, and the gradients (include/fagq_rope.h).
//
// y = R(p) (x rstd w), rstd = 1 / sqrt(mean(x^2) + eps).  R(p) is orthogonal, so the
// gradient of the normed row is dy rotated back, and with a = dn w
//   dx = rstd (a - x rstd^2 mean(a x)),   dw = sum over rows of dn x rstd.
// rstd is recomputed from x, which the backward reads anyway.
//
// Both directions are bound by HBM: 2 (3) tensors at one read or write each (16384 tokens, 64 + 8
// heads of 128, bf16: 98.5 us, 6.2 TB/s; backward, 8192 tokens, 32 + 8: 43.6 us, 5.9 TB/s, and 4.8
// for the sums of the weights' gradients).  A row of D
// elements belongs to LPR = D / 16 lanes (a power of two, 4 to 32), 16 elements each in two
// chunks of 8: for pairs (i, i + R / 2) lane l holds elements 8 l.. and R / 2 + 8 l.., for
// adjacent pairs 16 l.. and 16 l + 8.., so that both halves of every pair are in one lane
// and every access is 16 bytes.  A wave takes 64 / LPR heads of one token at a time (a "pass").
#include <hip/hip_runtime.h>

#include <cstdint>

#include "fagq.h"
#include "fagq_dispatch.hpp"
#include "fagq_rope.h"

namespace fagq {
namespace rope {
namespace {

constexpr int kWaves = 4;             // waves per workgroup
// Workgroups of the backward, two for each CU, each with its own sum of a weight's gradient (8192
// tokens, 32 + 8 heads of 128, us from HBM / from the caches: 53.7 / 47.5, three for each CU 54.4 /
// 48.1).
constexpr int kMaxBwdGroups = 512;
constexpr int kSumRows = 64;          // partial sums that a column's threads share out

struct Args {
  const void* q;
  const void* k;
  const void* qw;
  const void* kw;
  const float* cos;
  const float* sin;
  const void* pos;
  void* qo;          // forward: q_out; backward: dq
  void* ko;
  const void* dq;    // backward: dq_out, dk_out
  const void* dk;
  float* sums;       // backward: [workgroups][D]
  int64_t table_rows;
  int32_t qs[2], ks[2], qos[2], kos[2], dqs[2], dks[2];   // {token, head} strides, elements
  int32_t T, Hq, Hk, D, R;
  int32_t gq;        // backward: workgroups of q
  int32_t idx64;
  float eps;
};

template <int E> struct Elem { using type = uint16_t; };
template <> struct Elem<ET_F32> { using type = float; };

// Eight consecutive elements as fp32, and back (one rounding to nearest even).
template <int E>
struct Raw8 {
  u32x4 v[E == ET_F32 ? 2 : 1];
};
template <int E>
__device__ __forceinline__ Raw8<E> load8(const typename Elem<E>::type* p) {
  Raw8<E> r;
  r.v[0] = *reinterpret_cast<const u32x4*>(p);
  if constexpr (E == ET_F32) r.v[1] = *reinterpret_cast<const u32x4*>(p + 4);
  return r;
}
template <int E>
__device__ __forceinline__ Raw8<E> zero8() {
  Raw8<E> r;
  r.v[0] = u32x4{0, 0, 0, 0};
  if constexpr (E == ET_F32) r.v[1] = u32x4{0, 0, 0, 0};
  return r;
}
template <int E>
__device__ __forceinline__ void unpack8(const Raw8<E>& r, float* f) {
  if constexpr (E == ET_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(r.v[i / 4][i % 4]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = lo16<E>(r.v[0][i]);
      f[2 * i + 1] = hi16<E>(r.v[0][i]);
    }
  }
}
// NT: streamed past the caches.
template <bool NT>
__device__ __forceinline__ void store_b128(void* p, u32x4 v) {
  if constexpr (NT) __builtin_nontemporal_store(v, static_cast<u32x4*>(p));
  else *static_cast<u32x4*>(p) = v;
}
template <int E, bool NT>
__device__ __forceinline__ void store8(typename Elem<E>::type* p, const float* f) {
  if constexpr (E == ET_F32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(f[4 * h + i]);
      store_b128<NT>(p + 4 * h, v);
    }
  } else {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pack16<E>(f[2 * i], f[2 * i + 1]);
    store_b128<NT>(p, v);
  }
}

// Sum over the LPR lanes of a row; every lane receives the same value.
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
  v += __uint_as_float(dpp_u32<0xB1>(__float_as_uint(v)));    // quad_perm [1,0,3,2]
  v += __uint_as_float(dpp_u32<0x4E>(__float_as_uint(v)));    // quad_perm [2,3,0,1]
  if constexpr (LPR >= 8) v += __uint_as_float(dpp_u32<0x141>(__float_as_uint(v)));
  if constexpr (LPR >= 16) v += __uint_as_float(dpp_u32<0x140>(__float_as_uint(v)));
  if constexpr (LPR >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// What a lane knows of every row: where its two chunks are, and its pairs' angles.
struct Lane {
  int sub;        // lane within the row
  int row;        // row within a pass
  int c0, c1;     // first elements of its chunks
  bool on;        // the lane holds elements
};

template <int LPR, bool INTER>
__device__ __forceinline__ Lane lane_of(int lane, int D, int R) {
  Lane l;
  l.sub = lane & (LPR - 1);
  l.row = lane / LPR;
  l.on = 16 * l.sub < D;
  const bool pairs_apart = !INTER && 16 * l.sub < R;
  l.c0 = pairs_apart ? 8 * l.sub : 16 * l.sub;
  l.c1 = pairs_apart ? R / 2 + 8 * l.sub : 16 * l.sub + 8;
  return l;
}

// cos and sin of the lane's eight pairs (1 and 0 where its elements are not rotated).
struct Turn {
  float c[8], s[8];
};
__device__ __forceinline__ Turn load_turn(const Args& a, const Lane& l, int64_t pos, bool real) {
  Turn t;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    t.c[i] = 1.0f;
    t.s[i] = 0.0f;
  }
  if (real && 16 * l.sub < a.R) {      // padding may have no table row to read
    const int64_t at = pos * (a.R / 2) + 8 * l.sub;
    unpack8<ET_F32>(load8<ET_F32>(a.cos + at), t.c);
    unpack8<ET_F32>(load8<ET_F32>(a.sin + at), t.s);
  }
  return t;
}

// Rotates the lane's 16 elements (chunk 0, chunk 1) in place; BACK: the other way.
template <bool INTER, bool BACK>
__device__ __forceinline__ void rotate(float (&n)[16], const Turn& t) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int ia = INTER ? 2 * i : i, ib = INTER ? 2 * i + 1 : i + 8;
    const float x = n[ia], y = n[ib], s = BACK ? -t.s[i] : t.s[i];
    n[ia] = __builtin_fmaf(x, t.c[i], -(y * s));
    n[ib] = __builtin_fmaf(y, t.c[i], x * s);
  }
}

// 1 / sqrt(v) to an ulp; v_rsq_f32 takes no subnormals.
__device__ __forceinline__ float rsqrt_of(float v) {
  const bool tiny = v < 0x1p-100f;
  const float r = __builtin_amdgcn_rsqf(tiny ? v * 0x1p100f : v);
  return tiny ? r * 0x1p50f : r;
}

// A scalar load: positions are constant during the kernel, which the compiler cannot know of one
// that stores.
__device__ __forceinline__ int64_t position(const Args& a, int t) {
  using C64 = const __attribute__((address_space(4))) int64_t;
  using C32 = const __attribute__((address_space(4))) int32_t;
  const uintptr_t p = reinterpret_cast<uintptr_t>(a.pos);
  return a.idx64 ? reinterpret_cast<C64*>(p)[t] : (int64_t) reinterpret_cast<C32*>(p)[t];
}

// The heads of q or of k, for one wave: where they start and how far apart.
template <int E>
struct Heads {
  using T = typename Elem<E>::type;
  const T* x;
  const T* dy;               // backward
  T* y;                      // forward: result; backward: dx
  int32_t xh, dyh, yh;       // head strides
  int32_t H;
};
template <int E, bool BWD>
__device__ __forceinline__ Heads<E> heads_of(const Args& a, bool isq, int t) {
  using T = typename Elem<E>::type;
  Heads<E> h;
  h.x = static_cast<const T*>(isq ? a.q : a.k) + (int64_t)t * (isq ? a.qs[0] : a.ks[0]);
  h.y = static_cast<T*>(isq ? a.qo : a.ko) + (int64_t)t * (isq ? a.qos[0] : a.kos[0]);
  h.xh = isq ? a.qs[1] : a.ks[1];
  h.yh = isq ? a.qos[1] : a.kos[1];
  h.dy = nullptr;
  h.dyh = 0;
  if constexpr (BWD) {
    h.dy = static_cast<const T*>(isq ? a.dq : a.dk) + (int64_t)t * (isq ? a.dqs[0] : a.dks[0]);
    h.dyh = isq ? a.dqs[1] : a.dks[1];
  }
  h.H = isq ? a.Hq : a.Hk;
  return h;
}

// The lane's 16 elements of a row (a weight: the row at p itself).
template <int E>
struct Raw16 {
  Raw8<E> a, b;
};
template <int E>
__device__ __forceinline__ Raw16<E> load16(const typename Elem<E>::type* p, const Lane& l, bool on) {
  Raw16<E> r = {zero8<E>(), zero8<E>()};
  if (on) {
    r.a = load8<E>(p + l.c0);
    r.b = load8<E>(p + l.c1);
  }
  return r;
}
template <int E>
__device__ __forceinline__ void unpack16(const Raw16<E>& r, float (&f)[16]) {
  unpack8<E>(r.a, f);
  unpack8<E>(r.b, f + 8);
}
template <int E, bool NT>
__device__ __forceinline__ void store16(typename Elem<E>::type* p, const Lane& l, const float (&f)[16]) {
  store8<E, NT>(p + l.c0, f);
  store8<E, NT>(p + l.c1, f + 8);
}

// One pass for each wave, in the order of memory: waves that walk a token's heads each by
// themselves spread the loads under way over more of HBM's pages (16384 tokens, 72 heads of 128:
// 99 us with one pass for each wave, 102 with two, 108 with five, 115 with the whole token).
template <int E, int LPR, bool INTER>
__global__ __launch_bounds__(64 * kWaves) void qk_norm_rope_fwd(Args a) {
  using T = typename Elem<E>::type;
  constexpr int kRows = 64 / LPR;
  const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * kWaves + threadIdx.x / 64));
  const int pq = (a.Hq + kRows - 1) / kRows, passes = pq + (a.Hk + kRows - 1) / kRows;
  const int t = wave / passes;
  if (t >= a.T) return;
  const int p = wave - t * passes;
  const bool isq = p < pq;
  const Lane l = lane_of<LPR, INTER>(threadIdx.x & 63, a.D, a.R);
  const Heads<E> s = heads_of<E, false>(a, isq, t);
  const int h = (isq ? p : p - pq) * kRows + l.row;
  const bool on = l.on && h < s.H;
  const Raw16<E> raw = load16<E>(s.x + (int64_t)h * s.xh, l, on);
  const Raw16<E> raw_w = load16<E>(static_cast<const T*>(isq ? a.qw : a.kw), l, on);
  const int64_t pos = position(a, t);
  const bool real = pos >= 0 && pos < a.table_rows;
  const Turn turn = load_turn(a, l, pos, real);
  float n[16], g[16];
  unpack16<E>(raw, n);
  unpack16<E>(raw_w, g);
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) ss = __builtin_fmaf(n[i], n[i], ss);
  const float rstd = rsqrt_of(row_sum<LPR>(ss) / (float)a.D + a.eps);
#pragma unroll
  for (int i = 0; i < 16; ++i) n[i] = n[i] * rstd * g[i];
  rotate<INTER, false>(n, turn);
  if (!real) {
#pragma unroll
    for (int i = 0; i < 16; ++i) n[i] = 0.0f;
  }
  if (on) store16<E, true>(s.y + (int64_t)h * s.yh, l, n);
}

// A workgroup works on q (the first a.gq of them) or on k, so that it holds one weight and one sum:
// its waves walk the passes of that side in the order of memory, each pass's position read one
// ahead (its angles would wait for it otherwise).
template <int E, int LPR, bool INTER>
__global__ __launch_bounds__(64 * kWaves, 3) void qk_norm_rope_bwd(Args a) {
  using T = typename Elem<E>::type;
  constexpr int kRows = 64 / LPR;
  extern __shared__ float sums[];               // [waves][D]
  const bool isq = (int)blockIdx.x < a.gq;
  const int wg_wave = threadIdx.x / 64;
  const int group = isq ? (int)blockIdx.x : (int)blockIdx.x - a.gq;
  const int wave = __builtin_amdgcn_readfirstlane(group * kWaves + wg_wave);
  const int waves = (isq ? a.gq : (int)gridDim.x - a.gq) * kWaves;
  const Lane l = lane_of<LPR, INTER>(threadIdx.x & 63, a.D, a.R);
  const int passes = ((isq ? a.Hq : a.Hk) + kRows - 1) / kRows;
  const Raw16<E> weight = load16<E>(static_cast<const T*>(isq ? a.qw : a.kw), l, l.on);
  const float inv_d = 1.0f / (float)a.D;
  float dw[16] = {};
  const int items = a.T * passes;
  int64_t next_pos = wave < items ? position(a, wave / passes) : 0;
  for (int item = wave; item < items; item += waves) {
    const int t = item / passes;
    const Heads<E> s = heads_of<E, true>(a, isq, t);
    const int h = (item - t * passes) * kRows + l.row;
    const bool on = l.on && h < s.H;
    const Raw16<E> raw = load16<E>(s.x + (int64_t)h * s.xh, l, on);
    const Raw16<E> raw_d = load16<E>(s.dy + (int64_t)h * s.dyh, l, on);
    const int64_t pos = next_pos;
    const bool real = pos >= 0 && pos < a.table_rows;
    const Turn turn = load_turn(a, l, pos, real);
    if (item + waves < items) next_pos = position(a, (item + waves) / passes);
    float n[16], d[16], g[16];
    unpack16<E>(raw, n);
    unpack16<E>(raw_d, d);
    unpack16<E>(weight, g);
    rotate<INTER, true>(d, turn);
    float ss = 0.0f, ax = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      ss = __builtin_fmaf(n[i], n[i], ss);
      ax = __builtin_fmaf(d[i] * g[i], n[i], ax);
    }
    const float rstd = rsqrt_of(row_sum<LPR>(ss) * inv_d + a.eps);
    const float back = row_sum<LPR>(ax) * inv_d * rstd * rstd;
    if (real) {
      // Rows past the last head hold zeros: they add nothing, or 0 * inf where eps is 0.
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float gx = d[i] * (n[i] * rstd);
        dw[i] += h < s.H ? gx : 0.0f;
        n[i] = rstd * __builtin_fmaf(-n[i], back, d[i] * g[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) n[i] = 0.0f;
    }
    // Through the caches, for who reads the gradients next (past them: 52.0 / 50.0 us).
    if (on) store16<E, false>(s.y + (int64_t)h * s.yh, l, n);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
#pragma unroll
    for (int m = LPR; m < 64; m *= 2) dw[i] += __shfl_xor(dw[i], m);
  }
  if ((threadIdx.x & 63) < LPR && l.on) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sums[wg_wave * a.D + l.c0 + i] = dw[i];
      sums[wg_wave * a.D + l.c1 + i] = dw[8 + i];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.D; i += 64 * kWaves) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += sums[w * a.D + i];
    a.sums[(int64_t)blockIdx.x * a.D + i] = s;
  }
}

struct SumArgs {
  const float* sums;    // [gq + gk][D]
  float* dqw;
  float* dkw;
  int32_t gq, gk, D;
};

// The workgroups' sums of 16 columns: 64 threads of each column take every 64th one, then
// add their own in LDS in a fixed order.  blockIdx.y: q or k.
__global__ __launch_bounds__(16 * kSumRows) void weight_sums(SumArgs a) {
  __shared__ float part[kSumRows][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + c;          // D is a multiple of 16
  const bool isq = blockIdx.y == 0;
  const int n = isq ? a.gq : a.gk;
  const float* sums = a.sums + (isq ? 0 : (int64_t)a.gq * a.D) + col;
  float s = 0.0f;
#pragma unroll 8
  for (int i = r; i < n; i += kSumRows) s += sums[(int64_t)i * a.D];
  part[r][c] = s;
  __syncthreads();
  for (int half = kSumRows / 2; half > 0; half /= 2) {
    if (r < half) part[r][c] += part[r + half][c];
    __syncthreads();
  }
  if (r == 0) (isq ? a.dqw : a.dkw)[col] = part[0][c];
}

// ---------------------------------------------------------------------------------- host

bool aligned(const void* p, uintptr_t a) {
  return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}

// Rows of D elements at token and head strides.
struct Rows {
  const void* p;
  int64_t H, st, sh;
};

int64_t span(const Rows& r, int64_t T, int64_t D) {
  return (T - 1) * r.st + (r.H - 1) * r.sh + D;
}

// Whether two sets of rows share an element (told exactly for heads that lie within a token's
// stride, as views of one fused buffer do; otherwise by their ranges).
bool overlap(const Rows& a, const Rows& b, int64_t T, int64_t D, int64_t es) {
  const intptr_t pa = reinterpret_cast<intptr_t>(a.p), pb = reinterpret_cast<intptr_t>(b.p);
  if (pa + span(a, T, D) * es <= pb || pb + span(b, T, D) * es <= pa) return false;
  const int64_t wa = ((a.H - 1) * a.sh + D) * es, wb = ((b.H - 1) * b.sh + D) * es;
  const int64_t s = a.st * es;
  if (a.st != b.st || T < 2 || wa > s || wb > s) return true;
  const int64_t off = ((pb - pa) % s + s) % s;       // b's heads start here in a's token
  return off < wa || (off != 0 && s - off < wb);
}

bool overlap_range(const Rows& a, int64_t T, int64_t D, int64_t es, const void* p, int64_t n) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(a.p), q = reinterpret_cast<uintptr_t>(p);
  return lo < q + (uintptr_t)n && q < lo + (uintptr_t)(span(a, T, D) * es);
}

// Rows that are written must not share an element among themselves.
bool self_overlap(const Rows& r, int64_t T, int64_t D) {
  const bool heads = r.H < 2 || r.sh >= D, tokens = T < 2 || r.st >= D;
  if (!heads || !tokens) return true;
  if (r.H < 2 || T < 2) return false;
  return r.st < (r.H - 1) * r.sh + D && r.sh < (T - 1) * r.st + D;
}

bool same(const Rows& a, const Rows& b) { return a.p == b.p && a.st == b.st && a.sh == b.sh; }

int check_sizes(int64_t T, int64_t Hq, int64_t Hk, int64_t D, int64_t R, int64_t table_rows) {
  if (T < 0 || Hq < 1 || Hk < 1 || D < 16 || D % 16 != 0 || R < 16 || R > D || R % 16 != 0 ||
      table_rows < 0)
    return FAGQ_E_SHAPE;
  if (D > FAGQ_ROPE_MAX_D || T > (1ll << 24) || Hq > 4096 || Hk > 4096 || table_rows > (1ll << 31))
    return FAGQ_E_TOO_LARGE;
  return FAGQ_OK;
}

int lanes_per_row(int64_t D) { return D <= 64 ? 4 : D <= 128 ? 8 : D <= 256 ? 16 : 32; }

template <int E, int LPR>
const void* kernel_for(bool inter, bool bwd) {
  if (bwd)
    return inter ? reinterpret_cast<const void*>(&qk_norm_rope_bwd<E, LPR, true>)
                 : reinterpret_cast<const void*>(&qk_norm_rope_bwd<E, LPR, false>);
  return inter ? reinterpret_cast<const void*>(&qk_norm_rope_fwd<E, LPR, true>)
               : reinterpret_cast<const void*>(&qk_norm_rope_fwd<E, LPR, false>);
}
template <int E>
const void* kernel_for(int lpr, bool inter, bool bwd) {
  switch (lpr) {
    case 4: return kernel_for<E, 4>(inter, bwd);
    case 8: return kernel_for<E, 8>(inter, bwd);
    case 16: return kernel_for<E, 16>(inter, bwd);
    default: return kernel_for<E, 32>(inter, bwd);
  }
}
const void* kernel_for(int dtype, int lpr, bool inter, bool bwd) {
  return dtype == FAGQ_DT_BF16  ? kernel_for<ET_BF16>(lpr, inter, bwd)
         : dtype == FAGQ_DT_F16 ? kernel_for<ET_F16>(lpr, inter, bwd)
                                : kernel_for<ET_F32>(lpr, inter, bwd);
}

int64_t passes_of(int64_t Hq, int64_t Hk, int64_t D) {
  const int64_t rows = 64 / lanes_per_row(D);
  return (Hq + rows - 1) / rows + (Hk + rows - 1) / rows;
}

// The backward's workgroups of q and of k, in proportion to their passes.
struct Split {
  int64_t gq, gk;
};
Split split_for(int64_t T, int64_t Hq, int64_t Hk, int64_t D) {
  const int64_t rows = 64 / lanes_per_row(D);
  const int64_t pq = (Hq + rows - 1) / rows, pk = (Hk + rows - 1) / rows;
  int64_t gq = (kMaxBwdGroups * pq + (pq + pk) / 2) / (pq + pk);
  gq = gq < 1 ? 1 : gq > kMaxBwdGroups - 1 ? kMaxBwdGroups - 1 : gq;
  const int64_t gk = kMaxBwdGroups - gq;
  const int64_t nq = (T * pq + kWaves - 1) / kWaves, nk = (T * pk + kWaves - 1) / kWaves;
  return {nq < gq ? nq : gq, nk < gk ? nk : gk};
}

int64_t bwd_bytes(const Split& s, int64_t D) { return (s.gq + s.gk) * D * 4; }

int check_common(const void* const* ptrs, int n, const int64_t* strides, int nstrides, int64_t T,
                 int64_t Hq, int64_t Hk, int64_t D, int64_t R, int64_t table_rows, float eps,
                 int dtype, int index_dtype, const void* positions) {
  for (int i = 0; i < n; ++i)
    if (!ptrs[i]) return FAGQ_E_NULL;
  if (!positions || !strides) return FAGQ_E_NULL;
  if (dtype != FAGQ_DT_BF16 && dtype != FAGQ_DT_F16 && dtype != FAGQ_DT_F32) return FAGQ_E_FORMAT;
  if (index_dtype != FAGQ_IDX_I32 && index_dtype != FAGQ_IDX_I64) return FAGQ_E_FORMAT;
  if (!(eps >= 0.0f) || eps > 3.0e38f) return FAGQ_E_EPS;
  const int sizes = check_sizes(T, Hq, Hk, D, R, table_rows);
  if (sizes != FAGQ_OK) return sizes;
  const int64_t unit = dtype == FAGQ_DT_F32 ? 4 : 8;
  for (int i = 0; i < nstrides; ++i) {
    if (strides[i] < 0) return FAGQ_E_SHAPE;
    if (strides[i] >= (1ll << 31)) return FAGQ_E_TOO_LARGE;
    if (strides[i] % unit != 0) return FAGQ_E_ALIGN;
  }
  for (int i = 0; i < n; ++i)
    if (!aligned(ptrs[i], 16)) return FAGQ_E_ALIGN;
  if (!aligned(positions, index_dtype == FAGQ_IDX_I64 ? 8 : 4)) return FAGQ_E_ALIGN;
  return FAGQ_OK;
}

void set_strides(int32_t (&to)[2], const int64_t* from) {
  to[0] = (int32_t)from[0];
  to[1] = (int32_t)from[1];
}

}  // namespace
}  // namespace rope
}  // namespace fagq

extern "C" {

FAGQ_API int fagq_qk_norm_rope_launch(const void* q, const void* k, const void* q_weight,
                                      const void* k_weight, const float* cos, const float* sin,
                                      const void* positions, void* q_out, void* k_out,
                                      const int64_t* strides, int64_t T, int64_t Hq, int64_t Hk,
                                      int64_t D, int64_t R, int64_t table_rows, float eps,
                                      int interleaved, int dtype, int index_dtype, void* stream) {
  using namespace fagq;
  using namespace fagq::rope;
  const void* ptrs[] = {q, k, q_weight, k_weight, cos, sin, q_out, k_out};
  const int v = check_common(ptrs, 8, strides, 8, T, Hq, Hk, D, R, table_rows, eps, dtype,
                             index_dtype, positions);
  if (v != FAGQ_OK) return v;
  if (T == 0) return FAGQ_OK;
  const int64_t es = dtype == FAGQ_DT_F32 ? 4 : 2;
  const Rows in[2] = {{q, Hq, strides[0], strides[1]}, {k, Hk, strides[2], strides[3]}};
  const Rows out[2] = {{q_out, Hq, strides[4], strides[5]}, {k_out, Hk, strides[6], strides[7]}};
  const void* rest[] = {q_weight, k_weight, cos, sin, positions};
  const int64_t nrest[] = {D * es, D * es, table_rows * R * 2, table_rows * R * 2,
                           T * (index_dtype == FAGQ_IDX_I64 ? 8 : 4)};
  if (overlap(out[0], out[1], T, D, es)) return FAGQ_E_ALIAS;
  for (int i = 0; i < 2; ++i) {
    if (self_overlap(out[i], T, D)) return FAGQ_E_ALIAS;
    for (int j = 0; j < 2; ++j)
      if (!(i == j && same(out[i], in[j])) && overlap(out[i], in[j], T, D, es)) return FAGQ_E_ALIAS;
    for (int j = 0; j < 5; ++j)
      if (overlap_range(out[i], T, D, es, rest[j], nrest[j])) return FAGQ_E_ALIAS;
  }
  const int dcheck = device_check();
  if (dcheck != FAGQ_OK) return dcheck;
  Args a = {};
  a.q = q, a.k = k, a.qw = q_weight, a.kw = k_weight, a.cos = cos, a.sin = sin, a.pos = positions;
  a.qo = q_out, a.ko = k_out, a.table_rows = table_rows;
  set_strides(a.qs, strides), set_strides(a.ks, strides + 2);
  set_strides(a.qos, strides + 4), set_strides(a.kos, strides + 6);
  a.T = (int32_t)T, a.Hq = (int32_t)Hq, a.Hk = (int32_t)Hk, a.D = (int32_t)D, a.R = (int32_t)R;
  a.idx64 = index_dtype == FAGQ_IDX_I64, a.eps = eps;
  void* args[] = {&a};
  const int64_t groups = (T * passes_of(Hq, Hk, D) + kWaves - 1) / kWaves;
  if (groups >= (1ll << 32) / (64 * kWaves)) return FAGQ_E_TOO_LARGE;
  return launch_kernel(kernel_for(dtype, lanes_per_row(D), interleaved != 0, false),
                       dim3((unsigned)groups), dim3(64 * kWaves), args, 0,
                       static_cast<hipStream_t>(stream));
}

FAGQ_API int64_t fagq_qk_norm_rope_bwd_workspace_bytes(int64_t T, int64_t Hq, int64_t Hk,
                                                       int64_t D) {
  using namespace fagq::rope;
  if (check_sizes(T, Hq, Hk, D, 16, 0) != FAGQ_OK) return -1;
  return bwd_bytes(split_for(T, Hq, Hk, D), D);
}

FAGQ_API int fagq_qk_norm_rope_bwd_launch(const void* dq_out, const void* dk_out, const void* q,
                                          const void* k, const void* q_weight,
                                          const void* k_weight, const float* cos, const float* sin,
                                          const void* positions, void* dq, void* dk,
                                          float* dq_weight, float* dk_weight, void* workspace,
                                          int64_t workspace_bytes, const int64_t* strides,
                                          int64_t T, int64_t Hq, int64_t Hk, int64_t D, int64_t R,
                                          int64_t table_rows, float eps, int interleaved,
                                          int dtype, int index_dtype, void* stream) {
  using namespace fagq;
  using namespace fagq::rope;
  const void* ptrs[] = {dq_out, dk_out, q,  k,  q_weight,  k_weight,
                        cos,    sin,    dq, dk, dq_weight, dk_weight};
  const int v = check_common(ptrs, 12, strides, 12, T, Hq, Hk, D, R, table_rows, eps, dtype,
                             index_dtype, positions);
  if (v != FAGQ_OK) return v;
  const Split s = split_for(T, Hq, Hk, D);
  const int64_t need = bwd_bytes(s, D);
  if (need > 0 && !workspace) return FAGQ_E_NULL;
  if (workspace_bytes < need) return FAGQ_E_SHAPE;
  if (!aligned(workspace, 16)) return FAGQ_E_ALIGN;
  const int64_t es = dtype == FAGQ_DT_F32 ? 4 : 2;
  const Rows in[4] = {{dq_out, Hq, strides[0], strides[1]},
                      {dk_out, Hk, strides[2], strides[3]},
                      {q, Hq, strides[4], strides[5]},
                      {k, Hk, strides[6], strides[7]}};
  const Rows out[2] = {{dq, Hq, strides[8], strides[9]}, {dk, Hk, strides[10], strides[11]}};
  const void* flat[] = {dq_weight, dk_weight, workspace, q_weight, k_weight, cos, sin, positions};
  const int64_t nflat[] = {D * 4, D * 4, need, D * es, D * es, table_rows * R * 2,
                           table_rows * R * 2, T * (index_dtype == FAGQ_IDX_I64 ? 8 : 4)};
  if (T > 0) {
    if (overlap(out[0], out[1], T, D, es)) return FAGQ_E_ALIAS;
    for (int i = 0; i < 2; ++i) {
      if (self_overlap(out[i], T, D)) return FAGQ_E_ALIAS;
      for (int j = 0; j < 4; ++j)
        if (overlap(out[i], in[j], T, D, es)) return FAGQ_E_ALIAS;
      for (int j = 0; j < 8; ++j)
        if (overlap_range(out[i], T, D, es, flat[j], nflat[j])) return FAGQ_E_ALIAS;
    }
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 3; ++j)
        if (overlap_range(in[i], T, D, es, flat[j], nflat[j])) return FAGQ_E_ALIAS;
  }
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 8; ++j) {
      const uintptr_t x = reinterpret_cast<uintptr_t>(flat[i]), y = reinterpret_cast<uintptr_t>(flat[j]);
      if (nflat[i] > 0 && nflat[j] > 0 && x < y + (uintptr_t)nflat[j] && y < x + (uintptr_t)nflat[i])
        return FAGQ_E_ALIAS;
    }
  const int dcheck = device_check();
  if (dcheck != FAGQ_OK) return dcheck;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (T > 0) {
    if (T * passes_of(Hq, Hk, D) >= (1ll << 31) - kWaves * kMaxBwdGroups) return FAGQ_E_TOO_LARGE;
    Args a = {};
    a.q = q, a.k = k, a.qw = q_weight, a.kw = k_weight, a.cos = cos, a.sin = sin;
    a.pos = positions, a.qo = dq, a.ko = dk, a.dq = dq_out, a.dk = dk_out;
    a.sums = static_cast<float*>(workspace), a.table_rows = table_rows;
    set_strides(a.dqs, strides), set_strides(a.dks, strides + 2);
    set_strides(a.qs, strides + 4), set_strides(a.ks, strides + 6);
    set_strides(a.qos, strides + 8), set_strides(a.kos, strides + 10);
    a.T = (int32_t)T, a.Hq = (int32_t)Hq, a.Hk = (int32_t)Hk, a.D = (int32_t)D, a.R = (int32_t)R;
    a.gq = (int32_t)s.gq;
    a.idx64 = index_dtype == FAGQ_IDX_I64, a.eps = eps;
    void* args[] = {&a};
    const int ls = launch_kernel(kernel_for(dtype, lanes_per_row(D), interleaved != 0, true),
                                 dim3((unsigned)(s.gq + s.gk)), dim3(64 * kWaves), args,
                                 (size_t)kWaves * D * 4, st);
    if (ls != FAGQ_OK) return ls;
  }
  SumArgs sa = {static_cast<const float*>(workspace), dq_weight, dk_weight, (int32_t)s.gq,
                (int32_t)s.gk, (int32_t)D};
  void* sargs[] = {&sa};
  return launch_kernel(reinterpret_cast<const void*>(&weight_sums), dim3((unsigned)(D / 16), 2),
                       dim3(16 * kSumRows), sargs, 0, st);
}

}  // extern "C"
