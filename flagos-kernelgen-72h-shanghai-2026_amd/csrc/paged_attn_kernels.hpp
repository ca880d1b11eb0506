// paged_attn_kernels.hpp - device code of the attention over the quantised paged cache
// (include/fagq_cache.h).
//
// One pass with a running maximum m and sum l of the softmax: for key j with score x (in units
// of log 2), p = 2^(x - m), l = sum p, o = sum p v; parts of a row's keys have m, l and o of
// their own and are joined by o = sum 2^(m_i - m) o_i.
//
// A unit of work is 16 R query rows that read the same keys (the rows of one sequence that share
// a cache head; for the shared prefix, those of the whole batch) times a chunk of keys.  R D <= 256:
// with more rows the registers hold one wave on a SIMD, whose loads and products wait for each
// other (64 rows of 64 sequences behind 32768 keys, heads of 128: R = 2 145 us, R = 4 234).  The four
// waves of a workgroup take its steps of 32 keys in turn, each with m, l and o of its own, and are
// joined through LDS; chunks are joined by a second kernel.
//
// Keys and values go from HBM straight into the registers that feed the matrix instructions
// (16 x 16 x 32), with no LDS and no shuffle on the way:
//   scores   S^T = K Q^T.  Lane (c, g), c = lane % 16, g = lane / 16, holds 16-byte pieces
//            64 h + 16 g of key c: which dim stands at which place of the product's sum does not
//            matter, as long as Q is laid out the same.  Result: lane (c, g) has query c's
//            scores of keys 4 g .. 4 g + 3 of each tile of 16.
//   output   O^T = V^T P^T.  The lane's own eight probabilities of two tiles are its eight
//            places of the sum over 32 keys, so lane (c, g) loads D / 16 bytes of values of each
//            of those eight keys (dims D / 16 c ..) and transposes them, byte by byte, within its
//            registers.  Result: lane (c, g) has query c's dims D / 16 (4 g + r) + j.
// Codes are exact in q's type and in fp16 (fp8's 4 and int8's 8 bits of significand), so products
// with them lose nothing; the keys' scales multiply the scores, the values' the probabilities, in
// fp32.  Probabilities times value scales are rounded to fp16 whatever q's type is: half a step
// of 2^-11 of each, where bf16's 2^-8 would be as large an error as the result's own rounding
// (measured against 64 bits: 2.4e-3 with bf16, 1.7e-3 with fp16, 1.7e-3 for the rounding alone).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "fagq_cache_index.hpp"
#include "fagq_dispatch.hpp"

namespace fagq {
namespace attn {

constexpr int kWaves = 4;
constexpr int kStep = 32;            // keys of a wave's step
constexpr float kLow = -3.0e38f;     // running maximum before the first key
// The running maximum follows a row's scores only where they pass it by this much (p <= 2^8 then,
// which neither the sums nor fp16 probabilities mind), so that o is rarely multiplied.
constexpr float kSlack = 8.0f;

struct Args {
  const uint16_t* q;
  const uint8_t* kc;
  const uint8_t* vc;
  const void* ks;
  const void* vs;
  const int32_t* table;
  const void* lens;
  const int32_t* prefix;
  uint16_t* out;             // one chunk for each row: the result itself
  float* part;               // else [rows][chunks][D], then m and l [rows][chunks][2]
  float* part_ml;
  int32_t num_pages;
  int32_t qs[3];             // {sequence, token, head} strides, elements
  int32_t B, S, Hq, H, group;
  int32_t page_shift;
  int32_t width;             // pages of a row of the table
  int32_t prefix_len;
  int32_t most;              // tokens of a sequence that are read at most
  int32_t chunk, prefix_chunk;        // keys of a chunk, multiples of kStep * kWaves
  int32_t chunks, prefix_chunks;      // chunks of a row: its own, and of the prefix
  int32_t tiles, prefix_tiles;        // row tiles of a sequence and cache head; of the batch
  int32_t prefix_items, items;        // workgroups of the prefix, ahead of the others
  int32_t idx64;
  float scale2;                       // sm_scale * log2(e)
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <int E>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (E == ET_BF16) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a),
                                                   __builtin_bit_cast(v8, b), c, 0, 0, 0);
  } else {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a),
                                                  __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
}

// Four codes -> four values of type E, exactly.
template <int E, int QF>
__device__ __forceinline__ u32x2 widen4(uint32_t v) {
  u32x2 r;
  if constexpr (QF == QF_FP8 && E == ET_BF16) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, true));
  } else if constexpr (QF == QF_FP8) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v, 1.0f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v, 1.0f, true));
  } else if constexpr (E == ET_F16) {
    // Code + 128 under the exponent byte 0x64 is 1024 + 128 + code; the subtraction is exact.
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const uint32_t u = v ^ 0x80808080u;
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
    const uint32_t hi = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    r[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, lo) - off);
    r[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, hi) - off);
  } else {
    // |code| <= 128 fits bf16's 8 bits: the upper halves of the fp32 values are exact.
    uint32_t f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __float_as_uint((float)(int8_t)(v >> (8 * i)));
    r[0] = __builtin_amdgcn_perm(f[1], f[0], 0x07060302u);
    r[1] = __builtin_amdgcn_perm(f[3], f[2], 0x07060302u);
  }
  return r;
}

template <int E, int QF>
__device__ __forceinline__ u32x4 widen8(uint32_t lo, uint32_t hi) {
  const u32x2 a = widen4<E, QF>(lo), b = widen4<E, QF>(hi);
  return u32x4{a[0], a[1], b[0], b[1]};
}

// Maximum (sum) over the four lanes c, c + 16, c + 32, c + 48; every one of them receives it.
__device__ __forceinline__ float cross_max(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const float m = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const uint32_t w = __float_as_uint(m);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float cross_sum(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const float m = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const uint32_t w = __float_as_uint(m);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The pages of a step's two tiles, -1: none.
struct Pages {
  int32_t p[2];
};

template <int NT>
__device__ __forceinline__ void load_bytes(const uint8_t* p, uint32_t (&v)[NT / 4]) {
  if constexpr (NT == 4) {
    v[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (NT == 8) {
    const u32x2 x = *reinterpret_cast<const u32x2*>(p);
    v[0] = x[0], v[1] = x[1];
  } else {
    const u32x4 x = *reinterpret_cast<const u32x4*>(p);
    v[0] = x[0], v[1] = x[1], v[2] = x[2], v[3] = x[3];
  }
}

// The table's entry for the tile of 16 keys at `tok`, past its end -1; not checked yet, so that
// nothing waits for it until `checked`.
__device__ __forceinline__ int32_t entry_of(const int32_t* pages, int32_t width, int shift,
                                            int32_t tok) {
  const int32_t p = tok >> shift;
  return p < width ? pages[p] : -1;
}
__device__ __forceinline__ int32_t checked(int32_t page, int32_t num_pages) {
  return page < num_pages ? page : -1;          // negative: no page
}

// First row (page, head, offset) of a tile.  One without a page reads page 0, which exists, and
// is masked.
__device__ __forceinline__ int64_t first_row(const Args& a, int h, int32_t page, int32_t tok) {
  return (((int64_t)(page < 0 ? 0 : page) * a.H + h) << a.page_shift) +
         (tok & ((1 << a.page_shift) - 1));
}

// Scales of four consecutive keys.
template <int SF>
struct Scales {
  using type = u32x4;
};
template <>
struct Scales<SF_UE8M0> {
  using type = uint32_t;
};
template <int SF>
__device__ __forceinline__ typename Scales<SF>::type load_scales(const void* s, int64_t row) {
  using T = typename Scales<SF>::type;
  return *reinterpret_cast<const T*>(static_cast<const uint8_t*>(s) + row * (sizeof(T) / 4));
}
template <int SF>
__device__ __forceinline__ float scale_of(const typename Scales<SF>::type& s, int i) {
  if constexpr (SF == SF_UE8M0) return __uint_as_float(((s >> (8 * i)) & 255u) << 23);
  else return __uint_as_float(s[i]);
}

// The keys' and the values' codes and scales of one step, as loaded.
template <int D, int SF>
struct RawKeys {
  u32x4 k[2][D / 64];          // key c of each tile: its pieces 64 h + 16 g
  typename Scales<SF>::type s[2];   // of keys 4 g .. of each tile
};
template <int D, int SF>
struct RawValues {
  uint32_t v[8][D / 64];       // keys 4 g + i of tile 0 and 1: dims D / 16 c ..
  typename Scales<SF>::type s[2];
};

template <int D, int SF>
__device__ __forceinline__ void load_keys(const Args& a, int h, int lane, int32_t tok,
                                          const Pages& pages, RawKeys<D, SF>& r) {
  const int c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int64_t row = first_row(a, h, pages.p[t], tok + 16 * t);
    const uint8_t* k = a.kc + row * D;
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
      r.k[t][i] = *reinterpret_cast<const u32x4*>(k + (uint32_t)(c * D + 16 * g + 64 * i));
    r.s[t] = load_scales<SF>(a.ks, row + 4 * g);
  }
}

template <int D, int SF>
__device__ __forceinline__ void load_values(const Args& a, int h, int lane, int32_t tok,
                                            const Pages& pages, RawValues<D, SF>& r) {
  constexpr int NT = D / 16;
  const int c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int64_t row = first_row(a, h, pages.p[t], tok + 16 * t);
    const uint8_t* v = a.vc + row * D;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      load_bytes<NT>(v + (uint32_t)((4 * g + i) * D + c * NT), r.v[4 * t + i]);
    r.s[t] = load_scales<SF>(a.vs, row + 4 * g);
  }
}

// The rows of a unit: each lane's query c of R tiles.  One tile's queries stay in registers; more
// of them lie in LDS in the order of the products (the waves of a workgroup have the same rows),
// which leaves the registers for two waves on each SIMD.
template <int E, int D, int R>
struct Rows {
  u32x4 q[D / 32];             // R == 1; lane (c, g): dims 64 h + 16 g + 8 i .. of step 2 h + i
  const u32x4* lds_q;          // R > 1: [R][D / 32][64]
  f32x4 o[R][D / 16];          // dims D / 16 (4 g + r) + j at [j][r]
  float m[R], l[R];            // l: of this lane's keys
  int32_t seen[R];             // keys that the row sees
  float unit, inv_unit;        // o is in units of `unit`, a power of two (see join)
};

// Products of one step's keys with the queries.
template <int E, int QF, int SF, int D, int R>
__device__ __forceinline__ void scores(int lane, const RawKeys<D, SF>& raw, const Rows<E, D, R>& s,
                                       f32x4 (&x)[R][2]) {
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < 2; ++t) x[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    u32x4 k[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
      k[t] = widen8<E, QF>(raw.k[t][i / 2][2 * (i & 1)], raw.k[t][i / 2][2 * (i & 1) + 1]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const u32x4 q = R == 1 ? s.q[i] : s.lds_q[(r * (D / 32) + i) * 64 + lane];
#pragma unroll
      for (int t = 0; t < 2; ++t) x[r][t] = mfma<E>(k[t], q, x[r][t]);
    }
  }
}

// The softmax and the values of one step: 32 keys from `tok` on, of which the unit's last row
// sees those below `end`; all rows see those below `all`.  ks: the keys' scales times scale2.
template <int E, int QF, int SF, int D, int R>
__device__ __forceinline__ void join(int lane, int32_t tok, int32_t all, int32_t end,
                                     const Pages& pages, f32x4 (&x)[R][2], float (&ks)[8],
                                     RawValues<D, SF>& raw, Rows<E, D, R>& s) {
  constexpr int NT = D / 16;
  const int g = lane >> 4;
  float vs[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) vs[i] = scale_of<SF>(raw.s[i / 4], i % 4);
  if (tok + kStep > all || pages.p[0] < 0 || pages.p[1] < 0) {
    // What no row sees may hold anything: its values and their scales become zeros.  What a row
    // does not see gets no weight, whatever the score and the key's scale are.
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int32_t at = tok + 16 * (i / 4) + 4 * g + i % 4;
      const bool page = pages.p[i / 4] >= 0, live = at < end && page;
      vs[i] = live ? vs[i] : 0.0f;
#pragma unroll
      for (int w = 0; w < NT / 4; ++w) raw.v[i][w] = live ? raw.v[i][w] : 0u;
#pragma unroll
      for (int r = 0; r < R; ++r)
        x[r][i / 4][i % 4] = at < s.seen[r] && page ? x[r][i / 4][i % 4] * ks[i] : -INFINITY;
      ks[i] = 1.0f;
    }
  }
  // Probabilities times value scales have to fit fp16: they are taken in units of the power of
  // two just above the largest value scale so far, and o with them.
  float most = fmaxf(fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3])),
                     fmaxf(fmaxf(vs[4], vs[5]), fmaxf(vs[6], vs[7])));
  if (__any(most > s.unit)) {
    const uint32_t bits =
        (uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(cross_max(most)));
    int32_t e = (int32_t)(bits >> 23) - 126;
    e = e < 127 ? e : 127;
    const float unit = __builtin_ldexpf(1.0f, e), f = s.unit * __builtin_ldexpf(1.0f, -e);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < NT; ++j) s.o[r][j] *= f;
    s.unit = unit;
    s.inv_unit = __builtin_ldexpf(1.0f, -e);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) vs[i] *= s.inv_unit;
  u32x4 p[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __builtin_fmaf(x[r][i / 4][i % 4], ks[i], -s.m[r]);
    const float top = fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])),
                            fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7])));
    if (__any(top > kSlack)) {
      float m = s.m[r];
#pragma unroll
      for (int i = 0; i < 8; ++i) m = fmaxf(m, x[r][i / 4][i % 4] * ks[i]);
      m = cross_max(m);
      const float f = __builtin_amdgcn_exp2f(s.m[r] - m);
      s.m[r] = m;
      s.l[r] *= f;
#pragma unroll
      for (int j = 0; j < NT; ++j) s.o[r][j] *= f;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = __builtin_fmaf(x[r][i / 4][i % 4], ks[i], -m);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = __builtin_amdgcn_exp2f(y[i]);
      s.l[r] += y[i];
      y[i] *= vs[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) p[r][i] = pack16<ET_F16>(y[2 * i], y[2 * i + 1]);
  }
#pragma unroll
  for (int w = 0; w < NT / 4; ++w) {
    // Bytes of 8 keys x 4 dims -> 4 dims x 8 keys.
    uint32_t d[4][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t a0 = raw.v[4 * t][w], a1 = raw.v[4 * t + 1][w];
      const uint32_t a2 = raw.v[4 * t + 2][w], a3 = raw.v[4 * t + 3][w];
      const uint32_t e0 = __builtin_amdgcn_perm(a1, a0, 0x05010400u);   // dims 0, 1 of keys 0, 1
      const uint32_t e1 = __builtin_amdgcn_perm(a1, a0, 0x07030602u);   // dims 2, 3
      const uint32_t f0 = __builtin_amdgcn_perm(a3, a2, 0x05010400u);
      const uint32_t f1 = __builtin_amdgcn_perm(a3, a2, 0x07030602u);
      d[0][t] = __builtin_amdgcn_perm(f0, e0, 0x05040100u);
      d[1][t] = __builtin_amdgcn_perm(f0, e0, 0x07060302u);
      d[2][t] = __builtin_amdgcn_perm(f1, e1, 0x05040100u);
      d[3][t] = __builtin_amdgcn_perm(f1, e1, 0x07060302u);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4 v = widen8<ET_F16, QF>(d[i][0], d[i][1]);
#pragma unroll
      for (int r = 0; r < R; ++r) s.o[r][4 * w + i] = mfma<ET_F16>(v, p[r], s.o[r][4 * w + i]);
    }
  }
}

// The query of a row of a unit.
struct Row {
  int32_t b, s, hq;
};

// Keys of a list of pages, for the rows of one unit.
struct Keys {
  const int32_t* pages;
  int32_t width;
  int32_t begin, end;          // of this workgroup
};

template <int E, int QF, int SF, int D, int R>
__device__ __forceinline__ void run_steps(const Args& a, const Keys& k, int h, int lane, int wave,
                                          int32_t all, int32_t end, Rows<E, D, R>& s) {
  int32_t tok = k.begin + wave * kStep;
  constexpr int32_t kNext = kStep * kWaves;
  if (tok >= k.end) return;
  // Table entries are read a step ahead of the loads that need them.
  auto entries = [&](int32_t t) {
    return Pages{{entry_of(k.pages, k.width, a.page_shift, t),
                  entry_of(k.pages, k.width, a.page_shift, t + 16)}};
  };
  auto check = [&](const Pages& p) {
    return Pages{{checked(p.p[0], a.num_pages), checked(p.p[1], a.num_pages)}};
  };
  Pages ahead;
  auto work = [&](RawKeys<D, SF>& keys, RawValues<D, SF>& values, const Pages& pages, auto between) {
    f32x4 x[R][2];
    float ks[8];
    scores<E, QF, SF, D, R>(lane, keys, s, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) ks[i] = scale_of<SF>(keys.s[i / 4], i % 4) * a.scale2;
    between();
    join<E, QF, SF, D, R>(lane, tok, all, end, pages, x, ks, values, s);
  };
  if constexpr (R * D <= 128) {
    // Bound by HBM: two sets of registers, the next step's loads all under way during this one.
    RawKeys<D, SF> keys[2];
    RawValues<D, SF> values[2];
    Pages pages[2];
    pages[0] = check(entries(tok));
    ahead = entries(tok + kNext);
    load_keys<D, SF>(a, h, lane, tok, pages[0], keys[0]);
    load_values<D, SF>(a, h, lane, tok, pages[0], values[0]);
    auto one = [&](int now, int then) {
      const int32_t next = tok + kNext;
      const bool more = next < k.end;
      pages[then] = check(ahead);
      ahead = entries(next + kNext);
      if (more) {
        load_keys<D, SF>(a, h, lane, next, pages[then], keys[then]);
        load_values<D, SF>(a, h, lane, next, pages[then], values[then]);
      }
      work(keys[now], values[now], pages[now], [] {});
      tok = next;
      return more;
    };
    while (one(0, 1) && one(1, 0)) {
    }
  } else {
    // Short of registers: one set each, the next step's keys under way during this one's softmax
    // and values, its values during the next scores.
    RawKeys<D, SF> keys;
    RawValues<D, SF> values;
    Pages pages = check(entries(tok));
    ahead = entries(tok + kNext);
    load_keys<D, SF>(a, h, lane, tok, pages, keys);
    load_values<D, SF>(a, h, lane, tok, pages, values);
    for (;;) {
      const int32_t next = tok + kNext;
      const bool more = next < k.end;
      const Pages next_pages = check(ahead);
      ahead = entries(next + kNext);
      work(keys, values, pages, [&] {
        if (more) load_keys<D, SF>(a, h, lane, next, next_pages, keys);
      });
      if (!more) return;
      load_values<D, SF>(a, h, lane, next, next_pages, values);
      tok = next;
      pages = next_pages;
    }
  }
}

// LDS of a workgroup: the queries during the steps, then the waves' o of one tile of 16 rows; m and
// l of all rows.
template <int D, int R>
struct Shared {
  union {
    u32x4 q[R > 1 ? R * (D / 32) * 64 : 1];
    float o[kWaves][D / 4][64];
  };
  float m[kWaves][16 * R], l[kWaves][16 * R];
};

// Which tile of which group (cache head and chunk, ...) a workgroup takes: the tiles of a group
// read the same keys, so they go to one XCD (workgroup b runs on XCD b % 8) next to each other
// and find them in its L2.
struct Place {
  int tile, group;
};
__device__ __forceinline__ Place place_of(int item, int items, int tiles) {
  const int full = items / (8 * tiles) * 8 * tiles;
  if (item >= full) return {(item - full) % tiles, (full + item - full) / tiles};
  const int j = item >> 3;
  return {j % tiles, j / tiles * 8 + (item & 7)};
}

// One unit and chunk.  `item`: workgroup number within its kind.
template <int E, int QF, int SF, int D, int R, bool PREFIX>
__device__ __forceinline__ void unit(const Args& a, int item, char* lds) {
  constexpr int NT = D / 16;
  Shared<D, R>& sh = *reinterpret_cast<Shared<D, R>*>(lds);
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int chunks = PREFIX ? a.prefix_chunks : a.chunks;
  const Place place = PREFIX ? place_of(item, a.prefix_items, a.prefix_tiles)
                             : place_of(item, a.items, a.tiles);
  const int tile = place.tile;
  const int chunk = place.group % chunks;
  const int h = place.group / chunks % a.H;
  const int b = place.group / chunks / a.H;     // own keys: the sequence
  const int per = a.S * a.group;                // rows of a sequence and cache head
  const int rows = PREFIX ? a.B * per : per;
  Keys k;
  int32_t len = 0;                              // a sequence's own keys
  if constexpr (PREFIX) {
    k.pages = a.prefix;
    k.width = ((a.prefix_len - 1) >> a.page_shift) + 1;
    k.begin = chunk * a.prefix_chunk;
    k.end = k.begin + a.prefix_chunk < a.prefix_len ? k.begin + a.prefix_chunk : a.prefix_len;
  } else {
    const int64_t n = a.idx64 ? static_cast<const int64_t*>(a.lens)[b]
                              : (int64_t) static_cast<const int32_t*>(a.lens)[b];
    len = (int32_t)cache::seen_tokens(n, a.most, 1, 0);
    k.pages = a.table + (int64_t)b * a.width;
    k.width = a.width;
    k.begin = chunk * a.chunk;
    k.end = k.begin + a.chunk < len ? k.begin + a.chunk : len;
    // The joining kernel reads as many chunks as the length has.  The first one is always
    // written, for rows without keys.
    if (k.begin >= len && chunk > 0) return;
  }
  // Row i of the unit: i = (b,) s, query head of the group.
  auto row_of = [&](int i) {
    Row r;
    const int bs = i / a.group;
    r.hq = h * a.group + (i - bs * a.group);
    r.b = PREFIX ? bs / a.S : b;
    r.s = PREFIX ? bs - r.b * a.S : bs;
    return r;
  };
  auto load_q = [&](const Row& w, int j) {
    const uint16_t* q = a.q + ((int64_t)w.b * a.qs[0] + (int64_t)w.s * a.qs[1] +
                               (int64_t)w.hq * a.qs[2]);
    return *reinterpret_cast<const u32x4*>(q + 64 * (j / 2) + 16 * g + 8 * (j & 1));
  };
  Rows<E, D, R> s;
  s.unit = 0.0f;
  s.inv_unit = 0.0f;
  int32_t all = k.end, end = k.end;             // keys that all rows see; that the last one sees
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = (tile * R + r) * 16 + c;
    const Row w = row_of(i < rows ? i : rows - 1);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      if constexpr (R == 1) s.q[j] = load_q(w, j);
      else if ((r * (D / 32) + j) % kWaves == wave) sh.q[(r * (D / 32) + j) * 64 + lane] = load_q(w, j);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) s.o[r][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    s.m[r] = kLow;
    s.l[r] = 0.0f;
    s.seen[r] = PREFIX ? k.end : (int32_t)cache::seen_tokens(len, a.most, a.S, w.s);
  }
  s.lds_q = sh.q;
  if constexpr (R > 1) __syncthreads();
  if constexpr (!PREFIX) {
    // Rows are in order of their tokens: the first sees least, the last most.
    all = __builtin_amdgcn_readfirstlane(s.seen[0]);
    const int last = tile * R * 16 + 16 * R - 1;
    end = (int32_t)cache::seen_tokens(len, a.most, a.S, row_of(last < rows ? last : rows - 1).s);
    if (k.end > end) k.end = end;
  }
  run_steps<E, QF, SF, D, R>(a, k, h, lane, wave, all, end, s);

  // Join the waves.
#pragma unroll
  for (int r = 0; r < R; ++r) {
    s.l[r] = cross_sum(s.l[r]);
    if (g == 0) {
      sh.m[wave][16 * r + c] = s.m[r];
      sh.l[wave][16 * r + c] = s.l[r];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float m = kLow;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, sh.m[w][16 * r + c]);
    const float f = __builtin_amdgcn_exp2f(s.m[r] - m) * s.unit;
    float l = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      l += sh.l[w][16 * r + c] * __builtin_amdgcn_exp2f(sh.m[w][16 * r + c] - m);
    if (r > 0) __syncthreads();                 // the last tile's o has been read
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int j = 0; j < NT; ++j) sh.o[wave][q * NT + j][lane] = s.o[r][j][q] * f;
    __syncthreads();
    // Wave w adds up dims NT (4 g + w) + j of query c.
    float o[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      o[j] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) o[j] += sh.o[w][wave * NT + j][lane];
    }
    const int i = (tile * R + r) * 16 + c;
    if (i < rows) {
      const Row w = row_of(i);
      const int64_t row = ((int64_t)w.b * a.S + w.s) * a.Hq + w.hq;
      const int d = NT * (4 * g + wave);
      const int n = a.prefix_chunks + a.chunks;
      if (n == 1) {
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        uint32_t* to = reinterpret_cast<uint32_t*>(a.out + row * D + d);
#pragma unroll
        for (int j = 0; j < NT; j += 2) to[j / 2] = pack16<E>(o[j] * inv, o[j + 1] * inv);
      } else {
        const int64_t at = row * n + (PREFIX ? chunk : a.prefix_chunks + chunk);
        float* to = a.part + at * D + d;
#pragma unroll
        for (int j = 0; j < NT; j += 4)
          *reinterpret_cast<f32x4*>(to + j) = f32x4{o[j], o[j + 1], o[j + 2], o[j + 3]};
        if (wave == 0 && g == 0) {
          a.part_ml[2 * at] = m;
          a.part_ml[2 * at + 1] = l;
        }
      }
    }
  }
}

// RP: row tiles of a unit of the prefix (0: there is none), R: of the others.
template <int E, int QF, int SF, int D, int R, int RP>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_attention(Args a) {
  constexpr int kRows = R > RP ? R : RP;
  __shared__ __align__(16) char lds[sizeof(Shared<D, kRows>)];
  const int item = (int)blockIdx.x;
  if constexpr (RP > 0) {
    if (item < a.prefix_items) {
      unit<E, QF, SF, D, RP, true>(a, item, lds);
      return;
    }
  }
  unit<E, QF, SF, D, R, false>(a, item - a.prefix_items, lds);
}

// Kernels for an element type (ET_BF16, ET_F16), code format (QF_FP8, QF_I8_RNE) and scale format:
// lookup_e<E>_q<QF>_s<SF>, one for each instantiation unit.
const void* lookup_e0_q0_s0(int D, int R, int RP);
const void* lookup_e0_q0_s1(int D, int R, int RP);
const void* lookup_e0_q1_s0(int D, int R, int RP);
const void* lookup_e0_q1_s1(int D, int R, int RP);
const void* lookup_e1_q0_s0(int D, int R, int RP);
const void* lookup_e1_q0_s1(int D, int R, int RP);
const void* lookup_e1_q1_s0(int D, int R, int RP);
const void* lookup_e1_q1_s1(int D, int R, int RP);

}  // namespace attn
}  // namespace fagq
