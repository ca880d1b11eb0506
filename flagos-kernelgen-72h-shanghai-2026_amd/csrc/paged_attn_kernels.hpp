// paged_attn_kernels.hpp - device code of the attention over the quantised paged cache
// (include/fagq_cache.h).
//
// One pass with a running maximum m and sum l of the softmax: for key j with score x (in units
// of log 2), p = 2^(x - m), l = sum p, o = sum p v; parts of a row's keys have m, l and o of
// their own and are joined by o = sum 2^(m_i - m) o_i.
//
// A unit of work is 16 R query rows that read the same keys: the rows of one sequence that share a
// cache head, or for the shared prefix those of the whole batch.  R D <= 256: with more rows the
// registers hold one wave on a SIMD, whose loads and products wait for each other (64 rows of 64
// sequences behind 32768 keys, heads of 128: R = 2 145 us, R = 4 234).  A workgroup takes a range
// of a unit's keys; its four waves take the steps of 32 keys in turn, each with m, l and o of its
// own, and are joined through LDS.  Units of many rows of heads of 128 and 256 are tall ones: four
// times as many rows, a quarter for each wave (see Tall).  How units are cut goes by the host's
// bound on the lengths (plan_for), which knows nothing of the lengths themselves:
//   scheduled  The rounds of 128 keys of all units in a row are shared out evenly, so that every
//              workgroup reads as much as the others however the lengths differ (64 sequences of
//              1400 to 8192 tokens: 115 us, with chunks 131).  Each workgroup works that out by
//              itself from the lengths.
//   static     Chunks of one size, chosen by the host: the prefix; sequences of more than 16 rows,
//              whose units cost more to begin and to end in the middle (64 of 1500 tokens, 8 heads of
//              128, 32 rows: 43 us, scheduled 51; 16 of 4096, 16 heads of 64, 64 rows: 48, 80); short
//              sequences; and calls of few rounds, where working out the shares takes longer than
//              uneven ones (a call of 4 sequences of 1000 tokens: 0.9 us longer).
// The parts of a cut unit are joined by a second kernel.
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
//
// Bound: decode batches by HBM (64 sequences of 8192 tokens, 64 + 8 heads of 128: 174 us, 6.4 TB/s);
// many rows by no one unit: VALU instructions (the softmax) take 43 % of a SIMD's cycles, products 26 %,
// LDS 26 %, and its one or two waves wait for loads, LDS and barriers a quarter of theirs (64
// sequences behind 32768 shared tokens 116 us, 600 TFLOP/s; 4 of 512 new tokens over 4096 keys,
// 32 + 8 heads of 128, 179 us, 720); small calls by two dependent launches (4 sequences of 1000
// tokens 9.2 us, of which the kernels are 5.8 and 3.6).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "fagq_cache_index.hpp"
#include "fagq_dispatch.hpp"

namespace fagq {
namespace attn {

constexpr int kWaves = 4;
constexpr int kStep = 32;            // keys of a wave's step
constexpr int kRound = kStep * kWaves;
constexpr float kLow = -3.0e38f;     // running maximum before the first key
// The running maximum follows a row's scores only where a weight (probability times value scale)
// could pass 2^kSlack, which neither the sums nor fp16 minds, so that o is rarely multiplied.
constexpr float kSlack = 8.0f;
// Value scales lie in [0, 2^64]; smaller ones than this count as this in the running maximum, so that p
// is at most 2^(64 + kSlack).  See softmax for what the two bounds are for.
constexpr float kLeastScale = 0x1p-64f;
constexpr float kPartCost = 15.0f;   // what a part costs the joining kernel, in keys of a workgroup

// kScheduledOnce: the codes are read past the caches (64 sequences of 8192 tokens, 64 + 8 heads of
// 128, 1.07 GB: 172 against 186 us); calls whose cache may still hold what the last one read
// lose by it (8 of 4000 tokens, 32 heads, 131 MB: 46 against 36 us).  It is taken by the bytes of
// the bound on the lengths, which a wide table makes larger than what is read.
enum Form { kStatic = 0, kScheduled = 1, kScheduledOnce = 2 };

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
  // Parts of cut units: o [index][D], then {m, l} [index][2].  Index: row * row_parts + i (i: chunk
  // of the prefix, then a chunk of its own keys or all of them), behind those
  // segment_at(workgroup, slot) + row of the unit.
  float* part;
  float* part_ml;
  int32_t* sched;            // scheduled: each sequence's first round, then the rounds of a workgroup
  int32_t num_pages;
  int32_t qs[3];             // {sequence, token, head} strides, elements
  int32_t B, S, Hq, H, group;
  int32_t page_shift;
  int32_t width;             // pages of a row of the table
  int32_t prefix_len;
  int32_t most;              // tokens of a sequence that are read at most
  int32_t chunk, prefix_chunk;        // keys of a chunk, multiples of kRound
  int32_t chunks, prefix_chunks;      // chunks of a row: its own (static), and of the prefix
  int32_t row_parts;
  int32_t tiles, prefix_tiles;        // row tiles of a sequence and cache head; of the batch
  int32_t prefix_items, items;        // workgroups of the prefix, ahead of the others
  int32_t slots;                      // workgroups that the schedule fills
  int32_t idx64;
  float scale2;                       // sm_scale * log2(e)
  const uint8_t* tree;                // [S][S] of each sequence, tree_next bytes apart (see Tree)
  int64_t tree_next;
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

// Bytes of 4 keys x 4 dims -> 4 dims x 4 keys.
__device__ __forceinline__ void transpose4(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                           uint32_t (&d)[4]) {
  const uint32_t e0 = __builtin_amdgcn_perm(a1, a0, 0x05010400u);   // dims 0, 1 of keys 0, 1
  const uint32_t e1 = __builtin_amdgcn_perm(a1, a0, 0x07030602u);   // dims 2, 3
  const uint32_t f0 = __builtin_amdgcn_perm(a3, a2, 0x05010400u);
  const uint32_t f1 = __builtin_amdgcn_perm(a3, a2, 0x07030602u);
  d[0] = __builtin_amdgcn_perm(f0, e0, 0x05040100u);
  d[1] = __builtin_amdgcn_perm(f0, e0, 0x07060302u);
  d[2] = __builtin_amdgcn_perm(f1, e1, 0x05040100u);
  d[3] = __builtin_amdgcn_perm(f1, e1, 0x07060302u);
}

// Own keys of a sequence: its length, as far as `most` of them are read.
__device__ __forceinline__ int32_t own_length(const void* lens, int idx64, int32_t most, int b) {
  const int64_t n = idx64 ? static_cast<const int64_t*>(lens)[b]
                          : (int64_t) static_cast<const int32_t*>(lens)[b];
  return (int32_t)cache::seen_tokens(n, most, 1, 0);
}
// Rounds of a sequence's units: one for a sequence without keys, whose rows are written too.
__device__ __forceinline__ int32_t rounds_of(int32_t len) {
  const int32_t n = (len + kRound - 1) / kRound;
  return n > 1 ? n : 1;
}

// First index of the parts that a workgroup leaves of units of 16 rows: slot 1 of the unit that it
// began and did not finish, slot 0 of the one that it did not begin.
constexpr int kSegmentRows = 16;
__device__ __forceinline__ int64_t segment_at(int64_t first, int wg, int slot) {
  return first + ((int64_t)wg * 2 + slot) * kSegmentRows;
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

// 2^d for d <= 0 as a product: what 2^d alone is too small for in fp32 keeps its value if it is multiplied
// by b, then by a.  b is 1 for d >= -64.
struct Power {
  float a, b;
};
__device__ __forceinline__ Power power_of(float d) {
  return {__builtin_amdgcn_exp2f(fmaxf(d, -64.0f)), __builtin_amdgcn_exp2f(fminf(d + 64.0f, 0.0f))};
}

// The pages of a step's two tiles, -1: none.
struct Pages {
  int32_t p[2];
};

// ONCE: the codes are read once and are too many to be found in a cache by the next call.
template <bool ONCE, typename T>
__device__ __forceinline__ T load_codes(const uint8_t* p) {
  if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
  else return *reinterpret_cast<const T*>(p);
}
template <int NT, bool ONCE>
__device__ __forceinline__ void load_bytes(const uint8_t* p, uint32_t (&v)[NT / 4]) {
  if constexpr (NT == 4) {
    v[0] = load_codes<ONCE, uint32_t>(p);
  } else if constexpr (NT == 8) {
    const u32x2 x = load_codes<ONCE, u32x2>(p);
    v[0] = x[0], v[1] = x[1];
  } else {
    const u32x4 x = load_codes<ONCE, u32x4>(p);
    v[0] = x[0], v[1] = x[1], v[2] = x[2], v[3] = x[3];
  }
}

// The table's entry for the tile of 16 keys at `tok`, past its end -1; not checked yet, so that
// nothing waits for it until `checked`.  A scalar load (the table is constant during the kernel,
// which the compiler cannot know of a kernel that stores): a vector load would stand in line with
// the codes' and be waited for with them.
__device__ __forceinline__ int32_t entry_of(const int32_t* pages, int32_t width, int shift,
                                            int32_t tok) {
  using Constant = const __attribute__((address_space(4))) int32_t;
  const int32_t p = tok >> shift;
  return p < width ? reinterpret_cast<Constant*>(reinterpret_cast<uintptr_t>(pages))[p] : -1;
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

// Where a step's two tiles are.
struct Rows2 {
  int64_t row[2];
};
__device__ __forceinline__ Rows2 rows_at(const Args& a, int h, const Pages& pages, int32_t tok) {
  return {{first_row(a, h, pages.p[0], tok), first_row(a, h, pages.p[1], tok + 16)}};
}

template <int D, int SF, bool ONCE>
__device__ __forceinline__ void load_keys(const Args& a, int lane, const Rows2& at,
                                          RawKeys<D, SF>& r) {
  const int c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint8_t* k = a.kc + at.row[t] * D;
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
      r.k[t][i] = load_codes<ONCE, u32x4>(k + (uint32_t)(c * D + 16 * g + 64 * i));
    r.s[t] = load_scales<SF>(a.ks, at.row[t] + 4 * g);
  }
}

template <int D, int SF, bool ONCE>
__device__ __forceinline__ void load_values(const Args& a, int lane, const Rows2& at,
                                            RawValues<D, SF>& r) {
  constexpr int NT = D / 16;
  const int c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint8_t* v = a.vc + at.row[t] * D;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      load_bytes<NT, ONCE>(v + (uint32_t)((4 * g + i) * D + c * NT), r.v[4 * t + i]);
    r.s[t] = load_scales<SF>(a.vs, at.row[t] + 4 * g);
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
};

// TREE: the newest S tokens are drafts.  Query s sees the len - S tokens before them and the drafts t
// (token len - S + t) whose byte [s][t] of the mask is not 0.  Rows::seen then is s S, where the
// row's bytes begin.
struct Tree {
  const uint8_t* mask;
  int32_t context, len;
};
// A draft that none of a wave's rows sees may hold anything, NaN among it, which a weight of 0 does not
// take away: its value scale and its values become zeros.  Element i of a lane's operand of values is
// key i of the lane's eight.
struct Kept {
  u32x4 bits = {~0u, ~0u, ~0u, ~0u};
  __device__ __forceinline__ void drop(int lane, int i, bool seen, float& scale) {
    if ((__ballot(seen) >> (lane & 48)) & 0xffffu) return;       // by one of the 16 rows of some tile
    scale = 0.0f;
    bits[i / 2] &= i % 2 ? 0x0000ffffu : 0xffff0000u;
  }
};
template <bool TREE>
__device__ __forceinline__ bool sees(int32_t seen, const Tree& tree, int32_t at) {
  if constexpr (TREE)
    return at < tree.context || (at < tree.len && tree.mask[seen + (at - tree.context)] != 0);
  else
    return at < seen;
}

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

// The softmax of one step: 32 keys from `tok` on, of which all rows see those below `all`.  From the
// products x, the keys' scales times scale2 and the values' scales (zeros for what no row sees) to
// the probabilities times value scales, as fp16 operands of the next product.
//
// m is the running maximum of score + log2(value scale), not of the score: p = 2^(x - m) times its
// value scale is at most 2^kSlack then, which fits fp16, and what fp16 loses of a small one is lost
// relative to the largest contribution to the row, however far apart the value scales are.  l is in the
// same units, so the bounds of the value scales keep it in fp32's range: m <= largest score + 64, so the
// largest score's p is 2^-64 or more and what is flushed below 2^-126 is 2^-62 of it; and p <= 2^72, so
// 2^31 keys add up to at most 2^103.  But from one m to the next l may fall by more than 2^-126 (keys of
// scale 0, then one of 2^64: 2^-128 at equal scores), where o, whose terms fall with it, may become 0
// and l may not: it takes the factor in two.
template <int E, int D, int R, bool TREE>
__device__ __forceinline__ void softmax(int lane, int32_t tok, int32_t all, const Pages& pages,
                                        f32x4 (&x)[R][2], float (&ks)[8], float (&vs)[8],
                                        const Tree& tree, Rows<E, D, R>& s, u32x4 (&p)[R],
                                        Kept& kept) {
  constexpr int NT = D / 16;
  const int g = lane >> 4;
  if (tok + kStep > all || pages.p[0] < 0 || pages.p[1] < 0) {
    // What a row does not see gets no weight, whatever the score and the key's scale are.
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int32_t at = tok + 16 * (i / 4) + 4 * g + i % 4;
      bool any = false;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool seen = sees<TREE>(s.seen[r], tree, at) && pages.p[i / 4] >= 0;
        x[r][i / 4][i % 4] = seen ? x[r][i / 4][i % 4] * ks[i] : -INFINITY;
        any |= seen;
      }
      ks[i] = 1.0f;
      if constexpr (TREE) kept.drop(lane, i, any, vs[i]);
    }
  }
  const float most = fmaxf(fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3])),
                           fmaxf(fmaxf(vs[4], vs[5]), fmaxf(vs[6], vs[7])));
  const float room = kSlack - __builtin_amdgcn_logf(fmaxf(most, kLeastScale));
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __builtin_fmaf(x[r][i / 4][i % 4], ks[i], -s.m[r]);
    const float top = fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])),
                            fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7])));
    if (__any(!(top <= room))) {
      float m = s.m[r];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        m = fmaxf(m, __builtin_fmaf(x[r][i / 4][i % 4], ks[i],
                                    __builtin_amdgcn_logf(fmaxf(vs[i], kLeastScale))));
      m = cross_max(m);
      const Power f = power_of(s.m[r] - m);
      s.m[r] = m;
      s.l[r] = s.l[r] * f.b * f.a;
#pragma unroll
      for (int j = 0; j < NT; ++j) s.o[r][j] *= f.a * f.b;
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
}

// One step of keys in registers, `end`: the unit's last row sees the keys below it.
template <int E, int QF, int SF, int D, int R, bool TREE>
__device__ __forceinline__ void join(int lane, int32_t tok, int32_t all, int32_t end,
                                     const Pages& pages, f32x4 (&x)[R][2], float (&ks)[8],
                                     RawValues<D, SF>& raw, const Tree& tree, Rows<E, D, R>& s) {
  constexpr int NT = D / 16;
  const int g = lane >> 4;
  float vs[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) vs[i] = scale_of<SF>(raw.s[i / 4], i % 4);
  if (tok + kStep > end || pages.p[0] < 0 || pages.p[1] < 0) {
    // What no row sees may hold anything: its values and their scales become zeros.
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool live = tok + 16 * (i / 4) + 4 * g + i % 4 < end && pages.p[i / 4] >= 0;
      vs[i] = live ? vs[i] : 0.0f;
#pragma unroll
      for (int w = 0; w < NT / 4; ++w) raw.v[i][w] = live ? raw.v[i][w] : 0u;
    }
  }
  u32x4 p[R];
  Kept kept;
  softmax<E, D, R, TREE>(lane, tok, all, pages, x, ks, vs, tree, s, p, kept);
#pragma unroll
  for (int w = 0; w < NT / 4; ++w) {
    uint32_t d[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
      transpose4(raw.v[4 * t][w], raw.v[4 * t + 1][w], raw.v[4 * t + 2][w], raw.v[4 * t + 3][w], d[t]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 v = widen8<ET_F16, QF>(d[0][i], d[1][i]);
      if constexpr (TREE)
        if (tok + kStep > all) v &= kept.bits;
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

template <int E, int QF, int SF, int D, int R, bool ONCE, bool TREE>
__device__ __forceinline__ void run_steps(const Args& a, const Keys& k, int h, int lane, int wave,
                                          int32_t all, int32_t end, const Tree& tree,
                                          Rows<E, D, R>& s) {
  int32_t tok = k.begin + wave * kStep;
  if (tok >= k.end) return;
  // Table entries are read a step ahead of the loads that need them.
  auto entries = [&](int32_t t) {
    return Pages{{entry_of(k.pages, k.width, a.page_shift, t),
                  entry_of(k.pages, k.width, a.page_shift, t + 16)}};
  };
  auto check = [&](const Pages& p) {
    return Pages{{checked(p.p[0], a.num_pages), checked(p.p[1], a.num_pages)}};
  };
  // One set of registers each: the next step's keys are under way during this one's softmax and
  // values, its values during the next scores.  (A second set, with both under way during all of a
  // step, changed nothing where HBM bounds: 187 against 186 us.)
  RawKeys<D, SF> keys;
  RawValues<D, SF> values;
  Pages pages = check(entries(tok));
  Pages ahead = entries(tok + kRound);
  Rows2 at = rows_at(a, h, pages, tok);
  load_keys<D, SF, ONCE>(a, lane, at, keys);
  load_values<D, SF, ONCE>(a, lane, at, values);
  for (;;) {
    const int32_t next = tok + kRound;
    const bool more = next < k.end;
    const Pages next_pages = check(ahead);
    // Behind the last step its own rows are loaded again: loads that are under way on one path only
    // would have every wait for older ones wait for them too.
    if (more) at = rows_at(a, h, next_pages, next);
    f32x4 x[R][2];
    float ks[8];
    scores<E, QF, SF, D, R>(lane, keys, s, x);
    // Behind the scores: their LDS reads would wait for a scalar load under way.
    ahead = entries(next + kRound);
#pragma unroll
    for (int i = 0; i < 8; ++i) ks[i] = scale_of<SF>(keys.s[i / 4], i % 4) * a.scale2;
    load_keys<D, SF, ONCE>(a, lane, at, keys);
    join<E, QF, SF, D, R, TREE>(lane, tok, all, end, pages, x, ks, values, tree, s);
    if (!more) return;
    load_values<D, SF, ONCE>(a, lane, at, values);
    tok = next;
    pages = next_pages;
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

// What a workgroup does at a time: a range of one unit's keys.
struct Segment {
  int b, h, tile;            // sequence (own keys), cache head, row tile
  int32_t len;               // own keys of the sequence
  Keys keys;
  int64_t to;                // index of row 0 of its part; kRowParts: of each row's own; kOut
  int row_part;              // kRowParts: which of a row's parts
};
constexpr int64_t kOut = -1;          // the result itself
constexpr int64_t kRowParts = -2;

template <bool TREE>
__device__ __forceinline__ Tree tree_of(const Args& a, int b, int32_t len) {
  if constexpr (TREE) return {a.tree + b * a.tree_next, len - a.S, len};
  else return {};
}

template <int E, int QF, int SF, int D, int R, bool PREFIX, bool ONCE, bool TREE>
__device__ __forceinline__ void run_segment(const Args& a, const Segment& seg, Shared<D, R>& sh) {
  constexpr int NT = D / 16;
  int lane = threadIdx.x & 63;
  // Opaque, so that what a segment derives from it is not kept in registers from one to the next.
  asm volatile("" : "+v"(lane));
  const int c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int h = seg.h, b = seg.b, tile = seg.tile;
  const int32_t len = seg.len;
  const int per = a.S * a.group;                // rows of a sequence and cache head
  const int rows = PREFIX ? a.B * per : per;
  Keys k = seg.keys;
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
    s.seen[r] = PREFIX ? k.end : TREE ? w.s * a.S : (int32_t)cache::seen_tokens(len, a.most, a.S, w.s);
  }
  s.lds_q = sh.q;
  if constexpr (R > 1) __syncthreads();
  const Tree tree = tree_of<TREE>(a, b, len);
  if constexpr (TREE) {
    all = tree.context;
    end = len;
  } else if constexpr (!PREFIX) {
    // Rows are in order of their tokens: the first sees least, the last most.
    all = __builtin_amdgcn_readfirstlane(s.seen[0]);
    const int last = tile * R * 16 + 16 * R - 1;
    end = (int32_t)cache::seen_tokens(len, a.most, a.S, row_of(last < rows ? last : rows - 1).s);
    if (k.end > end) k.end = end;
  }
  run_steps<E, QF, SF, D, R, ONCE, TREE>(a, k, h, lane, wave, all, end, tree, s);

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
    const float f = __builtin_amdgcn_exp2f(s.m[r] - m);
    float l = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const Power g = power_of(sh.m[w][16 * r + c] - m);
      l = __builtin_fmaf(sh.l[w][16 * r + c] * g.b, g.a, l);
    }
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
      if (seg.to == kOut) {
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        uint32_t* to = reinterpret_cast<uint32_t*>(a.out + row * D + d);
#pragma unroll
        for (int j = 0; j < NT; j += 2) to[j / 2] = pack16<E>(o[j] * inv, o[j + 1] * inv);
      } else {
        const int64_t at = seg.to == kRowParts ? row * a.row_parts + seg.row_part : seg.to + i;
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

// ------------------------------------------------------------------------- many rows

// Tall units: each wave has 16 R rows of its own (R D = 256), and the four waves see the same keys.
// A step's codes are widened once for all of them, a quarter by each wave, and handed on through LDS
// in the order of the products; the next steps' are staged while these are worked on.  The shorter
// units widen as much for 16 R rows as these do for 64 R, which is a third of their instructions.
// V's tile (h, i) of the product has the dims 64 h + 4 c + i.
template <int D>
struct Tall {
  static constexpr int R = 256 / D;
  // Steps between two barriers, as far as two workgroups' LDS fits a CU (heads of 128: one step
  // 188 us, two 181; heads of 256: 223, two 388).
  static constexpr int kSteps = 256 / D;
  static constexpr int kPieces = D / 32;        // 16-byte pieces of a step's keys; 4-key tiles of
                                                // 64 dims of its values
  static constexpr int kEach = kPieces / kWaves;
  static_assert(kPieces % kWaves == 0, "heads of 128 and 256");
  struct Lds {
    u32x4 k[2][kSteps][2 * (D / 32)][64];
    u32x4 v[2][kSteps][D / 16][64];
    float ks[2][kSteps][kStep], vs[2][kSteps][kStep];
  };
  struct Raw {
    u32x4 k[kEach];
    uint32_t v[kEach][4];
    float scale;               // wave 0: of key lane % 32, keys' below lane 32, values' above
    Pages pages;
    int32_t tok;
  };
  static __device__ __forceinline__ int piece(int wave, int n) { return wave + n * kWaves; }
};

template <int SF, int D>
__device__ __forceinline__ void load_tall(const Args& a, int h, int lane, int wave, int32_t tok,
                                          const Pages& pages, typename Tall<D>::Raw& r) {
  const int c = lane & 15, g = lane >> 4;
  const Rows2 at = rows_at(a, h, pages, tok);
  r.pages = pages;
  r.tok = tok;
#pragma unroll
  for (int n = 0; n < Tall<D>::kEach; ++n) {
    const int p = Tall<D>::piece(wave, n);
    r.k[n] = *reinterpret_cast<const u32x4*>(
        a.kc + (p < D / 64 ? at.row[0] : at.row[1]) * D +
        (uint32_t)(c * D + 16 * g + 64 * (p % (D / 64))));
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r.v[n][i] = *reinterpret_cast<const uint32_t*>(
          a.vc + (p & 1 ? at.row[1] : at.row[0]) * D +
          (uint32_t)((4 * g + i) * D + 64 * (p >> 1) + 4 * c));
  }
  if (wave == 0) {
    const void* s = lane < kStep ? a.ks : a.vs;
    const int64_t row = (lane & 16 ? at.row[1] : at.row[0]) + c;
    r.scale = SF == SF_UE8M0
                  ? __uint_as_float((uint32_t) static_cast<const uint8_t*>(s)[row] << 23)
                  : static_cast<const float*>(s)[row];
  }
}

template <int E, int QF, int D>
__device__ __forceinline__ void stage_tall(const Args& a, int lane, int wave, int32_t end,
                                           const typename Tall<D>::Raw& r,
                                           typename Tall<D>::Lds& sh, int buf, int step) {
  const int c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int n = 0; n < Tall<D>::kEach; ++n) {
    const int p = Tall<D>::piece(wave, n);
    const int at = p / (D / 64) * (D / 32) + 2 * (p % (D / 64));
    sh.k[buf][step][at][lane] = widen8<E, QF>(r.k[n][0], r.k[n][1]);
    sh.k[buf][step][at + 1][lane] = widen8<E, QF>(r.k[n][2], r.k[n][3]);
    const int t = p & 1;
    const bool page = (t ? r.pages.p[1] : r.pages.p[0]) >= 0;
    uint32_t v[4], d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = r.v[n][i];
    if (r.tok + kStep > end || !page) {
      // What no row sees may hold anything: it becomes zeros.
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = r.tok + 16 * t + 4 * g + i < end && page ? v[i] : 0u;
    }
    transpose4(v[0], v[1], v[2], v[3], d);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<u32x2*>(&sh.v[buf][step][4 * (p >> 1) + i][lane])[t] =
          widen4<ET_F16, QF>(d[i]);
  }
  if (wave == 0) {
    const int t = (lane >> 4) & 1;
    if (lane < kStep) {
      sh.ks[buf][step][lane] = r.scale * a.scale2;
    } else {
      const bool live = r.tok + 16 * t + c < end && (t ? r.pages.p[1] : r.pages.p[0]) >= 0;
      sh.vs[buf][step][lane - kStep] = live ? r.scale : 0.0f;
    }
  }
}

template <int E, int QF, int SF, int D, bool PREFIX, bool TREE>
__device__ __forceinline__ void run_tall(const Args& a, const Segment& seg,
                                         typename Tall<D>::Lds& sh) {
  constexpr int R = Tall<D>::R, NT = D / 16;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int per = a.S * a.group;
  const int rows = PREFIX ? a.B * per : per;
  const int first_row = (seg.tile * kWaves + wave) * 16 * R;
  Keys k = seg.keys;
  auto row_of = [&](int i) {
    Row r;
    const int bs = i / a.group;
    r.hq = seg.h * a.group + (i - bs * a.group);
    r.b = PREFIX ? bs / a.S : seg.b;
    r.s = PREFIX ? bs - r.b * a.S : bs;
    return r;
  };
  Rows<E, D, R> s;
  u32x4 q[R][D / 32];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = first_row + 16 * r + c;
    const Row w = row_of(i < rows ? i : rows - 1);
    const uint16_t* at = a.q + ((int64_t)w.b * a.qs[0] + (int64_t)w.s * a.qs[1] +
                                (int64_t)w.hq * a.qs[2]);
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
      q[r][j] = *reinterpret_cast<const u32x4*>(at + 64 * (j / 2) + 16 * g + 8 * (j & 1));
#pragma unroll
    for (int j = 0; j < NT; ++j) s.o[r][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    s.m[r] = kLow;
    s.l[r] = 0.0f;
    s.seen[r] = PREFIX ? k.end
                : TREE ? w.s * a.S
                       : (int32_t)cache::seen_tokens(seg.len, a.most, a.S, w.s);
  }
  int32_t all = k.end;                          // keys that all rows of this wave see
  const Tree tree = tree_of<TREE>(a, seg.b, seg.len);
  if constexpr (TREE) {
    all = tree.context;
  } else if constexpr (!PREFIX) {
    // Rows are in order of their tokens: the last one of the workgroup sees most.
    all = __builtin_amdgcn_readfirstlane(s.seen[0]);
    const int last = (seg.tile + 1) * kWaves * 16 * R - 1;
    const int32_t end =
        (int32_t)cache::seen_tokens(seg.len, a.most, a.S, row_of(last < rows ? last : rows - 1).s);
    if (k.end > end) k.end = end;
  }
  if (k.begin < k.end) {
    auto entries = [&](int32_t t) {
      return Pages{{entry_of(k.pages, k.width, a.page_shift, t),
                    entry_of(k.pages, k.width, a.page_shift, t + 16)}};
    };
    auto check = [&](const Pages& p) {
      return Pages{{checked(p.p[0], a.num_pages), checked(p.p[1], a.num_pages)}};
    };
    constexpr int kSteps = Tall<D>::kSteps, kKeys = kSteps * kStep;
    typename Tall<D>::Raw raw[kSteps];
    int32_t tok = k.begin;
    Pages pages[kSteps], next_pages[kSteps], ahead[kSteps];
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      pages[u] = check(entries(tok + u * kStep));
      next_pages[u] = check(entries(tok + kKeys + u * kStep));
      ahead[u] = entries(tok + 2 * kKeys + u * kStep);
    }
#pragma unroll
    for (int u = 0; u < kSteps; ++u)
      load_tall<SF, D>(a, seg.h, lane, wave, tok + u * kStep, pages[u], raw[u]);
#pragma unroll
    for (int u = 0; u < kSteps; ++u)
      stage_tall<E, QF, D>(a, lane, wave, k.end, raw[u], sh, 0, u);
    // Behind the last steps codes are loaded again: see run_steps.
    if (tok + kKeys < k.end) {
#pragma unroll
      for (int u = 0; u < kSteps; ++u)
        load_tall<SF, D>(a, seg.h, lane, wave, tok + kKeys + u * kStep, next_pages[u], raw[u]);
    }
    // The queries are waited for here: in the loop their first use would wait for all loads under
    // way, every time (heads of 128: 200 us, so 188).
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < D / 32; ++j) asm volatile("" : "+v"(q[r][j]));
    for (int buf = 0;; buf ^= 1) {
      const bool more = tok + kKeys < k.end, far = tok + 2 * kKeys < k.end;
      lds_barrier();                            // these steps are staged, the last ones done with
      if (more) {
#pragma unroll
        for (int u = 0; u < kSteps; ++u)
          stage_tall<E, QF, D>(a, lane, wave, k.end, raw[u], sh, buf ^ 1, u);
      }
      Pages now[kSteps];
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        now[u] = pages[u];
        pages[u] = next_pages[u];
        next_pages[u] = check(ahead[u]);
        load_tall<SF, D>(a, seg.h, lane, wave, (far ? tok + 2 * kKeys : tok) + u * kStep,
                         far ? next_pages[u] : now[u], raw[u]);
      }
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        f32x4 x[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int t = 0; t < 2; ++t) x[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const u32x4 k0 = sh.k[buf][u][i][lane], k1 = sh.k[buf][u][D / 32 + i][lane];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            x[r][0] = mfma<E>(k0, q[r][i], x[r][0]);
            x[r][1] = mfma<E>(k1, q[r][i], x[r][1]);
          }
        }
        float ks[8], vs[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ks[i] = sh.ks[buf][u][16 * (i / 4) + 4 * g + i % 4];
          vs[i] = sh.vs[buf][u][16 * (i / 4) + 4 * g + i % 4];
        }
        u32x4 p[R];
        Kept kept;
        softmax<E, D, R, TREE>(lane, tok + u * kStep, all, now[u], x, ks, vs, tree, s, p, kept);
        if (u == kSteps - 1) {
#pragma unroll
          for (int w = 0; w < kSteps; ++w) ahead[w] = entries(tok + 3 * kKeys + w * kStep);
        }
        // Two loops: with a branch in one, 32 x 32 drafts over 8192 tokens take 385 us, so 364.
        if (TREE && tok + (u + 1) * kStep > all) {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const u32x4 v = sh.v[buf][u][j][lane] & kept.bits;
#pragma unroll
            for (int r = 0; r < R; ++r) s.o[r][j] = mfma<ET_F16>(v, p[r], s.o[r][j]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const u32x4 v = sh.v[buf][u][j][lane];
#pragma unroll
            for (int r = 0; r < R; ++r) s.o[r][j] = mfma<ET_F16>(v, p[r], s.o[r][j]);
          }
        }
      }
      if (!more) break;
      tok += kKeys;
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float l = cross_sum(s.l[r]);
    const int i = first_row + 16 * r + c;
    if (i >= rows) continue;
    const Row w = row_of(i);
    const int64_t row = ((int64_t)w.b * a.S + w.s) * a.Hq + w.hq;
    const bool whole = seg.to == kOut;
    const int64_t at = whole ? 0 : row * a.row_parts + seg.row_part;
    const float f = whole ? (l > 0.0f ? 1.0f / l : 0.0f) : 1.0f;
#pragma unroll
    for (int hh = 0; hh < D / 64; ++hh) {       // dims 64 hh + 16 g + 4 r + i
      const int d = 64 * hh + 16 * g;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4 o = {s.o[r][4 * hh][e] * f, s.o[r][4 * hh + 1][e] * f,
                         s.o[r][4 * hh + 2][e] * f, s.o[r][4 * hh + 3][e] * f};
        if (whole)
          *reinterpret_cast<u32x2*>(a.out + row * D + d + 4 * e) =
              u32x2{pack16<E>(o[0], o[1]), pack16<E>(o[2], o[3])};
        else
          *reinterpret_cast<f32x4*>(a.part + at * D + d + 4 * e) = o;
      }
    }
    if (!whole && g == 0) {
      a.part_ml[2 * at] = s.m[r];
      a.part_ml[2 * at + 1] = l;
    }
  }
}

// One chunk of the prefix or (static) of a sequence's own keys.  `item`: workgroup number within
// its kind.
template <int E, int QF, int SF, int D, int R, bool PREFIX, bool TALL, bool TREE>
__device__ __forceinline__ void run_chunk(const Args& a, int item, char* lds) {
  const int chunks = PREFIX ? a.prefix_chunks : a.chunks;
  const Place place = PREFIX ? place_of(item, a.prefix_items, a.prefix_tiles)
                             : place_of(item, a.items, a.tiles);
  Segment s;
  s.tile = place.tile;
  const int chunk = place.group % chunks;
  s.h = place.group / chunks % a.H;
  s.b = place.group / chunks / a.H;
  s.len = 0;
  s.row_part = PREFIX ? chunk : a.prefix_chunks + chunk;
  s.to = a.row_parts > 1 ? kRowParts : kOut;
  if constexpr (PREFIX) {
    s.keys.pages = a.prefix;
    s.keys.width = ((a.prefix_len - 1) >> a.page_shift) + 1;
    s.keys.begin = chunk * a.prefix_chunk;
    s.keys.end = s.keys.begin + a.prefix_chunk < a.prefix_len ? s.keys.begin + a.prefix_chunk
                                                              : a.prefix_len;
  } else {
    s.len = own_length(a.lens, a.idx64, a.most, s.b);
    s.keys.pages = a.table + (int64_t)s.b * a.width;
    s.keys.width = a.width;
    s.keys.begin = chunk * a.chunk;
    s.keys.end = s.keys.begin + a.chunk < s.len ? s.keys.begin + a.chunk : s.len;
    // The joining kernel reads as many chunks as the length has.  The first one is always
    // written, for rows without keys.
    if (s.keys.begin >= s.len && chunk > 0) return;
  }
  if constexpr (TALL)
    run_tall<E, QF, SF, D, PREFIX, TREE>(a, s, *reinterpret_cast<typename Tall<D>::Lds*>(lds));
  else
    run_segment<E, QF, SF, D, R, PREFIX, false, TREE>(a, s, *reinterpret_cast<Shared<D, R>*>(lds));
}

// LDS of the schedule.
struct Schedule {
  int32_t sum[kWaves], most[kWaves];
  int32_t b, first;
};

// A workgroup's share of all units' rounds in a row (sequence, then head): [lo, hi), and the
// sequence of round lo with its first round.
struct Share {
  int32_t lo, hi, b, first;
};

// q rounds for each workgroup.  Few rounds for each leave many parts for each row to join: a part
// costs as much as kPartCost keys, so n rounds are best cut into parts of sqrt(n kPartCost / kRound).
__device__ __forceinline__ int32_t rounds_each(int32_t total, int32_t most, int32_t slots) {
  const int32_t q = (total + slots - 1) / slots;
  const int32_t least = (int32_t)(__builtin_sqrtf((float)most * (kPartCost / kRound)) + 0.5f);
  return q > least ? q : least > 1 ? least : 1;
}
__device__ __forceinline__ void cut_out(int wg, int32_t q, int32_t total, Share& s) {
  const int64_t lo = (int64_t)wg * q;
  s.lo = lo < total ? (int32_t)lo : total;
  s.hi = total - s.lo > q ? s.lo + q : total;
}
__device__ __forceinline__ int32_t scan64(int32_t v, int lane) {     // inclusive
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int32_t o = __shfl_up(v, d);
    v += lane >= d ? o : 0;
  }
  return v;
}
__device__ __forceinline__ int32_t max64(int32_t v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int32_t o = __shfl_xor(v, d);
    v = o > v ? o : v;
  }
  return v;
}

// Up to 64 sequences, one for each lane: every wave by itself.
__device__ __forceinline__ Share share_of_few(const Args& a, int wg, int32_t len) {
  const int lane = threadIdx.x & 63;
  const int32_t n = lane < a.B ? rounds_of(len) * a.H : 0;
  const int32_t upto = scan64(n, lane), first = upto - n;
  const int32_t total = __builtin_amdgcn_readlane(upto, 63);
  const int32_t q = rounds_each(total, max64(n) / a.H, a.slots);
  Share s;
  cut_out(wg, q, total, s);
  const uint64_t here = __ballot(s.lo >= first && s.lo < upto);
  s.b = here ? (int)__builtin_ctzll(here) : 0;
  s.first = __builtin_amdgcn_readlane(first, s.b);
  if (wg == 0 && threadIdx.x < 64) {
    if (lane < a.B) a.sched[lane] = first;
    if (lane == 0) a.sched[a.B] = q;
  }
  return s;
}

// Any number of sequences: the workgroup's threads together, twice over the lengths.
__device__ __forceinline__ Share share_of_many(const Args& a, int wg, Schedule& sc) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t sum = 0, most = 0;
  for (int b = tid; b < a.B; b += 64 * kWaves) {
    const int32_t n = rounds_of(own_length(a.lens, a.idx64, a.most, b));
    sum += n;
    most = n > most ? n : most;
  }
  sum = scan64(sum, lane);
  most = max64(most);
  if (lane == 63) {
    sc.sum[wave] = sum;
    sc.most[wave] = most;
  }
  if (tid == 0) {
    sc.b = 0;
    sc.first = 0;
  }
  __syncthreads();
  int32_t total = 0;
  most = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    total += sc.sum[w];
    most = sc.most[w] > most ? sc.most[w] : most;
  }
  total *= a.H;
  const int32_t q = rounds_each(total, most, a.slots);
  Share s;
  cut_out(wg, q, total, s);
  // The sequence that holds round lo; workgroup 0 writes all sequences' first rounds down.
  int32_t base = 0;
  for (int b0 = 0; b0 < a.B && (wg == 0 || base <= s.lo); b0 += 64 * kWaves) {
    const int b = b0 + tid;
    const int32_t n = b < a.B ? rounds_of(own_length(a.lens, a.idx64, a.most, b)) * a.H : 0;
    const int32_t upto = scan64(n, lane);
    __syncthreads();                            // the sums of before have been read
    if (lane == 63) sc.sum[wave] = upto;
    __syncthreads();
    int32_t first = base + upto - n;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      first += w < wave ? sc.sum[w] : 0;
      base += sc.sum[w];
    }
    if (b < a.B) {
      if (wg == 0) a.sched[b] = first;
      if (s.lo >= first && s.lo < first + n) {
        sc.b = b;
        sc.first = first;
      }
    }
  }
  if (wg == 0 && tid == 0) a.sched[a.B] = q;
  __syncthreads();
  s.b = __builtin_amdgcn_readfirstlane(sc.b);
  s.first = __builtin_amdgcn_readfirstlane(sc.first);
  return s;
}

template <int E, int QF, int SF, int D, bool ONCE>
__device__ __forceinline__ void run_share(const Args& a, int wg, Shared<D, 1>& sh, Schedule& sc) {
  const int lane = threadIdx.x & 63;
  const bool few = a.B <= 64;
  const int32_t lens = few ? own_length(a.lens, a.idx64, a.most, lane < a.B ? lane : 0) : 0;
  const Share share = few ? share_of_few(a, wg, lens) : share_of_many(a, wg, sc);
  const int32_t lo = share.lo, hi = share.hi;
  int b = share.b;
  int32_t first = share.first;
  for (int32_t pos = lo; pos < hi;) {
    Segment s;
    s.b = b;
    s.tile = 0;
    s.len = few ? __builtin_amdgcn_readlane(lens, b)
                : __builtin_amdgcn_readfirstlane(own_length(a.lens, a.idx64, a.most, b));
    const int32_t n = rounds_of(s.len);
    s.h = (pos - first) / n;
    const int32_t r0 = pos - first - s.h * n;
    const int32_t r1 = n - r0 < hi - pos ? n : r0 + (hi - pos);
    s.keys.pages = a.table + (int64_t)b * a.width;
    s.keys.width = a.width;
    s.keys.begin = r0 * kRound;
    s.keys.end = r1 == n ? s.len : r1 * kRound;
    s.row_part = a.prefix_chunks;
    s.to = r0 > 0 || r1 < n
               ? segment_at((int64_t)a.B * a.S * a.Hq * a.row_parts, wg, r0 > 0 ? 0 : 1)
           : a.prefix_len > 0 ? kRowParts
                              : kOut;
    if (pos > lo) __syncthreads();              // the last segment's LDS has been read
    run_segment<E, QF, SF, D, 1, false, ONCE, false>(a, s, sh);
    pos += r1 - r0;
    if (r1 == n && s.h == a.H - 1) {
      first += n * a.H;
      ++b;
    }
  }
}

// R: row tiles of a unit of the sequences' own keys, RP: of the prefix (0: there is none); kTall:
// tall units.
constexpr int kTall = 8;
template <int D, int R>
constexpr int lds_of() {
  if constexpr (R == 0) return 0;
  else if constexpr (R == kTall) return sizeof(typename Tall<D>::Lds);
  else return sizeof(Shared<D, R>);
}

template <int E, int QF, int SF, int D, int R, int RP, int FORM, bool TREE>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_attention(Args a) {
  constexpr int kLds = lds_of<D, R>() > lds_of<D, RP>() ? lds_of<D, R>() : lds_of<D, RP>();
  __shared__ __align__(16) char lds[kLds];
  const int item = (int)blockIdx.x;
  if constexpr (RP > 0) {
    if (item < a.prefix_items) {
      run_chunk<E, QF, SF, D, RP == kTall ? 1 : RP, true, RP == kTall, false>(a, item, lds);
      return;
    }
  }
  if constexpr (FORM == kStatic) {
    run_chunk<E, QF, SF, D, R == kTall ? 1 : R, false, R == kTall, TREE>(a, item - a.prefix_items, lds);
  } else {
    __shared__ Schedule sc;
    static_assert(R == 1 && !TREE, "units of 16 rows, no trees");
    run_share<E, QF, SF, D, FORM == kScheduledOnce>(
        a, item - a.prefix_items, *reinterpret_cast<Shared<D, 1>*>(lds), sc);
  }
}

// Kernels for an element type (ET_BF16, ET_F16), code format (QF_FP8, QF_I8_RNE) and scale format:
// lookup_e<E>_q<QF>_s<SF>, one for each instantiation unit.  tree: of drafted trees, static.
const void* lookup_e0_q0_s0(int D, int R, int RP, int form, bool tree);
const void* lookup_e0_q0_s1(int D, int R, int RP, int form, bool tree);
const void* lookup_e0_q1_s0(int D, int R, int RP, int form, bool tree);
const void* lookup_e0_q1_s1(int D, int R, int RP, int form, bool tree);
const void* lookup_e1_q0_s0(int D, int R, int RP, int form, bool tree);
const void* lookup_e1_q0_s1(int D, int R, int RP, int form, bool tree);
const void* lookup_e1_q1_s0(int D, int R, int RP, int form, bool tree);
const void* lookup_e1_q1_s1(int D, int R, int RP, int form, bool tree);

}  // namespace attn
}  // namespace fagq
