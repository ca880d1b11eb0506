// prompt_attn_bwd.hip - gradients of the causal attention of packed prompts (include/fagq_prompt.h).
//
// Two passes over the pairs of query and key, so that every sum has one owner and one order (no
// atomics): seven products for the five of the formulas.
//   prompt_dq     A workgroup takes 128 queries of one head, keys and values come through LDS.
//                 S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T.  It also leaves what the other
//                 pass needs of each query: lse in units of log 2, and -delta.  Where there are
//                 few workgroups, the keys are cut into parts of their own sums.
//   prompt_dkdv   A workgroup takes 128 keys of one head of k and v, the queries of all heads of
//                 the group come through LDS.  S = Q K^T, dP = dO V^T, dV^T += dO^T P,
//                 dK^T += Q^T dS.  Two teams of four waves share the steps of a tile and join
//                 their sums through LDS; where there are few workgroups, the steps are cut into
//                 parts besides.
//   prompt_join   adds the parts up, in order.
// 8192 tokens, 32 + 8 heads of 128, in 1.87 ms: dq 860 us, bound by power (the matrix units busy 73 % of
// the cycles at 1.8 GHz), dk and dv 1000 (59 %): what is between their products are LDS reads, the
// exponentials and the steps' barriers.  dS enters dq's product in two terms of 16 bits, without which dq
// would be 1.7 times as far off as its own rounding makes it.
// Calls of few rows, where a launch is what counts, take both passes in one (prompt_bwd_small): the
// second then works out lse and delta of its queries by itself.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "fagq.h"
#include "fagq_dispatch.hpp"
#include "fagq_prompt.h"
#include "prompt_attn.hpp"

namespace fagq {
namespace prompt {
namespace {

struct Args {
  const uint16_t* dout;
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* out;
  const float* lse;
  Sequences queries, keys;           // tiles of queries, of keys
  uint16_t* dq;
  uint16_t* dk;
  uint16_t* dv;
  float* lse2;                       // [Hq, T]; +inf for a query without keys.  Null: small calls
  float* delta;                      // [Hq, T], negative
  float* part;                       // [parts][Tk][H][D] of dk, then of dv
  float* dq_part;                    // [dq_parts][T][Hq][D]
  int64_t dos[2], qs[2], ks[2], vs[2], dqs[2], dks[2], dvs[2];   // {token, head} strides, elements
  int32_t Hq, H, group, fill, parts, dq_parts;
  int32_t dq_items;                  // small calls: workgroups of the first pass
  int32_t first;                     // of the second pass in this launch
  float scale, scale2;               // sm_scale, and times log2(e)
};

template <int D>
__device__ __forceinline__ void fill_tail(uint16_t* out, const int64_t (&s)[2], int head, int32_t rows,
                                          const Place& p) {
  const int64_t first = (int64_t)p.end + (int64_t)p.tile * kTile;
  for (int i = threadIdx.x; i < kTile * (D / 8); i += 64 * kWaves) {
    const int64_t row = first + i / (D / 8);
    if (row >= rows) break;
    *reinterpret_cast<u32x4*>(out + row * s[0] + (int64_t)head * s[1] + i % (D / 8) * 8) = u32x4{0, 0, 0, 0};
  }
}

// An lse in units of log 2, as the exponentials take it.
__device__ __forceinline__ float lse_in_2(float lse) { return lse == -INFINITY ? INFINITY : lse * kLog2e; }

// fp16 has neither the range nor the small values for dS, whose size is that of dout, nor for the weights
// of long sequences: dS goes into its product times a power of two (Scaled), P for dv times 2^kShift,
// which the dq pass takes off the lse2 that it leaves (P is at most 1 and a rounding of the exponent, so
// 2^14 keeps a factor of four to infinity, and weights above 2^-28 keep all their bits).
template <int E>
constexpr float kShift = E == ET_F16 ? 14.0f : 0.0f;

// What a lane's column of dS is multiplied by before it is packed: as much as leaves its largest element
// below 2^15.  It falls as that element rises, to put it in 2^8 to 2^9, as a softmax's running maximum does,
// and the column's sums with it: elements above 2^-22 of the largest keep all their bits.  A power of two,
// so nothing is rounded.  bf16 has fp32's range, and none of this.  (fp16, us, with / without: 4096 tokens,
// 32 + 8 heads of 64 327 / 304, of 128 565 / 532, 16 + 4 of 256 684 / 654; 100 tokens, 16 + 4 of 256 51 / 44.)
struct Scaled {
  float f = 0x1p60f;
  __device__ __forceinline__ float inverse() const {
    return __uint_as_float((2u * 127u << 23) - __float_as_uint(f));
  }
  // Multiplies a column's elements, half of which are in each of two lanes.  Whether the sums of some
  // column are to be multiplied too, and by what in this lane.
  __device__ __forceinline__ bool operator()(f32x16& x, float* change) {
    float top = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(x[r]));
    top *= f;
    const bool falls = __any(top > 0x1p15f);
    if (falls) {
      top = cross_max(top);
      const uint32_t exponent = __float_as_uint(top) >> 23;         // top is 2^(exponent - 127) and up
      *change = top > 0x1p15f ? __uint_as_float((2 * 127 + 8 - exponent) << 23) : 1.0f;
      f *= *change;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] *= f;
    return falls;
  }
};
// Sums times f.
template <int N>
__device__ __forceinline__ void rescale(f32x16 (&sum)[N], float f) {
#pragma unroll
  for (int d = 0; d < N; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[d][r] *= f;
}
// 16 of them by way of LDS, for sums in the accumulation half of the register file: multiplied in place they
// cost dk and dv of heads of 256 134 spilled registers (fp16, 4096 tokens, 16 + 4 heads: 1512 us in all).
using Room = f32x4[4][64];           // of a wave
__device__ __forceinline__ void rescale_through(Room& room, int lane, f32x16& x, float f) {
#pragma unroll
  for (int r = 0; r < 4; ++r) room[r][lane] = f32x4{x[4 * r], x[4 * r + 1], x[4 * r + 2], x[4 * r + 3]};
  asm volatile("" ::: "memory");
#pragma unroll
  for (int r = 0; r < 4; ++r) room[r][lane] *= f;
  asm volatile("" ::: "memory");
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const f32x4 v = room[r][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * r + e] = v[e];
  }
  asm volatile("" ::: "memory");
}

template <int D>
struct DqLds {
  char tile[2][2][Tile<D>::kBytes];
};

template <int E, int D>
__device__ __forceinline__ void run_dq(const Args& a, int item, DqLds<D>& shared) {
  auto& lds = shared.tile;
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int wave = scalar((int)(threadIdx.x >> 6));
  // Workgroup b runs on XCD b % 8: heads that share keys stay on one.
  const int kvh = item % a.H, heads = item / a.H;
  const int hq = kvh * a.group + heads % a.group, rest = heads / a.group, part = rest % a.dq_parts;
  const Place p = place_of<true>(a.queries, rest / a.dq_parts);
  if (p.b < 0) {
    if (part == 0 && (a.fill & FAGQ_FILL_DQ)) fill_tail<D>(a.dq, a.dqs, hq, a.queries.T, p);
    return;
  }
  const int32_t ahead = p.m - p.n;               // query i sees the keys up to i + ahead
  const int32_t q0 = p.tile * kTile, mine = q0 + wave * kRows;
  const int32_t i = mine + c, row = p.row + (i < p.n ? i : p.n - 1);
  auto seen_by = [&](int32_t query) {
    const int32_t n = query + ahead + 1;
    return n < 0 ? 0 : n < p.m ? n : p.m;
  };
  const int32_t seen = i < p.n ? seen_by(i) : 0;
  const int32_t all = seen_by(mine);             // keys that every query of the wave sees
  const int32_t last = mine + kRows <= p.n ? mine + kRows - 1 : p.n - 1;
  const int32_t end = mine < p.n ? seen_by(last) : 0;                    // that one of them sees
  // Steps of the workgroup, this part's share of them.
  const int32_t steps = (seen_by(q0 + kTile <= p.n ? q0 + kTile - 1 : p.n - 1) + kStep - 1) / kStep;
  const int32_t from = (int32_t)((int64_t)steps * part / a.dq_parts) * kStep;
  const int32_t stop = (int32_t)((int64_t)steps * (part + 1) / a.dq_parts) * kStep;

  Copier<D> ck, cv;
  ck.init(a.k, (int64_t)p.other * a.ks[0] + (int64_t)kvh * a.ks[1], a.ks[0], lane, wave);
  cv.init(a.v, (int64_t)p.other * a.vs[0] + (int64_t)kvh * a.vs[1], a.vs[0], lane, wave);
  if (from < stop) {
    ck.issue(lds[0][0], wave, from, p.m - 1);
    cv.issue(lds[0][1], wave, from, p.m - 1);
  }
  u32x4 q[D / 16], g[D / 16];
  load_row<D>(a.q + (int64_t)row * a.qs[0] + (int64_t)hq * a.qs[1], h, q);
  load_row<D>(a.dout + (int64_t)row * a.dos[0] + (int64_t)hq * a.dos[1], h, g);
  float delta = 0.0f;
  {
    u32x4 out[D / 16];
    load_row<D>(a.out + ((int64_t)row * a.Hq + hq) * D, h, out);
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        delta = __builtin_fmaf(-lo16<E>(g[j][e]), lo16<E>(out[j][e]), delta);
        delta = __builtin_fmaf(-hi16<E>(g[j][e]), hi16<E>(out[j][e]), delta);
      }
  }
  delta = cross_sum(delta);
  const float lse = a.lse[(int64_t)hq * a.queries.T + row];
  const float lse2 = lse_in_2(lse);
  if (a.lse2 && part == 0 && h == 0 && i < p.n) {
    a.lse2[(int64_t)hq * a.queries.T + row] = lse2 - kShift<E>;
    a.delta[(int64_t)hq * a.queries.T + row] = delta;
  }
  f32x16 dq[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d) dq[d] = splat(0.0f);
  Scaled scaled;

  int buf = 0;
  for (int32_t tok = from; tok < stop; tok += kStep, buf ^= 1) {
    __builtin_amdgcn_s_waitcnt(kVmcnt0);         // this step's tiles have landed, of this wave
    lds_barrier();                               // of all; the last step's are done with
    if (tok + kStep < stop) {
      ck.issue(lds[buf ^ 1][0], wave, tok + kStep, p.m - 1);
      cv.issue(lds[buf ^ 1][1], wave, tok + kStep, p.m - 1);
    }
    if (tok >= end) continue;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x16 x = splat(0.0f), y = splat(delta);
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        x = mfma<E>(row_frag<D>(lds[buf][0], lane, t, j), q[j], x);
        y = mfma<E>(row_frag<D>(lds[buf][1], lane, t, j), g[j], y);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r)
        x[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], a.scale2, -lse2));
      if (tok + kStep > all) {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = tok + 32 * t + row_of(r, h) < seen ? x[r] : 0.0f;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] *= y[r];
      if constexpr (E == ET_F16)
        if (float f; scaled(x, &f)) rescale(dq, f);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const u32x4 w = pack8<E>(x, u), rest = pack_rest8<E>(x, u, w);
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
          const u32x4 k = col_frag<D>(lds[buf][0], lane, d, 2 * t + u);
          dq[d] = mfma<E>(k, w, dq[d]);
          dq[d] = mfma<E>(k, rest, dq[d]);
        }
      }
    }
  }
  if constexpr (E == ET_F16) rescale(dq, scaled.inverse());
  if (a.dq_parts == 1) {
    store_row<E, D>(a.dq + (int64_t)row * a.dqs[0] + (int64_t)hq * a.dqs[1], h, dq, a.scale, i < p.n);
  } else if (i < p.n) {
    float* to = a.dq_part + (((int64_t)part * a.queries.T + row) * a.Hq + hq) * D;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<f32x4*>(to + 32 * d + row_of(r, h)) =
            f32x4{dq[d][r], dq[d][r + 1], dq[d][r + 2], dq[d][r + 3]};
  }
}

template <int E, int D>
__global__ __launch_bounds__(64 * kWaves, 2) void prompt_dq(Args a) {
  __shared__ __align__(16) DqLds<D> lds;
  run_dq<E, D>(a, (int)blockIdx.x, lds);
}

// Teams of four waves in a workgroup, which share its steps and join their sums through LDS.
constexpr int teams(int64_t D, bool small) { return D == 256 || small ? 1 : 2; }
constexpr int queries(int64_t D) { return D == 128 ? 32 : 64; }   // of a team in LDS at a time

template <int D, bool SMALL>
struct DkdvLds {
  static constexpr bool kInLds = D <= 128;                // k and v; else in registers
  char tile[teams(D, SMALL)][2][2][Tile<D, queries(D)>::kBytes];
  char kv[2][kInLds ? Tile<D, kTile>::kBytes : 16];
  float stats[teams(D, SMALL)][2][2][queries(D)];         // lse2, -delta
  char room[kInLds ? 16 : kWaves * sizeof(Room)];         // of rescale_through
};

// SMALL: one team, lse2 and delta worked out here, and two terms (of 16 bits each) of P and dS, as dq
// always has.  One leaves dk and dv 1.4 times the error that their own rounding makes, as long as
// there are many roundings to average over, and takes a quarter of the products less.
template <int E, int D, bool SMALL>
__device__ __forceinline__ void run_dkdv(const Args& a, int item, DkdvLds<D, SMALL>& shared) {
  constexpr int kQueries = queries(D), kTeams = teams(D, SMALL);
  using L = Tile<D, kQueries>;
  using KV = Tile<D, kTile>;
  constexpr bool kInLds = DkdvLds<D, SMALL>::kInLds;
  auto& lds_kv = shared.kv;
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int waves = scalar((int)(threadIdx.x >> 6)), wave = waves % kWaves, team = waves / kWaves;
  auto& lds = shared.tile[team];
  auto& stats = shared.stats[team];
  const int kvh = item % a.H, rest = item / a.H;
  const int part = rest % a.parts;
  const Place p = place_of<false>(a.keys, rest / a.parts);
  if (p.b < 0) {
    if (part == 0 && (a.fill & FAGQ_FILL_DK)) fill_tail<D>(a.dk, a.dks, kvh, a.keys.T, p);
    if (part == 0 && (a.fill & FAGQ_FILL_DV)) fill_tail<D>(a.dv, a.dvs, kvh, a.keys.T, p);
    return;
  }
  // n keys, m queries; query i sees the keys up to i + ahead.
  const int32_t ahead = p.n - p.m, k0 = p.tile * kTile, mine = k0 + wave * kRows;
  const int32_t j0 = mine + c;
  const int32_t first = k0 > ahead ? k0 - ahead : 0;       // query that sees one of the tile's keys
  const int32_t steps = first < p.m ? (p.m - first + kQueries - 1) / kQueries : 0;
  // Steps of all heads in a row, head by head: this part's share, and its longest team's number.
  const int64_t total = (int64_t)steps * a.group;
  const int32_t shares = a.parts * kTeams, share = part * kTeams + team;
  const int32_t from = (int32_t)(total * share / shares), to = (int32_t)(total * (share + 1) / shares);
  const int32_t rounds = (int32_t)((total + shares - 1) / shares);

  Copier<D, kQueries> cq, cg;
  cq.init(a.q, (int64_t)p.other * a.qs[0] + (int64_t)kvh * a.group * a.qs[1], a.qs[0], lane, wave);
  cg.init(a.dout, (int64_t)p.other * a.dos[0] + (int64_t)kvh * a.group * a.dos[1], a.dos[0], lane, wave);
  int32_t head = steps > 0 ? from / steps : 0, step = from - head * steps;   // of the next copies
  auto issue = [&](int buf, int32_t head, int32_t step) {
    const int32_t i0 = first + step * kQueries;
    Copier<D, kQueries> x = cq, y = cg;
    x.base += (int64_t)head * a.qs[1] * 2;
    y.base += (int64_t)head * a.dos[1] * 2;
    x.issue(lds[buf][0], wave, i0, p.m - 1);
    y.issue(lds[buf][1], wave, i0, p.m - 1);
    if (!SMALL && wave < 2 && lane < kQueries) {
      const int64_t at = (int64_t)(kvh * a.group + head) * a.keys.Tother + p.other + i0;
      const int32_t most = p.m - 1 - i0;
      copy4(buffer_at((wave == 0 ? a.lse2 : a.delta) + at),
            reinterpret_cast<char*>(wave == 0 ? stats[buf][0] : stats[buf][1]),
            (uint32_t)(lane < most ? lane : most) * 4u);
    }
  };
  // SMALL: dout, out and lse of the step under way; kThreads have a row.
  constexpr int kThreads = 64 * kWaves / kQueries, kOwn = SMALL ? D / kThreads / 8 : 1;
  const int own_row = (int)threadIdx.x / kThreads, own_at = (int)threadIdx.x % kThreads * (D / kThreads);
  u32x4 own_g[kOwn], own_o[kOwn];
  float own_lse = 0.0f;
  auto load_stats = [&](int32_t head, int32_t step) {
    const int32_t i = first + step * kQueries + own_row;
    const int64_t row = p.other + (i < p.m ? i : p.m - 1);
    const int hq = kvh * a.group + head;
    const uint16_t* g = a.dout + row * a.dos[0] + (int64_t)hq * a.dos[1] + own_at;
    const uint16_t* o = a.out + (row * a.Hq + hq) * D + own_at;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      own_g[i] = *reinterpret_cast<const u32x4*>(g + 8 * i);
      own_o[i] = *reinterpret_cast<const u32x4*>(o + 8 * i);
    }
    own_lse = a.lse[(int64_t)hq * a.keys.Tother + row];
  };
  auto store_stats = [&](int buf) {
    float delta = 0.0f;
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        delta = __builtin_fmaf(-lo16<E>(own_g[i][e]), lo16<E>(own_o[i][e]), delta);
        delta = __builtin_fmaf(-hi16<E>(own_g[i][e]), hi16<E>(own_o[i][e]), delta);
      }
#pragma unroll
    for (int d = 1; d < kThreads; d *= 2) delta += __shfl_xor(delta, d);
    if (own_at == 0) {
      stats[buf][0][own_row] = lse_in_2(own_lse) - kShift<E>;
      stats[buf][1][own_row] = delta;
    }
  };
  u32x4 k[kInLds ? 1 : D / 16], v[kInLds ? 1 : D / 16];
  if constexpr (!kInLds) {
    const int64_t row = p.row + (j0 < p.n ? j0 : p.n - 1);
    load_row<D>(a.k + row * a.ks[0] + (int64_t)kvh * a.ks[1], h, k);
    load_row<D>(a.v + row * a.vs[0] + (int64_t)kvh * a.vs[1], h, v);
  }
  if (kInLds && team == 0) {
    Copier<D, kTile> cv;
    cv.init(a.v, (int64_t)p.row * a.vs[0] + (int64_t)kvh * a.vs[1], a.vs[0], lane, wave);
    cv.issue(lds_kv[1], wave, k0, p.n - 1);
    cv.init(a.k, (int64_t)p.row * a.ks[0] + (int64_t)kvh * a.ks[1], a.ks[0], lane, wave);
    cv.issue(lds_kv[0], wave, k0, p.n - 1);
  }
  int32_t i0 = first + step * kQueries;          // of the step that is worked on
  if (from < to) {
    issue(0, head, step);
    if constexpr (SMALL) {
      load_stats(head, step);
      store_stats(0);
    }
  }
  const char* tk = lds_kv[0] + wave * kRows * KV::kRowBytes;
  const char* tv = lds_kv[1] + wave * kRows * KV::kRowBytes;
  f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d) dk[d] = dv[d] = splat(0.0f);
  Scaled scaled;

  int buf = 0;
  for (int32_t round = 0; round < rounds; ++round, buf ^= 1, i0 += kQueries) {
    const int32_t it = from + round;
    if (i0 >= p.m) i0 = first;
    __builtin_amdgcn_s_waitcnt(kVmcnt0);         // this step's tiles have landed, of this wave
    lds_barrier();                               // of all; the last step's are done with
    if (++step == steps) step = 0, ++head;
    if (it + 1 < to) {
      issue(buf ^ 1, head, step);
      if constexpr (SMALL && kInLds) load_stats(head, step);
    }
#pragma unroll 1
    for (int t = 0; t < kQueries / 32; ++t) {
      const int32_t query = i0 + 32 * t;
      if (mine >= p.n || it >= to || query >= p.m || query + 31 + ahead < mine) continue;
      const char* tq = lds[buf][0] + t * 32 * L::kRowBytes;
      const char* tg = lds[buf][1] + t * 32 * L::kRowBytes;
      f32x16 x = splat(0.0f), y;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        if constexpr (kInLds) x = mfma<E>(row_frag<D>(tq, lane, 0, j), row_frag<D>(tk, lane, 0, j), x);
        else x = mfma<E>(row_frag<D>(tq, lane, 0, j), k[j], x);
      }
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const f32x4 s = *reinterpret_cast<const f32x4*>(&stats[buf][1][32 * t + row_of(r, h)]);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[r + e] = s[e];
      }
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        if constexpr (kInLds) y = mfma<E>(row_frag<D>(tg, lane, 0, j), row_frag<D>(tv, lane, 0, j), y);
        else y = mfma<E>(row_frag<D>(tg, lane, 0, j), v[j], y);
      }
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const f32x4 s = *reinterpret_cast<const f32x4*>(&stats[buf][0][32 * t + row_of(r, h)]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[r + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r + e], a.scale2, -s[e]));
      }
      if constexpr (kInLds) read_ahead<8, 2, D / 8>();
      if (query + 32 > p.m || query + ahead < mine + kRows - 1) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int32_t i = query + row_of(r, h);
          x[r] = i < p.m && j0 <= i + ahead ? x[r] : 0.0f;
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const u32x4 w = pack8<E>(x, u);
        u32x4 rest;
        if constexpr (SMALL) rest = pack_rest8<E>(x, u, w);
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
          const u32x4 g = col_frag<D>(tg, lane, d, u);
          dv[d] = mfma<E>(g, w, dv[d]);
          if constexpr (SMALL) dv[d] = mfma<E>(g, rest, dv[d]);
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] *= y[r];
      if constexpr (E == ET_F16) {
        if (float f; scaled(x, &f)) {
          if constexpr (kInLds) {
            rescale(dk, f);
          } else {
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
              rescale_through(reinterpret_cast<Room*>(shared.room)[wave], lane, dk[d], f);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const u32x4 w = pack8<E>(x, u);
        u32x4 rest;
        if constexpr (SMALL) rest = pack_rest8<E>(x, u, w);
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
          const u32x4 q = col_frag<D>(tq, lane, d, u);
          dk[d] = mfma<E>(q, w, dk[d]);
          if constexpr (SMALL) dk[d] = mfma<E>(q, rest, dk[d]);
        }
      }
      if constexpr (kInLds) read_ahead<8, 2, D / 8>();
    }
    if (SMALL && it + 1 < to) {
      if constexpr (SMALL && !kInLds) load_stats(head, step);   // no registers to hold them that long
      store_stats(buf ^ 1);
    }
  }
  float fk = 1.0f, fv = 1.0f;                    // what the sums still have to be multiplied by
  if constexpr (E == ET_F16) {
    fv = 0x1p-14f, fk = fv * scaled.inverse();
    if constexpr (kTeams > 1) {
      rescale(dk, fk);
      rescale(dv, fv);
      fk = fv = 1.0f;
    }
  }
  if constexpr (kTeams > 1) {
    // The second team hands its sums over, dk's, then dv's.
    f32x4* sums = reinterpret_cast<f32x4*>(shared.tile);
    static_assert(sizeof(shared.tile) >= kWaves * D / 32 * 4 * 64 * sizeof(f32x4), "room for one of them");
    auto hand = [&](f32x16 (&x)[D / 32]) {
      __syncthreads();
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          f32x4& at = sums[((wave * (D / 32) + d) * 4 + r) * 64 + lane];
          if (team) at = f32x4{x[d][4 * r], x[d][4 * r + 1], x[d][4 * r + 2], x[d][4 * r + 3]};
        }
      __syncthreads();
      if (team) return;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x4 v = sums[((wave * (D / 32) + d) * 4 + r) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[d][4 * r + e] += v[e];
        }
    };
    hand(dk);
    hand(dv);
    if (team) return;
  }
  const int64_t row = p.row + j0;
  if (a.parts == 1) {
    store_row<E, D>(a.dk + row * a.dks[0] + (int64_t)kvh * a.dks[1], h, dk, a.scale * fk, j0 < p.n);
    store_row<E, D>(a.dv + row * a.dvs[0] + (int64_t)kvh * a.dvs[1], h, dv, fv, j0 < p.n);
  } else if (j0 < p.n) {
    const int64_t plane = (int64_t)a.keys.T * a.H * D;
    float* to_k = a.part + part * plane + (row * a.H + kvh) * D;
    float* to_v = to_k + a.parts * plane;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        *reinterpret_cast<f32x4*>(to_k + 32 * d + row_of(r, h)) =
            f32x4{dk[d][r] * fk, dk[d][r + 1] * fk, dk[d][r + 2] * fk, dk[d][r + 3] * fk};
        *reinterpret_cast<f32x4*>(to_v + 32 * d + row_of(r, h)) =
            f32x4{dv[d][r] * fv, dv[d][r + 1] * fv, dv[d][r + 2] * fv, dv[d][r + 3] * fv};
      }
  }
}

template <int E, int D>
__global__ __launch_bounds__(64 * kWaves * teams(D, false), teams(D, false)) void prompt_dkdv(Args a) {
  __shared__ __align__(16) DkdvLds<D, false> lds;
  run_dkdv<E, D, false>(a, a.first + (int)blockIdx.x, lds);
}

template <int E, int D>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 1 : 2) void prompt_bwd_small(Args a) {
  __shared__ __align__(16) union {
    DqLds<D> dq;
    DkdvLds<D, true> dkdv;
  } lds;
  if ((int)blockIdx.x < a.dq_items) run_dq<E, D>(a, (int)blockIdx.x, lds.dq);
  else run_dkdv<E, D, true>(a, (int)blockIdx.x - a.dq_items, lds.dkdv);
}

// Sums of the parts.  A thread has 8 elements of dk or dv, where they have parts, or of dq.
template <int E>
__global__ __launch_bounds__(256) void prompt_join(Args a, int32_t D) {
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t keys = a.parts > 1 ? (int64_t)a.keys.T * a.H * D / 8 : 0;
  const int64_t queries = a.dq_parts > 1 ? (int64_t)a.queries.T * a.Hq * D / 8 : 0;
  if (item >= 2 * keys + queries) return;
  const bool of_q = item >= 2 * keys, values = !of_q && item >= keys;
  const Sequences& s = of_q ? a.queries : a.keys;
  const int32_t heads = of_q ? a.Hq : a.H, parts = of_q ? a.dq_parts : a.parts;
  const int64_t plane = (int64_t)s.T * heads * D;
  const int64_t at = (item - (of_q ? 2 * keys : values ? keys : 0)) * 8;
  const int64_t row = at / ((int64_t)heads * D);
  const int32_t rest = (int32_t)(at - row * heads * D), head = rest / D, d = rest - head * D;
  if (row >= clamped(s.cu[s.B], s.T)) return;
  const float* part = (of_q ? a.dq_part : values ? a.part + parts * plane : a.part) + at;
  f32x4 sum[2] = {};
  for (int i = 0; i < parts; ++i, part += plane) {
    sum[0] += *reinterpret_cast<const f32x4*>(part);
    sum[1] += *reinterpret_cast<const f32x4*>(part + 4);
  }
  const float f = values ? 1.0f : a.scale;
  const int64_t* strides = of_q ? a.dqs : values ? a.dvs : a.dks;
  uint16_t* to = (of_q ? a.dq : values ? a.dv : a.dk) + row * strides[0] + (int64_t)head * strides[1];
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack16<E>(sum[i / 2][2 * i % 4] * f, sum[i / 2][2 * i % 4 + 1] * f);
  *reinterpret_cast<u32x4*>(to + d) = w;
}

// ---------------------------------------------------------------------------------- host

constexpr int64_t kCUs = 256;        // a workgroup on each

// Calls of few rows and few pairs of query and key: both passes in one launch, with one team and two
// terms (32 + 8 heads of 128, us, in one launch / in two: 1 token 15 / 17, 200 tokens 26 / 36, 4 x 128
// 30 / 34, 4 x 200 58 / 41; 16 heads of 64, 1000 tokens 39 / 51; 8 heads of 128, 100 tokens behind 3000
// 32 / 41, 1024 behind 1024 88 / 79; 24 + 8 of 256, 5 and 70 behind 4000 200 / 177).  The more a head
// has, the fewer of the one launch's waves run at once.  Not with more tiles than a grid may hold of both
// passes, which few rows have in many empty sequences only.
bool small(int64_t B, int64_t T, int64_t Tk, int64_t Hq, int64_t D) {
  return T * Hq <= 16384 && B * Hq <= kMostGroups / 64 && (double)(T * Hq * D * D) * (double)Tk <= 0x1p36 * (double)std::max<int64_t>(1, B);
}

// Parts of a key tile's steps: as many as let the tile with most of them, twice the average, not take
// longer than all together, but four steps for each team.
int64_t parts_for(int64_t B, int64_t T, int64_t Tk, int64_t Hq, int64_t H, int64_t D) {
  const int64_t groups = std::max<int64_t>(1, (Tk + kTile - 1) / kTile * H);
  const int64_t steps = Hq / H * ((T + queries(D) - 1) / queries(D)) / std::max<int64_t>(1, B);
  return std::max<int64_t>(
      1, std::min<int64_t>({2 * kCUs / groups, steps / (4 * teams(D, small(B, T, Tk, Hq, D))), kMostParts}));
}

// Parts of a query tile's keys (us, with parts / without: 8 + 2 heads of 128, 10 tokens behind 8000
// 31 / 247; 8 heads of 64, 64 behind 1000 16 / 24; 4 of 128, 200 behind 2000 29 / 74, of 64, 4 x 300
// behind 3000 43 / 65; but 8 + 1 of 256, 2048 tokens 180 / 157).  In one launch the keys' workgroups
// run at the same time: one on a CU for heads of 128 and 256, two for those of 64.
int64_t dq_parts_for(int64_t B, int64_t T, int64_t Tk, int64_t Hq, int64_t H, int64_t D) {
  const bool one_launch = small(B, T, Tk, Hq, D);
  int64_t slots = D == 256 || (D == 128 && one_launch) ? kCUs : 2 * kCUs;
  if (one_launch) {
    const int64_t others = (Tk + kTile - 1) / kTile * H * parts_for(B, T, Tk, Hq, H, D);
    slots = std::max(slots - others, slots / 4);
  }
  return key_parts(B, T, Tk, Hq, slots);
}

int check_bwd_sizes(int64_t B, int64_t T, int64_t Tk, int64_t Hq, int64_t H, int64_t D) {
  const int st = check_sizes(B, T, Tk, Hq, H, D);
  if (st != FAGQ_OK) return st;
  // There are parts, and a joining kernel, where workgroups are few only.
  const int64_t dq_items = tile_slots(T, B) * Hq * dq_parts_for(B, T, Tk, Hq, H, D);
  const int64_t dkdv_items = tile_slots(Tk, B) * H * parts_for(B, T, Tk, Hq, H, D);
  const bool large =
      dq_items >= kMostGroups || dkdv_items + (small(B, T, Tk, Hq, D) ? dq_items : 0) >= kMostGroups;
  return large ? FAGQ_E_TOO_LARGE : FAGQ_OK;
}

struct Space {                       // elements of fp32 in the workspace
  int64_t stats, part, dq_part;
  int64_t bytes() const { return (stats + part + dq_part) * 4; }
};
Space space_for(int64_t parts, int64_t dq_parts, int64_t B, int64_t T, int64_t Tk, int64_t Hq, int64_t H,
                int64_t D) {
  return {small(B, T, Tk, Hq, D) ? 0 : (2 * Hq * T + 3) / 4 * 4, parts > 1 ? 2 * parts * Tk * H * D : 0,
          dq_parts > 1 ? dq_parts * T * Hq * D : 0};
}

template <int E>
const void* dq_for(int64_t D) {
  return D == 64    ? reinterpret_cast<const void*>(&prompt_dq<E, 64>)
         : D == 128 ? reinterpret_cast<const void*>(&prompt_dq<E, 128>)
                    : reinterpret_cast<const void*>(&prompt_dq<E, 256>);
}
template <int E>
const void* dkdv_for(int64_t D) {
  return D == 64    ? reinterpret_cast<const void*>(&prompt_dkdv<E, 64>)
         : D == 128 ? reinterpret_cast<const void*>(&prompt_dkdv<E, 128>)
                    : reinterpret_cast<const void*>(&prompt_dkdv<E, 256>);
}
template <int E>
const void* small_for(int64_t D) {
  return D == 64    ? reinterpret_cast<const void*>(&prompt_bwd_small<E, 64>)
         : D == 128 ? reinterpret_cast<const void*>(&prompt_bwd_small<E, 128>)
                    : reinterpret_cast<const void*>(&prompt_bwd_small<E, 256>);
}

}  // namespace
}  // namespace prompt
}  // namespace fagq

extern "C" {

FAGQ_API int64_t fagq_prompt_attention_bwd_workspace_bytes(int64_t B, int64_t T, int64_t Tk,
                                                           int64_t Hq, int64_t H, int64_t D) {
  using namespace fagq::prompt;
  if (check_bwd_sizes(B, T, Tk, Hq, H, D) != FAGQ_OK) return -1;
  return space_for(parts_for(B, T, Tk, Hq, H, D), dq_parts_for(B, T, Tk, Hq, H, D), B, T, Tk, Hq, H, D).bytes();
}

FAGQ_API int fagq_prompt_attention_bwd_launch(const void* dout, const void* q, const void* k,
                                              const void* v, const void* out, const float* lse,
                                              const int32_t* cu_seqlens,
                                              const int32_t* cu_seqlens_k, void* dq, void* dk,
                                              void* dv, void* workspace, int64_t workspace_bytes,
                                              const int64_t* strides, int64_t B, int64_t T,
                                              int64_t Tk, int64_t Hq, int64_t H, int64_t D,
                                              float sm_scale, int dtype, int fill, void* stream) {
  using namespace fagq;
  using namespace fagq::prompt;
  if ((T > 0 && (!dout || !q || !out || !lse || !dq)) || (Tk > 0 && (!k || !v || !dk || !dv)) ||
      !cu_seqlens || !strides)
    return FAGQ_E_NULL;
  if (dtype != FAGQ_DT_BF16 && dtype != FAGQ_DT_F16) return FAGQ_E_FORMAT;
  if (fill & ~(FAGQ_FILL_DQ | FAGQ_FILL_DK | FAGQ_FILL_DV)) return FAGQ_E_FORMAT;
  if (!std::isfinite(sm_scale)) return FAGQ_E_SHAPE;
  const int sizes = check_bwd_sizes(B, T, Tk, Hq, H, D);
  if (sizes != FAGQ_OK) return sizes;
  if (!cu_seqlens_k && T != Tk) return FAGQ_E_SHAPE;
  const int strided = check_strides(strides, 14);
  if (strided != FAGQ_OK) return strided;
  for (const void* p : {dout, q, k, v, out, (const void*)dq, (const void*)dk, (const void*)dv,
                        (const void*)workspace})
    if (!aligned(p, 16)) return FAGQ_E_ALIGN;
  if (!aligned(lse, 4) || !aligned(cu_seqlens, 4) || !aligned(cu_seqlens_k, 4)) return FAGQ_E_ALIGN;
  const int64_t parts = parts_for(B, T, Tk, Hq, H, D), dq_parts = dq_parts_for(B, T, Tk, Hq, H, D);
  const Space space = space_for(parts, dq_parts, B, T, Tk, Hq, H, D);
  const int64_t need = space.bytes();
  if (workspace_bytes < need) return FAGQ_E_SHAPE;
  if (need > 0 && !workspace) return FAGQ_E_NULL;
  if (T == 0 && Tk == 0) return FAGQ_OK;
  Rows rows[7];
  const void* const tensors[7] = {dout, q, k, v, dq, dk, dv};
  for (int i = 0; i < 7; ++i) {
    const bool kv = i == 2 || i == 3 || i > 4;
    rows[i] = {tensors[i], kv ? Tk : T, kv ? H : Hq, D, strides[2 * i], strides[2 * i + 1]};
  }
  const void* flat[5] = {out, lse, cu_seqlens, cu_seqlens_k, workspace};
  const int64_t nflat[5] = {T * Hq * D * 2, T * Hq * 4, (B + 1) * 4, cu_seqlens_k ? (B + 1) * 4 : 0, need};
  for (int i = 4; i < 7; ++i) {
    if (rows[i].T == 0) continue;
    if (self_overlap(rows[i])) return FAGQ_E_ALIAS;
    for (int j = 0; j < i; ++j)
      if (rows[j].T > 0 && overlap(rows[i], rows[j])) return FAGQ_E_ALIAS;
    for (int j = 0; j < 5; ++j)
      if (overlap(rows[i].p, rows[i].bytes(), flat[j], nflat[j])) return FAGQ_E_ALIAS;
  }
  for (int j = 0; j < 4; ++j)
    if (overlap(rows[j].p, rows[j].bytes(), workspace, need) || overlap(flat[j], nflat[j], workspace, need))
      return FAGQ_E_ALIAS;
  const int dcheck = device_check();
  if (dcheck != FAGQ_OK) return dcheck;
  Args a = {};
  a.dout = static_cast<const uint16_t*>(dout), a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<const uint16_t*>(out), a.lse = lse;
  const int32_t* cu_k = cu_seqlens_k ? cu_seqlens_k : cu_seqlens;
  a.queries = {cu_seqlens, cu_k, (int32_t)B, (int32_t)T, (int32_t)Tk};
  a.keys = {cu_k, cu_seqlens, (int32_t)B, (int32_t)Tk, (int32_t)T};
  a.dq = static_cast<uint16_t*>(dq), a.dk = static_cast<uint16_t*>(dk), a.dv = static_cast<uint16_t*>(dv);
  const bool one_launch = small(B, T, Tk, Hq, D);
  float* const room = static_cast<float*>(workspace);
  if (!one_launch) a.lse2 = room, a.delta = room + Hq * T;
  a.part = room + space.stats, a.dq_part = a.part + space.part;
  int64_t(*to[7])[2] = {&a.dos, &a.qs, &a.ks, &a.vs, &a.dqs, &a.dks, &a.dvs};
  for (int i = 0; i < 7; ++i) (*to[i])[0] = strides[2 * i], (*to[i])[1] = strides[2 * i + 1];
  a.Hq = (int32_t)Hq, a.H = (int32_t)H, a.group = (int32_t)(Hq / H);
  a.fill = fill, a.parts = (int32_t)parts, a.dq_parts = (int32_t)dq_parts;
  a.scale = sm_scale, a.scale2 = sm_scale * kLog2e;
  int32_t dim = (int32_t)D;
  void* args[] = {&a, &dim};
  const bool bf16 = dtype == FAGQ_DT_BF16;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t dq_items = T > 0 ? tile_slots(T, B) * Hq * dq_parts : 0;
  const int64_t dkdv_items = Tk > 0 ? tile_slots(Tk, B) * H * parts : 0;
  if (one_launch) {
    a.dq_items = (int32_t)dq_items;
    const int ls = launch_kernel(bf16 ? small_for<ET_BF16>(D) : small_for<ET_F16>(D),
                                 dim3((unsigned)(a.dq_items + dkdv_items)), dim3(64 * kWaves), args, 0, st);
    if (ls != FAGQ_OK) return ls;
  } else {
    int ls = FAGQ_OK;
    if (dq_items > 0)
      ls = launch_kernel(bf16 ? dq_for<ET_BF16>(D) : dq_for<ET_F16>(D), dim3((unsigned)dq_items),
                         dim3(64 * kWaves), args, 0, st);
    // With two teams a grid of kMostGroups would be too large.
    for (int64_t first = 0; first < dkdv_items && ls == FAGQ_OK; first += kMostGroups / 4) {
      a.first = (int32_t)first;
      ls = launch_kernel(bf16 ? dkdv_for<ET_BF16>(D) : dkdv_for<ET_F16>(D),
                         dim3((unsigned)std::min(dkdv_items - first, kMostGroups / 4)),
                         dim3((unsigned)(64 * kWaves * teams(D, false))), args, 0, st);
    }
    if (ls != FAGQ_OK) return ls;
  }
  const int64_t items = (parts > 1 ? 2 * Tk * H * (D / 8) : 0) + (dq_parts > 1 ? T * Hq * (D / 8) : 0);
  if (items == 0) return FAGQ_OK;
  return launch_kernel(bf16 ? reinterpret_cast<const void*>(&prompt_join<ET_BF16>)
                            : reinterpret_cast<const void*>(&prompt_join<ET_F16>),
                       dim3((unsigned)((items + 255) / 256)), dim3(256), args, 0, st);
}

}  // extern "C"
