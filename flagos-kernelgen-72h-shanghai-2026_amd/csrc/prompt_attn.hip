// prompt_attn.hip - causal attention of packed prompts (include/fagq_prompt.h).
//
// One pass with a running maximum m and sum l of the softmax: for key j with score x (in units of
// log 2), p = 2^(x - m), l = sum p, o = sum p v.  A workgroup takes 128 queries of one head, each
// wave 32; keys and values come through LDS in tiles of 64 (heads of 256: 32), the next ones under
// way while these are worked on.
//   scores   S^T = K Q^T: lane (c, h) has query c's scores of half of the keys.
//   output   O^T = V^T P^T: the packed probabilities are its B operand as they are.
// Where there are few workgroups, each one's keys are cut into parts with m, l and o of their own,
// which prompt_attention_join puts together: o = sum 2^(m_i - m) o_i.
//
// Bound by power where calls are long: 16384 tokens, 64 + 8 heads of 128, 3.87 ms, 1.14 PFLOP/s, the
// matrix units busy 59 % of the cycles at 1.75 GHz.  Tiles of 128 queries: a CU then reads 32 KB of keys
// and values in the time of 4.2 MFLOP from its L2.  Two workgroups a CU, so that one's softmax runs under
// the other's products; three, with steps of 32 keys, take as long.  P is rounded to the element type
// for its product: the output is 1.1 to 1.4 times as far off as its own rounding makes it.
// Heads of 256 have their keys in tiles of 32: of 64, one workgroup fills a CU's LDS (4 chunks of 512
// tokens over 4096, 16 + 4 heads, 175 us).
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

constexpr float kLow = -3.0e38f;     // running maximum before the first key
// The running maximum follows a row's scores only where p could pass 2^kMost, which neither the sums nor
// 16 bits mind, so that o is rarely multiplied.  It is kept kLift below them: fp16 loses bits of weights
// under 2^-14, which thousands of keys behind one that takes nearly all of the weight have, so there the
// largest is 2^11 to 2^15, and weights above 2^-25 of it keep all their bits.  (16384 tokens, 64 + 8 heads
// of 128, in fp16: 4.46 ms, 4.42 with a lift of 0 and 2^8, 4.50 with 13.)
template <int E>
constexpr float kLift = E == ET_F16 ? 11.0f : 0.0f;
template <int E>
constexpr float kMost = E == ET_F16 ? 15.0f : 8.0f;

struct Args {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  Sequences seq;
  uint16_t* out;
  float* lse;
  float* part;                       // [parts][T][Hq][D], then {m, l} [parts][T][Hq][2]
  int64_t qs[2], ks[2], vs[2];       // {token, head} strides, elements
  int32_t Hq, H, group, fill, parts;
  float scale2;                      // |sm_scale| log2(e), not 0
  uint32_t flip;                     // signs of a pair of queries' values, where sm_scale < 0
};

// Rows behind the last sequence.
template <int D>
__device__ __forceinline__ void fill_tail(const Args& a, const Place& p, int hq) {
  const int64_t first = (int64_t)p.end + (int64_t)p.tile * kTile;
  for (int i = threadIdx.x % (64 * kWaves); i < kTile * (D / 8); i += 64 * kWaves) {
    const int64_t row = first + i / (D / 8);
    if (row >= a.seq.T) break;
    if (a.fill & FAGQ_FILL_OUT)
      *reinterpret_cast<u32x4*>(a.out + (row * a.Hq + hq) * D + i % (D / 8) * 8) = u32x4{0, 0, 0, 0};
    if (a.lse && (a.fill & FAGQ_FILL_LSE) && i % (D / 8) == 0) a.lse[(int64_t)hq * a.seq.T + row] = -INFINITY;
  }
}

// TEAMS: of four waves, each with a head of its own, of those that share keys.
template <int E, int D, int TEAMS>
__global__ __launch_bounds__(64 * kWaves * TEAMS, 2) void prompt_attention(Args a) {
  constexpr int kKeys = D == 256 ? 32 : 64;      // in LDS at a time
  using L = Tile<D, kKeys>;
  __shared__ __align__(16) char lds[2][2][L::kBytes];
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int waves = scalar((int)(threadIdx.x >> 6)), wave = waves % kWaves, team = waves / kWaves;
  // Workgroup b runs on XCD b % 8: heads that share keys stay on one.
  const int item = (int)blockIdx.x, kvh = item % a.H, heads = item / a.H, sets = a.group / TEAMS;
  const int hq = kvh * a.group + heads % sets * TEAMS + team, rest = heads / sets, part = rest % a.parts;
  const Place p = place_of<true>(a.seq, rest / a.parts);
  if (p.b < 0) {
    if (a.fill && part == 0) fill_tail<D>(a, p, hq);
    return;
  }
  const int32_t ahead = p.m - p.n;               // query i sees the keys up to i + ahead
  const int32_t q0 = p.tile * kTile, mine = q0 + wave * kRows;
  const int32_t i = mine + c;
  auto seen_by = [&](int32_t query) {
    const int32_t n = query + ahead + 1;
    return n < 0 ? 0 : n < p.m ? n : p.m;
  };
  const int32_t seen = i < p.n ? seen_by(i) : 0;
  const int32_t all = seen_by(mine);             // keys that every query of the wave sees
  const int32_t last = mine + kRows <= p.n ? mine + kRows - 1 : p.n - 1;
  const int32_t end = mine < p.n ? seen_by(last) : 0;                    // that one of them sees
  // Steps of the workgroup, this part's share of them.
  const int32_t steps = (seen_by(q0 + kTile <= p.n ? q0 + kTile - 1 : p.n - 1) + kKeys - 1) / kKeys;
  const int32_t from = (int32_t)((int64_t)steps * part / a.parts) * kKeys;
  const int32_t stop = (int32_t)((int64_t)steps * (part + 1) / a.parts) * kKeys;

  Copier<D, kKeys> ck, cv;
  ck.init(a.k, (int64_t)p.other * a.ks[0] + (int64_t)kvh * a.ks[1], a.ks[0], lane, wave);
  cv.init(a.v, (int64_t)p.other * a.vs[0] + (int64_t)kvh * a.vs[1], a.vs[0], lane, wave);
  auto issue = [&](int buf, int32_t tok) {       // two teams: keys, values
    if (TEAMS == 1 || team == 0) ck.issue(lds[buf][0], wave, tok, p.m - 1);
    if (TEAMS == 1 || team == 1) cv.issue(lds[buf][1], wave, tok, p.m - 1);
  };
  if (from < stop) issue(0, from);
  u32x4 q[D / 16];
  load_row<D>(a.q + (int64_t)(p.row + (i < p.n ? i : p.n - 1)) * a.qs[0] + (int64_t)hq * a.qs[1], h, q);
#pragma unroll
  for (int j = 0; j < D / 16; ++j) q[j] ^= a.flip;
  f32x16 o[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d) o[d] = splat(0.0f);
  float m = kLow, l = 0.0f;

  int buf = 0;
  for (int32_t tok = from; tok < stop; tok += kKeys, buf ^= 1) {
    __builtin_amdgcn_s_waitcnt(kVmcnt0);         // this step's tiles have landed, of this wave
    lds_barrier();                               // of all; the last step's are done with
    if (tok + kKeys < stop) issue(buf ^ 1, tok + kKeys);
    if (tok >= end) continue;
    f32x16 x[kKeys / 32];
#pragma unroll
    for (int t = 0; t < kKeys / 32; ++t) {
      x[t] = splat(0.0f);
#pragma unroll
      for (int j = 0; j < D / 16; ++j) x[t] = mfma<E>(row_frag<D>(lds[buf][0], lane, t, j), q[j], x[t]);
    }
    read_ahead<4, 1, kKeys / 32 * (D / 16)>();
    if (tok + kKeys > all) {
#pragma unroll
      for (int t = 0; t < kKeys / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          x[t][r] = tok + 32 * t + row_of(r, h) < seen ? x[t][r] : -INFINITY;
    }
    float top = x[0][0];
#pragma unroll
    for (int r = 1; r < kKeys / 2; ++r) top = fmaxf(top, x[r / 16][r % 16]);
    if (__any(__builtin_fmaf(top, a.scale2, -m) > kMost<E>)) {
      const float next = fmaxf(m, cross_max(top) * a.scale2 - kLift<E>);
      const float f = __builtin_amdgcn_exp2f(m - next);
      m = next;
      l *= f;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= f;
    }
    u32x4 w[kKeys / 16];
    float sum = 0.0f;                            // by itself: one large weight does not swallow single ones
#pragma unroll
    for (int t = 0; t < kKeys / 32; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][r], a.scale2, -m));
        sum += x[t][r];
      }
      w[2 * t] = pack8<E>(x[t], 0);
      w[2 * t + 1] = pack8<E>(x[t], 1);
    }
    l += sum;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int t = 0; t < kKeys / 16; ++t)
        o[d] = mfma<E>(col_frag<D>(lds[buf][1], lane, d, t), w[t], o[d]);
    read_ahead<8, 2, kKeys / 16 * (D / 32)>();
  }
  l = cross_sum(l);
  const int64_t row = p.row + i;
  if (a.parts == 1) {
    store_row<E, D>(a.out + (row * a.Hq + hq) * D, h, o, l > 0.0f ? 1.0f / l : 0.0f, i < p.n);
    if (a.lse && h == 0 && i < p.n)
      a.lse[(int64_t)hq * a.seq.T + row] =
          l > 0.0f ? (m + __builtin_amdgcn_logf(l)) * (1.0f / kLog2e) : -INFINITY;
  } else if (i < p.n) {
    const int64_t at = ((int64_t)part * a.seq.T + row) * a.Hq + hq;
    float* to = a.part + at * D;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<f32x4*>(to + 32 * d + row_of(r, h)) =
            f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
    if (h == 0) {
      float* ml = a.part + (int64_t)a.parts * a.seq.T * a.Hq * D + 2 * at;
      ml[0] = m;
      ml[1] = l;
    }
  }
}

// Joins the parts of a query's keys.  D / 8 threads have a query and head, each 8 of its values.
template <int E, int D>
__global__ __launch_bounds__(256) void prompt_attention_join(Args a) {
  constexpr int kThreads = D / 8;
  const int64_t item = (int64_t)blockIdx.x * (256 / kThreads) + threadIdx.x / kThreads;
  const int d = threadIdx.x % kThreads * 8;
  const int64_t rows = (int64_t)a.seq.T * a.Hq, row = item / a.Hq;
  if (row >= clamped(a.seq.cu[a.seq.B], a.seq.T)) return;
  const float* ml = a.part + a.parts * rows * D + 2 * item;
  float m = kLow;
  for (int i = 0; i < a.parts; ++i) m = fmaxf(m, ml[2 * i * rows]);
  float l = 0.0f;
  f32x4 o[2] = {};
  for (int i = 0; i < a.parts; ++i) {
    const float f = __builtin_amdgcn_exp2f(ml[2 * i * rows] - m);
    const float* part = a.part + (i * rows + item) * D + d;
    l = __builtin_fmaf(ml[2 * i * rows + 1], f, l);
    o[0] += *reinterpret_cast<const f32x4*>(part) * f;
    o[1] += *reinterpret_cast<const f32x4*>(part + 4) * f;
  }
  const float f = l > 0.0f ? 1.0f / l : 0.0f;
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack16<E>(o[i / 2][2 * i % 4] * f, o[i / 2][2 * i % 4 + 1] * f);
  *reinterpret_cast<u32x4*>(a.out + item * D + d) = w;
  if (a.lse && d == 0)
    a.lse[item % a.Hq * a.seq.T + row] =
        l > 0.0f ? (m + __builtin_amdgcn_logf(l)) * (1.0f / kLog2e) : -INFINITY;
}

// Two workgroups run on a CU (us, so / in parts of 16 steps at least: 8 + 8 heads of 128, 100 tokens
// behind 1500 17 / 31; 4 + 4, 200 behind 2000 19 / 27; 4 + 1, prompts of 3000 and 500 tokens 33 / 53;
// 16 + 8 of 256, 20 behind 1800 23 / 34; 8 + 1 of 256, 2048 tokens 58 / 53).
constexpr int64_t kSlots = 512;
int64_t parts_for(int64_t B, int64_t T, int64_t Tk, int64_t Hq) { return key_parts(B, T, Tk, Hq, kSlots); }

// Two teams, and half as many workgroups, read keys once for two heads: for long calls of heads of 128 (us,
// two / one, 32 + 8 heads: 4096 tokens 148 / 159, 8192 503 / 511, 8 x 512 behind 4096 265 / 278; 16 + 2,
// 8192 251 / 275; but 2048 tokens 59 / 51, 16 x 1024 198 / 187).  For heads of 256 they take longer
// there too (4 x 512 behind 4096, 16 + 4 heads 164 / 157), for heads of 64 within 2 % of as long.
int teams_for(int64_t B, int64_t T, int64_t Tk, int64_t Hq, int64_t H, int64_t D) {
  return D == 128 && B > 0 && Hq / H % 2 == 0 && query_tiles(B, T, Hq) >= 2 * kSlots &&
                 steps_of_tile(B, T, Tk) >= 32 ? 2 : 1;
}

int check_fwd_sizes(int64_t B, int64_t T, int64_t Tk, int64_t Hq, int64_t H, int64_t D) {
  const int st = check_sizes(B, T, Tk, Hq, H, D);
  if (st != FAGQ_OK) return st;
  return tile_slots(T, B) * Hq * parts_for(B, T, Tk, Hq) >= kMostGroups ? FAGQ_E_TOO_LARGE : FAGQ_OK;
}

int64_t bytes_for(int64_t B, int64_t T, int64_t Tk, int64_t Hq, int64_t D) {
  const int64_t parts = parts_for(B, T, Tk, Hq);
  return parts > 1 ? parts * T * Hq * (D + 2) * 4 : 0;
}

template <int E>
const void* kernel_for(int64_t D, int teams) {
  return D == 64      ? reinterpret_cast<const void*>(&prompt_attention<E, 64, 1>)
         : D == 256   ? reinterpret_cast<const void*>(&prompt_attention<E, 256, 1>)
         : teams == 2 ? reinterpret_cast<const void*>(&prompt_attention<E, 128, 2>)
                      : reinterpret_cast<const void*>(&prompt_attention<E, 128, 1>);
}
template <int E>
const void* join_for(int64_t D) {
  return D == 64    ? reinterpret_cast<const void*>(&prompt_attention_join<E, 64>)
         : D == 128 ? reinterpret_cast<const void*>(&prompt_attention_join<E, 128>)
                    : reinterpret_cast<const void*>(&prompt_attention_join<E, 256>);
}

}  // namespace
}  // namespace prompt
}  // namespace fagq

extern "C" {

FAGQ_API int64_t fagq_prompt_attention_workspace_bytes(int64_t B, int64_t T, int64_t Tk,
                                                       int64_t Hq, int64_t H, int64_t D) {
  using namespace fagq::prompt;
  return check_fwd_sizes(B, T, Tk, Hq, H, D) == FAGQ_OK ? bytes_for(B, T, Tk, Hq, D) : -1;
}

FAGQ_API int fagq_prompt_attention_launch(const void* q, const void* k, const void* v,
                                          const int32_t* cu_seqlens, const int32_t* cu_seqlens_k,
                                          void* out, float* lse, void* workspace,
                                          int64_t workspace_bytes, const int64_t* strides,
                                          int64_t B, int64_t T, int64_t Tk, int64_t Hq, int64_t H,
                                          int64_t D, float sm_scale, int dtype, int fill,
                                          void* stream) {
  using namespace fagq;
  using namespace fagq::prompt;
  if (!q || (Tk > 0 && (!k || !v)) || !cu_seqlens || !out || !strides) return FAGQ_E_NULL;
  if (dtype != FAGQ_DT_BF16 && dtype != FAGQ_DT_F16) return FAGQ_E_FORMAT;
  if (fill & ~(FAGQ_FILL_OUT | FAGQ_FILL_LSE)) return FAGQ_E_FORMAT;
  if (!std::isfinite(sm_scale)) return FAGQ_E_SHAPE;
  const int sizes = check_fwd_sizes(B, T, Tk, Hq, H, D);
  if (sizes != FAGQ_OK) return sizes;
  if (!cu_seqlens_k && T != Tk) return FAGQ_E_SHAPE;
  const int st = check_strides(strides, 6);
  if (st != FAGQ_OK) return st;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) || !aligned(lse, 4) ||
      !aligned(cu_seqlens, 4) || !aligned(cu_seqlens_k, 4) || !aligned(workspace, 16))
    return FAGQ_E_ALIGN;
  const int64_t need = bytes_for(B, T, Tk, Hq, D);
  if (workspace_bytes < need) return FAGQ_E_SHAPE;
  if (need > 0 && !workspace) return FAGQ_E_NULL;
  if (T == 0) return FAGQ_OK;
  const Rows rows[3] = {{q, T, Hq, D, strides[0], strides[1]},
                        {k, Tk, H, D, strides[2], strides[3]},
                        {v, Tk, H, D, strides[4], strides[5]}};
  const void* ins[5] = {q, k, v, cu_seqlens, cu_seqlens_k};
  const int64_t nin[5] = {rows[0].bytes(), rows[1].bytes(), rows[2].bytes(), (B + 1) * 4,
                          cu_seqlens_k ? (B + 1) * 4 : 0};
  const int64_t nout = T * Hq * D * 2, nlse = lse ? T * Hq * 4 : 0;
  for (int i = 0; i < 5; ++i)
    if (overlap(out, nout, ins[i], nin[i]) || overlap(lse, nlse, ins[i], nin[i]) ||
        overlap(workspace, need, ins[i], nin[i]))
      return FAGQ_E_ALIAS;
  if (overlap(out, nout, lse, nlse) || overlap(workspace, need, out, nout) ||
      overlap(workspace, need, lse, nlse))
    return FAGQ_E_ALIAS;
  const int dcheck = device_check();
  if (dcheck != FAGQ_OK) return dcheck;
  Args a = {};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v);
  a.seq = {cu_seqlens, cu_seqlens_k ? cu_seqlens_k : cu_seqlens, (int32_t)B, (int32_t)T, (int32_t)Tk};
  a.out = static_cast<uint16_t*>(out), a.lse = lse;
  for (int i = 0; i < 2; ++i) a.qs[i] = strides[i], a.ks[i] = strides[2 + i], a.vs[i] = strides[4 + i];
  a.Hq = (int32_t)Hq, a.H = (int32_t)H, a.group = (int32_t)(Hq / H);
  a.fill = fill;
  // What a query does not see has the score -inf, which times 0 would be no number.
  a.scale2 = std::fmax(std::fabs(sm_scale) * kLog2e, 0x1p-126f);
  a.flip = sm_scale < 0.0f ? 0x80008000u : 0u;
  a.parts = (int32_t)parts_for(B, T, Tk, Hq), a.part = static_cast<float*>(workspace);
  void* args[] = {&a};
  const bool bf16 = dtype == FAGQ_DT_BF16;
  hipStream_t to = static_cast<hipStream_t>(stream);
  const int teams = teams_for(B, T, Tk, Hq, H, D);
  const int ls = launch_kernel(bf16 ? kernel_for<ET_BF16>(D, teams) : kernel_for<ET_F16>(D, teams),
                               dim3((unsigned)(tile_slots(T, B) * Hq / teams * a.parts)),
                               dim3((unsigned)(64 * kWaves * teams)), args, 0, to);
  if (ls != FAGQ_OK || a.parts == 1) return ls;
  return launch_kernel(bf16 ? join_for<ET_BF16>(D) : join_for<ET_F16>(D),
                       dim3((unsigned)((T * Hq * (D / 8) + 255) / 256)), dim3(256), args, 0, to);
}

}  // extern "C"
