// paged_attn.hip - attention over the quantised paged cache (include/fagq_cache.h): the split of
// the work, the kernel that joins its parts, and the C entry points.  The attention itself is in
// paged_attn_kernels.hpp.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "fagq.h"
#include "fagq_cache.h"
#include "fagq_cache_index.hpp"
#include "fagq_dispatch.hpp"
#include "paged_attn_kernels.hpp"

namespace fagq {
namespace attn {
namespace {

constexpr int64_t kCUs = 256;
constexpr int64_t kSlots = 2 * kCUs;   // workgroups of a round
// Which way is taken goes by `most`, the caller's bound on the lengths: a loose one takes the way of the
// lengths that it allows (512 ragged sequences of 300 tokens, 32 + 8 heads of 128: 43 us with a close
// bound, 95 with room for 32768 tokens; 4 sequences of 2000, 4 tokens, 64 + 8 heads: 16.5, 39.5).
// Shares are for long lists of keys: with short ones a workgroup has several units, one after the
// other, that chunks give to as many workgroups at once (chunks / shares, us: 8 heads of 128, 64
// sequences of 4096 keys 102 / 97, of 3000 77 / 74, 256 of 2048 199 / 205, ragged 79 / 71, 56 / 58 and
// 136 / 164, 512 ragged ones of 300 53 / 105; 8 heads of 64, 64 of 6000 77 / 73, of
// 4096 54 / 54, 16 heads, 16 of 4096: 28 / 32), and for many rounds altogether (8 heads of 128, 4 of
// 32768 keys 57 / 55, 8 of 8192 28.7 / 30.2).
constexpr int64_t kLongUnit = 32, kLongUnit64 = 40;   // rounds; of heads of 64
constexpr int64_t kFewRounds = 8 * kSlots;            // of all units
constexpr int64_t kCacheBytes = 256ll << 20;    // of the cache behind the XCDs' L2

constexpr int64_t kMostGroups = (1ll << 32) / (64 * kWaves);   // a grid of 2^32 threads is too large

struct JoinArgs {
  const float* part;
  const float* ml;
  const void* lens;
  const int32_t* sched;      // null: static
  uint16_t* out;
  int32_t B, S, Hq, H;
  int32_t prefix_chunks, row_parts, chunk, most;
  int32_t idx64;
};

// The parts of a row's keys, joined by o = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i.  W waves for
// each query row take every W-th part, a lane D / 64 dims; a workgroup has kWaves / W rows.  The
// first kAhead parts of a wave are loaded at once; of static chunks before the length says how many
// hold keys (those that do not are not used): the kernel is a chain of waits.
constexpr int kAhead = 8;

template <int E, int D, int W>
__global__ __launch_bounds__(64 * kWaves) void paged_attention_join(JoinArgs a) {
  constexpr int N = D / 64;
  __shared__ float joined[W > 1 ? W : 1][D];
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64));
  const int row = (int)blockIdx.x * (kWaves / W) + wave / W, sub = wave % W;
  if (row >= a.B * a.S * a.Hq) return;          // W > 1: no workgroup is cut
  const int lane = threadIdx.x & 63;
  const int bs = row / a.Hq, hq = row - bs * a.Hq, b = bs / a.S;
  const int32_t len = own_length(a.lens, a.idx64, a.most, b);
  const int64_t mine = (int64_t)row * a.row_parts;
  // Own parts: n - prefix_chunks, from index `own` on, the first one at own_first, each next one
  // `apart` further.
  int n, apart = 1;
  int64_t own_first = mine + a.prefix_chunks, own = own_first;
  if (a.sched) {
    const int32_t rounds = rounds_of(len), q = a.sched[a.B];
    const int group = a.Hq / a.H, h = hq / group;
    const int32_t begin = a.sched[b] + h * rounds;
    const int wg = begin / q, cuts = (begin + rounds - 1) / q - wg;
    if (cuts == 0 && a.prefix_chunks == 0) return;       // written already
    if (cuts > 0) {
      const int i = (bs - b * a.S) * group + (hq - h * group);   // row of the unit
      const int64_t behind = (int64_t)a.B * a.S * a.Hq * a.row_parts + i;
      own_first = segment_at(behind, wg, 1);
      own = segment_at(behind, wg, 0);         // + 1 workgroup: the next ones
      apart = 2 * kSegmentRows;
    }
    n = a.prefix_chunks + cuts + 1;
  } else {
    n = a.row_parts;                            // at most; what the length says, below
  }
  auto index = [&](int i) {
    const int k = i - a.prefix_chunks;
    return k < 0 ? mine + i : k == 0 ? own_first : own + (int64_t)k * apart;
  };
  const f32x2* ml = reinterpret_cast<const f32x2*>(a.ml);
  const float* part = a.part + lane * N;
  float ahead[kAhead][N];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const int i = sub + u * W;
    const int64_t at = index(i < n ? i : 0);
#pragma unroll
    for (int j = 0; j < N; ++j) ahead[u][j] = part[at * D + j];
  }
  const f32x2 first = ml[index(lane < n ? lane : 0)];
  if (!a.sched) {
    const int chunks = (len + a.chunk - 1) / a.chunk;
    n = a.prefix_chunks + (chunks > 1 ? chunks : 1);
  }
  float m = lane < n ? first[0] : kLow;
  for (int i = 64 + lane; i < n; i += 64) m = fmaxf(m, ml[index(i)][0]);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
  float o[N] = {}, l = 0.0f;
  for (int i0 = 0; i0 < n; i0 += 64) {
    float w = 0.0f;
    if (i0 + lane < n) {
      const f32x2 v = i0 == 0 ? first : ml[index(i0 + lane)];
      const Power f = power_of(v[0] - m);
      w = f.a * f.b;
      l = __builtin_fmaf(v[1] * f.b, f.a, l);
    }
    const int stop = n - i0 < 64 ? n - i0 : 64;
    int i = sub;
    if (i0 == 0) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (sub + u * W >= stop) break;
        const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), sub + u * W));
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = __builtin_fmaf(f, ahead[u][j], o[j]);
      }
      i += kAhead * W;
    }
#pragma unroll 8
    for (; i < stop; i += W) {
      const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), i));
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] = __builtin_fmaf(f, part[index(i0 + i) * D + j], o[j]);
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) l += __shfl_xor(l, d);
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  if constexpr (W > 1) {
#pragma unroll
    for (int j = 0; j < N; ++j) joined[sub][lane * N + j] = o[j];
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int w = 1; w < W; ++w) o[j] += joined[w][lane * N + j];
  }
  uint16_t* out = a.out + (int64_t)row * D + lane * N;
  if constexpr (N == 1) {
    out[0] = (uint16_t)pack16<E>(o[0] * inv, 0.0f);
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 2)
      *reinterpret_cast<uint32_t*>(out + j) = pack16<E>(o[j] * inv, o[j + 1] * inv);
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

// Rounds that a schedule may have, at most.
int64_t most_rounds(int64_t B, int64_t H, int64_t most) {
  const int64_t n = (most + kRound - 1) / kRound;
  return B * H * (n > 1 ? n : 1);
}

int check_sizes(int64_t B, int64_t S, int64_t Hq, int64_t H, int64_t D, int64_t prefix_len,
                int64_t max_kv_len) {
  if (B < 0 || S < 1 || H < 1 || Hq < H || Hq % H != 0 || (D != 64 && D != 128 && D != 256) ||
      prefix_len < 0 || max_kv_len < 0)
    return FAGQ_E_SHAPE;
  // The joining kernel may have a workgroup for each row.
  if (B > 65535 || S > 65535 || Hq > 4096 || B * S * Hq >= kMostGroups ||
      prefix_len > (1ll << 30) || max_kv_len > (1ll << 30) ||
      most_rounds(B, H, max_kv_len) >= (1ll << 31) - kSlots)
    return FAGQ_E_TOO_LARGE;
  return FAGQ_OK;
}

// How a call's rows and keys are cut (see paged_attn_kernels.hpp).
struct Plan {
  int R, RP, form;
  int64_t rows, tiles, prefix_tiles;
  int64_t chunk, prefix_chunk, chunks, prefix_chunks;   // chunks: static
  int64_t items, prefix_items;                          // workgroups
  int64_t row_parts, parts;                             // of a row; of the workspace
};

// Rows of a unit.
int64_t height(int R, int64_t D) { return R == kTall ? kWaves * 16 * (256 / D) : 16 * R; }

// What a workgroup's keys cost, in keys of a short unit's workgroup / 5, and what it costs besides.
constexpr int64_t kShortKey = 5, kTallKey = 14, kFixed = 5 * 128;

int64_t key_cost(int R) { return R == kTall ? kTallKey : kShortKey; }

// What one more part of each of so many rows costs the joining kernel: a step of its chain, or its
// bytes, of which HBM moves 35 KB in the time of a key.
int64_t part_cost(int64_t rows, int64_t D) {
  const int64_t bytes = rows * D * 5 / (68 * 128);
  return bytes > 5 * (int64_t)kPartCost ? bytes : 5 * (int64_t)kPartCost;
}

// Cuts a unit's keys into the number of chunks that takes least time where each of the `units`
// becomes so many workgroups and the GPU runs them in rounds of kSlots; returns that time.  With w
// rounds, n chunks cost w (key keys / n + kFixed) + part n, least at sqrt(w key keys / part): tried for
// each w, as far as w rounds go (all n cost the host 19 us for one unit of 524288 keys).
int64_t cut(int64_t keys, int64_t units, int64_t key, int64_t part, int64_t* chunk, int64_t* chunks) {
  const int64_t most = (keys + kRound - 1) / kRound;
  int64_t best = -1;
  *chunk = kRound, *chunks = 0;
  auto consider = [&](int64_t n) {
    n = n < most ? n : most;
    if (n < 1) return;
    int64_t c = (keys + n - 1) / n;
    c = (c + kRound - 1) / kRound * kRound;
    const int64_t got = (keys + c - 1) / c;
    const int64_t time =
        (units * got + kSlots - 1) / kSlots * (c * key + kFixed) + part * got;
    if (best < 0 || time < best) {
      best = time;
      *chunk = c;
      *chunks = got;
    }
  };
  consider(1);
  for (int64_t w = 1; w <= 16; ++w) {
    const int64_t fit = w * kSlots / units;
    if (fit == 0) continue;
    const int64_t n = (int64_t)std::sqrt((double)(w * keys * key) / (double)part);
    consider(n < fit ? n : fit);
    consider(n + 1 < fit ? n + 1 : fit);
  }
  return best;
}

// The units of so many rows that see the same keys, in each of `lists` lists of so many: short ones, of
// as few row tiles as hold the rows, or for heads of 128 and 256 tall ones where that takes less time.
// (Heads of 64 are bound by the softmax, which is the same in both: 8 sequences of 256 tokens, 32 + 8
// heads, 4096 keys 113 us short, 133 tall.)  Tall units read and widen codes once for four times as
// many rows, but leave four times as many parts where workgroups are few, and waste more of their
// last rows.  Short / tall, us: 16 sequences of 4096 keys, 8 heads of 128: 64 rows 47 / 60, 96 rows
// 76 / 65, 256 rows 126 / 116; 4 heads of 256: 32 rows 38 / 43, 96 rows 95 / 74; 2 sequences, 8
// heads of 128, 256 rows 28 / 37; a prefix, 8 heads of 128: 512 rows of 32768 keys 122 / 114, of
// 4096 35 / 45.  The costs were fitted to 73 such pairs: over them the choice is 0.4 % off the best.
int row_tiles(int64_t rows, int64_t D, int64_t lists, int64_t keys) {
  int R = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  R = R * D <= 256 ? R : (int)(256 / D);
  auto units = [&](int r) { return lists * ((rows + height(r, D) - 1) / height(r, D)); };
  // A tall unit never takes less time than two short ones.
  if (D == 64 || units(R) <= 2 * units(kTall)) return R;
  int64_t chunk, chunks;
  const int64_t part = part_cost(lists * rows, D);
  const int64_t tall = cut(keys, units(kTall), key_cost(kTall), part, &chunk, &chunks);
  return tall < cut(keys, units(R), key_cost(R), part, &chunk, &chunks) ? kTall : R;
}

Plan plan_for(int64_t B, int64_t S, int64_t Hq, int64_t H, int64_t D, int64_t prefix_len,
              int64_t most) {
  Plan p = {};
  const int64_t per = S * (Hq / H);
  p.rows = B * S * Hq;
  p.R = row_tiles(per, D, B * H, most);
  if (prefix_len > 0) {
    p.RP = row_tiles(B * per, D, H, prefix_len);
    if (p.R > 1 && p.RP != kTall) p.R = p.RP;
    p.prefix_tiles = (B * per + height(p.RP, D) - 1) / height(p.RP, D);
    cut(prefix_len, H * p.prefix_tiles, key_cost(p.RP), part_cost(p.rows, D), &p.prefix_chunk,
        &p.prefix_chunks);
    p.prefix_items = H * p.prefix_tiles * p.prefix_chunks;
  }
  p.tiles = (per + height(p.R, D) - 1) / height(p.R, D);
  if (p.tiles > 1 || p.R > 1 || most_rounds(1, 1, most) < (D == 64 ? kLongUnit64 : kLongUnit) ||
      most_rounds(B, H, most) <= kFewRounds) {
    p.form = kStatic;
    cut(most, B * H * p.tiles, key_cost(p.R), part_cost(p.rows, D), &p.chunk, &p.chunks);
    if (p.chunks < 1) p.chunks = 1;     // rows without keys are written all the same
    p.items = B * H * p.tiles * p.chunks;
    p.row_parts = p.prefix_chunks + p.chunks;
    p.parts = p.row_parts > 1 ? p.rows * p.row_parts : 0;
  } else {
    p.form = prefix_len == 0 && 2 * B * most * H * D >= kCacheBytes ? kScheduledOnce : kScheduled;
    p.items = kSlots;
    p.row_parts = prefix_len > 0 ? p.prefix_chunks + 1 : 0;
    p.parts = p.rows * p.row_parts + p.items * 2 * kSegmentRows;
  }
  return p;
}

// o, {m, l} of each part, and the schedule.
int64_t bytes_of(const Plan& p, int64_t B, int64_t D) {
  return p.parts * (D + 2) * 4 + (p.form == kStatic ? 0 : (B + 1) * 4);
}

const void* kernel_for(int dtype, int q_format, int scale_format, int D, const Plan& p) {
  using Lookup = const void* (*)(int, int, int, int);
  static constexpr Lookup table[8] = {lookup_e0_q0_s0, lookup_e0_q0_s1, lookup_e0_q1_s0, lookup_e0_q1_s1,
                                      lookup_e1_q0_s0, lookup_e1_q0_s1, lookup_e1_q1_s0, lookup_e1_q1_s1};
  const int e = dtype == FAGQ_DT_BF16 ? 0 : 1, q = q_format == FAGQ_Q_FP8_E4M3FN ? 0 : 1;
  const int s = scale_format == FAGQ_SCALE_F32 ? 0 : 1;
  return table[4 * e + 2 * q + s](D, p.R, p.RP, p.form);
}

template <int E, int W>
const void* join_for(int64_t D) {
  return D == 64    ? reinterpret_cast<const void*>(&paged_attention_join<E, 64, W>)
         : D == 128 ? reinterpret_cast<const void*>(&paged_attention_join<E, 128, W>)
                    : reinterpret_cast<const void*>(&paged_attention_join<E, 256, W>);
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
  if (B == 0) return 0;
  const Plan p = plan_for(B, S, Hq, H, D, prefix_len, max_kv_len);
  return p.prefix_items + p.items < kMostGroups ? bytes_of(p, B, D) : -1;
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
  if (num_pages < 1 || table_width < 0 || page_size < FAGQ_CACHE_MIN_PAGE ||
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
      !aligned(k_scale, ss * 4) || !aligned(v_scale, ss * 4) || !aligned(page_table, 4) ||
      !aligned(kv_lens, is) || !aligned(prefix_pages, 4) || !aligned(out, 16))
    return FAGQ_E_ALIGN;
  const Plan p = B > 0 ? plan_for(B, S, Hq, H, D, prefix_len, max_kv_len) : Plan{};
  if (p.prefix_items + p.items >= kMostGroups) return FAGQ_E_TOO_LARGE;
  const int64_t need = B > 0 ? bytes_of(p, B, D) : 0;
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
  a.num_pages = (int32_t)num_pages;
  for (int i = 0; i < 3; ++i) a.qs[i] = (int32_t)strides[i];
  a.B = (int32_t)B, a.S = (int32_t)S, a.Hq = (int32_t)Hq, a.H = (int32_t)H;
  a.group = (int32_t)(Hq / H);
  a.page_shift = log2_of(page_size), a.width = (int32_t)table_width;
  a.prefix_len = (int32_t)prefix_len;
  const int64_t room = table_width > (max_kv_len >> a.page_shift) ? max_kv_len
                                                                  : table_width << a.page_shift;
  a.most = (int32_t)(room < max_kv_len ? room : max_kv_len);
  a.idx64 = index_dtype == FAGQ_IDX_I64;
  a.scale2 = sm_scale * 1.44269504088896340736f;
  a.chunk = (int32_t)p.chunk, a.chunks = (int32_t)p.chunks, a.tiles = (int32_t)p.tiles;
  a.prefix_chunk = (int32_t)p.prefix_chunk, a.prefix_chunks = (int32_t)p.prefix_chunks;
  a.prefix_tiles = (int32_t)p.prefix_tiles, a.prefix_items = (int32_t)p.prefix_items;
  a.items = (int32_t)p.items;
  a.row_parts = (int32_t)p.row_parts, a.slots = (int32_t)kSlots;
  if (need > 0) {
    a.part = static_cast<float*>(workspace);
    a.part_ml = a.part + p.parts * D;
    a.sched = p.form == kStatic ? nullptr : reinterpret_cast<int32_t*>(a.part_ml + 2 * p.parts);
  }
  void* args[] = {&a};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int ls = launch_kernel(kernel_for(dtype, q_format, scale_format, (int)D, p),
                               dim3((unsigned)(p.prefix_items + p.items)), dim3(64 * kWaves), args,
                               0, st);
  if (ls != FAGQ_OK || p.parts == 0) return ls;
  JoinArgs j = {};
  j.part = a.part, j.ml = a.part_ml, j.lens = kv_lens, j.sched = a.sched, j.out = a.out;
  j.B = a.B, j.S = a.S, j.Hq = a.Hq, j.H = a.H;
  j.prefix_chunks = a.prefix_chunks, j.row_parts = a.row_parts, j.chunk = a.chunk, j.most = a.most;
  j.idx64 = a.idx64;
  void* jargs[] = {&j};
  // A workgroup for each row where one may have more than kAhead parts.
  const int64_t rounds = (max_kv_len + kRound - 1) / kRound;
  const int64_t own = p.form == kStatic ? p.chunks : B * H >= kSlots ? 2 : rounds;
  const bool wide = p.prefix_chunks + own > kAhead;
  const void* fn = dtype == FAGQ_DT_BF16 ? (wide ? join_for<ET_BF16, kWaves>(D) : join_for<ET_BF16, 1>(D))
                                         : (wide ? join_for<ET_F16, kWaves>(D) : join_for<ET_F16, 1>(D));
  const int64_t groups = wide ? p.rows : (p.rows + kWaves - 1) / kWaves;
  return launch_kernel(fn, dim3((unsigned)groups), dim3(64 * kWaves), jargs, 0, st);
}

}  // extern "C"
