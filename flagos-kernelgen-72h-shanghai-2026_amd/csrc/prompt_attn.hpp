// prompt_attn.hpp - device code shared by the attention of prompts and its gradients
// (include/fagq_prompt.h): which rows a workgroup takes, tiles in LDS, operands of the matrix
// instructions, and the host's checks.
//
// Matrix instructions are 32 x 32 x 16.  Lane (c, h), c = lane % 32, h = lane / 32:
//   A, B     row (column) c, places 8 h .. 8 h + 7 of the sum over 16
//   C        column c, rows (r % 4) + 8 (r / 4) + 4 h at register r
// A product's result therefore is the B operand of the next one as it stands: registers 8 t .. of
// a lane are 8 of 16 places of the sum over the result's rows, and the A operand only has to have
// the same rows there, 4 h + 0..3 and 8 + 4 h + 0..3 of each 16.  A tile that lies in LDS row by
// row gives both kinds of operand: rows as they are (16-byte reads), columns by the transposed
// 8-byte read (a lane receives 4 rows of its column).
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "fagq.h"
#include "fagq_dispatch.hpp"

namespace fagq {
namespace prompt {

constexpr int kWaves = 4;
constexpr int kRows = 32;                       // of a wave
constexpr int kTile = kRows * kWaves;           // of a workgroup
constexpr int kStep = 64;                       // rows of the other side that are in LDS at a time
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int64_t kMostGroups = 1ll << 24;      // a grid of 2^32 threads is too large
constexpr int64_t kMostTokens = (1ll << 31) - 1024;   // a tile past the last token has 32-bit numbers
constexpr int kVmcnt0 = 0x0F70;                 // s_waitcnt vmcnt(0), other counters not waited; + n < 16

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <int E>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (E == ET_BF16) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a),
                                                   __builtin_bit_cast(v8, b), c, 0, 0, 0);
  } else {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a),
                                                  __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
}

__device__ __forceinline__ f32x16 splat(float v) {
  f32x16 r;
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = v;
  return r;
}

__device__ __forceinline__ int32_t scalar(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// Row of a 32 x 32 result at register r.
__device__ __forceinline__ int row_of(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

// Maximum (sum) over the lanes c and c + 32; both receive it.
__device__ __forceinline__ float cross_max(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float cross_sum(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// ------------------------------------------------------------------------- tiles in LDS

// A tile of ROWS rows of D elements, row by row, in 16-byte chunks; chunk c of row r lies at chunk
// c ^ swizzle(r) of it.  256 bytes of LDS (16 chunks) are read at once without a conflict: the 16
// rows of a 16-byte read at one c, and the 4 rows x 4 chunks of a transposed read.
template <int D, int ROWS = kStep>
struct Tile {
  static constexpr int kChunks = D / 8;
  static constexpr int kRowBytes = D * 2;
  static constexpr int kBytes = ROWS * kRowBytes;
  static constexpr int kCopyRows = 64 / kChunks;              // rows that one copy brings
  static constexpr int kCopies = ROWS / kCopyRows / kWaves;  // of each wave
  static __device__ __forceinline__ int swizzle(int r) {
    if constexpr (D == 64) return ((r >> 1) & 1) << 2 | ((r >> 2) & 3);   // two rows in 256 bytes
    else return (r & 3) << 2 | ((r >> 2) & 3);
  }
};

// 16 (4) bytes a lane from `rs` at voff + soff past the registers to LDS, lane by lane from `lds` on
// (which m0 tells the instruction; it is put back, the compiler keeps it).  In assembly, so that only
// the kernel's own waits are for it: of the builtin the compiler has every transposed read of LDS
// wait for all copies under way, the ones for the next step among them (dk and dv of 8192 tokens,
// 32 + 8 heads of 128: 1075 us, with the builtin 1145; the other kernels take as long with either).
__device__ __forceinline__ void copy16(const u32x4& rs, char* lds, uint32_t voff, uint32_t soff) {
  uint32_t old;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t"
               "buffer_load_dwordx4 %2, %3, %4 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(old)
               : "s"((uint32_t)(uintptr_t)(lds_void_t*)lds), "v"(voff), "s"(rs), "s"(soff)
               : "memory");
}
__device__ __forceinline__ void copy4(const u32x4& rs, char* lds, uint32_t voff) {
  uint32_t old;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t"
               "buffer_load_dword %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(old)
               : "s"((uint32_t)(uintptr_t)(lds_void_t*)lds), "v"(voff), "s"(rs)
               : "memory");
}
// A buffer from p on, of any size: callers keep their offsets inside the tensor.
__device__ __forceinline__ u32x4 buffer_at(const void* p) {
  const uintptr_t v = reinterpret_cast<uintptr_t>(p);
  return {(uint32_t)scalar((int32_t)(uint32_t)v), (uint32_t)scalar((int32_t)(uint32_t)(v >> 32)) & 0xffffu,
          0xffffffffu, kRsrcWord3};
}

// Copies rows [first, first + ROWS) of one head, row `last` in place of those behind it, from HBM
// into LDS, past the registers.  Copy n of wave w brings rows (4 n + w) kCopyRows ..
template <int D, int ROWS = kStep>
struct Copier {
  using L = Tile<D, ROWS>;
  const char* base;            // row 0 of the sequence
  uint32_t stride;             // bytes of a row
  int row;                     // within the copies of this wave, of this lane
  uint32_t chunk[2];           // byte in the row, for even and odd n
  __device__ __forceinline__ void init(const void* p, int64_t element, int64_t token_stride, int lane,
                                       int wave) {
    base = static_cast<const char*>(p) + element * 2;
    stride = (uint32_t)token_stride * 2u;
    row = wave * L::kCopyRows + lane / L::kChunks;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      chunk[i] = (uint32_t)((lane % L::kChunks) ^ L::swizzle(row + i * kWaves * L::kCopyRows)) * 16u;
  }
  __device__ __forceinline__ void issue(char* lds, int wave, int first, int last) const {
    const u32x4 rs = buffer_at(base + (int64_t)first * stride);
    if (first + ROWS - 1 <= last) {
      const uint32_t off = (uint32_t)row * stride;
#pragma unroll
      for (int n = 0; n < L::kCopies; ++n)
        copy16(rs, lds + (n * kWaves + wave) * 1024, off + chunk[n & 1],
               (uint32_t)(n * kWaves * L::kCopyRows) * stride);
    } else {
#pragma unroll
      for (int n = 0; n < L::kCopies; ++n) {
        const int r = row + n * kWaves * L::kCopyRows, most = last - first;
        copy16(rs, lds + (n * kWaves + wave) * 1024, (uint32_t)(r < most ? r : most) * stride + chunk[n & 1],
               0);
      }
    }
  }
};

// Row operand: rows 32 t .. of a tile, places 16 i .. of the sum over D.
template <int D>
__device__ __forceinline__ u32x4 row_frag(const char* tile, int lane, int t, int i) {
  const int c = lane & 31, h = lane >> 5;
  const int at = c * Tile<D>::kRowBytes + (((2 * i) ^ (h ^ Tile<D>::swizzle(c))) << 4);
  return *reinterpret_cast<const u32x4*>(tile + at + t * 32 * Tile<D>::kRowBytes);
}

// Column operand: columns 32 d .. of a tile, rows 16 t .. as the places of the sum.
template <int D>
__device__ __forceinline__ u32x4 col_frag(const char* tile, int lane, int d, int t) {
  const int i = lane & 15, g = (lane >> 4) & 1, h = lane >> 5;
  u32x4 r;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int row = 8 * u + 4 * h + (i >> 2);
    const int chunk = (4 * d + 2 * g + ((i >> 1) & 1)) ^ Tile<D>::swizzle(row);
    const char* p = tile + row * Tile<D>::kRowBytes + chunk * 16 + (i & 1) * 8 +
                    t * 16 * Tile<D>::kRowBytes;
    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    r[2 * u] = w[0], r[2 * u + 1] = w[1];
  }
  return r;
}

// The order of a stretch of N products: FIRST reads of LDS ahead of the first, EACH between any two.
template <int FIRST, int EACH, int N>
__device__ __forceinline__ void read_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, FIRST, 0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);
  }
}

// Registers 8 t .. of a result as the B operand of the next product.
template <int E>
__device__ __forceinline__ u32x4 pack8(const f32x16& x, int t) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = pack16<E>(x[8 * t + 2 * i], x[8 * t + 2 * i + 1]);
  return r;
}

// What packing lost of them, packed: a product with both terms has twice the bits.
template <int E>
__device__ __forceinline__ u32x4 pack_rest8(const f32x16& x, int t, const u32x4& w) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = pack16<E>(x[8 * t + 2 * i] - lo16<E>(w[i]), x[8 * t + 2 * i + 1] - hi16<E>(w[i]));
  return r;
}

// A row in global memory as row operands: places 16 i + 8 h ..
template <int D>
__device__ __forceinline__ void load_row(const uint16_t* row, int h, u32x4 (&f)[D / 16]) {
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
    f[i] = *reinterpret_cast<const u32x4*>(row + 16 * i + 8 * h);
}

// A lane's column of a transposed result [D x 32] times f, as a row in global memory.  The halves
// exchange four rows each, so that every lane stores 16 bytes.
template <int E, int D>
__device__ __forceinline__ void store_row(uint16_t* row, int h, const f32x16 (&o)[D / 32], float f,
                                          bool live) {
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int p = 0; p < 2; ++p) {               // rows 16 p ..: 4 h .. and 8 + 4 h ..
      uint32_t a[2], b[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        a[i] = pack16<E>(o[d][8 * p + 2 * i] * f, o[d][8 * p + 2 * i + 1] * f);
        b[i] = pack16<E>(o[d][8 * p + 4 + 2 * i] * f, o[d][8 * p + 4 + 2 * i + 1] * f);
      }
      // Lane c keeps rows 0 .. 3 and receives 4 .. 7; lane c + 32 receives 8 .. 11, keeps 12 .. 15.
      const auto x = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
      if (live)
        *reinterpret_cast<u32x4*>(row + 32 * d + 16 * p + 8 * h) = u32x4{x[0], y[0], x[1], y[1]};
    }
}

// ------------------------------------------------------------------------- sequences

struct Sequences {
  const int32_t* cu;           // of the rows that tiles are made of
  const int32_t* other;        // of the other side's
  int32_t B, T, Tother;
};

struct Place {
  int32_t b;                   // -1: a tile behind the last one
  int32_t tile;                // of the sequence; behind the last one: which
  int32_t row, n;              // first row and length of the sequence
  int32_t other, m;            // of the other side
  int32_t end;                 // rows of all sequences
};

__device__ __forceinline__ int32_t clamped(int32_t v, int32_t most) {
  return v < 0 ? 0 : v < most ? v : most;
}

// Tile number `slot` of all sequences'.  Late tiles have most work (LATE: tiles of queries), or early
// ones: of up to 64 sequences of up to kLevels tiles those with most come first, whichever sequence
// they are of, so that the last workgroups to start are the shortest (32 + 8 heads of 128, us, so /
// sequence by sequence: dk and dv of 16 sequences of 166 to 1000 tokens 141 / 180, four prompts of 800
// 36 / 42).  Of more, or longer ones, the tiles come sequence by sequence, each one's in that order.
// Up to 64 sequences a lane has everything about its own in registers, and one trip to memory is
// enough; more are looked through kAtOnce to a lane at a time, lane by lane next to each other (us, so /
// a run of them to each lane: 256 of 100 tokens, 8 heads 46 / 49, 1000 of 60 146 / 201, 4096 of 30, 4 heads
// 223 / 662).
constexpr int kLevels = 64, kAtOnce = 4;
template <bool LATE>
__device__ __forceinline__ Place place_of(const Sequences& s, int32_t slot) {
  const int lane = threadIdx.x & 63;
  struct Sequence {
    int32_t row, n, other, m;
  };
  auto sequence = [&](int i) {                   // i: in the order of the tiles
    const int b = LATE ? s.B - 1 - i : i;
    const int32_t lo = clamped(s.cu[b], s.T), hi = clamped(s.cu[b + 1], s.T);
    const int32_t lo2 = clamped(s.other[b], s.Tother), hi2 = clamped(s.other[b + 1], s.Tother);
    return Sequence{lo, hi > lo ? hi - lo : 0, lo2, hi2 > lo2 ? hi2 - lo2 : 0};
  };
  auto tiles_of = [](int32_t n) { return (n + kTile - 1) / kTile; };
  // Sums of this lane and those before it.
  auto sums = [&](int32_t v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int32_t o = __shfl_up(v, d);
      v += lane >= d ? o : 0;
    }
    return v;
  };
  Place p = {};
  p.end = scalar(clamped(s.cu[s.B], s.T));
  int i = 0;
  int32_t at = slot;                             // of those from sequence i on
  if (s.B > 64) {
    bool found = false;
    for (; i < s.B && !found;) {
      int32_t n[kAtOnce], mine = 0;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int j = i + 64 * u + lane, jj = j < s.B ? j : s.B - 1, b = LATE ? s.B - 1 - jj : jj;
        const int32_t lo = clamped(s.cu[b], s.T), hi = clamped(s.cu[b + 1], s.T);
        n[u] = j < s.B && hi > lo ? tiles_of(hi - lo) : 0;
        mine += n[u];
      }
      // Lengths that overlap may add up to any number: cut, so that 64 lanes' do not pass 31 bits.  No
      // grid has as many workgroups.
      const int32_t all = __builtin_amdgcn_readlane(sums(clamped(mine, (int32_t)kMostGroups)), 63);
      if (at >= all) {
        at -= all;
        i += 64 * kAtOnce;
        continue;
      }
      found = true;                              // these have more than `at`
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int32_t upto = sums(n[u]);
        const uint64_t here = __ballot(at >= upto - n[u] && at < upto);
        if (here) {
          const int l = (int)__builtin_ctzll(here);
          at -= __builtin_amdgcn_readlane(upto - n[u], l);
          i += l;
          break;
        }
        at -= __builtin_amdgcn_readlane(upto, 63);
        i += 64;
      }
    }
    if (!found) {
      p.b = -1;
      p.tile = at;
      return p;
    }
    const Sequence q = sequence(i);
    p.row = scalar(q.row), p.n = scalar(q.n), p.other = scalar(q.other), p.m = scalar(q.m);
  } else {
    const Sequence mine = lane < s.B ? sequence(lane) : Sequence{};
    const int32_t count = tiles_of(mine.n), upto = sums(count);
    const int32_t total = __builtin_amdgcn_readlane(upto, 63);
    if (slot >= total) {
      p.b = -1;
      p.tile = slot - total;
      return p;
    }
    if (__ballot(count > kLevels) == 0 && __popcll(__ballot(count > 0)) > 1) {
      // Tile `at` counted from the one with most work: tiles with as many behind them in their
      // sequence as a level says, from the highest level on.
      int32_t left = slot, most = 0;
#pragma unroll
      for (int bit = kLevels; bit > 0; bit /= 2)
        if (__ballot(count >= most + bit)) most += bit;
      uint64_t mask = 0;
      for (at = most - 1; at >= 0; --at) {       // ends before: slot < total
        mask = __ballot(count > at);
        const int n = __popcll(mask);
        if (left < n) break;
        left -= n;
      }
      const bool here = (mask >> lane & 1) && __popcll(mask & ((1ull << lane) - 1)) == left;
      i = (int)__builtin_ctzll(__ballot(here));
      at = __builtin_amdgcn_readlane(count, i) - 1 - at;
    } else {
      i = (int)__builtin_ctzll(__ballot(slot >= upto - count && slot < upto));
      at = slot - __builtin_amdgcn_readlane(upto - count, i);
    }
    p.row = __builtin_amdgcn_readlane(mine.row, i), p.n = __builtin_amdgcn_readlane(mine.n, i);
    p.other = __builtin_amdgcn_readlane(mine.other, i), p.m = __builtin_amdgcn_readlane(mine.m, i);
  }
  p.b = LATE ? s.B - 1 - i : i;
  p.tile = LATE ? tiles_of(p.n) - 1 - at : at;
  return p;
}

// Tiles that a grid has room for: every sequence may end in a tile of its own.  Those behind the
// last one are as many as the rows behind the last sequence fill, at least.
inline int64_t tile_slots(int64_t T, int64_t B) { return (T + B * (kTile - 1) + kTile - 1) / kTile; }

// ------------------------------------------------------------------------- host

inline bool aligned(const void* p, uintptr_t a) {
  return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}
inline bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na > 0 && nb > 0 && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

// Tiles of queries of all heads, and a tile's steps of keys, for sequences of average length.
inline int64_t query_tiles(int64_t B, int64_t T, int64_t Hq) {
  return B * ((T + B * kTile - 1) / (B * kTile)) * Hq;
}
inline int64_t steps_of_tile(int64_t B, int64_t T, int64_t Tk) {
  return std::max(Tk - T / 2, Tk / 2) / B / kStep;
}

// Parts that a query tile's keys are cut into, each a workgroup's: as many as let `slots` workgroups run
// at once, but four steps of 64 keys for each, on average.  What a part costs the join goes by the rows,
// what it saves by the steps: with time a steps / n + b rows n, n = sqrt(a / b steps / rows) is best.  a / b =
// 8192: over twelve sizes, of 10 to 3500 queries of 4 to 32 heads on 1000 to 65536 keys, an eighth of it takes up
// to 1.6 times as long (4 + 1 heads of 128, prompts of 3000 and 500 tokens: 53 / 34 us), eight times it
// as long within 4 %.  Lengths are taken as the average over B: empty sequences make calls look shorter.
constexpr int64_t kMostParts = 16;
inline int64_t key_parts(int64_t B, int64_t T, int64_t Tk, int64_t Hq, int64_t slots) {
  if (B < 1 || T < 1) return 1;
  const int64_t groups = query_tiles(B, T, Hq), steps = steps_of_tile(B, T, Tk);
  const int64_t best = std::lround(std::sqrt(8192.0 * (double)steps / ((double)T * (double)Hq)));
  return std::max<int64_t>(1, std::min<int64_t>({slots / groups, steps / 4, best, kMostParts}));
}

// T tokens of H rows of D elements of 16 bits, at token and head strides.
struct Rows {
  const void* p;
  int64_t T, H, D, st, sh;
  int64_t bytes() const { return T > 0 ? ((T - 1) * st + (H - 1) * sh + D) * 2 : 0; }
};

// Whether two sets of rows share an element (told exactly for heads that lie within a token's
// stride, as views of one fused buffer do; otherwise by their ranges).
inline bool overlap(const Rows& a, const Rows& b) {
  if (!overlap(a.p, a.bytes(), b.p, b.bytes())) return false;
  const int64_t wa = ((a.H - 1) * a.sh + a.D) * 2, wb = ((b.H - 1) * b.sh + b.D) * 2, s = a.st * 2;
  if (a.st != b.st || a.T < 2 || b.T < 2 || wa > s || wb > s) return true;
  const intptr_t pa = reinterpret_cast<intptr_t>(a.p), pb = reinterpret_cast<intptr_t>(b.p);
  const int64_t off = ((pb - pa) % s + s) % s;   // b's heads start here in a's token
  return off < wa || (off != 0 && s - off < wb);
}

// Rows that are written must not share an element among themselves.
inline bool self_overlap(const Rows& r) {
  const bool tokens_outside = (r.T < 2 || r.st >= (r.H - 1) * r.sh + r.D) && (r.H < 2 || r.sh >= r.D);
  const bool heads_outside = (r.H < 2 || r.sh >= (r.T - 1) * r.st + r.D) && (r.T < 2 || r.st >= r.D);
  return !tokens_outside && !heads_outside;
}

// {token, head} strides in elements.
inline int check_strides(const int64_t* strides, int n) {
  for (int i = 0; i < n; ++i) {
    if (strides[i] < 0) return FAGQ_E_SHAPE;
    if (strides[i] >= (i % 2 ? 1ll << 31 : 1ll << 24)) return FAGQ_E_TOO_LARGE;
    if (strides[i] % 8 != 0) return FAGQ_E_ALIGN;
  }
  return FAGQ_OK;
}

inline int check_sizes(int64_t B, int64_t T, int64_t Tk, int64_t Hq, int64_t H, int64_t D) {
  if (B < 0 || T < 0 || Tk < 0 || H < 1 || Hq < H || Hq % H != 0 || (D != 64 && D != 128 && D != 256))
    return FAGQ_E_SHAPE;
  if (B > (1ll << 24) || T > kMostTokens || Tk > kMostTokens || Hq > 4096 ||
      tile_slots(T, B) * Hq >= kMostGroups)
    return FAGQ_E_TOO_LARGE;
  return FAGQ_OK;
}

}  // namespace prompt
}  // namespace fagq
