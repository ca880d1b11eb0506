// batch_tables.hip - the index tensors of a step from its requests' lengths (include/fagq_cache.h).
//
// Everything follows from running sums over the requests, of new tokens, new pages and keys.  One
// launch: every workgroup works the sums out for itself (8 bytes a request, from L2) and then writes
// its share of the tokens and of the new pages, so none waits for another.
//
// Bound by latency: the lengths, then a page of the table, each a trip to memory, and between them one
// exchange of sums (the page that a request's first new token goes to is read ahead of it, by the
// thread that has the request, so that a decode step needs no search).  256 requests of one token: 5.1 us
// in the kernel, 64 of 16384 tokens 9.2 (7.6 MB written).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fagq.h"
#include "fagq_cache.h"
#include "fagq_dispatch.hpp"

namespace fagq {
namespace tables {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kEach = 4;                        // requests of a thread, at most
constexpr int kRequests = kThreads * kEach;     // of a pass
constexpr int kRun = 4;                         // tokens that a thread writes at a time
constexpr int64_t kMostGroups = 1024;           // workgroups: four on each CU
constexpr int64_t kTokensEach = kThreads * kRun;   // of a workgroup, at least
constexpr int32_t kMost = 0x7fffffff;

struct Args {
  const void* context;
  const void* fresh;
  const int32_t* free_pages;
  const int32_t* free_start;
  int32_t* table;
  int32_t* cu;
  int32_t* cu_k;
  int32_t* lens;
  int32_t* positions;
  int64_t* slots;
  int32_t* free_end;
  int64_t num_free, width;
  int32_t B, rows, shift, idx64;
  int32_t wide;              // positions and slots are 16-byte aligned
};

__device__ __forceinline__ int64_t length(const void* p, int idx64, int b, int64_t most) {
  const int64_t n = idx64 ? static_cast<const int64_t*>(p)[b]
                          : (int64_t) static_cast<const int32_t*>(p)[b];
  return n < 0 ? 0 : n < most ? n : most;
}

// Three sums at once: of the threads before this one, and of all.
struct Sums {
  int64_t tokens, pages, keys;
};
__device__ __forceinline__ Sums operator+(const Sums& a, const Sums& b) {
  return {a.tokens + b.tokens, a.pages + b.pages, a.keys + b.keys};
}
__device__ __forceinline__ Sums before(const Sums& mine, Sums (&waves)[kWaves], Sums* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Sums v = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const Sums o = {__shfl_up(v.tokens, d), __shfl_up(v.pages, d), __shfl_up(v.keys, d)};
    if (lane >= d) v = v + o;
  }
  __syncthreads();                              // the last sums have been read
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  v = {v.tokens - mine.tokens, v.pages - mine.pages, v.keys - mine.keys};
  *all = {};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) v = v + waves[w];
    *all = *all + waves[w];
  }
  return v;
}

// The request b of n with first[b] <= i < first[b + 1], where first[0] <= i < first[n].
template <typename T>
__device__ __forceinline__ int owner(const T* first, int n, T i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kThreads) void batch_tables(Args a) {
  __shared__ Sums waves[kWaves];
  __shared__ int32_t row[kRequests + 1], context[kRequests], have[kRequests];
  __shared__ int64_t page[kRequests + 1];       // new pages of the requests before
  const int tid = threadIdx.x, groups = gridDim.x, me = blockIdx.x;
  const int64_t each = (((int64_t)a.rows + groups - 1) / groups + kRun - 1) / kRun * kRun;
  const int64_t lo = me * each < a.rows ? me * each : a.rows, hi = lo + each < a.rows ? lo + each : a.rows;
  const int64_t start = a.free_start ? (a.free_start[0] > 0 ? a.free_start[0] : 0) : 0;
  const int64_t unit = 1ll << a.shift;
  Sums so_far = {};
  auto pages_of = [&](int64_t tokens) { return std::min(a.width, (tokens + unit - 1) >> a.shift); };
  auto free_page = [&](int64_t i) {
    i += start;
    return i < a.num_free ? a.free_pages[i] : -1;
  };
  auto put = [&](int64_t r, int64_t at, int64_t p) {
    a.positions[r] = (int32_t)(at < kMost ? at : kMost);
    a.slots[r] = p < 0 ? -1 : (p << a.shift) + (at & (unit - 1));
  };
  if (me == 0 && tid == 0) a.cu[0] = a.cu_k[0] = 0;
  for (int b0 = 0; b0 < a.B; b0 += kRequests) {
    const int n = a.B - b0 < kRequests ? a.B - b0 : kRequests, k = (n + kThreads - 1) / kThreads;
    const int s0 = tid * k;                     // this thread's requests: s0 .. s0 + k - 1
    int64_t ctx[kEach], mine[kEach];
    int32_t next[kEach];                        // the page that the first new token goes to, if it is there
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const bool live = i < k && s0 + i < n;
      ctx[i] = live ? length(a.context, a.idx64, b0 + s0 + i, kMost) : 0;
      mine[i] = live ? length(a.fresh, a.idx64, b0 + s0 + i, a.rows) : 0;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      next[i] = mine[i] > 0 && (ctx[i] >> a.shift) < pages_of(ctx[i])
                    ? a.table[(int64_t)(b0 + s0 + i) * a.width + (ctx[i] >> a.shift)] : -1;
    auto sums = [&] {
      Sums t = {};
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int64_t len = ctx[i] + mine[i] < kMost ? ctx[i] + mine[i] : kMost;
        t = t + Sums{mine[i], pages_of(len) - pages_of(ctx[i]), i < k && s0 + i < n ? len : 0};
      }
      return t;
    };
    Sums all, from = before(sums(), waves, &all);
    if (so_far.tokens + all.tokens > a.rows) {
      // Rows behind the last one there is room for are no part of this step.
      int64_t at = so_far.tokens + from.tokens;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int64_t room = a.rows > at ? a.rows - at : 0;
        at += mine[i];
        mine[i] = mine[i] < room ? mine[i] : room;
      }
      from = before(sums(), waves, &all);
    }
    __syncthreads();                            // the last requests' tables have been read
    Sums at = so_far + from;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int s = s0 + i;
      if (i < k && s < n) {
        const int64_t len = ctx[i] + mine[i] < kMost ? ctx[i] + mine[i] : kMost;
        const int64_t old = pages_of(ctx[i]);
        row[s] = (int32_t)at.tokens;
        page[s] = at.pages;
        context[s] = (int32_t)ctx[i];
        have[s] = (int32_t)old;
        if (mine[i] > 0 && at.tokens >= lo && at.tokens < hi) {
          const int64_t first = ctx[i] >> a.shift;
          put(at.tokens, ctx[i], first < old ? next[i] : first < a.width ? free_page(at.pages + (first - old)) : -1);
        }
        at = at + Sums{mine[i], pages_of(len) - old, len};
        if (me == 0) {
          a.cu[b0 + s + 1] = (int32_t)at.tokens;
          a.cu_k[b0 + s + 1] = (int32_t)(at.keys < kMost ? at.keys : kMost);
          a.lens[b0 + s] = (int32_t)len;
        }
      }
    }
    const Sums end = so_far + all;
    if (tid == 0) {
      row[n] = (int32_t)end.tokens;
      page[n] = end.pages;
    }
    bool two = false;                           // whether some request has two new tokens
#pragma unroll
    for (int i = 0; i < kEach; ++i) two |= mine[i] > 1;
    const bool more = __syncthreads_or(two);
    // Tokens behind their request's first.
    const int64_t stop = end.tokens < hi ? end.tokens : hi;
    for (int64_t r0 = lo + tid * kRun; more && r0 < stop; r0 += kThreads * kRun) {
      const int64_t r1 = r0 + kRun < stop ? r0 + kRun : stop;
      int64_t r = r0 > so_far.tokens ? r0 : so_far.tokens;
      if (r >= r1) continue;
      int s = owner(row, n, (int32_t)r);
      const bool whole = r == r0 && r1 == r0 + kRun && a.wide;
      int32_t positions[kRun];
      int64_t slots[kRun];
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        if (r0 + i < r || r0 + i >= r1) continue;
        while (r0 + i >= row[s + 1]) ++s;       // ends: row[n] is larger
        const int64_t at = (int64_t)context[s] + (r0 + i - row[s]), g = at >> a.shift;
        int64_t p = -1;
        if (g < have[s]) p = a.table[(int64_t)(b0 + s) * a.width + g];
        else if (g < a.width) p = free_page(page[s] + (g - have[s]));
        if (!whole) put(r0 + i, at, p);
        positions[i] = (int32_t)(at < kMost ? at : kMost);
        slots[i] = p < 0 ? -1 : (p << a.shift) + (at & (unit - 1));
      }
      if (whole) {
        typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
        typedef int64_t i64x2 __attribute__((ext_vector_type(2)));
        *reinterpret_cast<i32x4*>(a.positions + r0) = i32x4{positions[0], positions[1], positions[2], positions[3]};
        *reinterpret_cast<i64x2*>(a.slots + r0) = i64x2{slots[0], slots[1]};
        *reinterpret_cast<i64x2*>(a.slots + r0 + 2) = i64x2{slots[2], slots[3]};
      }
    }
    const int64_t first = so_far.pages + all.pages * me / groups;
    const int64_t last = so_far.pages + all.pages * (me + 1) / groups;
    for (int64_t f = first + tid; f < last; f += kThreads) {
      const int s = owner(page, n, f);
      a.table[(int64_t)(b0 + s) * a.width + have[s] + (f - page[s])] = free_page(f);
    }
    so_far = end;
  }
  for (int64_t r = (so_far.tokens > lo ? so_far.tokens : lo) + tid; r < hi; r += kThreads) {
    a.positions[r] = -1;
    a.slots[r] = -1;
  }
  if (me == 0 && tid == 0)
    a.free_end[0] = (int32_t)(start + so_far.pages < kMost ? start + so_far.pages : kMost);
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na > 0 && nb > 0 && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

}  // namespace
}  // namespace tables
}  // namespace fagq

extern "C" {

FAGQ_API int fagq_batch_tables_launch(
    const void* context_lens, const void* new_lens, const int32_t* free_pages,
    const int32_t* free_start, int32_t* page_table, int32_t* cu_seqlens, int32_t* cu_seqlens_k,
    int32_t* kv_lens, int32_t* positions, int64_t* slots, int32_t* free_end, int64_t B,
    int64_t rows, int64_t num_free, int64_t page_size, int64_t table_width, int index_dtype,
    void* stream) {
  using namespace fagq;
  using namespace fagq::tables;
  if (B < 0 || rows < 0 || num_free < 0 || table_width < 0 || page_size < FAGQ_CACHE_MIN_PAGE ||
      (page_size & (page_size - 1)) != 0)
    return FAGQ_E_SHAPE;
  if (!cu_seqlens || !cu_seqlens_k || !free_end || (B > 0 && (!context_lens || !new_lens || !kv_lens)) ||
      (rows > 0 && (!positions || !slots)) || (num_free > 0 && !free_pages) ||
      (B > 0 && table_width > 0 && !page_table))
    return FAGQ_E_NULL;
  if (index_dtype != FAGQ_IDX_I32 && index_dtype != FAGQ_IDX_I64) return FAGQ_E_FORMAT;
  if (page_size > FAGQ_CACHE_MAX_PAGE || B > (1ll << 24) || rows > (1ll << 31) - 1 ||
      num_free > (1ll << 31) - 1 || table_width > (1ll << 31) - 1)
    return FAGQ_E_TOO_LARGE;
  const int64_t is = index_dtype == FAGQ_IDX_I64 ? 8 : 4;
  const void* ins[4] = {context_lens, new_lens, free_pages, free_start};
  const int64_t nin[4] = {B * is, B * is, num_free * 4, free_start ? 4 : 0};
  const void* outs[7] = {page_table, cu_seqlens, cu_seqlens_k, kv_lens, positions, slots, free_end};
  const int64_t nout[7] = {B * table_width * 4, (B + 1) * 4, (B + 1) * 4, B * 4, rows * 4, rows * 8, 4};
  for (int i = 0; i < 4; ++i)
    if (!aligned(ins[i], i < 2 ? is : 4)) return FAGQ_E_ALIGN;
  for (int i = 0; i < 7; ++i) {
    if (!aligned(outs[i], i == 5 ? 8 : 4)) return FAGQ_E_ALIGN;
    for (int j = 0; j < 4; ++j)
      if (overlap(outs[i], nout[i], ins[j], nin[j])) return FAGQ_E_ALIAS;
    for (int j = 0; j < i; ++j)
      if (overlap(outs[i], nout[i], outs[j], nout[j])) return FAGQ_E_ALIAS;
  }
  const int dcheck = device_check();
  if (dcheck != FAGQ_OK) return dcheck;
  Args a = {context_lens, new_lens,  free_pages, free_start, page_table, cu_seqlens,
            cu_seqlens_k, kv_lens,   positions,  slots,      free_end,   num_free,
            table_width,  (int32_t)B, (int32_t)rows, 0, index_dtype == FAGQ_IDX_I64, 0};
  while ((1ll << a.shift) < page_size) ++a.shift;
  a.wide = aligned(positions, 16) && aligned(slots, 16);
  void* args[] = {&a};
  const int64_t groups = std::max<int64_t>(1, std::min(kMostGroups, (rows + kTokensEach - 1) / kTokensEach));
  return launch_kernel(reinterpret_cast<const void*>(&batch_tables), dim3((unsigned)groups),
                       dim3(kThreads), args, 0, static_cast<hipStream_t>(stream));
}

}  // extern "C"
