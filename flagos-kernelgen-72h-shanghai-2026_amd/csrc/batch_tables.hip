// batch_tables.hip - the index tensors of a step from its requests' lengths (include/fagq_cache.h).
//
// Everything follows from two running sums over the requests, of new tokens and of new pages.  One
// launch: every workgroup works the sums out for itself (8 bytes a request, from L2) and then writes
// its share of the tokens and of the new pages, so none waits for another.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fagq.h"
#include "fagq_cache.h"
#include "fagq_dispatch.hpp"

namespace fagq {
namespace tables {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int64_t kMostGroups = 256;            // workgroups: one on each CU
constexpr int64_t kTokensEach = 2048;           // of a workgroup, at least
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
};

__device__ __forceinline__ int64_t length(const void* p, int idx64, int b, int64_t most) {
  const int64_t n = idx64 ? static_cast<const int64_t*>(p)[b]
                          : (int64_t) static_cast<const int32_t*>(p)[b];
  return n < 0 ? 0 : n < most ? n : most;
}

// Inclusive sum over the workgroup's threads.
__device__ __forceinline__ int64_t scan(int64_t v, int64_t (&sums)[kWaves]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t o = __shfl_up(v, d);
    v += lane >= d ? o : 0;
  }
  __syncthreads();                              // the last sums have been read
  if (lane == 63) sums[wave] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v += w < wave ? sums[w] : 0;
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
  __shared__ int64_t sums[kWaves];
  __shared__ int32_t row[kThreads + 1], context[kThreads], have[kThreads];
  __shared__ int64_t page[kThreads + 1];        // new pages of the requests before
  const int tid = threadIdx.x, groups = gridDim.x, me = blockIdx.x;
  const int32_t each = (a.rows + groups - 1) / groups;
  const int64_t lo = (int64_t)me * each, hi = lo + each < a.rows ? lo + each : a.rows;
  const int64_t start = a.free_start ? (a.free_start[0] > 0 ? a.free_start[0] : 0) : 0;
  int64_t rows = 0, pages = 0, keys = 0;        // of the requests so far
  auto free_page = [&](int64_t i) {
    i += start;
    return i < a.num_free ? a.free_pages[i] : -1;
  };
  if (me == 0 && tid == 0) a.cu[0] = a.cu_k[0] = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + tid, n = a.B - b0 < kThreads ? a.B - b0 : kThreads;
    const int64_t ctx = b < a.B ? length(a.context, a.idx64, b, kMost) : 0;
    const int64_t want = b < a.B ? length(a.fresh, a.idx64, b, a.rows) : 0;
    // Rows behind the last one there is room for are no part of this step.
    const int64_t upto = rows + scan(want, sums), from = upto - want;
    const int64_t end = upto < a.rows ? upto : a.rows, mine = end - (from < a.rows ? from : a.rows);
    const int64_t len = ctx + mine < kMost ? ctx + mine : kMost;
    const int64_t unit = 1ll << a.shift;
    const int64_t old = std::min(a.width, (ctx + unit - 1) >> a.shift);
    const int64_t all = std::min(a.width, (len + unit - 1) >> a.shift);
    const int64_t need = all > old ? all - old : 0;
    const int64_t pages_upto = pages + scan(need, sums);
    const int64_t keys_upto = keys + scan(b < a.B ? len : 0, sums);
    __syncthreads();                            // the last requests' have been read
    if (tid == 0) {
      row[0] = (int32_t)rows;
      page[0] = pages;
    }
    row[tid + 1] = (int32_t)end;
    page[tid + 1] = pages_upto;
    context[tid] = (int32_t)ctx;
    have[tid] = (int32_t)old;
    if (me == 0 && b < a.B) {
      a.cu[b + 1] = (int32_t)end;
      a.cu_k[b + 1] = (int32_t)(keys_upto < kMost ? keys_upto : kMost);
      a.lens[b] = (int32_t)len;
    }
    __syncthreads();
    const int64_t stop = row[n] < hi ? row[n] : hi;
    for (int64_t r = (rows > lo ? rows : lo) + tid; r < stop; r += kThreads) {
      const int s = owner(row, n, (int32_t)r);
      const int64_t at = (int64_t)context[s] + (r - row[s]), i = at >> a.shift;
      int64_t p = -1;
      if (i < have[s]) p = a.table[(int64_t)(b0 + s) * a.width + i];
      else if (i < a.width) p = free_page(page[s] + (i - have[s]));
      a.positions[r] = (int32_t)(at < kMost ? at : kMost);
      a.slots[r] = p < 0 ? -1 : (p << a.shift) + (at & (unit - 1));
    }
    const int64_t fresh = page[n] - page[0];
    const int64_t first = page[0] + fresh * me / groups, last = page[0] + fresh * (me + 1) / groups;
    for (int64_t f = first + tid; f < last; f += kThreads) {
      const int s = owner(page, n, f);
      a.table[(int64_t)(b0 + s) * a.width + have[s] + (f - page[s])] = free_page(f);
    }
    rows = row[n];
    pages = page[n];
    // The last scan's sums are still there.
#pragma unroll
    for (int w = 0; w < kWaves; ++w) keys += sums[w];
  }
  for (int64_t r = (rows > lo ? rows : lo) + tid; r < hi; r += kThreads) {
    a.positions[r] = -1;
    a.slots[r] = -1;
  }
  if (me == 0 && tid == 0) a.free_end[0] = (int32_t)(start + pages < kMost ? start + pages : kMost);
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
            table_width,  (int32_t)B, (int32_t)rows, 0, index_dtype == FAGQ_IDX_I64};
  while ((1ll << a.shift) < page_size) ++a.shift;
  void* args[] = {&a};
  const int64_t groups = std::max<int64_t>(1, std::min(kMostGroups, (rows + kTokensEach - 1) / kTokensEach));
  return launch_kernel(reinterpret_cast<const void*>(&batch_tables), dim3((unsigned)groups),
                       dim3(kThreads), args, 0, static_cast<hipStream_t>(stream));
}

}  // extern "C"
