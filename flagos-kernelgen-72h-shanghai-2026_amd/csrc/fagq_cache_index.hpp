// fagq_cache_index.hpp - the index arithmetic of the paged cache, shared by its kernels and
// by the host-side diagnostic that checks it.  Indexes read from memory (page tables, lengths,
// slots) are never trusted: whatever they hold, what comes out is in range or negative.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fagq {
namespace cache {

constexpr int64_t kNoPage = -1;   // a token without a page: reads as zeros
constexpr int64_t kNoRow = -2;    // a row that belongs to no sequence: left as it was

// The sequence b with cu[b] <= r < cu[b + 1], -1 if r lies outside all of them.  Ends for any
// content of cu.
__host__ __device__ inline int sequence_of(const int32_t* cu, int B, int64_t r) {
  if (B < 1 || r < cu[0] || r >= cu[B]) return -1;
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (cu[mid] <= r) lo = mid;
    else hi = mid;
  }
  return r >= cu[lo] && r < cu[lo + 1] ? lo : -1;
}

// The slot (page * page_size + offset) of token j >= 0 of a list of `width` pages.
__host__ __device__ inline int64_t slot_of(const int32_t* pages, int64_t width, int64_t num_pages,
                                           int page_shift, int64_t j) {
  const int64_t p = j >> page_shift;
  if (p >= width) return kNoPage;
  const int64_t page = pages[p];
  if (page < 0 || page >= num_pages) return kNoPage;
  return (page << page_shift) + (j & ((1 << page_shift) - 1));
}

// The slot that row r of a gathered batch reads, kNoPage or kNoRow.
__host__ __device__ inline int64_t gathered_slot(const int32_t* cu, const int32_t* table, int B,
                                                 int64_t width, int64_t num_pages, int page_shift,
                                                 int64_t r) {
  const int b = sequence_of(cu, B, r);
  if (b < 0) return kNoRow;
  return slot_of(table + (int64_t)b * width, width, num_pages, page_shift, r - cu[b]);
}

// How many of its own tokens query s of the newest S of a sequence of kv_len tokens sees, where
// no more than `most` of them are read.
__host__ __device__ inline int64_t seen_tokens(int64_t kv_len, int64_t most, int S, int s) {
  const int64_t read = kv_len < 0 ? 0 : kv_len < most ? kv_len : most;
  const int64_t n = read - S + s + 1;
  return n > 0 ? n : 0;
}

}  // namespace cache
}  // namespace fagq
