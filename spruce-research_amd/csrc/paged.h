// The ragged batch over a paged K/V cache that the append and the chunk
// attention share, and the lookups in it.
#pragma once

#include "common.h"

namespace spruce {

// x / d == (x * magic) >> shift for 0 <= x < 2^31.  With l = ceil(log2(d)),
// magic = floor(2^(31 + l) / d) + 1 exceeds 2^(31 + l) / d by at most 1, so
// x * magic / 2^(31 + l) exceeds x / d by less than 2^-l <= 1 / d: the floor is
// the same.
struct Divisor {
  uint32_t magic;
  int shift;
  __device__ __forceinline__ int of(int x) const { return (int)(((uint64_t)(uint32_t)x * magic) >> shift); }
};
inline Divisor divisor(int64_t d) {  // 1 <= d < 2^31
  int l = 0;
  while (((int64_t)1 << l) < d) ++l;
  return Divisor{(uint32_t)((((uint64_t)1 << (31 + l)) / (uint64_t)d) + 1), 31 + l};
}

// Sequences s = 0..S-1 with their new tokens at rows q_starts[s] ..
// q_starts[s + 1) of the packed tensors and kv_lens[s] cached keys, those of
// the new tokens included: new token i stands at position kv_lens[s] - n + i
// of n.  Position p lies in slot p % page of page page_table[s][p / page].
// Everything is read on the device; what a caller may have wrong there (a
// page outside [0, pages), lengths past the table, starts past the packed
// rows) is bounded where it is read and never addresses memory.
struct PagedBatch {
  const int32_t* table;
  int64_t table_stride;
  const int32_t* q_starts;
  const int32_t* kv_lens;
  int S, N, page, pages;
  int cap;  // positions the table holds: width * page
  Divisor by_page;
};

inline int prepare_batch(PagedBatch& b, const int32_t* table, int64_t table_stride, int64_t width,
                         const int32_t* q_starts, const int32_t* kv_lens, int64_t S, int64_t N, int64_t page,
                         int64_t pages) {
  SPRUCE_REQUIRE((table || width == 0) && q_starts && kv_lens, "page_table, q_starts and kv_lens must be non-null device pointers");
  SPRUCE_REQUIRE(S >= 1 && S < (int64_t)1 << 20, "sequences must be in [1, 2^20), got %lld", (long long)S);
  SPRUCE_REQUIRE(N >= 0 && N < (int64_t)1 << 30, "invalid token count %lld", (long long)N);
  SPRUCE_REQUIRE(page >= 1 && page < (int64_t)1 << 30, "invalid page size %lld", (long long)page);
  SPRUCE_REQUIRE(pages >= 0 && pages < (int64_t)1 << 31, "invalid page count %lld", (long long)pages);
  // (Stride 0: one row for all sequences.)
  SPRUCE_REQUIRE(width >= 0 && (table_stride == 0 || table_stride >= width), "page_table rows (%lld) overlap (stride %lld)",
                 (long long)width, (long long)table_stride);
  // The kernels reach up to a tile past the last position in 32 bits.
  SPRUCE_REQUIRE(width <= (((int64_t)1 << 31) - 1024) / page, "page_table covers 2^31 - 1024 positions or more");
  b.table = table;
  b.table_stride = table_stride;
  b.q_starts = q_starts;
  b.kv_lens = kv_lens;
  b.S = (int)S;
  b.N = (int)N;
  b.page = (int)page;
  b.pages = (int)pages;
  b.cap = (int)(width * page);
  b.by_page = divisor(page);
  return SPRUCE_OK;
}

// Whether no two of the rows of D values that a call writes share memory: `n`
// dims of sizes[i] rows at strides[i], in whatever order; each dim of more than
// one row has to step over all that those with smaller strides span.  (Dims that
// interleave without meeting are taken for overlapping.)
inline bool rows_apart(const int64_t* strides, const int64_t* sizes, int n, int64_t D) {
  int order[4], dims = 0;
  for (int i = 0; i < n; ++i) {
    if (sizes[i] == 0) return true;
    if (sizes[i] == 1) continue;
    int at = dims++;
    for (; at > 0 && strides[order[at - 1]] > strides[i]; --at) order[at] = order[at - 1];
    order[at] = i;
  }
  int64_t span = D;
  for (int i = 0; i < dims; ++i) {
    const int64_t stride = strides[order[i]];
    int64_t steps;
    if (stride < span || __builtin_mul_overflow(sizes[order[i]] - 1, stride, &steps) ||
        __builtin_add_overflow(steps, span, &span))
      return false;
  }
  return true;
}

__device__ __forceinline__ int page_of(const PagedBatch& b, int pos) { return b.by_page.of(pos); }

// q_starts[s] brought into range.
__device__ __forceinline__ int clamp_start(const PagedBatch& b, int v) { return v < 0 ? 0 : (v > b.N ? b.N : v); }

// The table's entry for position pos (0 <= pos < cap) of sequence s, and
// whether it names a page: apart, so that a caller can look entries up ahead
// and wait for them where it uses them.
__device__ __forceinline__ int page_entry(const PagedBatch& b, int s, int pos) {
  return b.table[(int64_t)s * b.table_stride + page_of(b, pos)];
}
__device__ __forceinline__ bool is_page(const PagedBatch& b, int entry) { return (uint32_t)entry < (uint32_t)b.pages; }

// The sequence of packed row n, wave-uniform: the starts at or below n are
// counted 64 at a time.  -1 for rows before the first or behind the last.
__device__ __forceinline__ int sequence_of(const PagedBatch& b, int n, int lane) {
  int below = 0;
  for (int s0 = 0; s0 <= b.S; s0 += 64) {
    const int s = s0 + lane;
    below += __builtin_popcountll(__ballot(s <= b.S && b.q_starts[s] <= n));
  }
  return below == 0 || below > b.S ? -1 : below - 1;
}

}  // namespace spruce
