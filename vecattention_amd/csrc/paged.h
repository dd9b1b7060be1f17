// Index arithmetic of the paged key-value cache, shared by the plan, the cache
// writes and the decode attention.  Host code compiles it too
// (tests/test_paged_host.py runs it there).
//
// A cache holds num_pages pages of page_size slots; slot s is row s % page_size
// of page s / page_size.  Row i of a block table lists the pages of request i in
// order: its token t lives in page table[i][t / page_size], row t % page_size.
#pragma once
#include "common.h"

namespace va {

// floor(n / d) for 0 <= n < 2^31 by one 32x32 multiplication: with
// s = ceil(log2 d) and m = floor(2^(31+s) / d) + 1, m*d = 2^(31+s) + e with
// 0 < e <= d <= 2^s, so n*m / 2^(31+s) = n/d + n*e / (d * 2^(31+s)), and the
// excess is below 1/d because n*e < 2^(31+s).  m < 2^32 since 2^s < 2d.
struct FastDiv {
  uint32_t d = 1, m = 0;
  int shift = 31;
  FastDiv() = default;
  __host__ explicit FastDiv(uint32_t divisor) : d(divisor) {
    int s = 0;
    while ((uint64_t(1) << s) < divisor) ++s;
    shift = 31 + s;
    m = uint32_t((uint64_t(1) << shift) / divisor + 1);
  }
  __host__ __device__ uint32_t div(uint32_t n) const {
    return uint32_t((uint64_t(n) * m) >> shift);
  }
};

// Tokens and pages of one request in a step: `len` tokens are in the cache,
// `fresh` are added, the table has room for `width` pages.  Negative lengths
// count as 0; pages past the table are not taken.
struct PlanRow {
  uint32_t len, fresh, held, need;
  __host__ __device__ PlanRow(int32_t l, int32_t n, uint32_t page, uint32_t width) {
    len = l > 0 ? uint32_t(l) : 0u;
    fresh = n > 0 ? uint32_t(n) : 0u;
    const uint32_t end = len + fresh;  // < 2^32
    held = len / page + (len % page != 0);
    uint32_t total = end / page + (end % page != 0);
    if (total > width) total = width;
    need = total > held ? total - held : 0u;
  }
};

// Pages that `len` tokens take of a table of `width` entries.
__host__ __device__ inline uint32_t held_pages(int32_t len, uint32_t page, uint32_t width) {
  if (len <= 0) return 0;
  const uint32_t n = uint32_t(len) / page + (uint32_t(len) % page != 0);
  return n < width ? n : width;
}
// The entry whose page holds tokens and has room for more, or -1: where a row's
// next token goes beside some of its own.
__host__ __device__ inline int64_t open_page(int32_t len, uint32_t page, uint32_t width) {
  if (len <= 0 || uint32_t(len) % page == 0) return -1;
  const uint32_t at = uint32_t(len) / page;
  return at < width ? int64_t(at) : -1;
}
__host__ __device__ inline bool is_page(int32_t id, int64_t pages) { return id >= 0 && id < pages; }

// Entry `at` of the list of free pages: -1 past its ends.
__host__ __device__ inline int32_t free_page(const int32_t* free_pages, int64_t count, int64_t at) {
  return at >= 0 && at < count ? free_pages[at] : -1;
}

// Slot of position `pos` of a request, or -1 where it has no page: pages it
// holds come from its table row, new ones from the free list at `first`.
__host__ __device__ inline int64_t plan_slot(const PlanRow& r, uint32_t pos, uint32_t page,
                                             uint32_t width, const int32_t* row,
                                             const int32_t* free_pages, int64_t count,
                                             int64_t first) {
  const uint32_t p = pos / page;
  if (p >= width) return -1;
  const int32_t id =
      p < r.held ? row[p] : free_page(free_pages, count, first + int64_t(p - r.held));
  return id < 0 ? -1 : int64_t(id) * page + int64_t(pos % page);
}

// Work of the decode attention.  A segment is one (request, kv head, tile of
// query heads); its keys are cut into units of `unit` keys, at least one per
// segment, so that an empty request's rows have a writer.  The units of all
// segments in order are dealt to `groups` work-groups in contiguous shares whose
// sizes differ by at most one.  Fewer than 2^31 units: a 64-bit division
// costs a wave half a microsecond.
struct PagedShare {
  uint32_t groups, each, more;  // the first `more` shares hold one unit more than `each`
  __host__ __device__ PagedShare(uint32_t total, uint32_t g)
      : groups(g), each(total / g), more(total - each * g) {}
  __host__ __device__ uint32_t begin(uint32_t w) const { return w * each + (w < more ? w : more); }
  // Work-group whose share holds unit u.
  __host__ __device__ uint32_t owner(uint32_t u) const {
    const uint32_t cut = more * (each + 1);
    return u < cut ? u / (each + 1) : more + (u - cut) / each;  // each > 0 where u >= cut
  }
};

// Keys a request's rows see: its length, 0 if negative; -1 (not a number comes
// out) when it is longer than its table row can hold.
__host__ __device__ inline int32_t paged_keys(int32_t len, int64_t capacity) {
  return len <= 0 ? 0 : int64_t(len) > capacity ? -1 : len;
}
__host__ __device__ inline uint32_t paged_units(int32_t keys, uint32_t unit) {
  return keys <= 0 ? 1 : (uint32_t(keys) + unit - 1) / unit;
}

}  // namespace va
