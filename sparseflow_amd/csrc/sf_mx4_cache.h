// The paged cache in the microscaled 4-bit format on the device.  gfx950 only.
#pragma once

#include "sf_mx4.h"

namespace sf {
namespace {

// Where a row of keys or values lies: token t of a sequence is row t % page of its page
// table[t / page]; a page holds [heads, page] rows.  -1: no such page.
__device__ __forceinline__ int64_t cache_row(const CacheView& c, const int32_t* __restrict__ table, int64_t t, int head) {
  const int64_t p = table[t >> c.page_shift];
  if (p < 0 || p >= c.pages) return -1;
  return (((p * c.heads + head) << c.page_shift)) + (t & ((1 << c.page_shift) - 1));
}

// The tokens that a sequence's table has room for.
__device__ __forceinline__ int64_t cache_room(const CacheView& c) { return (int64_t)c.width << c.page_shift; }

}  // namespace
}  // namespace sf
