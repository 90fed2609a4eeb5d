// Address arithmetic of the paged KV cache, shared by the kernels that write, read and attend to it, and by the CPU
// test that tries it with bad pages. Plain C++: no HIP header needed.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define ZTVM_HD __host__ __device__ __forceinline__
#else
#define ZTVM_HD inline
#endif

namespace ztvm {

// x / d for x < 2^31 as one multiplication and a shift. With l = ceil(log2 d), mul = ceil(2^(31+l) / d) fits 32 bits
// (d > 2^(l-1)) and exceeds the quotient by e/d, e < d <= 2^l: the error x*e/(d*2^(31+l)) stays below 1/d.
struct FastDiv {
  uint32_t d, mul, shift;
};
inline FastDiv make_fast_div(uint32_t d) {
  uint32_t l = 0;
  while (l < 32 && (1ull << l) < d) l++;
  FastDiv f;
  f.d = d;
  f.shift = 31 + l;
  f.mul = (uint32_t)(((1ull << (31 + l)) + d - 1) / d);
  return f;
}
ZTVM_HD uint32_t fast_div(const FastDiv& f, uint32_t x) { return (uint32_t)(((uint64_t)x * f.mul) >> f.shift); }

// Both formats as byte strides: row (page, head, slot, side) starts at page*page_bytes + head*head_bytes +
// slot*slot_bytes + side*side_bytes behind `pages`. All offsets of a row are 64 bits wide: a long cache passes 4 GiB.
struct KvView {
  char* pages;      // page 0
  uint16_t* scales;  // scale of page 0, head 0, slot 0, K (int8 only)
  uint64_t page_bytes, head_bytes, side_bytes;
  uint32_t slot_bytes;
  uint32_t num_pages;  // pages that lie whole inside the bound memory
  uint32_t kv_heads, head_dim, page_size, int8;
  FastDiv by_page;
};

ZTVM_HD uint64_t kv_row_offset(const KvView& c, uint32_t page, uint32_t head, uint32_t slot, uint32_t side) {
  return (uint64_t)page * c.page_bytes + (uint64_t)head * c.head_bytes + (uint64_t)slot * c.slot_bytes + (uint64_t)side * c.side_bytes;
}
ZTVM_HD uint64_t kv_scale_index(const KvView& c, uint32_t page, uint32_t head, uint32_t slot, uint32_t side) {
  return (((uint64_t)page * c.kv_heads + head) * c.page_size + slot) * 2u + side;
}
// page and slot of a cache slot number; false where it is negative or outside the cache
ZTVM_HD bool kv_locate(const KvView& c, int32_t where, uint32_t& page, uint32_t& slot) {
  if (where < 0) return false;
  page = fast_div(c.by_page, (uint32_t)where);
  slot = (uint32_t)where - page * c.page_size;
  return page < c.num_pages;
}

// How many pages lie whole inside the capacities (elements / words and scales, from `pages` on).
inline uint32_t kv_whole_pages(uint64_t capacity, uint64_t offset, uint64_t stride, uint64_t used) {
  if (capacity < offset || capacity - offset < used || !stride) return 0;
  const uint64_t n = (capacity - offset - used) / stride + 1;
  return n > 0x7FFFFFFFull ? 0x7FFFFFFFu : (uint32_t)n;
}

}  // namespace ztvm
