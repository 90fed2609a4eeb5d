// The page arithmetic of the kernels, on the CPU: division by any page size, bad slots and pages, 64-bit offsets.
#include "../../zero-tvm_amd/csrc/kv_cache.h"

#include <cstdio>
#include <cstdlib>

using namespace ztvm;

#define CHECK(x)                                             \
  do {                                                       \
    if (!(x)) {                                              \
      std::printf("failed at line %d: %s\n", __LINE__, #x);  \
      std::exit(1);                                          \
    }                                                        \
  } while (0)

int main() {
  const uint32_t divisors[] = {1, 2, 3, 5, 7, 12, 16, 17, 31, 48, 64, 100, 127, 128, 255, 256, 1000, 4097, 65535, 65536, 1000003, 0x40000000u, 0x7FFFFFFEu, 0x7FFFFFFFu};
  const uint32_t values[] = {0, 1, 2, 3, 15, 16, 17, 99, 100, 4095, 4096, 65534, 65535, 65536, 1234567, 0x3FFFFFFFu, 0x40000000u, 0x7FFFFFFDu, 0x7FFFFFFEu, 0x7FFFFFFFu};
  for (uint32_t d : divisors) {
    const FastDiv f = make_fast_div(d);
    for (uint32_t x : values) CHECK(fast_div(f, x) == x / d);
    for (uint32_t k = 1; k < 400; k++) {  // around multiples
      const uint64_t m = (uint64_t)d * k;
      for (uint64_t x = m ? m - 1 : 0; x <= m + 1 && x < 0x80000000ull; x++) CHECK(fast_div(f, (uint32_t)x) == x / d);
    }
    for (uint32_t k = 0; k < 3; k++) {
      const uint64_t m = (0x7FFFFFFFull / d - k) * d;
      if (m && m < 0x80000000ull) CHECK(fast_div(f, (uint32_t)m) == m / d && fast_div(f, (uint32_t)m - 1) == (m - 1) / d);
    }
  }
  KvView c{};
  c.page_size = 16;
  c.num_pages = 5;
  c.by_page = make_fast_div(16);
  uint32_t page, slot;
  CHECK(kv_locate(c, 0, page, slot) && page == 0 && slot == 0);
  CHECK(kv_locate(c, 79, page, slot) && page == 4 && slot == 15);
  CHECK(!kv_locate(c, 80, page, slot));
  CHECK(!kv_locate(c, -1, page, slot));
  CHECK(!kv_locate(c, 0x7FFFFFFF, page, slot));
  CHECK(!kv_locate(c, -0x7FFFFFFF - 1, page, slot));
  // a long cache: offsets past 32 bits
  c.kv_heads = 8;
  c.page_bytes = 65536;
  c.head_bytes = 4096;
  c.side_bytes = 32768;
  c.slot_bytes = 256;
  CHECK(kv_row_offset(c, 1000000, 7, 15, 1) == 1000000ull * 65536 + 7 * 4096 + 15 * 256 + 32768);
  CHECK(kv_scale_index(c, 50000000, 7, 15, 1) == ((50000000ull * 8 + 7) * 16 + 15) * 2 + 1);
  // whole pages only
  CHECK(kv_whole_pages(100, 0, 30, 30) == 3);
  CHECK(kv_whole_pages(100, 0, 30, 10) == 4);
  CHECK(kv_whole_pages(100, 10, 30, 30) == 3);
  CHECK(kv_whole_pages(100, 11, 30, 30) == 2);
  CHECK(kv_whole_pages(29, 0, 30, 30) == 0);
  CHECK(kv_whole_pages(30, 31, 30, 30) == 0);
  CHECK(kv_whole_pages(~0ull, 0, 1, 1) == 0x7FFFFFFFu);
  std::printf("kv cache arithmetic ok\n");
  return 0;
}
