// What the kernels of the paged cache may read, and how their blocks share units, at the edges.
#include <cstdint>
#include <cstdio>

#include "paged_cache.h"

using namespace fbgemm_b200;

static int failures = 0;
#define CHECK(x)                                         \
  do {                                                   \
    if (!(x)) {                                          \
      std::printf("%s:%d: %s\n", __FILE__, __LINE__, #x); \
      ++failures;                                        \
    }                                                    \
  } while (0)

// The pieces of a row are its bytes, each once, and none behind its end.
static void pieces() {
  for (int row_bytes = 4; row_bytes <= 512; row_bytes += 4) {
    int sum = 0;
    for (int piece = 0; piece < 34; ++piece) {
      const int n = piece_bytes(row_bytes, piece);
      CHECK(n >= 0 && n <= 16 && (n == 0 || 16 * piece + n <= row_bytes));
      sum += n;
    }
    CHECK(sum == row_bytes);
  }
}

// Blocks' shares are all units, each once; blocks of a second set that has none, or behind the last unit, have no share.
static void blocks() {
  for (int64_t total : {1, 5, 443, 444, 4440, 17000, 17760, 17761, 60000, 1000000}) {
    for (int32_t of_block : {2, 4}) {
      for (bool two : {false, true}) {
        const int64_t blocks = 444 / of_block;
        const UnitSplit s = split_units(total, blocks * of_block, two);
        int64_t sum = 0;
        for (int64_t b = 0; b < 2 * blocks; ++b) {
          const BlockShare share = block_share(s, b, of_block, total);
          int64_t units = 0;
          int32_t active = 0;
          for (int32_t w = 0; w < of_block; ++w) {  // worker by worker
            const int64_t first = s.first(b * of_block + w), end = first + s.units_of(b * of_block + w);
            const int64_t n = (end < total ? end : total) - first;
            units += n > 0 ? n : 0;
            active += n > 0;
          }
          CHECK(share.units == units && share.active == active);
          CHECK(b < blocks || s.small > 0 || share.active == 0);
          sum += share.units;
        }
        CHECK(sum == total);
      }
    }
  }
}

// Workers of either size: where rows are waited for, with many items and long lines of units.
static void sizes() {
  for (int bits : {16, 8}) {
    CHECK(two_sizes(bits, 8, 64, 40 * 1776, 1776) && two_sizes(bits, 8, 4096, 1000 * 1776, 1776));
    CHECK(!two_sizes(bits, 8, 63, 1000 * 1776, 1776) && !two_sizes(bits, 8, 64, 40 * 1776 - 1, 1776));
    CHECK(!two_sizes(bits, 16, 4096, 1000 * 1776, 1776) && !two_sizes(bits, 32, 4096, 1000 * 1776, 1776));
  }
  CHECK(!two_sizes(4, 8, 4096, 1000 * 1776, 1776));
}

int main() {
  pieces();
  sizes();
  blocks();
  std::printf(failures ? "%d failures\n" : "ok\n", failures);
  return failures != 0;
}
