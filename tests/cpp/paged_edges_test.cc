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

int main() {
  pieces();
  std::printf(failures ? "%d failures\n" : "ok\n", failures);
  return failures != 0;
}
