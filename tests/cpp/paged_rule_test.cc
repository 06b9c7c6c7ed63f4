// How paged attention is split over workers: every unit of every request belongs to one worker, and the worker that
// begins an item names as many followers as there are.
#include <cstdint>
#include <cstdio>
#include <vector>

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

int main() {
  // rows that a token sees
  CHECK(span_of(0, 0, 100).first == 0 && span_of(0, 0, 100).end == 0);
  CHECK(span_of(-3, 5, 100).first == 0 && span_of(-3, 5, 100).end == 0);
  CHECK(span_of(7, 0, 100).first == 0 && span_of(7, 0, 100).end == 7);
  CHECK(span_of(7, 7, 100).first == 0 && span_of(7, 6, 100).first == 1);
  CHECK(span_of(2147483647, 0, 2147483647).end == 2147483647);
  CHECK(span_of(2147483647, 10, 2147483647).first == 2147483637);
  CHECK(span_of(101, 0, 100).end == 100);
  // units
  CHECK(units_of(span_of(0, 0, 9), 64) == 1 && units_of(span_of(1, 0, 9), 64) == 1);
  CHECK(units_of(span_of(64, 0, 999), 64) == 1 && units_of(span_of(65, 0, 999), 64) == 2);
  CHECK(aligned_first(span_of(100, 71, 999)) == 0 && units_of(span_of(100, 71, 999), 64) == 2);
  CHECK(aligned_first(span_of(100, 61, 999)) == 32 && units_of(span_of(100, 61, 999), 64) == 2);
  CHECK(units_of(span_of(96, 64, 999), 64) == 1 && units_of(span_of(95, 64, 999), 64) == 2);
  CHECK(units_of(span_of(2147483647, 0, 2147483647), 64) == 33554432);
  CHECK(split_units(0, 444, true).big == 1 && split_units(444, 444, true).big == 1 && split_units(445, 444, true).big == 2);
  CHECK(split_units(444 * 39, 444, true).small == 0 && split_units(444 * 40, 444, true).small == 10);
  CHECK(split_units(444 * 40, 444, false).small == 0);

  CHECK(blocks_of_item(0, 1, 444) == 1 && blocks_of_item(127, 1, 444) == 1 && blocks_of_item(512, 444, 444) == 1);
  CHECK(blocks_of_item(512, 445, 444) == 0 && blocks_of_item(1, 1 << 20, 444) == 0);
  CHECK(blocks_of_item(128, 1, 444) == 2 && blocks_of_item(512, 1, 444) == 8 && blocks_of_item(512, 37, 444) == 4);
  CHECK(blocks_of_item(513, 222, 444) == 2 && blocks_of_item(513, 223, 444) == 0);
  CHECK(blocks_of_item(4096, 55, 444) == 8 && blocks_of_item(4096, 56, 444) == 0 && blocks_of_item(4097, 1, 444) == 0);

  const std::vector<std::vector<int32_t>> batches = {
      {1}, {0}, {131072}, {0, 0, 0}, {1, 64, 65, 0, 5000}, std::vector<int32_t>(1000, 77), {5, 100000, 3, 3, 70000, 0}};
  for (const auto& lengths : batches) {
    for (int heads : {1, 3, 8}) {
      for (int64_t workers : {1, 7, 296, 444}) {
        std::vector<int64_t> start;  // of each item, in units
        std::vector<int32_t> units;
        int64_t total = 0;
        for (int32_t n : lengths) {
          for (int h = 0; h < heads; ++h) {
            start.push_back(total);
            units.push_back(units_of(span_of(n, 0, 1 << 30), 64));
            total += units.back();
          }
        }
        for (bool two : {false, true}) {
          const UnitSplit s = split_units(total, workers, two);
          // every unit has one worker, and each worker's are neighbours
          int64_t next = 0;
          for (int64_t w = 0; w < 2 * workers; ++w) {
            CHECK(s.small == 0 && w >= workers ? s.units_of(w) == 0 : s.first(w) == next);
            const int64_t end = s.first(w) + s.units_of(w);
            for (int64_t u : {s.first(w), end - 1}) {
              CHECK(u >= total || s.units_of(w) == 0 || s.worker_of(u) == w);
            }
            next = end > next ? end : next;
          }
          CHECK(next >= total);
          for (size_t i = 0; i < start.size(); ++i) {
            const int64_t first = s.worker_of(start[i]), last = s.worker_of(start[i] + units[i] - 1);
            CHECK(first <= last && last < 2 * workers);
            if (units[i] == 1) {
              CHECK(first == last);  // an item of one unit needs no joining
            }
          }
        }
      }
    }
  }
  std::printf(failures ? "%d failures\n" : "ok\n", failures);
  return failures != 0;
}
