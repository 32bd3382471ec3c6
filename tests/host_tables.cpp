// Host unit test of csrc/hpx_tables.h (compiled and run by tests/test_tables.py).
#include "hpx_tables.h"

#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#define CHECK(c)                                                            \
  do {                                                                      \
    if (!(c)) {                                                             \
      std::printf("%s:%d: %s\n", __FILE__, __LINE__, #c);                   \
      std::exit(1);                                                         \
    }                                                                       \
  } while (0)

namespace {
struct Seg {
  int item;
  int64_t from, n;
};

// Lays items of `sizes` elements out in parts of `part`, tiles of `tile` elements; checks every table and that the segments
// are the items, whole and in order.  Returns the number of launches.
template <int CAP>
int lay_out(const std::vector<int64_t>& sizes, int64_t part, int64_t tile, int32_t most) {
  int launches = 0, item = 0;
  int64_t at = 0;
  bool ended = false;
  const int rc = hpx::for_tables<Seg, CAP>(
      int(sizes.size()), most,
      [&](int i, int64_t* from, Seg& s) -> int64_t {
        s.item = i;
        s.from = *from;
        if (sizes[size_t(i)] == 0) return 0;
        s.n = hpx::next_part(sizes[size_t(i)], from, part);
        return (s.n + tile - 1) / tile;
      },
      [&](const hpx::Table<Seg, CAP>& a, int tiles, bool last) -> int {
        CHECK(!ended && a.nseg >= 0 && a.nseg <= CAP && tiles <= most && a.tile_start[0] == 0);
        launches++;
        ended = last;
        for (int k = 0; k < a.nseg; k++) {
          const Seg& s = a.seg[k];
          while (size_t(item) < sizes.size() && sizes[size_t(item)] == 0) item++;
          CHECK(s.item == item && s.from == at && s.n > 0 && s.n <= part);
          CHECK(a.tile_start[k + 1] - a.tile_start[k] == (s.n + tile - 1) / tile);
          at += s.n;
          if (at == sizes[size_t(item)]) {
            at = 0;
            item++;
          }
        }
        CHECK(tiles == a.tile_start[a.nseg]);
        if (launches > 1) CHECK(a.nseg > 0);
        return HPX_OK;
      });
  CHECK(rc == HPX_OK && ended && at == 0);
  while (size_t(item) < sizes.size() && sizes[size_t(item)] == 0) item++;
  CHECK(size_t(item) == sizes.size());
  return launches;
}
}  // namespace

int main() {
  // fewer than 2^32 lanes in a launch
  static_assert(uint64_t(hpx::most_tiles(256)) * 256 < (uint64_t(1) << 32) && uint64_t(hpx::most_tiles(256) + 1) * 256 >= (uint64_t(1) << 32), "");
  static_assert(uint64_t(hpx::most_tiles(512)) * 512 < (uint64_t(1) << 32), "");
  // a part of any tensor, in the smallest tiles that are launched with a workgroup each, goes into a table
  static_assert(hpx::kPartElements / 1024 + 1 <= hpx::most_tiles(256), "");

  CHECK(lay_out<4>({}, 100, 10, 50) == 1);
  CHECK(lay_out<4>({0, 0}, 100, 10, 50) == 1);
  CHECK(lay_out<4>({5, 0, 7, 1, 9, 0, 0}, 100, 10, 50) == 1);     // a full table, and nothing behind it
  CHECK(lay_out<4>({5, 5, 5, 5, 5}, 100, 10, 50) == 2);
  CHECK(lay_out<4>({1000}, 100, 10, 50) == 3);                    // ten parts of ten tiles: four, four, two
  CHECK(lay_out<4>({1000}, 100, 10, 10) == 10);
  CHECK(lay_out<4>({1001}, 100, 10, 10) == 11);
  CHECK(lay_out<8>({100, 100, 100}, 100, 10, 29) == 2);           // by tiles, not by segments
  // the elements of 137 GB of fp32 and of as many again, in tiles of 2048
  const int64_t n = int64_t(1) << 35;
  CHECK(lay_out<8>({n + 4099, n}, hpx::kPartElements, 2048, hpx::most_tiles(256)) == 3);
  CHECK(lay_out<320>({n + 4099, n}, hpx::kPartElements, 2048, hpx::most_tiles(256)) == 3);

  std::mt19937 gen(1);
  for (int trial = 0; trial < 20000; trial++) {
    std::vector<int64_t> sizes(gen() % 12);
    for (auto& s : sizes) s = gen() % 3 == 0 ? 0 : int64_t(gen() % 300);
    const int64_t tile = 1 + gen() % 9, part = tile * (1 + gen() % 8);
    lay_out<3>(sizes, part, tile, int32_t(part / tile + gen() % 20));
  }

  // an error ends the list
  int calls = 0;
  CHECK((hpx::for_tables<Seg, 2>(5, 10, [](int, int64_t*, Seg&) -> int64_t { return 1; },
                                 [&](const hpx::Table<Seg, 2>&, int, bool) { return ++calls == 2 ? HPX_ERR_HIP : HPX_OK; }) == HPX_ERR_HIP));
  CHECK(calls == 2);
  std::puts("OK");
  return 0;
}
