// Lists of tensors laid out as the argument tables of kernel launches.  Host code only.
#ifndef HPX_TABLES_H_
#define HPX_TABLES_H_

#include <algorithm>
#include <cstdint>

#include "hpx.h"

namespace hpx {

// Segments and the exclusive prefix of their tiles.
template <typename Seg, int CAP>
struct Table {
  int32_t nseg;
  int32_t tile_start[CAP + 1];
  Seg seg[CAP];
};

// The lanes of a launch are counted in 32 bits, and a launch of more is no error: it runs what their number leaves modulo 2^32 (2^24
// workgroups of 256 lanes and a few: the few).  So this is the most tiles of a table that is launched with a workgroup of `threads`
// lanes for each.
constexpr int32_t most_tiles(int threads) { return int32_t(UINT32_MAX / uint32_t(threads)); }

// A tensor goes into such tables in parts of this many elements, a multiple of every tile: a part then begins on the same place of
// a tile as the tensor does, and is far from filling a launch.
constexpr int64_t kPartElements = int64_t(1) << 32;

// The elements of the part that begins at element *at; moves *at behind it, to 0 where the tensor ends.
inline int64_t next_part(int64_t size, int64_t* at, int64_t part = kPartElements) {
  const int64_t from = *at, n = std::min(part, size - from);
  *at = from + n < size ? from + n : 0;
  return n;
}

// Fills tables of at most CAP segments and `most` tiles from items [0, count) and hands each to `launch(table, tiles, last)`.
// fill(i, at, seg) describes what of item i begins at *at, moves *at behind it (to 0 where the item ends) and returns its tiles: 0
// to leave it out, `most` at most.  At least one launch is made, of an empty table if need be.
template <typename Seg, int CAP, typename Fill, typename Launch>
int for_tables(int count, int32_t most, Fill fill, Launch launch) {
  Table<Seg, CAP> a;
  int i = 0;
  int64_t at = 0;
  do {
    a.nseg = 0;
    a.tile_start[0] = 0;
    while (i < count) {  // to the next item that has tiles, also when the table is full: a launch knows whether it is the last
      Seg seg;
      int64_t next = at;
      const int64_t tiles = fill(i, &next, seg);
      if (tiles > 0) {
        if (a.nseg == CAP || a.tile_start[a.nseg] + tiles > most) break;
        a.seg[a.nseg] = seg;
        a.tile_start[a.nseg + 1] = a.tile_start[a.nseg] + int32_t(tiles);
        a.nseg++;
      }
      at = next;
      if (at == 0) i++;
    }
    const int rc = launch(a, a.tile_start[a.nseg], i == count);
    if (rc != HPX_OK) return rc;
  } while (i < count);
  return HPX_OK;
}

}  // namespace hpx
#endif  // HPX_TABLES_H_
