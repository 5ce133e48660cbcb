// The index arithmetic of the paged cache's kernels (pages_args.h) against divisions:
// the page of a tile for every page size, and what is left out.
#include "pages_args.h"

#include <cstdio>
#include <cstdlib>

#define CHECK(x)                                            \
  do {                                                      \
    if (!(x)) {                                             \
      std::printf("line %d: %s\n", __LINE__, #x);           \
      std::exit(1);                                         \
    }                                                       \
  } while (0)

int main() {
  PagesBatch b{};
  for (int size = 16; size <= 4096; size += 16) {
    b.page_size = size;
    b.tiles = size / 16;
    b.tiles_inv = b.tiles == 1 ? 0 : (uint32_t)((0xffffffffull + b.tiles) / b.tiles);
    for (int tile = 0; tile < 1 << 20; tile += tile < 5000 ? 1 : 61)
      CHECK(page_of_tile(b, tile) == tile / b.tiles);
    const int last = ((1 << 20) - 1) / b.tiles * b.tiles;
    for (int tile = last - b.tiles; tile <= last; ++tile)
      if (tile >= 0) CHECK(page_of_tile(b, tile) == tile / b.tiles);
    CHECK(page_of_tile(b, (1 << 20) - 1) == ((1 << 20) - 1) / b.tiles);
  }
  b.rows = 10;
  b.max_rows = 4;
  CHECK(rows_of(b, 0, 4) == 4 && rows_of(b, 6, 10) == 4 && rows_of(b, 3, 3) == 0);
  CHECK(rows_of(b, 0, 5) == 0 && rows_of(b, -1, 2) == 0 && rows_of(b, 8, 11) == 0);
  CHECK(rows_of(b, 4, 3) == 0 && rows_of(b, -2147483647, 2147483647) == 0);
  CHECK(rows_of(b, 2147483647, -2147483647) == 0);
  b.slots = 96;
  b.pages = 7;
  CHECK(slot_ok(b, 0) && slot_ok(b, 95) && !slot_ok(b, 96) && !slot_ok(b, -1));
  CHECK(!slot_ok(b, 1ll << 40) && !slot_ok(b, -(1ll << 40)));
  CHECK(page_ok(b, 0) && page_ok(b, 6) && !page_ok(b, 7) && !page_ok(b, -1));
  CHECK(slots_seen(b, 5, 1, 0) == 5 && slots_seen(b, 5, 3, 0) == 3 && slots_seen(b, 5, 3, 2) == 5);
  CHECK(slots_seen(b, 1, 3, 0) == 0 && slots_seen(b, 1, 3, 2) == 1 && slots_seen(b, 0, 1, 0) == 0);
  CHECK(slots_seen(b, 2147483647, 1, 0) == 96 && slots_seen(b, -2147483647 - 1, 256, 255) == 0);
  CHECK(slots_seen(b, 2147483647, 4, 3) == 96);
  std::printf("ok\n");
  return 0;
}
