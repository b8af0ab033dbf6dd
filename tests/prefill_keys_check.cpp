// Every key that the tiles of prompt attention would read, as their kernel works it out: none but visible ones, and no
// entry of the block table but those that were copied.
#include <stdio.h>

#include "attention_prefill_keys.h"

int main() {
  const int pages[] = {8, 16, 24, 32, 40, 64}, widths[] = {1, 2, 5, 7, 13, 40}, runs[] = {32, 64, 128};
  const int windows[] = {0, 1, 8, 20, 50, 300, -8, -16, -100}, tiles[] = {32, 64, 128}, counts[] = {1, 2, 33, 64, 100, 200};
  const int starts[] = {0, 1, 7, 39, 64, 92, 111, 300, 1000};
  long blocks = 0, read = 0, empty = 0;
  for (int page : pages)
    for (int width : widths)
      for (int run : runs)
        for (int window : windows)
          for (int tile : tiles)
            for (int count : counts)
              for (int start : starts)
                for (int q0 = 0; q0 < count; q0 += tile)
                  for (int ranges : {1, 2, 5, 16})
                    for (int range = 0; range < ranges; ++range) {
                      int shift = -1;
                      if ((page & (page - 1)) == 0)
                        for (shift = 0; (1 << shift) < page;) ++shift;
                      const int room = width * page, last_q = q0 + tile - 1 < count ? q0 + tile - 1 : count - 1;
                      PrefillKeys keys = prefill_keys(start, q0, last_q, window, room, page, shift, run);
                      const int begin = keys.first, total = keys.tiles;
                      if (ranges > 1) prefill_range(keys, range, ranges, run);
                      ++blocks;
                      empty += total <= 0;
                      for (int t = 0; t < keys.tiles; ++t)
                        for (int local = 0; local < run; ++local) {
                          const int asked = keys.first + t * run + local, key = prefill_key(keys, asked);
                          const int entry = prefill_entry(key, page, shift) - keys.first_entry;
                          const bool seen = key >= first_visible_key(start + q0, window) && key <= start + last_q;
                          ++read;
                          if (entry < 0 || entry >= keys.entries || keys.first_entry + entry >= width || key < 0 || !seen) {
                            printf("pages of %d, %d of them, runs of %d, window %d, queries %d .. %d behind %d, range %d of %d: "
                                   "key %d is read from entry %d of %d\n", page, width, run, window, q0, last_q, start, range,
                                   ranges, key, entry, keys.entries);
                            return 1;
                          }
                        }
                      // every key that a query sees lies in a run of some range
                      if (range == 0)
                        for (int key = keys.begin; key < keys.end; ++key)
                          if (key < begin || key >= begin + total * run) {
                            printf("key %d of %d .. %d lies in no run\n", key, keys.begin, keys.end);
                            return 1;
                          }
                    }
  printf("%ld blocks, %ld keys, %ld blocks without any\n", blocks, read, empty);
  return empty > 0 ? 0 : 1;
}
