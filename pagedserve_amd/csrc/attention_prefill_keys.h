// Which keys a tile of queries reads, and where the block table has them: plain arithmetic, the same on host and device.
#pragma once

#include "common.h"

struct PrefillKeys {
  int begin, end;              // from the first key that one of the queries sees to the one behind the last
  int first_entry, entries;    // of the block table, those of these keys
  int first, tiles;            // keys are taken in runs of one length: where the first run begins, and how many there are
};

__host__ __device__ inline int prefill_entry(int key, int page_size, int page_shift) {
  return page_shift >= 0 ? key >> page_shift : key / page_size;
}

// Queries q0 .. last_q of a portion whose first token stands at position `start`; `room`: as many keys have a place in the
// block table (positions behind it see what it has); `run`: keys of a run.
__host__ __device__ inline PrefillKeys prefill_keys(int start, int q0, int last_q, int window, int room, int page_size,
                                                    int page_shift, int run) {
  PrefillKeys keys;
  keys.begin = first_visible_key(start + q0, window);
  keys.end = start + last_q + 1 < room ? start + last_q + 1 : room;
  keys.first_entry = prefill_entry(keys.begin, page_size, page_shift);
  keys.entries = prefill_entry(keys.end - 1, page_size, page_shift) - keys.first_entry + 1;
  keys.first = keys.begin / run * run;
  // (none where no query sees a key: no entry of the table is kept then, and none may be asked for)
  keys.tiles = keys.begin < keys.end ? (keys.end - keys.first + run - 1) / run : 0;
  return keys;
}

// Those of range `range` of `ranges` (none or fewer than the others: a range without keys).
__host__ __device__ inline void prefill_range(PrefillKeys& keys, int range, int ranges, int run) {
  const int per = (keys.tiles + ranges - 1) / ranges;
  keys.first += range * per * run;
  keys.tiles -= range * per;
  keys.tiles = keys.tiles < per ? keys.tiles : per;
}

// The key that is read in the place of key `key` of a run, one that some query sees; and its entry, counted from the
// first of `keys`.
__host__ __device__ inline int prefill_key(const PrefillKeys& keys, int key) {
  return key < keys.begin ? keys.begin : (key >= keys.end ? keys.end - 1 : key);
}
