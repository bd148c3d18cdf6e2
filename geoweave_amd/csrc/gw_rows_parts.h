// Part lengths of the few-rows attention, kept free of HIP headers so that the same code is compiled for the
// kernels and by a host-side test.
//
// The keys of all row tiles of a call (`total`: the sum of each tile's keys, below 2^59) are cut into about `want`
// parts, each a multiple of kRowsPart keys of one tile. A tile whose keys exceed the length is cut. Then there are at
// most tiles + want parts, and fewer than 2 want of them belong to cut tiles.
#pragma once

#include <stdint.h>

namespace gw {

constexpr int kRowsPart = 256;               // 4 waves x 32 keys, twice
constexpr int64_t kRowsKeysMax = 0x7FFFF000;  // keys of a sequence at most; a multiple of kRowsPart

// Formed in 64 bits: total / want passes 2^31 where many row tiles share long sequences. No sequence is
// longer than kRowsKeysMax, so a longer part is none.
constexpr int rows_part_keys(int64_t total, int want) {
  int64_t len = (total + want - 1) / want;
  if (len < kRowsPart) len = kRowsPart;
  if (len > kRowsKeysMax) len = kRowsKeysMax;
  return (int)((len + kRowsPart - 1) / kRowsPart * kRowsPart);
}

// Parts of a row tile of lk keys (one if it has none).
constexpr int rows_parts(int lk, int len) {
  const int64_t n = ((int64_t)lk + len - 1) / len;
  return n > 1 ? (int)n : 1;
}

}  // namespace gw
