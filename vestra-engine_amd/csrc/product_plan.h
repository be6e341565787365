// Which form a product of product_nt.h takes, from its sizes alone.  Plain C++, so
// that a host without a GPU evaluates the same rules.
#pragma once

namespace vkp {

constexpr int kGroupRows = 1024;  // rows of a that an XCD walks the columns with
constexpr int kFewRows = 32;      // most rows of the few-row kernels

enum TileSize { kTile64 = 0, kTile128 = 1, kTile256 = 2 };

struct Plan {
  bool few;
  TileSize tile;
};

inline long long tiles_of(int tile, long long m, long long n) {
  return ((m + tile - 1) / tile) * ((n + tile - 1) / tile);
}

// n: rows of b.
inline Plan plan(int cus, long long m, long long n, long long k_bytes) {
  (void)k_bytes;
  Plan p{m <= kFewRows, kTile64};
  if (tiles_of(256, m, n) >= cus) p.tile = kTile256;
  else if (tiles_of(128, m, n) >= cus) p.tile = kTile128;
  return p;
}

}  // namespace vkp
