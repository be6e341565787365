// Which form a product of product_nt.h takes, from its sizes alone.  Plain C++, so
// that a host without a GPU evaluates the same rules.
#pragma once

#include <cstddef>

namespace vkp {

constexpr int kGroupRows = 1024;  // rows of a that an XCD walks the columns with
constexpr int kFewRows = 32;      // most rows of the few-row kernels
// Rows of x that every workgroup of the 8-bit linear quantises for itself: a launch less, against
// reading them that many times.
constexpr int kOwnRows = 4, kOwnBytes = 4096;
inline bool own_rows(size_t rows, size_t bytes) { return rows <= kOwnRows && bytes <= kOwnBytes; }

// Tiles of 64 x 64 by one group of two waves or by four groups that share k, of 128 x 128 and
// of 256 x 256.
enum TileSize { kTile64 = 0, kTile64K = 1, kTile128 = 2, kTile256 = 3 };

struct Plan {
  bool few;
  TileSize tile;
};

inline long long tiles_of(int tile, long long m, long long n) {
  return ((m + tile - 1) / tile) * ((n + tile - 1) / tile);
}

// The cheapest by what a CU's share of the tiles took on a card of 256 CUs, in us: a tile's
// stages of 128 bytes and its two ends.  n: rows of b.
inline Plan plan(int cus, long long m, long long n, long long k_bytes) {
  const double stages = static_cast<double>((k_bytes + 127) / 128);
  const auto share = [&](int tile) { return (tiles_of(tile, m, n) + cus - 1) / cus; };
  const double n64 = static_cast<double>(share(64)), n128 = static_cast<double>(share(128)),
               n256 = static_cast<double>(share(256));
  Plan p{m <= kFewRows, kTile64};
  double best = n64 == 1 ? 0.47 * stages + 3 : n64 * (0.2 * stages + 0.7);
  const auto offer = [&](TileSize tile, double us) {
    if (us < best) {
      best = us;
      p.tile = tile;
    }
  };
  offer(kTile64K, n64 * (0.25 * stages + 3));
  offer(kTile128, n128 == 1 ? 0.57 * stages + 3 : n128 * (0.45 * stages + 2));
  offer(kTile256, n256 == 1 ? 1.1 * stages + 5 : n256 * (1.3 * stages + 5));
  return p;
}

}  // namespace vkp
