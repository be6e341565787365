// Which form a product of product_nt.h takes, from its sizes alone.  Plain C++, so
// that a host without a GPU evaluates the same rules.
#pragma once

#include <cstddef>
#include <initializer_list>

namespace vkp {

constexpr int kGroupRows = 1024;  // rows of a that an XCD walks the columns with
constexpr int kFewRows = 32;      // most rows of the few-row kernels
// Rows of x that every workgroup of the 8-bit linear quantises for itself: a launch less, against
// reading them that many times (from L2: 64 KiB of f32 at most).
constexpr int kOwnRows = 16, kOwnBytes = 16384;
inline bool own_rows(size_t rows, size_t bytes) {
  return rows <= kOwnRows && rows * bytes <= kOwnBytes;
}

// Tiles of 64 x 64 by one group of two waves or by four groups that share k, of 128 x 128 and
// of 256 x 256.
enum TileSize { kTile64 = 0, kTile64K = 1, kTile128 = 2, kTile256 = 3 };

constexpr int kSide[] = {64, 64, 128, 256};

inline long long tiles_of(int tile, long long m, long long n) {
  return ((m + tile - 1) / tile) * ((n + tile - 1) / tile);
}

// A product's sizes; n: rows of b.
struct Shape {
  long long m, n, k_bytes;
};

// Us of one tile's stages of 128 bytes and its two ends where it has a CU to itself, and a CU's us a
// tile where it has many, as measured on a card of 256 CUs (866 and 10,392 rows, 384 to 8192 wide).
struct TileCost {
  double alone, many;
};
inline TileCost tile_cost(TileSize tile, long long k_bytes) {
  const double s = static_cast<double>((k_bytes + 127) / 128);
  switch (tile) {
    case kTile64: return {0.47 * s + 3, 0.2 * s + 0.7};
    case kTile64K: return {0.23 * s + 3, 0.25 * s + 3};
    case kTile128: return {0.62 * s + 4, 0.45 * s + 2};
    default: return {1.1 * s + 6, 1.3 * s + 5};
  }
}

// Us of up to two products in one launch of one tile.
inline double launch_cost(int cus, TileSize tile, std::initializer_list<Shape> products) {
  double longest = 0, total = 0, end = 0, tiles = 0;
  for (const Shape& p : products) {
    if (p.m <= 0) continue;
    const double n = static_cast<double>(tiles_of(kSide[tile], p.m, p.n));
    const TileCost c = tile_cost(tile, p.k_bytes);
    longest = c.alone > longest ? c.alone : longest;
    end = c.many > end ? c.many : end;
    total += n * c.many;
    tiles += n;
  }
  const double share = tiles / cus;  // neighbours on a CU slow a tile down
  const double crowded = longest * (share > 1 ? 1 + 0.15 * (share - 1) : 1);
  const double busy = share > 1 ? total / cus + 0.5 * end : 0;
  return crowded > busy ? crowded : busy;
}

inline TileSize cheapest(int cus, std::initializer_list<Shape> products, double* us) {
  TileSize best = kTile64;
  for (TileSize t : {kTile64, kTile64K, kTile128, kTile256}) {
    const double c = launch_cost(cus, t, products);
    if (t != kTile64 && c >= *us) continue;
    *us = c;
    best = t;
  }
  return best;
}

struct Plan {
  bool few;
  TileSize tile;
};

inline Plan plan(int cus, long long m, long long n, long long k_bytes) {
  double us = 0;
  return Plan{m <= kFewRows, cheapest(cus, {Shape{m, n, k_bytes}}, &us)};
}

// Two products that do not wait for one another: in one launch of one tile, or each in its own, which
// costs a launch more.
struct PlanTwo {
  bool together;
  TileSize first, second;
};
inline PlanTwo plan_two(int cus, const Shape& a, const Shape& b) {
  double both = 0, one = 0, two = 0;
  const TileSize t = cheapest(cus, {a, b}, &both);
  const TileSize first = cheapest(cus, {a}, &one), second = cheapest(cus, {b}, &two);
  if (a.m <= 0 || b.m <= 0 || both <= one + two + 3) return PlanTwo{true, t, t};
  return PlanTwo{false, first, second};
}

}  // namespace vkp
