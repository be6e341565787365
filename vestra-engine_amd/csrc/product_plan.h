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

// A product as launched: `splits` workgroups share out a tile's k.
struct Job {
  Shape shape;
  int splits;
};

inline long long tiles_of(TileSize tile, const Shape& p) {
  return p.m > 0 ? tiles_of(kSide[tile], p.m, p.n) : 0;
}

// Bytes of a split tile's sums, of all workgroups.
inline long long split_bytes(TileSize tile, const Job& j) {
  return j.splits > 1 ? tiles_of(tile, j.shape) * j.splits * kSide[tile] * kSide[tile] * 4LL : 0;
}

// Us of one workgroup where it has a CU to itself, and a CU's us a workgroup where it has many, as
// measured on a card of 256 CUs (866 and 10,392 rows, 384 to 8192 wide): stages of 128 bytes, the
// two ends, and the last one's reading of its tile's parts.
struct TileCost {
  double alone, many;
};
inline TileCost tile_cost(TileSize tile, const Job& j) {
  const long long stages = (j.shape.k_bytes + 127) / 128;
  const double s = static_cast<double>((stages + j.splits - 1) / j.splits);
  const double join = j.splits > 1 ? 4 + j.splits * (kSide[tile] == 64 ? 0.4 : 1.3) : 0;
  switch (tile) {
    case kTile64: return {0.47 * s + 3 + join, 0.2 * s + 0.7};
    case kTile64K: return {0.23 * s + 3 + join, 0.25 * s + 3};
    case kTile128: return {0.62 * s + 4 + join, 0.45 * s + 2};
    default: return {1.1 * s + 6 + join, 1.3 * s + 5};
  }
}

// Us of up to two products in one launch of one tile.
inline double launch_cost(int cus, TileSize tile, std::initializer_list<Job> jobs) {
  double longest = 0, total = 0, end = 0, wgs = 0, sums = 0;
  for (const Job& j : jobs) {
    if (j.shape.m <= 0) continue;
    const double n = static_cast<double>(tiles_of(tile, j.shape) * j.splits);
    const TileCost c = tile_cost(tile, j);
    longest = c.alone > longest ? c.alone : longest;
    end = c.many > end ? c.many : end;
    total += n * c.many;
    wgs += n;
    sums += static_cast<double>(split_bytes(tile, j)) / 2e6;  // written and read
  }
  const double share = wgs / cus;  // neighbours on a CU slow a tile down
  const double crowded = longest * (share > 1 ? 1 + 0.15 * (share - 1) : 1);
  const double busy = share > 1 ? total / cus + 0.5 * end : 0;
  return (crowded > busy ? crowded : busy) + sums;
}

constexpr int kMostTilesSplit = 1024;  // of a product, by its counters

// How many workgroups a tile: no more than two to a CU.
inline int splits_for(int cus, TileSize tile, const Shape& p) {
  const long long tiles = tiles_of(tile, p);
  if (tile == kTile256 || tiles == 0 || tiles > kMostTilesSplit) return 1;
  int best = 1;
  double least = launch_cost(cus, tile, {Job{p, 1}});
  for (int c : {2, 3, 4, 6, 8, 12, 16, 24, 32}) {
    if (tiles * c > 2 * cus || 2 * c > (p.k_bytes + 127) / 128) break;
    const double us = launch_cost(cus, tile, {Job{p, c}});
    if (us < least) {
      least = us;
      best = c;
    }
  }
  return best;
}

struct Plan {
  bool few;
  TileSize tile;
  int splits;
};

inline Plan plan(int cus, const Shape& p, double* us) {
  Plan best{p.m <= kFewRows, kTile64, 1};
  for (TileSize t : {kTile64, kTile64K, kTile128, kTile256}) {
    const int splits = splits_for(cus, t, p);
    const double c = launch_cost(cus, t, {Job{p, splits}});
    if (t != kTile64 && c >= *us) continue;
    *us = c;
    best.tile = t;
    best.splits = splits;
  }
  return best;
}

inline Plan plan(int cus, long long m, long long n, long long k_bytes) {
  double us = 0;
  return plan(cus, Shape{m, n, k_bytes}, &us);
}

// Two products that do not wait for one another: in one launch of one tile, or each in its own,
// which costs a launch more.
struct PlanTwo {
  bool together;
  TileSize tile[2];
  int splits[2];
};
inline PlanTwo plan_two(int cus, const Shape& a, const Shape& b) {
  double one = 0, two = 0, least = 0;
  const Plan first = plan(cus, a, &one), second = plan(cus, b, &two);
  PlanTwo both{true, {kTile64, kTile64}, {1, 1}};
  for (TileSize t : {kTile64, kTile64K, kTile128, kTile256}) {
    const int sa = splits_for(cus, t, a), sb = splits_for(cus, t, b);
    const double us = launch_cost(cus, t, {Job{a, sa}, Job{b, sb}});
    if (t != kTile64 && us >= least) continue;
    least = us;
    both = PlanTwo{true, {t, t}, {sa, sb}};
  }
  if (a.m <= 0 || b.m <= 0 || least <= one + two + 3) return both;
  return PlanTwo{false, {first.tile, second.tile}, {first.splits, second.splits}};
}

}  // namespace vkp
