// Which form a product of product_nt.h takes, from its sizes alone.  Plain C++, so
// that a host without a GPU evaluates the same rules.
#pragma once

#include <cstddef>
#include <initializer_list>

namespace vkp {

constexpr int kGroupRows = 1024;  // rows of a that an XCD walks the columns with
constexpr int kFewRows = 32;  // most rows of the few-row kernels
// Rows of x that every workgroup of the 8-bit linear quantises for itself: a launch less, against
// reading them that many times (from L2: 64 KiB of f32 at most).  4 rows, 2272 -> 128: 6.2 us, 8
// rows, which take two launches: 8.1; 16 rows, 1024 -> 128: 6.8, 17 rows: 8.0.
constexpr int kOwnRows = 16, kOwnBytes = 16384;
inline bool own_rows(size_t rows, size_t bytes) {
  return rows <= kOwnRows && rows * bytes <= kOwnBytes;
}

// Tiles of 64 x 64 by one group of two waves or by two groups that share k, of 128 x 128, of
// 256 x 192 (gates and partners: 192 x 256) and of 256 x 256.
enum TileSize { kTile64 = 0, kTile64K = 1, kTile128 = 2, kTile192 = 3, kTile256 = 4 };
constexpr TileSize kTiles[] = {kTile64, kTile64K, kTile128, kTile192, kTile256};

// A product's sizes; n: rows of b, paired: gates and partners.
struct Shape {
  long long m, n, k_bytes;
  bool paired = false;
};

struct Sides {
  int m, n;
};
constexpr Sides sides(TileSize tile, bool paired) {
  switch (tile) {
    case kTile64:
    case kTile64K: return {64, 64};
    case kTile128: return {128, 128};
    case kTile192: return paired ? Sides{192, 256} : Sides{256, 192};
    default: return {256, 256};
  }
}

// A product as launched: `splits` workgroups share out a tile's k.
struct Job {
  Shape shape;
  int splits;
};

inline long long tiles_of(TileSize tile, const Shape& p) {
  const Sides s = sides(tile, p.paired);
  return p.m > 0 ? ((p.m + s.m - 1) / s.m) * ((p.n + s.n - 1) / s.n) : 0;
}

// Bytes of a split tile's sums, of all workgroups.
inline long long split_bytes(TileSize tile, const Job& j) {
  const Sides s = sides(tile, j.shape.paired);
  return j.splits > 1 ? tiles_of(tile, j.shape) * j.splits * s.m * s.n * 4LL : 0;
}

// What a launch takes, in us, as measured on a card of 256 CUs (866 to 10,392 rows, 384 to 8192
// wide).  A CU holds `held` workgroups of a tile, by their stage buffers and the columns' values
// beside them (64 x 64: 32 KiB and some, so four; 1,024 of them over k 2048 in bf16 take 24.7 us,
// 1,056 take 38.7, and 128 x 128 tiles of the same product 23.9 and 28.0); a stage of 128 bytes
// takes `lone` where a CU has one (none but it, for the tiles that fill a CU: where the rest of the
// card idles, whose power it then has) and `full` where all are there, in between in proportion. 
// To each round of workgroups comes `between`, to the last one `end`.
struct TileCost {
  int held;
  double lone, full, between, end;
};
constexpr TileCost tile_cost(TileSize tile) {
  switch (tile) {
    case kTile64: return {4, 0.47, 0.77, 3, 3};
    case kTile64K: return {1, 0.23, 0.25, 3, 3};
    case kTile128: return {2, 0.62, 0.9, 4, 4};
    case kTile192: return {1, 0.85, 1.25, 4, 6};
    default: return {1, 1.05, 1.5, 6, 6};
  }
}

// The launch of up to two products.  Workgroups come in rounds of as many as the card holds; the
// last round of two different products is half full, as it were.
inline double launch_cost(int cus, TileSize tile, std::initializer_list<Job> jobs) {
  const TileCost c = tile_cost(tile);
  const double room = static_cast<double>(cus) * c.held;
  double wgs = 0, longest = 0, rounds = 0, sums = 0, join = 0;
  int products = 0;
  for (const Job& j : jobs) {
    const long long n = tiles_of(tile, j.shape) * j.splits;
    if (n == 0) continue;
    ++products;
    const long long stages = (j.shape.k_bytes + 127) / 128;
    const auto s = static_cast<double>((stages + j.splits - 1) / j.splits);
    wgs += static_cast<double>(n);
    rounds += static_cast<double>(n) / room * (c.full * s + c.between);
    longest = s > longest ? s : longest;
    if (j.splits > 1) {  // the last one's reading of its tile's parts; they are written and read
      const double parts = 4 + j.splits * (tile < kTile128 ? 0.4 : 1.3);
      join = parts > join ? parts : join;
      sums += static_cast<double>(split_bytes(tile, j)) / 2e6;
    }
  }
  const auto last = [&](double n) {  // of n workgroups
    const double u = n / cus, from = c.held > 1 ? 1 : 0;
    const double x = u > from ? (u - from) / (c.held - from) : 0;
    return (c.lone + (c.full - c.lone) * x) * longest + c.end;
  };
  double us = 0;
  if (wgs <= room) {
    us = last(wgs);
  } else if (products == 1) {
    const double whole = static_cast<double>(static_cast<long long>(wgs / room));
    const double rest = wgs - whole * room;
    us = whole * (c.full * longest + c.between) + (rest > 0 ? last(rest) : c.end - c.between);
  } else {
    us = rounds + 0.5 * last(room);
  }
  return us + join + sums;
}

constexpr int kMostTilesSplit = 1024;  // of a product, by its counters

// How many workgroups a tile: no more than two to a CU.
inline int splits_for(int cus, TileSize tile, const Shape& p) {
  const long long tiles = tiles_of(tile, p);
  if (tile >= kTile192 || tiles == 0 || tiles > kMostTilesSplit) return 1;
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

// The few-row kernels: a CU takes in 42 bytes of operands a ns, whoever shares them out, so that
// few columns of a long k are better cut into tiles whose k many workgroups share (17 rows, 64
// hidden columns, bf16, us: k 1024 5.4 against 6.9, 2272 7.5 against 9.3, 4096 13.3 against 10.3,
// 8192 24.6 against 10.4; 4096 hidden columns: 5.4 against 7.1, 8.1 against 10.9, 15.1 against
// 16.1, 26 against 24.5).  `prepare`: what the tiles need before, in us.
inline bool few_rows(int cus, const Shape& p, double tiles_us, double prepare) {
  if (p.m > kFewRows) return false;
  const double cols = p.paired ? 32 : 16, turns = static_cast<double>(p.n) / cols / cus;
  const double us = 4 + (turns > 1 ? turns : 1) * 0.024 * (cols + static_cast<double>(p.m)) *
                            static_cast<double>(p.k_bytes) / 1024;
  return us <= 0.85 * (tiles_us > 4.5 ? tiles_us : 4.5) + 1.2 + prepare;
}

// `largest`: of the tiles to choose from.
inline Plan plan(int cus, const Shape& p, double* us, double prepare = 0,
                 TileSize largest = kTile256) {
  Plan best{false, kTile64, 1};
  for (TileSize t : kTiles) {
    if (t > largest) break;
    const int splits = splits_for(cus, t, p);
    const double c = launch_cost(cus, t, {Job{p, splits}});
    if (t != kTile64 && c >= *us) continue;
    *us = c;
    best.tile = t;
    best.splits = splits;
  }
  best.few = few_rows(cus, p, *us, prepare);
  return best;
}

inline Plan plan(int cus, const Shape& p, double prepare = 0) {
  double us = 0;
  return plan(cus, p, &us, prepare);
}

// Two products that do not wait for one another: in one launch of one tile, or each in its own.
// What the second launch costs is `kLaunch`, with the first one's end that covers nothing (110
// sizes of 34 to 9,735 rows, both ways timed: 6.3 us where both are one round of tiles; with 8 the
// choice loses 0.5% against the better one on average, with 3 1.5%).
constexpr double kLaunch = 8;
struct PlanTwo {
  bool together;
  TileSize tile[2];
  int splits[2];
};
inline PlanTwo plan_two(int cus, const Shape& a, const Shape& b) {
  double one = 0, two = 0, least = 0;
  const Plan first = plan(cus, a, &one), second = plan(cus, b, &two);
  PlanTwo both{true, {kTile64, kTile64}, {1, 1}};
  for (TileSize t : kTiles) {
    const int sa = splits_for(cus, t, a), sb = splits_for(cus, t, b);
    const double us = launch_cost(cus, t, {Job{a, sa}, Job{b, sb}});
    if (t != kTile64 && us >= least) continue;
    least = us;
    both = PlanTwo{true, {t, t}, {sa, sb}};
  }
  if (a.m <= 0 || b.m <= 0 || least <= one + two + kLaunch) return both;
  return PlanTwo{false, {first.tile, second.tile}, {first.splits, second.splits}};
}

}  // namespace vkp
