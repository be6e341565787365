// Products out[m, n] = sum_k a[m, k] b[n, k] on the gfx950 matrix cores: int8 with
// int32 sums, f16 and bf16 with f32 sums.  An operand's rows are contiguous in k, or (16-bit
// types) its columns are: then a stage lies in LDS as it lies in memory, and fragments are read
// with the transposing LDS reads, so that a backward pass needs no transposed copies.
//
// All three types share one kernel, because they share one layout in bytes: an
// operand of v_mfma_*_32x32x{32 int8, 16 f16/bf16} is 16 bytes a lane, lane l
// holding k bytes 16 (l / 32) .. + 16 of row l % 32.  What a lane calls k only has
// to agree between a and b.
//
// A workgroup owns a TM x TN tile and walks k in stages of 128 bytes a row: both operands go from
// memory straight into LDS (16 bytes a lane, no registers), two stage buffers (four where a tile is
// alone on its CU and short of work), one barrier a stage.  Between two matrix instructions goes
// one fragment read of the next step and one load of a later stage, so that neither LDS nor
// the load path holds the matrix pipe up (10,392 x 1536 x 8192 in bf16: reads and loads in
// bursts 237 us, one by one 204).  In LDS a row is 128 bytes, its 16-byte pieces permuted by
// (piece ^ row / 2 % 8): a fragment read, whose lanes read the same piece of 32 rows, then
// touches all 64 banks once with any 16 lanes that it takes together (0-3, 12-15, 20-23 and
// 24-27 among them).  The permutation is applied to the addresses that the loads read from.
//
// What bounds it.  Large products: the stages' loads, which the L2s deliver at 10.5-11 TB/s (the
// loads of the product above alone take 190 us, its matrix instructions alone some 150), and the
// card's power (the same product of zeros: 154 us).  Bigger tiles load less but leave a larger
// part of a last round of workgroups idle; product_plan.h weighs that.  It reaches 1,280 TFLOP/s
// in bf16 and 1,770 TOP/s in int8 (with its gated end) where a library's plain product of the
// same sizes reaches 1,415 and one of 8192^3 2,076.  Few tiles: the chain of stages, 0.23-0.47 us
// each, which groups of waves share (Tile::KG) and, for a long k, workgroups (Split).  A few rows:
// reading b (few_product).
#pragma once

#include <type_traits>

#include "common.h"
#include "product_plan.h"

namespace vkp {

enum Kind { kI8 = 0, kF16 = 1, kBF16 = 2 };

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <Kind KIND>
struct Ops {
  typedef f32x4 Acc4;
  typedef f32x16 Acc16;
  static __device__ __forceinline__ Acc16 mma32(i32x4 a, i32x4 b, Acc16 c) {
    if constexpr (KIND == kF16)
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                    __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                     __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ Acc4 mma16(i32x4 a, i32x4 b, Acc4 c) {
    if constexpr (KIND == kF16)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                    __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                     __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Ops<kI8> {
  typedef i32x4 Acc4;
  typedef i32x16 Acc16;
  static __device__ __forceinline__ Acc16 mma32(i32x4 a, i32x4 b, Acc16 c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ Acc4 mma16(i32x4 a, i32x4 b, Acc4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  }
};

// An operand in memory; base and pitch are multiples of 16 bytes.
//   Rows (k contiguous): row r at base + r * pitch, k_bytes of k; what lies between k_bytes and
//     the next multiple of 16 is zeros.
//   Columns (16-bit types): k's values at base + k * pitch, `rows` of them, a multiple of
//     8; `ks` of k.  With k_half > 0 (a multiple of 64) k comes in two halves: k < k_half is line
//     k where that is below ks / 2, k >= k_half line ks / 2 + k - k_half where that is below ks;
//     zeros otherwise.
struct Operand {
  const char* base;
  int rows;
  uint32_t pitch;
  int ks = 0, k_half = 0;
};

constexpr int kStage = 128;            // bytes of k of a stage
constexpr uint32_t kOutside = 0xfffffff0u;  // a lane offset past every buffer: reads zeros
constexpr uint32_t kMostBytes = 0x7ffffff0u;

// A tile's shape: WM x WN waves of MT x NT tiles of 32 x 32.  PAIRED: the tile's
// columns are TN / 2 gates and the TN / 2 partners of the same hidden columns, b
// rows h and hidden + h; a wave's first NT / 2 column tiles are gates, the others
// the partners.
// KG groups of waves share k out by stages and are added in their order at the end: for
// grids of few tiles.
template <int WM_, int WN_, int MT_, int NT_, bool PAIRED_, int R_, int KG_>
struct Tile {
  static constexpr int WM = WM_, WN = WN_, MT = MT_, NT = NT_, KG = KG_;
  static constexpr int R = R_;  // stage buffers
  static constexpr bool PAIRED = PAIRED_;
  static constexpr int kWaves = WM * WN;  // of a group
  static constexpr int kThreads = 64 * kWaves * KG;
  static constexpr int TM = 32 * WM * MT, TN = 32 * WN * NT;
  static constexpr int kHeld = PAIRED ? TN / 2 : TN;  // columns of the result
  static constexpr int kRows = 1024 / kStage;  // rows of a wave's load
  static constexpr int kALoads = TM / kRows / kWaves, kBLoads = TN / kRows / kWaves;
  static constexpr int kGroupBytes = (TM + TN) * kStage, kBytes = KG * kGroupBytes;
  static_assert((KG - 1) * TM * TN * 4 <= kBytes, "a group's sums fit a stage buffer");
  static constexpr int kWavesASimd = MT * NT > 8 ? 1 : 2;  // by the registers of the sums
  static_assert(kALoads * kWaves * kRows == TM && kBLoads * kWaves * kRows == TN,
                "loads divide evenly");
  static_assert(!PAIRED || NT % 2 == 0, "gates and partners");
  // First row of b, within the tile, of a wave's column tile.
  static __device__ __forceinline__ constexpr int b_row(int wn, int nt) {
    if (PAIRED) {
      constexpr int kHalf = NT / 2 > 0 ? NT / 2 : 1;
      return (nt / kHalf) * (TN / 2) + (wn * kHalf + nt % kHalf) * 32;
    }
    return (wn * NT + nt) * 32;
  }
};

// The tile of a plan's size.  16-bit results leave as whole lines where a wave has an even number
// of 32-column tiles of them (gates and partners: of hidden columns, which only the largest tile
// has), as halves of lines with the others.
template <bool PAIRED, typename F>
void with_tile(TileSize size, F go) {
  if (size == kTile192) {
    if constexpr (PAIRED) go(Tile<2, 4, 3, 2, true, 2, 1>{});
    else go(Tile<4, 2, 2, 3, false, 2, 1>{});
  } else if (size == kTile256) {
    if constexpr (PAIRED) go(Tile<4, 2, 2, 4, true, 2, 1>{});
    else go(Tile<2, 4, 4, 2, false, 2, 1>{});
  } else if (size == kTile128) {
    go(Tile<2, 2, 2, 2, PAIRED, 2, 1>{});
  } else if (size == kTile64K) {
    go(Tile<2, 1, 1, 2, PAIRED, 4, 2>{});
  } else {
    go(Tile<2, 1, 1, 2, PAIRED, 2, 1>{});
  }
}

typedef __attribute__((address_space(3))) void* lds_ptr;

constexpr int kReadsDone = 0xc07f;  // s_waitcnt lgkmcnt(0)

// All but the wave's last COUNT loads into LDS have landed, then all waves'.
template <int COUNT>
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(COUNT) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// Everyone is done with the stage buffers.
__device__ __forceinline__ void tile_done() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The stage buffers of a kernel: arrays of their own, so that the compiler sees that a load
// into one and a read of another do not meet.
#define VK_STAGES(T)                                                     \
  __shared__ __align__(16) char s0_[T::kBytes];                          \
  __shared__ __align__(16) char s1_[T::kBytes];                          \
  __shared__ __align__(16) char s2_[T::R > 2 ? T::kBytes : 16];          \
  __shared__ __align__(16) char s3_[T::R > 3 ? T::kBytes : 16];          \
  char* const stages_[4] = {s0_, s1_, s2_, s3_}

// A buffer resource's parts.
struct Source {
  const char* base;
  uint32_t bytes;
};

// Rows r0 .. of an operand.
__device__ __forceinline__ Source rows_of(const Operand& o, int r0) {
  const size_t from = static_cast<size_t>(r0) * o.pitch;
  const size_t left = static_cast<size_t>(o.rows) * o.pitch - from;
  return Source{o.base + from, left < kMostBytes ? static_cast<uint32_t>(left) : kMostBytes};
}

// 16 bytes a lane from source + lane offset (zeros past its bytes) + k into LDS.  BY_HAND: the
// instruction itself, which the compiler does not count: it would wait for every load under way
// before a transposing read, whose buffer it does not see.  No register is written, and what has to
// be waited for is waited for by stage_barrier and tile_done.  (The s_nop covers scalar operands
// that a vector instruction may just have written.)
template <bool BY_HAND>
__device__ __forceinline__ void load_lds(const Source& s, char* to, uint32_t lane_off, int k) {
  if constexpr (BY_HAND) {
    const uint64_t base = reinterpret_cast<uint64_t>(s.base);
    const i32x4 r = {static_cast<int>(base), static_cast<int>((base >> 32) & 0xffff),
                     static_cast<int>(s.bytes), 0x00020000};
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr)(to)))),
                   "v"(lane_off), "s"(r), "s"(k)
                 : "memory", "m0");
  } else {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(vkd::buffer_rsrc(s.base, s.bytes), (lds_ptr)(to), 16,
                                             static_cast<int>(lane_off), k, 0, 0);
  }
}

// Columns: a stage is 64 lines of W values.  In LDS a line's 16-byte pieces are permuted by
// piece ^ 4 (k % 4) (where two lines differ by half of the 64 banks, of 64 and 192 values: by
// 4 (k / 2 % 2)): the 32 lanes of a transposing read take 64 bytes each of four neighbouring lines,
// all banks once.
template <int W>
__device__ __forceinline__ constexpr int column_turn(int k) {
  return W % 128 ? ((k >> 1) & 1) * 4 : (k & 3) * 4;
}

// The lines of stage st, up to the last; none from stage `stop` on.
__device__ __forceinline__ Source columns_of(const Operand& o, int st, int stop) {
  int line = st * 64, end = o.ks;
  if (o.k_half > 0) {
    end = o.ks / 2;
    if (line >= o.k_half) {
      line += end - o.k_half;
      end = o.ks;
    }
  }
  const int lines = line < end && st < stop ? (end - line < 64 ? end - line : 64) : 0;
  return Source{o.base + static_cast<size_t>(line) * o.pitch,
                static_cast<uint32_t>(lines) * o.pitch};
}

// A lane's offsets in a stage's lines, of values c0 ...
template <int W, int WAVES, int N>
__device__ __forceinline__ void columns_at(const Operand& o, int c0, int lane, int wave,
                                           uint32_t (&v)[N]) {
  constexpr int kPieces = W / 8;  // of a line
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at_piece = (wave + i * WAVES) * 64 + lane, line = at_piece / kPieces;
    const int piece = (at_piece % kPieces) ^ column_turn<W>(line);
    const int c = c0 + piece * 8;
    const uint32_t at = static_cast<uint32_t>(line) * o.pitch + 2u * static_cast<uint32_t>(c);
    v[i] = c < o.rows ? at : kOutside;
  }
}

// The fragment of step ks, rows r0 .. of the tile: sixteen lanes read four lines of sixteen
// values and get a value's four k each; two reads make eight.
template <int W>
__device__ __forceinline__ i32x4 read_columns(const char* from, int lane, int ks, int r0) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4* lds_s4;
  const int line = 16 * ks + 8 * (lane >> 5) + ((lane >> 2) & 3);  // and 4 more: the same turn
  const int piece = (r0 >> 3) + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
  const char* p = from + line * 2 * W + ((piece ^ column_turn<W>(line)) << 4) + 8 * (lane & 1);
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + 8 * W));
  const int2 a = __builtin_bit_cast(int2, lo), b = __builtin_bit_cast(int2, hi);
  return i32x4{a.x, a.y, b.x, b.y};
}

// Where a wave stands: in group `group` of those that share k, wave `wave`, with the rows
// and columns of (wm, wn).
template <typename T>
struct Place {
  int lane, group, wave, wm, wn;
  __device__ __forceinline__ Place() {
    const int tid = threadIdx.x;
    __builtin_assume(tid < T::kThreads);
    lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    group = w / T::kWaves;
    wave = w % T::kWaves;
    wm = wave / T::WN;
    wn = wave % T::WN;
  }
};

// A launch may share a tile's k out over `count` workgroups: each leaves its sums in `partial`, and
// the one that arrives last adds all of them, in their order whoever it is, and goes on.  For few
// tiles of a long k.
struct Split {
  int count;
  char* partial;       // [count][tiles][a tile's sums]
  unsigned* arrivals;  // [tiles], zeros before and after a launch
};

// Leaves a wave's sums; whether its workgroup is its tile's last one, whose acc is then the sum of
// all parts'.  Nobody waits for anybody.  The sums go past the L2 of the XCD, 8 bytes at a time, in
// both directions (agent scope), so that they are where every XCD sees them once the wave's stores
// have returned, and a fence, which would write back and drop the whole L2, is not needed: with
// fences a launch of this kind took 44 us in place of 11.
template <Kind KIND, typename T>
__device__ __forceinline__ bool last_of_split(const Split& split, int part, int tile, int tiles,
                                              const Place<T>& at,
                                              typename Ops<KIND>::Acc16 (&acc)[T::MT][T::NT]) {
  typedef decltype(typename Ops<KIND>::Acc4{}[0] + 0) S;
  typedef S S2 __attribute__((ext_vector_type(2)));
  // pairs of a lane, a tile
  constexpr int kPairs = T::MT * T::NT * 8, kSums = T::kWaves * kPairs * 64;
  __shared__ unsigned arrived;
  uint64_t* mine = reinterpret_cast<uint64_t*>(split.partial) + static_cast<size_t>(tile) * kSums +
                   at.wave * kPairs * 64 + at.lane;
  const size_t part_sums = static_cast<size_t>(tiles) * kSums;
#pragma unroll
  for (int e = 0; e < kPairs; ++e) {
    const auto& v = acc[e / 8 / T::NT][e / 8 % T::NT];
    const S2 pair = {v[e % 8 * 2], v[e % 8 * 2 + 1]};
    __hip_atomic_store(mine + part * part_sums + e * 64, __builtin_bit_cast(uint64_t, pair),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's sums have arrived, then the count
  __syncthreads();
  if (threadIdx.x == 0)
    arrived = __hip_atomic_fetch_add(&split.arrivals[tile], 1u, __ATOMIC_RELAXED,
                                     __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (arrived + 1 != static_cast<unsigned>(split.count)) return false;
  if (threadIdx.x == 0)
    __hip_atomic_store(&split.arrivals[tile], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int i = 0; i < T::MT; ++i)
#pragma unroll
    for (int j = 0; j < T::NT; ++j) acc[i][j] = typename Ops<KIND>::Acc16{};
  // (a round trip for several parts together, as many as the registers hold)
  constexpr int kAtOnce = kPairs <= 16 ? 4 : 2;
  for (int p = 0; p < split.count; p += kAtOnce) {
    uint64_t w[kAtOnce][kPairs];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
      for (int e = 0; e < kPairs; ++e)
        w[u][e] = __hip_atomic_load(mine + (p + u < split.count ? p + u : p) * part_sums + e * 64,
                                    __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (p + u >= split.count) break;
#pragma unroll
      for (int e = 0; e < kPairs; ++e) {
        auto& v = acc[e / 8 / T::NT][e / 8 % T::NT];
        const S2 pair = __builtin_bit_cast(S2, w[u][e]);
        v[e % 8 * 2] += pair[0];
        v[e % 8 * 2 + 1] += pair[1];
      }
    }
  }
  return true;
}

// acc[mt][nt] of this wave: the tile's rows from m0, columns from n0 (of the
// hidden ones, where PAIRED), over all of k, where the wave is to go on with them: with KG > 1
// those of group 0, with a split those of the tile's last workgroup.  AC, BC: a, b as columns.
template <Kind KIND, typename T, bool AC = false, bool BC = false>
__device__ __forceinline__ bool product_tile(const Operand& a, const Operand& b, int k_bytes,
                                             int m0, int n0, const Split& split, int part, int tile,
                                             int tiles, const Place<T>& at,
                                             char* const (&stages_)[4],
                                             typename Ops<KIND>::Acc16 (&acc)[T::MT][T::NT]) {
  constexpr int S = kStage, R = T::R, KG = T::KG, KS = S / 32;
  const int lane = at.lane, wave = at.wave, wm = at.wm, wn = at.wn;
  char* buf[R];
#pragma unroll
  for (int i = 0; i < R; ++i) buf[i] = stages_[i] + at.group * T::kGroupBytes;

  // Loads of rows: 1 KiB an instruction, a lane 16 bytes.  Bit 3 of a row is the lowest of the
  // wave (rows from 8 (wave + i kWaves)).
  static_assert(T::kWaves % 2 == 0, "the permutation of a lane's rows is one");
  const int lr = lane >> 3;
  const uint32_t piece = 16u * static_cast<uint32_t>((lane & 7) ^ (4 * (wave & 1) + (lr >> 1)));
  uint32_t av[T::kALoads], bv[T::kBLoads];
  Source sa{}, sb{};
  if constexpr (!AC) sa = rows_of(a, m0);
  if constexpr (!BC) sb = rows_of(b, n0);
  if constexpr (AC) {
    columns_at<T::TM, T::kWaves>(a, m0, lane, wave, av);
  } else {
#pragma unroll
    for (int i = 0; i < T::kALoads; ++i) {
      const int r = (wave + i * T::kWaves) * T::kRows + lr;
      av[i] = m0 + r < a.rows ? static_cast<uint32_t>(r) * a.pitch + piece : kOutside;
    }
  }
  if constexpr (BC) {
    static_assert(!T::PAIRED, "gates and partners come as rows");
    columns_at<T::TN, T::kWaves>(b, n0, lane, wave, bv);
  } else {
#pragma unroll
    for (int i = 0; i < T::kBLoads; ++i) {
      const int r = (wave + i * T::kWaves) * T::kRows + lr;
      if constexpr (T::PAIRED) {
        const int hidden = b.rows / 2, j = r % T::kHeld;
        const uint32_t row = static_cast<uint32_t>(r < T::kHeld ? j : hidden + j);
        bv[i] = n0 + j < hidden ? row * b.pitch + piece : kOutside;
      } else {
        bv[i] = n0 + r < b.rows ? static_cast<uint32_t>(r) * b.pitch + piece : kOutside;
      }
    }
  }
  const int every = (k_bytes + S - 1) / S, mine = (every + split.count - 1) / split.count;
  const int start = part * mine, stop = start + mine < every ? start + mine : every;
  const int stages = (mine + KG - 1) / KG;  // of a group
  // the lane's bytes of stage t: t S < last
  const int last = (stop < every ? stop * S : k_bytes) - static_cast<int>(piece);
  // Load i of stage t (past the last stage they read zeros: their number stays the same).
  constexpr int kLoads = T::kALoads + T::kBLoads;
  auto load = [&](char* to, int t, int i) {
    const int st = start + t * KG + at.group, k = st * S;
    const bool in = k < last;
    constexpr bool kByHand = AC || BC;
    if (i < T::kALoads) {
      char* lds = to + (wave + i * T::kWaves) * 1024;
      if constexpr (AC)
        load_lds<kByHand>(columns_of(a, st, stop), lds, av[i], 0);
      else
        load_lds<kByHand>(sa, lds, in ? av[i] : kOutside, k);
    } else {
      const int j = i - T::kALoads;
      char* lds = to + T::TM * S + (wave + j * T::kWaves) * 1024;
      if constexpr (BC)
        load_lds<kByHand>(columns_of(b, st, stop), lds, bv[j], 0);
      else
        load_lds<kByHand>(sb, lds, in ? bv[j] : kOutside, k);
    }
  };

  // Fragment reads: step ks of a stage is pieces 2 ks + lane / 32.
  const int fr = lane & 31;
  const int at0 = fr * S + (((lane >> 5) ^ ((fr >> 1) & 7)) << 4);
  const int a0 = at0 + wm * T::MT * 32 * S;
  i32x4 fa[2][T::MT], fb[2][T::NT];
  constexpr int kReads = T::MT + T::NT;
  auto read = [&](const char* from, int ks, int i) {
    if (i < T::NT) {
      const char* fb_at = from + T::TM * S;
      if constexpr (BC)
        fb[ks & 1][i] = read_columns<T::TN>(fb_at, lane, ks, T::b_row(wn, i));
      else
        fb[ks & 1][i] = *reinterpret_cast<const i32x4*>(fb_at + (at0 ^ (ks << 5)) +
                                                        T::b_row(wn, i) * S);
    } else {
      const int r = i - T::NT;
      if constexpr (AC)
        fa[ks & 1][r] = read_columns<T::TM>(from, lane, ks, (wm * T::MT + r) * 32);
      else
        fa[ks & 1][r] = *reinterpret_cast<const i32x4*>(from + (a0 ^ (ks << 5)) + r * 32 * S);
    }
  };
  // The products of a step, and between them the reads of the step after it (`next`, step
  // nks) and the loads of stage t into `to`: one at a time, so that neither LDS nor the
  // load path holds the matrix pipe up.
  auto step = [&](auto reads, auto loads, int ks, const char* next, int nks, char* to, int t) {
    constexpr int kTiles = T::MT * T::NT;
    constexpr int kReadsEach = (kReads + kTiles - 1) / kTiles;
    constexpr int kLoadsEach = (kLoads + kTiles - 1) / kTiles;
#pragma unroll
    for (int e = 0; e < kTiles; ++e) {
      const int i = e / T::NT, j = e % T::NT;
      acc[i][j] = Ops<KIND>::mma32(fb[ks & 1][j], fa[ks & 1][i], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (reads.value)
#pragma unroll
        for (int r = e * kReadsEach; r < (e + 1) * kReadsEach && r < kReads; ++r)
          read(next, nks, r);
      if constexpr (loads.value)
#pragma unroll
        for (int l = e * kLoadsEach; l < (e + 1) * kLoadsEach && l < kLoads; ++l) load(to, t, l);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr int kFlying = (R - 2) * kLoads;
  constexpr std::true_type kYes{};
  constexpr std::false_type kNo{};
  // Stage t from `cur`: its last step's products run behind the barrier.
  auto stage = [&](char* cur, const char* next, int t) {
#pragma unroll
    for (int ks = 0; ks + 1 < KS; ++ks) step(kYes, kNo, ks, cur, ks + 1, nullptr, 0);
    __builtin_amdgcn_s_waitcnt(kReadsDone);
    stage_barrier<kFlying>();  // the next stage has landed, and nobody reads this one any more
    step(kYes, kYes, KS - 1, next, 0, cur, t + R);
  };
#pragma unroll
  for (int i = 0; i < T::MT; ++i)
#pragma unroll
    for (int j = 0; j < T::NT; ++j) acc[i][j] = typename Ops<KIND>::Acc16{};
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int l = 0; l < kLoads; ++l) load(buf[i], i, l);
  stage_barrier<kFlying + kLoads>();
#pragma unroll
  for (int i = 0; i < kReads; ++i) read(buf[0], 0, i);
  // To a multiple of R: stages past the last one are zeros, and a loop that does not branch
  // keeps the sums in one place.
  for (int t = 0; t < stages; t += R)
#pragma unroll
    for (int i = 0; i < R; ++i) stage(buf[i], buf[(i + 1) % R], t + i);
  tile_done();
  if constexpr (KG > 1) {
    typedef typename Ops<KIND>::Acc4 Acc4;
    constexpr int kTiles = T::MT * T::NT, kWaveSums = kTiles * 4 * 64;
    Acc4* sums = reinterpret_cast<Acc4*>(stages_[R - 1]) + wave * kWaveSums + lane;
#pragma unroll
    for (int e = 0; e < kTiles * 4; ++e) {
      const auto& v = acc[e / 4 / T::NT][e / 4 % T::NT];
      const int r = e % 4 * 4;
      if (at.group > 0)
        sums[(at.group - 1) * T::kWaves * kWaveSums + e * 64] =
            Acc4{v[r], v[r + 1], v[r + 2], v[r + 3]};
    }
    tile_done();
    if (at.group > 0) return false;
#pragma unroll
    for (int e = 0; e < kTiles * 4; ++e) {
      auto& v = acc[e / 4 / T::NT][e / 4 % T::NT];
#pragma unroll
      for (int o = 0; o < KG - 1; ++o) {
        const Acc4 w = sums[o * T::kWaves * kWaveSums + e * 64];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[e % 4 * 4 + i] += w[i];
      }
    }
  }
  // (not for the largest tiles: 192 KiB of sums a workgroup and more cost more than they save)
  if constexpr (T::TM < 192)
    if (split.count > 1) return last_of_split<KIND, T>(split, part, tile, tiles, at, acc);
  return true;
}

// A wave's sums lie with a row of a in each lane (lane % 32) and 16 columns in its registers:
// register 4 q + e is column 8 q + 4 (lane / 32) + e of its 32.  Results leave through LDS, 32 rows
// at a time, so that a row's columns go to memory as lines or halves of them: a Chunk is a wave's
// own 32 rows of 32 J columns, in the stage buffers that the products are done with, its 16-byte
// pieces permuted as the stages' are.
template <typename V, int J>
struct Chunk {
  typedef V V4 __attribute__((ext_vector_type(4)));
  static constexpr int kRowBytes = 32 * J * static_cast<int>(sizeof(V));
  static constexpr int kPieces = kRowBytes / 16, kPer = 16 / static_cast<int>(sizeof(V));
  static constexpr int kBytes = 32 * kRowBytes;
  static_assert(kRowBytes == 128 || kRowBytes == 64, "rows of a line or half of one");
  static __device__ __forceinline__ int slot(int row, int piece) {
    return row * kRowBytes + ((piece ^ (kPieces == 8 ? (row >> 1) & 7 : (row >> 2) & 3)) << 4);
  }
  // The four columns 32 j + 8 q + 4 (lane / 32) .. of the lane's row.
  static __device__ __forceinline__ V4* at(char* c, int lane, int j, int q) {
    const int byte = (32 * j + 8 * q + 4 * (lane >> 5)) * static_cast<int>(sizeof(V));
    return reinterpret_cast<V4*>(c + slot(lane & 31, byte >> 4) + (byte & 15));
  }
  // From rows m0 .., columns n0 .. of a matrix (zeros outside), through registers, so that the
  // loads of the next rows can be under way: fetch, then fill.  Rows may start anywhere: 16 bytes
  // go to and from any address, and only a row's last piece goes value by value.
  static constexpr int kFetch = kBytes / 1024;
  static __device__ __forceinline__ void fetch(i32x4 (&v)[kFetch], int lane, const V* from,
                                               size_t pitch, int m0, int M, int n0, int N) {
#pragma unroll
    for (int p = 0; p < kFetch; ++p) {
      v[p] = i32x4{};
      const int m = m0 + p * (64 / kPieces) + lane / kPieces, n = n0 + lane % kPieces * kPer;
      if (m >= M || n >= N) continue;
      const V* at = from + static_cast<size_t>(m) * pitch + n;
      if (n + kPer <= N) {
        __builtin_memcpy(&v[p], at, 16);
      } else {
        V e[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) e[i] = n + i < N ? at[i] : static_cast<V>(0.0f);
        __builtin_memcpy(&v[p], e, 16);
      }
    }
  }
  static __device__ __forceinline__ void fill(char* c, int lane, const i32x4 (&v)[kFetch]) {
#pragma unroll
    for (int p = 0; p < kFetch; ++p)
      *reinterpret_cast<i32x4*>(c + slot(p * (64 / kPieces) + lane / kPieces, lane % kPieces)) =
          v[p];
  }
  // To rows m0 .. of `out` (pitch values a row), columns n0 .., of those below M and N.  ADD: added
  // to what is there (f32).
  template <bool ADD>
  static __device__ __forceinline__ void store(char* c, int lane, V* out, size_t pitch, int m0,
                                               int M, int n0, int N) {
#pragma unroll
    for (int p = 0; p < kFetch; ++p) {
      const int row = p * (64 / kPieces) + lane / kPieces, piece = lane % kPieces;
      const int m = m0 + row, n = n0 + piece * kPer;
      i32x4 v = *reinterpret_cast<const i32x4*>(c + slot(row, piece));
      if (m >= M || n >= N) continue;
      V* to = out + static_cast<size_t>(m) * pitch + n;
      if (n + kPer <= N) {
        if constexpr (ADD) {
          f32x4 old;
          __builtin_memcpy(&old, to, 16);
          v = __builtin_bit_cast(i32x4, old + __builtin_bit_cast(f32x4, v));
        }
        __builtin_memcpy(to, &v, 16);
      } else {
        V e[kPer];
        __builtin_memcpy(e, &v, 16);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          if (n + i >= N) continue;
          if constexpr (ADD)
            to[i] = to[i] + e[i];
          else
            to[i] = e[i];
        }
      }
    }
  }
};

// Sums over lanes 0 .. 31 and over lanes 32 .. 63 of N = 32 R values a lane: lane l is left with
// the sums of values R (l % 32) .. + R.  A step adds half of the values of two lanes that
// differ in one more bit (lanes l and l ^ 16, 15, 7, 3, 1), in a fixed order.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf,
                                                            0xf, true));
}
template <int N, int CTRL>
__device__ __forceinline__ void halve(float* v, bool upper) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float keep = upper ? v[k + N] : v[k], send = upper ? v[k] : v[k + N];
    v[k] = keep + dpp<CTRL>(send);
  }
}
template <int R>
__device__ __forceinline__ void sum_rows(float* v, int lane) {
#pragma unroll
  for (int k = 0; k < 16 * R; ++k) {  // lanes l and l ^ 16
    const bool upper = lane & 16;
    const float keep = upper ? v[k + 16 * R] : v[k], send = upper ? v[k] : v[k + 16 * R];
    v[k] = keep + __shfl_xor(send, 16, 64);
  }
  halve<8 * R, 0x140>(v, lane & 8);  // row_mirror
  halve<4 * R, 0x141>(v, lane & 4);  // row_half_mirror
  halve<2 * R, 0x1b>(v, lane & 2);   // quad_perm 3, 2, 1, 0
  halve<R, 0xb1>(v, lane & 1);       // quad_perm 1, 0, 3, 2
}

// Tile `tile` of a product, XCD-major in groups of rows that a 4 MiB L2 holds together
// with the columns being walked: in a group, rows fastest.
__device__ __forceinline__ void tile_at(int tile, int gm, int gn, int group, int* mt, int* nt) {
  const int t = vkd::xcd_tile(tile, gm * gn);
  const int per = group * gn;
  const int g = t / per, r = t - g * per;
  const int left = gm - g * group, rows = left < group ? left : group;
  *mt = g * group + r % rows;
  *nt = r / rows;
}

// ---------------------------------------------------------------- activations
// Phi(g), the normal distribution's integral, and e^(-g^2 / 2), which act' takes too.  From the
// tail Phi(-a) = e^(-a^2 / 2) t P(t), t = 1 / (1 + 0.3055 a): P is of degree 7, fitted here to the
// least relative error over a of 0 to 14.5 (1.4 u, u = 2^-24), so that gates far out keep their
// value, where 1 + erf would cancel.  In f32 Phi(-a) is off by (19 + 1.3 a^2) u of itself (a^2 by
// the exponent's own rounding), 1 - Phi(-a) by what that is of it; below 2^-126 (a > 12.9) it is 0.
__device__ __forceinline__ float normal_below(float g, float* e) {
  const float a = fabsf(g);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3055f, a, 1.0f));
  float p = __builtin_fmaf(0.0366840921f, t, -0.152139843f);
  p = __builtin_fmaf(p, t, 0.183085442f);
  p = __builtin_fmaf(p, t, -0.0360131003f);
  p = __builtin_fmaf(p, t, 0.120097294f);
  p = __builtin_fmaf(p, t, 0.103812955f);
  p = __builtin_fmaf(p, t, 0.122632049f);
  p = __builtin_fmaf(p, t, 0.121841155f);
  *e = __builtin_amdgcn_exp2f(a * a * -0.72134752f);
  const float q = p * t * *e;
  return g < 0.0f ? q : 1.0f - q;
}

// act(g): SiLU g / (1 + e^-g), GELU g Phi(g).  The exponential is v_exp_f32 of g log2(e) and
// quotients v_rcp_f32, each 2 u off: some 20 instructions less than a correctly rounded
// quotient and expf.  SiLU's exponent is rounded too, which takes it (8 + 2 |g|) u off where g is
// below 0; below -87 it is 0 (e^-g above 2^126).
template <int ACT>
__device__ __forceinline__ float gate(float g) {
  float e;
  if constexpr (ACT == VK_GATE_SILU)
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504f));
  else
    return g * normal_below(g, &e);
}

// act(g) and its derivative: SiLU's is s (1 + g (1 - s)), s = 1 / (1 + e^-g); GELU's
// Phi(g) + g phi(g).
template <int ACT>
__device__ __forceinline__ void gate_slope(float g, float* act, float* slope) {
  if constexpr (ACT == VK_GATE_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504f));
    *act = g * s;
    *slope = s * __builtin_fmaf(g, 1.0f - s, 1.0f);
  } else {
    float e;
    const float phi = normal_below(g, &e);
    *act = g * phi;
    *slope = __builtin_fmaf(g * 0.39894228f, e, phi);
  }
}

// f(std::integral_constant<int, ACT>) for the activation of a launch: one branch, so that the
// values of a tile's end overlap one another's latencies.
template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {
  if (act == VK_GATE_SILU)
    f(std::integral_constant<int, VK_GATE_SILU>{});
  else
    f(std::integral_constant<int, VK_GATE_GELU>{});
}

// ---------------------------------------------------------------- 16-bit values
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(_Float16 v) { return static_cast<float>(v); }
__device__ __forceinline__ float widen(__bf16 v) { return static_cast<float>(v); }

template <Kind KIND>
struct Value;
template <>
struct Value<kF16> {
  typedef _Float16 type;
};
template <>
struct Value<kBF16> {
  typedef __bf16 type;
};

// ---------------------------------------------------------------- few rows
// Products of at most 16 RT rows: a workgroup owns 16 columns (of the hidden ones,
// where PAIRED), its eight waves share out the 128-byte stages of k and their sums are
// added in wave order through LDS.  Lane l holds row l % 16 of a 16 x 16 tile, and of
// each stage the 32 bytes of k from 32 (l / 16): a row's stage is one line read
// once.  Bound by reading b; what counts is loads in flight, U stages of a wave.
constexpr int kFewWaves = 8, kFewThreads = 64 * kFewWaves;

template <Kind KIND, int RT, bool PAIRED>
struct FewSums {
  typename Ops<KIND>::Acc4 v[PAIRED ? 2 : 1][RT];
};

// The 16 bytes of a row from byte k, zeros where they are not all below `whole`, the row's whole
// pieces (one at least).  The row may lie at any address.  No branch: a load in one would be waited
// for there.
__device__ __forceinline__ i32x4 row_piece(const char* row, int k, int whole) {
  i32x4 v;
  const bool in = k < whole;
  __builtin_memcpy(&v, row + (in ? k : 0), 16);
  return in ? v : i32x4{0, 0, 0, 0};
}

// The 16-bit values behind a row's whole pieces, zeros from its end on.
__device__ __forceinline__ i32x4 row_rest(const char* row, int k_bytes) {
  uint16_t e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int k = (k_bytes & ~15) + 2 * i;
    uint16_t v;
    __builtin_memcpy(&v, row + (k < k_bytes ? k : 0), 2);
    e[i] = k < k_bytes ? v : uint16_t{0};
  }
  i32x4 v;
  __builtin_memcpy(&v, e, 16);
  return v;
}

// The stages of a workgroup's k from stage `first` on, around to it again: b's rows often lie a
// power of two apart, where the same k of all of them is in one of the L2's channels, and
// workgroups that all began at 0 would ask the same few of them together (8 rows, 8192 -> 4096 in
// bf16: 27 us against 21; where the weights are in L2, no difference).
struct FewStages {
  int count, first, whole;  // whole: the bytes of k
  // First byte of the t-th one; past the last: none.
  __device__ __forceinline__ int at(int t) const {
    const int s = t + first;
    return t < count ? (s < count ? s : s - count) * kStage : whole;
  }
};

// Loads of b for U stages t, t + 8, ...: zeros past k and past the last stage.
template <bool PAIRED, int U>
struct FewColumns {
  i32x4 v[U][PAIRED ? 2 : 1][2];
  __device__ __forceinline__ void load(const char* const (&row)[2], int q, int t,
                                       const FewStages& stages) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int p = 0; p < (PAIRED ? 2 : 1); ++p)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          v[u][p][h] = row_piece(row[p], stages.at(t + u * kFewWaves) + q * 32 + h * 16,
                                 stages.whole);
  }
};

// The sums of all waves: thread i < 256 RT has (p, row, column) element i of each p.
template <Kind KIND, int RT, bool PAIRED>
__device__ __forceinline__ void few_join(const FewSums<KIND, RT, PAIRED>& s, char* smem, int wave,
                                         int lane) {
  typedef typename Ops<KIND>::Acc4 Acc4;
  Acc4* red = reinterpret_cast<Acc4*>(smem);
#pragma unroll
  for (int p = 0; p < (PAIRED ? 2 : 1); ++p)
#pragma unroll
    for (int r = 0; r < RT; ++r)
      red[((wave * (PAIRED ? 2 : 1) + p) * RT + r) * 64 + lane] = s.v[p][r];
  __syncthreads();
}

// Element (row, column) of part p after few_join.
template <Kind KIND, int RT, bool PAIRED>
__device__ __forceinline__ auto few_sum(const char* smem, int p, int row, int column) {
  typedef decltype(typename Ops<KIND>::Acc4{}[0] + 0) S;
  const S* red = reinterpret_cast<const S*>(smem);
  const int lane = column + 16 * ((row & 15) >> 2);
  S sum = 0;
#pragma unroll
  for (int w = 0; w < kFewWaves; ++w)
    sum += red[(((w * (PAIRED ? 2 : 1) + p) * RT + (row >> 4)) * 64 + lane) * 4 + (row & 3)];
  return sum;
}

template <Kind KIND, int RT, bool PAIRED>
constexpr int few_bytes() {
  return kFewWaves * (PAIRED ? 2 : 1) * RT * 64 * 16;
}

// The product of the columns n0 .. with at most 16 RT rows: a_at(r, k) is the lane's 16 bytes from
// k of row 16 r + lane % 16, zeros outside, a_rest(r) the values behind the whole pieces of a row
// of 16-bit ones.  The first columns are on their way before `first()` runs, the next ones while a
// stage's products do.
template <Kind KIND, int RT, bool PAIRED, typename A, typename R, typename F>
__device__ __forceinline__ void few_product(const Operand& b, int k_bytes, int n0, char* smem,
                                            F first, A a_at, R a_rest) {
  constexpr int U = 2, P = PAIRED ? 2 : 1;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  // (columns past the last one read the last one)
  const int held = b.rows / P, n = n0 + c < held ? n0 + c : held - 1;
  const char* const rows[2] = {b.base + static_cast<size_t>(n) * b.pitch,
                               b.base + static_cast<size_t>(n + (PAIRED ? held : 0)) * b.pitch};
  FewSums<KIND, RT, PAIRED> s{};
  const int whole = k_bytes & ~15, count = (whole + kStage - 1) / kStage;
  const FewStages stages{count, count > 0 ? static_cast<int>(blockIdx.x % count) : 0, whole};
  FewColumns<PAIRED, U> fb;
  if (count > 0) fb.load(rows, q, wave, stages);
  first();
  for (int t = wave; t < count; t += U * kFewWaves) {
    const FewColumns<PAIRED, U> now = fb;
    i32x4 fa[U][RT][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          fa[u][r][h] = a_at(r, stages.at(t + u * kFewWaves) + q * 32 + h * 16);
    if (t + U * kFewWaves < count) fb.load(rows, q, t + U * kFewWaves, stages);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int r = 0; r < RT; ++r)
            s.v[p][r] = Ops<KIND>::mma16(fa[u][r][h], now.v[u][p][h], s.v[p][r]);
  }
  if constexpr (KIND != kI8) {
    if (k_bytes > whole && wave == kFewWaves - 1) {
      const i32x4 none = {0, 0, 0, 0};
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const i32x4 w = row_rest(rows[p], k_bytes);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const i32x4 x = a_rest(r);
          s.v[p][r] = Ops<KIND>::mma16(q == 0 ? x : none, q == 0 ? w : none, s.v[p][r]);
        }
      }
    }
  }
  few_join<KIND, RT, PAIRED>(s, smem, wave, lane);
}

// Rows 0 .. a.rows of a in memory (rows past the last one read the last one: their sums go
// nowhere).
template <Kind KIND, int RT, bool PAIRED>
__device__ __forceinline__ void few_product(const Operand& a, const Operand& b, int k_bytes, int n0,
                                            char* smem) {
  const int c = threadIdx.x & 15;
  const char* rows[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = r * 16 + c;
    rows[r] = a.base + static_cast<size_t>(row < a.rows ? row : a.rows - 1) * a.pitch;
  }
  few_product<KIND, RT, PAIRED>(
      b, k_bytes, n0, smem, [] {},
      [&](int r, int k) { return row_piece(rows[r], k, k_bytes & ~15); },
      [&](int r) { return row_rest(rows[r], k_bytes); });
}

}  // namespace vkp
