// Products out[m, n] = sum_k a[m, k] b[n, k] of two operands whose rows are
// contiguous in k, on the gfx950 matrix cores: int8 with int32 sums, f16 and
// bf16 with f32 sums.
//
// All three types share one kernel, because they share one layout in bytes: an
// operand of v_mfma_*_32x32x{32 int8, 16 f16/bf16} is 16 bytes a lane, lane l
// holding k bytes 16 (l / 32) .. + 16 of row l % 32.  What a lane calls k only has
// to agree between a and b.
//
// A workgroup owns a TM x TN tile and walks k in stages of 128 bytes a row:
// both operands go from memory straight into LDS (16 bytes a lane, no
// registers), two stage buffers, one barrier a stage -- a stage's loads run
// while the stage before it is multiplied.  In LDS a row is 128 bytes, its
// 16-byte pieces permuted by (piece ^ row % 8): a fragment read, whose eight
// neighbouring lanes read the same piece of eight rows, then touches all banks
// once.  The permutation is applied to the addresses that the loads read from.
#pragma once

#include "common.h"

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

// Rows of an operand: row r is `bytes` bytes at base + r * pitch; pitch and base are
// multiples of 16, what is read past `bytes` counts as zeros (in pieces of 16:
// between `bytes` and the next multiple of 16 the row holds zeros).
struct Operand {
  const char* base;
  int rows;
  uint32_t pitch;
};

constexpr int kStage = 128;            // bytes of k of a stage
constexpr uint32_t kOutside = 0xfffffff0u;  // a lane offset past every buffer: reads zeros
constexpr uint32_t kMostBytes = 0x7ffffff0u;

// A tile's shape: WM x WN waves of MT x NT tiles of 32 x 32.  PAIRED: the tile's
// columns are TN / 2 gates and the TN / 2 partners of the same hidden columns, b
// rows h and hidden + h; a wave's first NT / 2 column tiles are gates, the others
// the partners.
template <int WM_, int WN_, int MT_, int NT_, bool PAIRED_>
struct Tile {
  static constexpr int WM = WM_, WN = WN_, MT = MT_, NT = NT_;
  static constexpr bool PAIRED = PAIRED_;
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int TM = 32 * WM * MT, TN = 32 * WN * NT;
  static constexpr int kHeld = PAIRED ? TN / 2 : TN;  // columns of the result
  static constexpr int kALoads = TM / 8 / kWaves, kBLoads = TN / 8 / kWaves;
  static constexpr int kBytes = (TM + TN) * kStage;
  static_assert(kALoads * kWaves * 8 == TM && kBLoads * kWaves * 8 == TN, "loads divide evenly");
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

typedef __attribute__((address_space(3))) void* lds_ptr;

// Every load into LDS of the wave has landed, then all waves': the barrier's own fence does
// not count loads that go past the registers.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// acc[mt][nt] of this wave: the tile's rows from m0, columns from n0 (of the
// hidden ones, where PAIRED), over all of k.
template <Kind KIND, typename T>
__device__ __forceinline__ void product_tile(const Operand& a, const Operand& b, int k_bytes,
                                             int m0, int n0, char* s0, char* s1,
                                             typename Ops<KIND>::Acc16 (&acc)[T::MT][T::NT]) {
  const int tid = threadIdx.x;
  __builtin_assume(tid < T::kThreads);
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / T::WN, wn = wave % T::WN;

  // Loads: eight rows of 128 bytes an instruction, lane l row l / 8, piece
  // (l % 8) ^ (l / 8).
  const int lr = lane >> 3;
  const uint32_t piece = static_cast<uint32_t>((lane & 7) ^ lr) * 16u;
  const size_t a_at = static_cast<size_t>(m0) * a.pitch, b_at = static_cast<size_t>(n0) * b.pitch;
  const size_t a_left = static_cast<size_t>(a.rows) * a.pitch - a_at;
  const size_t b_left = static_cast<size_t>(b.rows) * b.pitch - b_at;
  const auto ra = vkd::buffer_rsrc(a.base + a_at, a_left < kMostBytes ? static_cast<uint32_t>(a_left) : kMostBytes);
  const auto rb = vkd::buffer_rsrc(b.base + b_at, b_left < kMostBytes ? static_cast<uint32_t>(b_left) : kMostBytes);
  uint32_t av[T::kALoads], bv[T::kBLoads];
#pragma unroll
  for (int i = 0; i < T::kALoads; ++i) {
    const int r = (wave + i * T::kWaves) * 8 + lr;
    av[i] = m0 + r < a.rows ? static_cast<uint32_t>(r) * a.pitch + piece : kOutside;
  }
#pragma unroll
  for (int i = 0; i < T::kBLoads; ++i) {
    const int r = (wave + i * T::kWaves) * 8 + lr;
    if constexpr (T::PAIRED) {
      const int hidden = b.rows / 2, j = r % T::kHeld;
      const uint32_t at = static_cast<uint32_t>(r < T::kHeld ? j : hidden + j);
      bv[i] = n0 + j < hidden ? at * b.pitch + piece : kOutside;
    } else {
      bv[i] = n0 + r < b.rows ? static_cast<uint32_t>(r) * b.pitch + piece : kOutside;
    }
  }
  const int stages = (k_bytes + kStage - 1) / kStage;
  const bool whole = (stages - 1) * kStage + static_cast<int>(piece) < k_bytes;
  auto issue = [&](char* to, int t) {
    const bool in = t < stages - 1 || whole;
    const int k = t * kStage;
#pragma unroll
    for (int i = 0; i < T::kALoads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          ra, (lds_ptr)(to + (wave + i * T::kWaves) * 1024), 16,
          static_cast<int>(in ? av[i] : kOutside), k, 0, 0);
#pragma unroll
    for (int i = 0; i < T::kBLoads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rb, (lds_ptr)(to + T::TM * kStage + (wave + i * T::kWaves) * 1024), 16,
          static_cast<int>(in ? bv[i] : kOutside), k, 0, 0);
    __builtin_amdgcn_sched_barrier(0);  // not behind the stage that is multiplied meanwhile
  };

  // Fragment reads: step ks of a stage is pieces 2 ks + lane / 32.
  const int fr = lane & 31;
  const int at0 = fr * kStage + (((lane >> 5) ^ (fr & 7)) << 4);
  const int a0 = at0 + wm * T::MT * 32 * kStage;
  auto compute = [&](const char* from) {
    i32x4 fa[2][T::MT], fb[2][T::NT];
    auto read = [&](int ks) {
#pragma unroll
      for (int i = 0; i < T::NT; ++i)
        fb[ks & 1][i] = *reinterpret_cast<const i32x4*>(
            from + T::TM * kStage + (at0 ^ (ks << 5)) + T::b_row(wn, i) * kStage);
#pragma unroll
      for (int i = 0; i < T::MT; ++i)
        fa[ks & 1][i] =
            *reinterpret_cast<const i32x4*>(from + (a0 ^ (ks << 5)) + i * 32 * kStage);
    };
    read(0);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks < 3) read(ks + 1);
      __builtin_amdgcn_sched_barrier(0);  // the next step's reads before this one's products
#pragma unroll
      for (int i = 0; i < T::MT; ++i)
#pragma unroll
        for (int j = 0; j < T::NT; ++j)
          acc[i][j] = Ops<KIND>::mma32(fa[ks & 1][i], fb[ks & 1][j], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

#pragma unroll
  for (int i = 0; i < T::MT; ++i)
#pragma unroll
    for (int j = 0; j < T::NT; ++j) acc[i][j] = typename Ops<KIND>::Acc16{};
  issue(s0, 0);
  int t = 0;
  for (; t + 1 < stages; t += 2) {
    stage_barrier();  // stage t has landed; everyone is done with the other buffer
    issue(s1, t + 1);
    compute(s0);
    stage_barrier();
    if (t + 2 < stages) issue(s0, t + 2);
    compute(s1);
  }
  if (t < stages) {
    stage_barrier();
    compute(s0);
  }
}

// Row of acc register r of a 32 x 32 tile (its column is lane % 32).
__device__ __forceinline__ int acc_row(int lane, int r) {
  return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
}

// The tile of workgroup t, XCD-major in groups of rows that a 4 MiB L2 holds together
// with the columns being walked: in a group, rows fastest.
__device__ __forceinline__ void tile_at(int gm, int gn, int group, int* mt, int* nt) {
  const int t = vkd::xcd_tile(blockIdx.x, gridDim.x);
  const int per = group * gn;
  const int g = t / per, r = t - g * per;
  const int left = gm - g * group, rows = left < group ? left : group;
  *mt = g * group + r % rows;
  *nt = r / rows;
}

// ---------------------------------------------------------------- activations
// act(g): SiLU g / (1 + e^-g), GELU g Phi(g) with the device erff.  The exponential is
// v_exp_f32 of g log2(e) and the quotient v_rcp_f32: some 2 ulp each, against
// results that are then multiplied and, but for f32 outputs, rounded to 16 bits.
template <int ACT>
__device__ __forceinline__ float gate(float g) {
  if constexpr (ACT == VK_GATE_SILU)
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504f));
  else
    return vkd::gelu1<1>(g);
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
    const float phi = 0.5f + 0.5f * erff(g * 0.70710678f);
    *act = g * phi;
    *slope = __builtin_fmaf(g * 0.39894228f, __builtin_amdgcn_exp2f(g * g * -0.72134752f), phi);
  }
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

// Loads of b for U stages t, t + 8, ...: zeros past k and past the last stage.
template <bool PAIRED, int U>
struct FewColumns {
  i32x4 v[U][PAIRED ? 2 : 1][2];
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rb, const uint32_t (&at)[2], int q,
                                       int t, int k_bytes) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int p = 0; p < (PAIRED ? 2 : 1); ++p)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = (t + u * kFewWaves) * kStage + q * 32 + h * 16;
          v[u][p][h] = __builtin_bit_cast(
              i32x4, vkd::buffer_load4(rb, k < k_bytes ? at[p] + static_cast<uint32_t>(k) : kOutside, 0));
        }
  }
};

// The resource and the lane's row offsets of the columns n0 .. n0 + 16.  Columns past
// the last one read the last one.
template <bool PAIRED>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t few_rows_of(const Operand& b, int n0, int c,
                                                              uint32_t (&at)[2]) {
  const int held = PAIRED ? b.rows / 2 : b.rows;
  const int n = n0 + c < held ? c : held - 1 - n0;
  at[0] = static_cast<uint32_t>(n) * b.pitch;
  at[1] = static_cast<uint32_t>(n + (PAIRED ? held : 0)) * b.pitch;
  const size_t from = static_cast<size_t>(n0) * b.pitch;
  const size_t left = static_cast<size_t>(b.rows) * b.pitch - from;
  return vkd::buffer_rsrc(b.base + from, left < kMostBytes ? static_cast<uint32_t>(left) : kMostBytes);
}

// The sums of all waves: thread i < 256 RT has (p, row, column) element i of each p.
template <Kind KIND, int RT, bool PAIRED>
__device__ __forceinline__ void few_join(const FewSums<KIND, RT, PAIRED>& s, char* smem, int wave,
                                         int lane) {
  typedef typename Ops<KIND>::Acc4 Acc4;
  Acc4* red = reinterpret_cast<Acc4*>(smem);
#pragma unroll
  for (int p = 0; p < (PAIRED ? 2 : 1); ++p)
#pragma unroll
    for (int r = 0; r < RT; ++r) red[((wave * (PAIRED ? 2 : 1) + p) * RT + r) * 64 + lane] = s.v[p][r];
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

// The product of rows 0 .. a.rows of a, read from memory.
template <Kind KIND, int RT, bool PAIRED>
__device__ __forceinline__ void few_product(const Operand& a, const Operand& b, int k_bytes, int n0,
                                            char* smem) {
  constexpr int U = 2;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  uint32_t at[2], aat[RT];
  const auto rb = few_rows_of<PAIRED>(b, n0, c, at);
  const size_t a_bytes = static_cast<size_t>(a.rows) * a.pitch;
  const auto ra = vkd::buffer_rsrc(a.base, a_bytes < kMostBytes ? static_cast<uint32_t>(a_bytes) : kMostBytes);
#pragma unroll
  for (int r = 0; r < RT; ++r)
    aat[r] = r * 16 + c < a.rows ? static_cast<uint32_t>(r * 16 + c) * a.pitch : kOutside;
  FewSums<KIND, RT, PAIRED> s{};
  const int stages = (k_bytes + kStage - 1) / kStage;
  for (int t = wave; t < stages; t += U * kFewWaves) {
    FewColumns<PAIRED, U> fb;
    fb.load(rb, at, q, t, k_bytes);
    i32x4 fa[U][RT][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = (t + u * kFewWaves) * kStage + q * 32 + h * 16;
          fa[u][r][h] = __builtin_bit_cast(
              i32x4, vkd::buffer_load4(ra, k < k_bytes && aat[r] != kOutside ? aat[r] + static_cast<uint32_t>(k) : kOutside, 0));
        }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int p = 0; p < (PAIRED ? 2 : 1); ++p)
#pragma unroll
          for (int r = 0; r < RT; ++r)
            s.v[p][r] = Ops<KIND>::mma16(fa[u][r][h], fb.v[u][p][h], s.v[p][r]);
  }
  few_join<KIND, RT, PAIRED>(s, smem, wave, lane);
}

}  // namespace vkp
