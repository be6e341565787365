// A gated feed-forward's first half in 16 bits (f16 or bf16) for gfx950, forward and
// backward.
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) * u          (w = [Wg; Wu])
//
// Forward is one kernel: a workgroup's tile holds the gates and their partners of the
// same hidden columns, so both products, the activation and the product of the two
// meet in registers; h is rounded once.
//
// Backward, from x, w, b and the gradient dh, with nothing kept from the forward:
//   1. g and u again, and in the same kernel dg = dh u act'(g), du = dh act(g), in
//      f32 up to one rounding to x's type: the two products below take 16-bit
//      operands.  That rounding is as large as the result's own (10,392 x 1536 -> 2 x 4096 in
//      bf16: off by 2.3e-3 of the norm with it, 1.7e-3 without); held as two 16-bit parts, the
//      products below would have to be made twice, 430 us of 930.  Written as rows dg | du, with
//      the f32 column sums of each tile.  In f16, whose range is short, they are written times a
//      power of two where their largest asks for it (Range);
//   2. dx = [dg du] [Wg; Wu], w's lines being k;
//   3. dw = [dg du]^T x, the lines of both being k;
//   4. db: the tiles' column sums added in order;
// the last three in one launch.
#include "product_nt.h"

namespace {

using vkp::Kind;
using vkp::kBF16;
using vkp::kF16;
using vkp::Operand;

// What f16 holds of dg and du.  Its numbers end at 65,504 and are whole multiples of 2^-24: a
// loss's scale moves gradients past either end while dx and dw would be held.  So the first launch
// of step 1 also finds the largest |dg|, |du| (a NaN aside): every workgroup leaves its tile's, the
// last one to arrive takes the largest of all and with it the power of two that d is to be written
// times. That is 1 from 2^-8 (below which values of a 64th of the largest would lose bits) to
// 65,504, and for an infinity; otherwise a second launch writes d again, its largest in [2^14,
// 2^15), and steps 2 and 3 take the power back in f32.  At a power of 1 the second launch ends at
// once.  A backward of 257 x 384 -> 2 x 1023 takes 23.6 us (29 written again, 19.6 with none of
// this), of 866 x 768 -> 2 x 2048 41.8 (52; 38.2), of 10,392 x 1536 -> 2 x 4096 715 (974; 690).
// bf16 has f32's range and none of this.
struct Range {
  float* power;  // and 1 / power behind it; null: none of this
  float* peaks;  // of each tile
  unsigned* arrivals;  // 1 + kPeakGroups counters, a line each; zero before and after a launch
  bool again;
};
// Tiles arrive by groups, and a group's last one for all of it: at one counter they would queue,
// some 14 ns each (866 x 768 -> 2 x 2048 in 896 tiles of 64 x 64: 26.4 us against 19.3).
constexpr int kPeakGroups = 32, kPeakLine = 16;
__device__ __forceinline__ float power_for(float peak) {
  const int e = static_cast<int>(__float_as_uint(peak) >> 23);
  const bool held = peak == 0.0f || (peak >= 0x1p-8f && peak <= 65504.0f) || e == 255;
  const int power = 268 - e < 240 ? 268 - e : 240;  // 2^14 over the peak's own power, biased
  return held ? 1.0f : __uint_as_float(static_cast<uint32_t>(power) << 23);
}

struct Args {
  Operand a, b;
  int k_bytes;
  const void* bias;  // 2 N values of the type, or null
  const void* grad;  // [M, N]
  void* out;         // [M, N]; null in the backward
  void* d;           // dg | du, rows of 2 d_half values, zeros from N to d_half of each half
  float* sums;       // [gm * WM, 2 N], or null
  int d_half;
  Range range;       // of d in f16
  int M, N;
  int act;
  int gm, gn, group;
  vkp::Split split;
};

template <Kind KIND>
__device__ __forceinline__ float bias_at(const Args& g, int n) {
  typedef typename vkp::Value<KIND>::type V;
  return g.bias ? vkp::widen(static_cast<const V*>(g.bias)[n]) : 0.0f;
}

// The tile's biases, gates then partners.
template <Kind KIND, typename T>
__device__ __forceinline__ void load_bias(const Args& g, int n0, float* to) {
  for (int c = threadIdx.x; c < T::TN; c += T::kThreads) {
    const int n = n0 + c % T::kHeld;
    to[c] = bias_at<KIND>(g, (n < g.N ? n : g.N - 1) + (c < T::kHeld ? 0 : g.N));
  }
}

// The forward's tiles.  A wave has gates and partners of the same columns in its sums, so nothing
// but h leaves.  10,392 x 1536 -> 2 x 4096 in bf16: 235 us with SiLU (1.11 PFLOP/s; a library's
// plain product of these sizes 278), 247 with GELU, whose Phi no other work covers; 866 x 1024 -> 2
// x 2736 in f16 16.5, one round of tiles.  Bound by the products (product_nt.h) and the tiles'
// ends.
template <Kind KIND, typename T>
__global__ __launch_bounds__(T::kThreads, T::kWavesASimd) void gated_kernel(Args g) {
  typedef typename vkp::Value<KIND>::type V;
  VK_STAGES(T);
  __shared__ __align__(16) float bias[T::TN];
  int mt, nt;
  const int tiles = g.gm * g.gn, tile = blockIdx.x % tiles, part = blockIdx.x / tiles;
  vkp::tile_at(tile, g.gm, g.gn, g.group, &mt, &nt);
  const int m0 = mt * T::TM, n0 = nt * T::kHeld;
  load_bias<KIND, T>(g, n0, bias);
  const vkp::Place<T> place;
  vkp::f32x16 acc[T::MT][T::NT];
  if (!vkp::product_tile<KIND, T>(g.a, g.b, g.k_bytes, m0, n0, g.split, part, tile, tiles, place,
                                  stages_, acc))
    return;
  const int lane = place.lane, wave = place.wave, wm = place.wm, wn = place.wn;
  constexpr int kCols = T::NT / 2;
  typedef vkp::Chunk<V, kCols> C;
  char* chunk = stages_[0] + wave * C::kBytes;
  vkp::with_act(g.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < T::MT; ++i) {
#pragma unroll
      for (int j = 0; j < kCols; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = T::b_row(wn, j) + 8 * q + 4 * (lane >> 5);
          const vkp::f32x4 bg = *reinterpret_cast<const vkp::f32x4*>(bias + c);
          const vkp::f32x4 bu = *reinterpret_cast<const vkp::f32x4*>(bias + T::kHeld + c);
          typename C::V4 h;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            h[e] = static_cast<V>(vkp::gate<act.value>(acc[i][j][4 * q + e] + bg[e]) *
                                  (acc[i][j + kCols][4 * q + e] + bu[e]));
          *C::at(chunk, lane, j, q) = h;
        }
      vkd::wave_lds_fence();
      C::template store<false>(chunk, lane, static_cast<V*>(g.out), g.N, m0 + (wm * T::MT + i) * 32,
                               g.M, n0 + T::b_row(wn, 0), g.N);
      vkd::wave_lds_fence();
    }
  });
}

// A workgroup's largest |dg|, |du|, from its waves'; behind the barrier wave 0 goes on alone, and
// the last tile's takes the power.  Stores and loads of peaks go past the XCD's L2, as those of
// shared sums do.
template <typename T>
__device__ __forceinline__ void leave_peak(const Range& range, int tile, int tiles, float peak,
                                           const vkp::Place<T>& at, float* waves) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) peak = fmaxf(peak, __shfl_xor(peak, d, 64));
  if (at.lane == 0) waves[at.wave] = peak;
  __syncthreads();
  if (at.wave > 0) return;
#pragma unroll
  for (int w = 0; w < T::kWaves; ++w) peak = fmaxf(peak, waves[w]);
  int last = 0;
  if (at.lane == 0) {
    __hip_atomic_store(&range.peaks[tile], peak, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the peak is there, then the count
    const auto arrive = [](unsigned* counter, int all) {
      const unsigned n = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED,
                                                __HIP_MEMORY_SCOPE_AGENT);
      if (n + 1 != static_cast<unsigned>(all)) return 0;
      __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      return 1;
    };
    const int group = tile % kPeakGroups, groups = tiles < kPeakGroups ? tiles : kPeakGroups;
    if (arrive(range.arrivals + (1 + group) * kPeakLine, (tiles - group - 1) / kPeakGroups + 1))
      last = arrive(range.arrivals, groups);
  }
  if (__builtin_amdgcn_readfirstlane(last) == 0) return;
  for (int t = at.lane; t < tiles; t += 64)
    peak = fmaxf(peak, __hip_atomic_load(&range.peaks[t], __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT));
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) peak = fmaxf(peak, __shfl_xor(peak, d, 64));
  if (at.lane == 0) {
    const float power = power_for(peak);
    range.power[0] = power;
    range.power[1] = 1.0f / power;
  }
}

// Step 1 of the backward: the forward's products, then dg and du where h would be, through the same
// LDS rows as e came in by.  10,392 x 1536 -> 2 x 4096 in bf16: 262-285 us, of which the 340 MB of
// d are some 40 that no product covers.
template <Kind KIND, typename T>
__global__ __launch_bounds__(T::kThreads, T::kWavesASimd) void gated_grad_kernel(Args g) {
  typedef typename vkp::Value<KIND>::type V;
  VK_STAGES(T);
  __shared__ __align__(16) float bias[T::TN];
  constexpr bool kRanged = KIND == kF16;
  float power = 1.0f, peak = 0.0f;
  if constexpr (kRanged) {
    if (g.range.again) {
      power = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(g.range.power[0])));
      if (power == 1.0f) return;
    }
  }
  int mt, nt;
  const int tiles = g.gm * g.gn, tile = blockIdx.x % tiles, part = blockIdx.x / tiles;
  vkp::tile_at(tile, g.gm, g.gn, g.group, &mt, &nt);
  const int m0 = mt * T::TM, n0 = nt * T::kHeld;
  load_bias<KIND, T>(g, n0, bias);
  const vkp::Place<T> place;
  vkp::f32x16 acc[T::MT][T::NT];
  if (!vkp::product_tile<KIND, T>(g.a, g.b, g.k_bytes, m0, n0, g.split, part, tile, tiles, place,
                                  stages_, acc))
    return;
  const int lane = place.lane, wave = place.wave, wm = place.wm, wn = place.wn;
  constexpr int kCols = T::NT / 2;
  typedef vkp::Chunk<V, kCols> C;
  char* chunk = stages_[0] + wave * C::kBytes;
  const V* grad = static_cast<const V*>(g.grad);
  V* d = static_cast<V*>(g.d);
  const size_t pitch = 2 * static_cast<size_t>(g.d_half);
  const int nb = n0 + T::b_row(wn, 0);
  float sum[kCols] = {};
  vkp::with_act(g.act, [&](auto act) {
    vkp::i32x4 dh[C::kFetch];
    C::fetch(dh, lane, grad, g.N, m0 + wm * T::MT * 32, g.M, nb, g.N);
#pragma unroll
    for (int i = 0; i < T::MT; ++i) {
      const int mb = m0 + (wm * T::MT + i) * 32;
      C::fill(chunk, lane, dh);
      if (i + 1 < T::MT) C::fetch(dh, lane, grad, g.N, mb + 32, g.M, nb, g.N);
      vkd::wave_lds_fence();
      // rows past M and columns past N have dh of 0; what their g and u are is finite only where
      // the others' are
      const bool in = mb + (lane & 31) < g.M;
      typename C::V4 du[kCols][4];
      float v[kCols * 32];
#pragma unroll
      for (int j = 0; j < kCols; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = T::b_row(wn, j) + 8 * q + 4 * (lane >> 5);
          const vkp::f32x4 bg = *reinterpret_cast<const vkp::f32x4*>(bias + c);
          const vkp::f32x4 bu = *reinterpret_cast<const vkp::f32x4*>(bias + T::kHeld + c);
          typename C::V4* at = C::at(chunk, lane, j, q);
          const typename C::V4 h4 = *at;
          typename C::V4 dg;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float a, s;
            vkp::gate_slope<act.value>(acc[i][j][4 * q + e] + bg[e], &a, &s);
            const float h = vkp::widen(h4[e]);
            const bool held = in && n0 + c + e < g.N;
            const float fg = held ? h * (acc[i][j + kCols][4 * q + e] + bu[e]) * s : 0.0f;
            const float fu = held ? h * a : 0.0f;
            v[j * 16 + 4 * q + e] = fg;
            v[kCols * 16 + j * 16 + 4 * q + e] = fu;
            if constexpr (kRanged) peak = fmaxf(fmaxf(peak, fabsf(fg)), fabsf(fu));
            dg[e] = static_cast<V>(kRanged ? fg * power : fg);
            du[j][q][e] = static_cast<V>(kRanged ? fu * power : fu);
          }
          *at = dg;
        }
      if (g.sums) {
        vkp::sum_rows<kCols>(v, lane);
#pragma unroll
        for (int k = 0; k < kCols; ++k) sum[k] += v[k];
      }
      if (d) {
        vkd::wave_lds_fence();
        C::template store<false>(chunk, lane, d, pitch, mb, g.M, nb, g.d_half);
        vkd::wave_lds_fence();
#pragma unroll
        for (int j = 0; j < kCols; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) *C::at(chunk, lane, j, q) = du[j][q];
        vkd::wave_lds_fence();
        C::template store<false>(chunk, lane, d + g.d_half, pitch, mb, g.M, nb, g.d_half);
      }
      vkd::wave_lds_fence();
    }
  });
  if (g.sums) {
    // value k of lane l: columns of dg, then of du, by j, q, e
#pragma unroll
    for (int k = 0; k < kCols; ++k) {
      const int at = kCols * (lane & 31) + k, part = at / (kCols * 16), j = at / 16 % kCols;
      const int n = n0 + T::b_row(wn, 0) + 32 * j + 8 * (at / 4 % 4) + 4 * (lane >> 5) + at % 4;
      if (n < g.N) g.sums[(static_cast<size_t>(mt * T::WM + wm) * 2 + part) * g.N + n] = sum[k];
    }
  }
  if constexpr (kRanged)
    if (g.range.power && !g.range.again)
      leave_peak<T>(g.range, tile, tiles, peak, place, reinterpret_cast<float*>(stages_[1]));
}

// One of the products of steps 2 and 3: out[m, n] = sum_k a[m, k] b[n, k], rounded to the type; a
// as rows or columns, b as columns.  With m_half > 0 a's rows come in two halves: row m < m_half is
// out's m where that is below M / 2, row m >= m_half out's M / 2 + m - m_half where that is below
// M.
struct Product {
  Operand a, b;
  int k_bytes;
  void* out;
  const float* back;  // what the sums are to be multiplied by, or null
  int M, N, m_half;
  int gm, gn, group;
  vkp::Split split;
};

template <Kind KIND, typename T, bool AC>
__device__ __forceinline__ void product(const Product& g, int wg, char* const (&stages_)[4]) {
  typedef typename vkp::Value<KIND>::type V;
  const int tiles = g.gm * g.gn, tile = wg % tiles, part = wg / tiles;
  int mt, nt;
  vkp::tile_at(tile, g.gm, g.gn, g.group, &mt, &nt);
  const int m0 = mt * T::TM, n0 = nt * T::TN;
  const vkp::Place<T> place;
  float back = 1.0f;
  if constexpr (KIND == kF16)
    back = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(*g.back)));
  vkp::f32x16 acc[T::MT][T::NT];
  if (!vkp::product_tile<KIND, T, AC, true>(g.a, g.b, g.k_bytes, m0, n0, g.split, part, tile, tiles,
                                            place, stages_, acc))
    return;
  const int lane = place.lane, wave = place.wave, wm = place.wm, wn = place.wn;
  constexpr int J = T::NT % 2 ? 1 : 2;  // column tiles of 32 that leave together
  typedef vkp::Chunk<V, J> C;
  char* chunk = stages_[0] + wave * C::kBytes;
#pragma unroll
  for (int i = 0; i < T::MT; ++i) {
    int mb = m0 + (wm * T::MT + i) * 32, end = g.M;
    if (g.m_half > 0) {  // 32 rows lie in one half: m_half is a multiple of 64
      end = g.M / 2;
      if (mb >= g.m_half) {
        mb += end - g.m_half;
        end = g.M;
      }
    }
#pragma unroll
    for (int jg = 0; jg < T::NT; jg += J) {
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          typename C::V4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = acc[i][jg + j][4 * q + e];
            w[e] = static_cast<V>(KIND == kF16 ? v * back : v);
          }
          *C::at(chunk, lane, j, q) = w;
        }
      vkd::wave_lds_fence();
      C::template store<false>(chunk, lane, static_cast<V*>(g.out), g.N, mb, end,
                               n0 + T::b_row(wn, jg), g.N);
      vkd::wave_lds_fence();
    }
  }
}

// dbias: the tiles' sums of COLS columns, eight runs of parts each in order, then the runs in
// order.
struct BiasSums {
  const float* sums;  // [parts, cols]
  int parts, cols;
  void* out;
};

template <Kind KIND, int COLS>
__device__ __forceinline__ void bias_gradient(const BiasSums& g, int block, char* smem) {
  float(*run)[COLS] = reinterpret_cast<float(*)[COLS]>(smem);
  const int x = threadIdx.x % COLS, y = threadIdx.x / COLS, c = block * COLS + x;
  const int from = g.parts * y / 8, to = g.parts * (y + 1) / 8;
  float part = 0.0f;
  if (c < g.cols)
#pragma unroll 8
    for (int p = from; p < to; ++p) part += g.sums[static_cast<size_t>(p) * g.cols + c];
  run[y][x] = part;
  __syncthreads();
  if (y > 0 || c >= g.cols) return;
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += run[i][x];
  static_cast<typename vkp::Value<KIND>::type*>(g.out)[c] =
      static_cast<typename vkp::Value<KIND>::type>(s);
}

// Steps 2 to 4 in one launch, dx apart where that is cheaper: they need the same step before them,
// and few rows leave the card half empty one after another.  The first n_dx workgroups are dx, the
// next n_dw dw, the others dbias: short ones, for the CUs that the tiles leave.  866 x 768 x 2048:
// 24 us (apart 16 + 13 and a launch); 10,392 x 1536 x 4096, apart: dx 205-213, dw 214-238 (a
// library's plain products 185 and 216).
template <Kind KIND, typename T>
__global__ __launch_bounds__(T::kThreads, T::kWavesASimd) void gradients_kernel(
    Product dx, Product dw, BiasSums bias, int n_dx, int n_dw) {
  VK_STAGES(T);
  const int wg = blockIdx.x;
  if (wg < n_dx)
    product<KIND, T, false>(dx, wg, stages_);
  else if (wg < n_dx + n_dw)
    product<KIND, T, true>(dw, wg - n_dx, stages_);
  else
    bias_gradient<KIND, T::kThreads / 8>(bias, wg - n_dx - n_dw, stages_[0]);
}

// Forward of at most 16 RT rows, one workgroup to 16 hidden columns: w is read once.  5 rows, 1024
// -> 2 x 2736 in bf16: 4.8 us, the launch and its chain; 8 rows, 8192 -> 2 x 4096: 21 us, 6.4 TB/s.
template <Kind KIND, int RT>
__global__ __launch_bounds__(vkp::kFewThreads) void gated_few_kernel(Args g) {
  typedef typename vkp::Value<KIND>::type V;
  __shared__ __align__(16) char smem[vkp::few_bytes<KIND, RT, true>()];
  const int n0 = blockIdx.x * 16;
  vkp::few_product<KIND, RT, true>(g.a, g.b, g.k_bytes, n0, smem);
  for (int e = threadIdx.x; e < 256 * RT; e += vkp::kFewThreads) {
    const int m = e >> 4, n = n0 + (e & 15);
    if (m >= g.M || n >= g.N) continue;
    const float gate = vkp::few_sum<KIND, RT, true>(smem, 0, m, e & 15) + bias_at<KIND>(g, n);
    const float up = vkp::few_sum<KIND, RT, true>(smem, 1, m, e & 15) + bias_at<KIND>(g, g.N + n);
    vkp::with_act(g.act, [&](auto act) {
      static_cast<V*>(g.out)[static_cast<size_t>(m) * g.N + n] =
          static_cast<V>(vkp::gate<act.value>(gate) * up);
    });
  }
}

// ---------------------------------------------------------------- layouts
// Rows of x, then of w, of `cols` 16-bit values into rows of 8 `pieces`, zeros behind.
__global__ __launch_bounds__(256) void pad16_kernel(const char* __restrict__ x,
                                                    const char* __restrict__ w, size_t x_rows,
                                                    size_t rows, int cols, int pieces,
                                                    char* __restrict__ to) {
  const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  const size_t row = i / static_cast<unsigned>(pieces);
  if (row >= rows) return;
  const int piece = static_cast<int>(i - row * static_cast<unsigned>(pieces));
  const char* from = row < x_rows ? x + row * 2 * cols : w + (row - x_rows) * 2 * cols;
  vkp::i32x4 v = {0, 0, 0, 0};
  if (16 * piece + 16 <= 2 * cols)
    __builtin_memcpy(&v, from + 16 * piece, 16);
  else if (16 * piece < 2 * cols)
    v = vkp::row_rest(from, 2 * cols);
  *reinterpret_cast<vkp::i32x4*>(to + i * 16) = v;
}

__global__ __launch_bounds__(256) void zero16_kernel(uint16_t* to, size_t n) {
  const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) to[i] = 0;
}

void zero16(const vk_runtime* rt, void* p, size_t n) {
  hipLaunchKernelGGL(zero16_kernel, dim3((n + 255) / 256), dim3(256), 0, rt->stream,
                     static_cast<uint16_t*>(p), n);
}

// ---------------------------------------------------------------- launches
constexpr size_t kPitchValues = 64;  // rows of workspace start on 128-byte lines
size_t padded(size_t n) { return (n + kPitchValues - 1) / kPitchValues * kPitchValues; }
constexpr size_t kMostPieces = size_t{0x7fffff} * 256;  // of 16 bytes, that a launch copies

template <bool PAIRED, typename F>
void with_tile(vkp::TileSize size, Args& g, F go) {
  vkp::with_tile<PAIRED>(size, [&](auto tile) {
    typedef decltype(tile) T;
    g.gm = (g.M + T::TM - 1) / T::TM;
    g.gn = (g.N + T::kHeld - 1) / T::kHeld;
    g.group = vkp::kGroupRows / T::TM;
    go(tile);
  });
}

vkp::Shape forward_shape(const Args& g) { return vkp::Shape{g.M, 2LL * g.N, g.k_bytes, true}; }

template <Kind KIND>
int launch_forward(vk_runtime* rt, Args& g, const vkp::Plan& p) {
  if (p.few) {
    const dim3 grid((g.N + 15) / 16), block(vkp::kFewThreads);
    if (g.M <= 16)
      hipLaunchKernelGGL((gated_few_kernel<KIND, 1>), grid, block, 0, rt->stream, g);
    else
      hipLaunchKernelGGL((gated_few_kernel<KIND, 2>), grid, block, 0, rt->stream, g);
    return vk::check_launch("gated_few_kernel");
  }
  g.split.count = p.splits;
  g.split.arrivals = rt->arrivals;
  with_tile<true>(p.tile, g, [&](auto tile) {
    typedef decltype(tile) T;
    hipLaunchKernelGGL((gated_kernel<KIND, T>), dim3(g.gm * g.gn * p.splits), dim3(T::kThreads), 0,
                       rt->stream, g);
  });
  return vk::check_launch("gated_kernel");
}

// x's and w's rows as operands: as they are, or where a row is no multiple of 16 bytes, copied into
// the work buffer with zeros behind.
size_t operands_room(size_t rows, size_t in, size_t hidden) {
  return in % 8 == 0 ? 0 : (rows + 2 * hidden) * padded(in) * 2;
}

// What the backward's launches are and what they keep in the work buffer: d, the biases' sums, d's
// power and peaks (f16), then split tiles' sums, of the first step and after it of the products.
struct BackwardPlan {
  vkp::Plan first;
  vkp::PlanTwo second;
  bool ranged;
  size_t range, work, dx_sums, bytes;
};
constexpr size_t kPowers = 64;  // bytes before the peaks
static_assert(2 * vkp::kMostTilesSplit + (1 + kPeakGroups) * kPeakLine <= vk::kArrivals,
              "counters of dx's and dw's shared tiles, then of the peaks");
// Of the first step in f16: a larger tile's sums leave no registers for the power and the peak.
constexpr vkp::TileSize kLargestRanged = vkp::kTile192;
BackwardPlan plan_backward(int cus, const Args& g, size_t in, bool f16, bool dx, bool dw,
                           bool dbias) {
  BackwardPlan p{};
  double us = 0;
  const size_t rows = g.M, half = padded(g.N);
  // the zeros up to d_half too
  const vkp::Shape step{g.M, static_cast<long long>(2 * half), g.k_bytes, true};
  p.ranged = f16 && (dx || dw);
  p.first = vkp::plan(cus, step, &us, 0, f16 ? kLargestRanged : vkp::kTile256);
  const auto D = static_cast<long long>(in);
  const vkp::Shape x{dx ? g.M : 0, D, static_cast<long long>(4 * half)};
  const vkp::Shape w{dw ? static_cast<long long>(2 * half) : 0, D, 2LL * g.M};
  p.second = vkp::plan_two(cus, x, w);
  const auto round = [](size_t n) { return (n + 255) / 256 * 256; };
  if (dx || dw) p.work += round(rows * 4 * half);
  // (a tile of 64 or 128 rows has two waves' sums, one of 256 four)
  if (dbias) p.work += round(((rows + 63) / 64 * 2 + 4) * 2 * g.N * 4);
  p.range = p.work;
  if (p.ranged) p.work += round(kPowers + vkp::tiles_of(p.first.tile, step) * 4);
  p.dx_sums = vkp::split_bytes(p.second.tile[0], vkp::Job{x, p.second.splits[0]});
  const size_t after =
      p.dx_sums + vkp::split_bytes(p.second.tile[1], vkp::Job{w, p.second.splits[1]});
  const size_t before = vkp::split_bytes(p.first.tile, vkp::Job{step, p.first.splits});
  p.bytes = p.work + (before > after ? before : after);
  return p;
}

template <Kind KIND>
int backward(vk_runtime* rt, Args& g, const BackwardPlan& plan, size_t rows, size_t in,
             size_t hidden, char* room, vk_tensor* dx, vk_tensor* dw, vk_tensor* dbias) {
  const size_t half = padded(hidden), d_bytes = dx || dw ? (rows * 4 * half + 255) / 256 * 256 : 0;
  if (dx || dw) {
    g.d = room;
    g.d_half = static_cast<int>(half);
  }
  if (dbias) g.sums = reinterpret_cast<float*>(room + d_bytes);
  const float* sums_of_tiles = g.sums;
  if (plan.ranged)
    g.range = Range{reinterpret_cast<float*>(room + plan.range),
                    reinterpret_cast<float*>(room + plan.range + kPowers),
                    rt->arrivals + 2 * vkp::kMostTilesSplit, false};
  g.split = vkp::Split{plan.first.splits, room + plan.work, rt->arrivals};
  int parts = 0;
  with_tile<true>(plan.first.tile, g, [&](auto tile) {
    typedef decltype(tile) T;
    if constexpr (KIND != kF16 || !std::is_same_v<T, vkp::Tile<4, 2, 2, 4, true, 2, 1>>) {
      parts = g.gm * T::WM;
      g.gn = (static_cast<int>(half) + T::kHeld - 1) / T::kHeld;  // the zeros up to d_half too
      const dim3 grid(g.gm * g.gn * g.split.count), block(T::kThreads);
      hipLaunchKernelGGL((gated_grad_kernel<KIND, T>), grid, block, 0, rt->stream, g);
      if (plan.ranged) {  // d again, where another power holds it better; the biases' sums stand
        g.range.again = true;
        g.sums = nullptr;
        hipLaunchKernelGGL((gated_grad_kernel<KIND, T>), grid, block, 0, rt->stream, g);
      }
    }
  });
  VK_TRY(vk::check_launch("gated_grad_kernel"));
  const char* d = static_cast<char*>(g.d);
  const auto pitch = static_cast<uint32_t>(4 * half);
  const int R = static_cast<int>(rows), values = static_cast<int>((in + 7) / 8 * 8);
  const int D = static_cast<int>(in), H2 = static_cast<int>(2 * hidden);
  const int both = static_cast<int>(2 * half);
  Product x{}, w{};
  if (dx) {
    x.a = Operand{d, R, pitch};
    x.b = g.b;  // w's lines are k
    x.b.rows = values;
    x.b.ks = H2;
    x.b.k_half = static_cast<int>(half);
    x.k_bytes = 2 * both;
    x.out = dx->ptr;
    if (plan.ranged) x.back = g.range.power + 1;
    x.M = R;
    x.N = D;
  }
  if (dw) {
    w.a = Operand{d, both, pitch, R};
    w.b = g.a;  // x's lines are k
    w.b.rows = values;
    w.b.ks = R;
    w.k_bytes = 2 * R;
    w.out = dw->ptr;
    if (plan.ranged) w.back = g.range.power + 1;
    w.M = H2;
    w.N = D;
    w.m_half = static_cast<int>(half);
  }
  BiasSums sums{sums_of_tiles, parts, H2, dbias ? dbias->ptr : nullptr};
  // (the first step's split sums are done with)
  const vkp::PlanTwo& two = plan.second;
  x.split = vkp::Split{two.splits[0], room + plan.work, rt->arrivals};
  w.split = vkp::Split{two.splits[1], room + plan.work + plan.dx_sums,
                       rt->arrivals + vkp::kMostTilesSplit};
  // one launch, or dx and dbias in one of their own
  for (int part = two.together ? 1 : 0; part < 2; ++part) {
    vkp::with_tile<false>(two.tile[part], [&](auto tile) {
      typedef decltype(tile) T;
      for (Product* p : {&x, &w}) {
        p->gm = (p->a.rows + T::TM - 1) / T::TM;
        p->gn = (p->N + T::TN - 1) / T::TN;
        p->group = vkp::kGroupRows / T::TM;
      }
      const int n_dx = part == 0 || two.together ? x.gm * x.gn * x.split.count : 0;
      const int n_dw = part == 0 ? 0 : w.gm * w.gn * w.split.count;
      constexpr int kCols = T::kThreads / 8;
      const int biases = dbias && part == (two.together ? 1 : 0) ? (H2 + kCols - 1) / kCols : 0;
      if (biases + n_dx + n_dw > 0)
        hipLaunchKernelGGL((gradients_kernel<KIND, T>), dim3(biases + n_dx + n_dw),
                           dim3(T::kThreads), 0, rt->stream, x, w, sums, n_dx, n_dw);
    });
    VK_TRY(vk::check_launch("gradients_kernel"));
  }
  return VK_OK;
}

// ---------------------------------------------------------------- arguments
int check16(const vk_runtime* rt, const vk_tensor* t, vk_dtype dtype, size_t len,
            const char* what) {
  VK_REQUIRE(t && t->dtype == dtype && t->len == len,
             "gated: %s must hold %zu values of x's type (holds %zu)", what, len, t ? t->len : 0);
  VK_REQUIRE(reinterpret_cast<uintptr_t>(t->ptr) % 16 == 0, "gated: %s must be 16-byte aligned",
             what);
  return vk::check_device(rt, t, what);
}

int check_inputs(vk_runtime* rt, const vk_tensor* x, const vk_tensor* w, const vk_tensor* bias,
                 size_t rows, size_t in, size_t hidden, int act) {
  VK_REQUIRE(x && w, "gated: null argument");
  VK_REQUIRE(x->dtype == VK_F16 || x->dtype == VK_BF16, "gated: x must be f16 or bf16");
  VK_REQUIRE(in > 0 && hidden > 0, "gated: empty weights");
  VK_REQUIRE(act == VK_GATE_SILU || act == VK_GATE_GELU, "gated: unknown activation %d", act);
  // a tile addresses its rows of an operand by 31 bits
  VK_UNSUPPORTED_IF(in > 0x100000 || hidden > 0x100000 || rows > 0x1000000,
                    "gated: %zu x %zu -> %zu", rows, in, hidden);
  VK_UNSUPPORTED_IF(2 * hidden * padded(in) * 2 > 0x7fffff00ULL, "gated: weights of %zu x %zu",
                    2 * hidden, in);
  VK_UNSUPPORTED_IF(((rows + 63) / 64) * ((hidden + 31) / 32) > 0x7fffffULL,
                    "gated: %zu x %zu outputs", rows, hidden);
  // the copies' launch (align_operands), a thread to 16 bytes
  VK_UNSUPPORTED_IF(in % 8 != 0 && (rows + 2 * hidden) * (padded(in) / 8) > kMostPieces,
                    "gated: %zu rows of %zu, no multiple of 8", rows + 2 * hidden, in);
  VK_TRY(check16(rt, x, x->dtype, rows * in, "x"));
  VK_TRY(check16(rt, w, x->dtype, 2 * hidden * in, "w"));
  if (bias) VK_TRY(check16(rt, bias, x->dtype, 2 * hidden, "bias"));
  return VK_OK;
}

Args forward_args(const vk_runtime* rt, const vk_tensor* x, const vk_tensor* w,
                  const vk_tensor* bias, size_t rows, size_t in, size_t hidden, int act) {
  Args g{};
  const char* xp = static_cast<const char*>(x->ptr);
  const char* wp = static_cast<const char*>(w->ptr);
  const auto pitch = static_cast<uint32_t>(2 * in);
  g.a = Operand{xp, static_cast<int>(rows), pitch};
  g.b = Operand{wp, static_cast<int>(2 * hidden), pitch};
  g.k_bytes = static_cast<int>(2 * in);
  g.bias = bias ? bias->ptr : nullptr;
  g.M = static_cast<int>(rows);
  g.N = static_cast<int>(hidden);
  g.act = act;
  return g;
}

// The tiles' operands: 16-byte aligned rows.
int align_operands(const vk_runtime* rt, Args& g, size_t in, char* room) {
  if (in % 8 == 0) return VK_OK;
  const size_t rows = g.a.rows, all = rows + g.b.rows, pieces = padded(in) / 8;
  hipLaunchKernelGGL(pad16_kernel, dim3((all * pieces + 255) / 256), dim3(256), 0, rt->stream,
                     g.a.base,
                     g.b.base, rows, all, static_cast<int>(in), static_cast<int>(pieces), room);
  g.a.pitch = g.b.pitch = static_cast<uint32_t>(2 * padded(in));
  g.a.base = room;
  g.b.base = room + rows * g.a.pitch;
  return vk::check_launch("pad16_kernel");
}

}  // namespace

extern "C" {

int vk_gated_forward(vk_runtime* rt, const vk_tensor* x, const vk_tensor* w, const vk_tensor* bias,
                     size_t rows, size_t in_features, size_t hidden, int activation,
                     vk_tensor* out) {
  VK_TRY(vk::bind(rt));
  VK_TRY(check_inputs(rt, x, w, bias, rows, in_features, hidden, activation));
  VK_TRY(check16(rt, out, x->dtype, rows * hidden, "out"));
  for (const vk_tensor* t : {x, w, bias})
    VK_REQUIRE(!vk::overlap(out, t), "gated: out overlaps an input");
  if (rows == 0) return VK_OK;
  Args g = forward_args(rt, x, w, bias, rows, in_features, hidden, activation);
  g.out = out->ptr;
  const vkp::Shape shape = forward_shape(g);
  // (rows that are no multiple of 16 bytes take a launch and its time to copy)
  const vkp::Plan p = vkp::plan(rt->cu_count, shape, in_features % 8 == 0 ? 0 : 4);
  if (!p.few) {
    const size_t room = operands_room(rows, in_features, hidden);
    const size_t sums = vkp::split_bytes(p.tile, vkp::Job{shape, p.splits});
    if (room + sums > 0) VK_TRY(vk::ensure_work(rt, (room + sums) / 4, "gated_forward"));
    char* work = reinterpret_cast<char*>(rt->work);
    VK_TRY(align_operands(rt, g, in_features, work));
    g.split.partial = work + room;
  }
  return x->dtype == VK_F16 ? launch_forward<kF16>(rt, g, p) : launch_forward<kBF16>(rt, g, p);
}

int vk_gated_backward(vk_runtime* rt, const vk_tensor* x, const vk_tensor* w, const vk_tensor* bias,
                      const vk_tensor* grad, size_t rows, size_t in_features, size_t hidden,
                      int activation, vk_tensor* dx, vk_tensor* dw, vk_tensor* dbias) {
  VK_TRY(vk::bind(rt));
  VK_TRY(check_inputs(rt, x, w, bias, rows, in_features, hidden, activation));
  VK_TRY(check16(rt, grad, x->dtype, rows * hidden, "grad"));
  VK_REQUIRE(dx || dw || dbias, "gated: no gradient to compute");
  if (dx) VK_TRY(check16(rt, dx, x->dtype, rows * in_features, "dx"));
  if (dw) VK_TRY(check16(rt, dw, x->dtype, 2 * hidden * in_features, "dw"));
  if (dbias) VK_TRY(check16(rt, dbias, x->dtype, 2 * hidden, "dbias"));
  const vk_tensor* outs[] = {dx, dw, dbias};
  for (int i = 0; i < 3; ++i) {
    for (const vk_tensor* t : {x, w, bias, grad})
      VK_REQUIRE(!vk::overlap(outs[i], t), "gated: a gradient overlaps an input");
    for (int j = 0; j < i; ++j)
      VK_REQUIRE(!vk::overlap(outs[i], outs[j]), "gated: gradients overlap");
  }
  if (rows == 0) {  // sums of nothing
    if (dw) zero16(rt, dw->ptr, dw->len);
    if (dbias) zero16(rt, dbias->ptr, dbias->len);
    return vk::check_launch("zero16_kernel");
  }
  const size_t room = operands_room(rows, in_features, hidden);
  Args g = forward_args(rt, x, w, bias, rows, in_features, hidden, activation);
  const BackwardPlan plan =
      plan_backward(rt->cu_count, g, in_features, x->dtype == VK_F16, dx, dw, dbias);
  VK_TRY(vk::ensure_work(rt, (room + plan.bytes + 3) / 4, "gated_backward"));
  char* work = reinterpret_cast<char*>(rt->work);
  VK_TRY(align_operands(rt, g, in_features, work));
  work += room;
  g.grad = grad->ptr;
  return x->dtype == VK_F16
             ? backward<kF16>(rt, g, plan, rows, in_features, hidden, work, dx, dw, dbias)
             : backward<kBF16>(rt, g, plan, rows, in_features, hidden, work, dx, dw, dbias);
}

}  // extern "C"
