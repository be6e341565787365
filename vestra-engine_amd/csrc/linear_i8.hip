// The linear in 8-bit integers for gfx950: weights as int8 codes with an f32 scale for
// each output channel, rows of x quantised as they come, with a scale for each token.
//
//   y[m, n] = (sum_k c[m, k] q[n, k]) * t[n] * s[m] + b[n]
//
// s[m] is the row's largest |x| / 127 rounded to f32 and c = x / s rounded to f32 and
// then to the nearest whole number (ties to even).  The sum is exact in int32.  Then
// the epilogues of the F32 linear (LayerScale, GELU, residual), or the gate: of out =
// 2 H columns, column h of the result is act(y[m, h]) * y[m, H + h].
#include <cmath>
#include <cstring>
#include <new>
#include <vector>

#include "product_nt.h"

struct vk_linear_i8 {
  vk_runtime* rt = nullptr;
  size_t in_features = 0, out_features = 0;
  size_t pitch = 0;          // bytes of a row of codes: in_features rounded up to 128
  int8_t* codes = nullptr;   // [out, pitch], zeros past in_features
  float* scale = nullptr;    // [out]
  float* bias = nullptr;     // [out] or null
  float* ls_gamma = nullptr; // [out] or null
  bool far = false;          // a scale of kFar or more
};

namespace {

using vkp::Kind;
using vkp::kBF16;
using vkp::kF16;
using vkp::kI8;
using vkp::Operand;

constexpr float kTop = 127.0f;
constexpr float kLeastScale = 0x1p-100f;  // below, a row is held as zeros (as the cache does)
constexpr float kFar = 0x1p96f;           // a channel's scale from which sums below 2^31 leave f32
constexpr size_t kMostK = 1 << 17;        // 127 * 128 * 2^17 < 2^31: the sum fits
constexpr size_t kMostRows = (1 << 24) - 1;  // a launch has less than 2^32 threads, 256 a row

enum End { kStore = 0, kGelu = 1, kResidual = 2, kGated = 3 };

struct Args {
  Operand a, b;  // codes of x and of the weights
  const float* sx;
  const float* sw;
  const float* bias;
  const float* ls;
  void* out;
  int M, N;  // N: columns of out
  int k_bytes;
  int act;  // VK_GATE_*
  bool far;  // a channel's scale is kFar or more
  const void* x;  // for workgroups that quantise for themselves: [M, K] of vk_dtype x_type
  int K, x_type;
  int gm, gn, group;
  vkp::Split split;
};

// ---------------------------------------------------------------- rows to codes
__device__ __forceinline__ uint32_t bits_abs(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const uint32_t o = static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), d, 64));
    v = o > v ? o : v;
  }
  return v;
}

// A row's scale from the bits of its largest |x| (a NaN is above an infinity is above
// every number), what to divide by and its reciprocal (0 where all codes are 0).
struct RowScale {
  float scale, by, inverse;
};
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
  const float d = __uint_as_float(top) / kTop;
  const bool odd = top >= 0x7f800000u;
  const bool none = odd || d < kLeastScale;
  return RowScale{odd ? __uint_as_float(0x7fc00000u) : (none ? 0.0f : d), none ? 1.0f : d,
                  none ? 0.0f : 1.0f / d};
}

// Four codes.  x / by rounded to f32 without a division each: with the correctly rounded
// reciprocal r and q = x r, q + (x - q by) r in two fused steps is the correctly rounded quotient
// (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000
// processor", 1990; by is 2^-100 to 2^122 here, and a quotient that could leave the normal
// numbers rounds to 0 either way).  Adding 1.5 x 2^23 then rounds it to a whole number, ties to
// even, whose lowest byte is the code.
__device__ __forceinline__ uint32_t codes_of(const float* x, const RowScale& s) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float v = s.inverse == 0.0f ? 0.0f : x[i];  // (an infinity times 0 is none)
    const float q = v * s.inverse;
    const float y = __builtin_fmaf(__builtin_fmaf(-q, s.by, v), s.inverse, q);
    c[i] = __float_as_uint(y + 12582912.0f);
  }
  const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0cu);
  return lo | hi;
}

// Eight values from x[i], zeros from the left-th on; x + i may lie anywhere.
template <typename XT>
__device__ __forceinline__ void load8(const XT* x, size_t i, int left, float (&v)[8]) {
  XT e[8];
  if (left >= 8) {
    __builtin_memcpy(e, x + i, sizeof(e));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = j < left ? x[i + j] : static_cast<XT>(0.0f);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = vkp::widen(e[j]);
}

__device__ __forceinline__ uint32_t top_of(const float (&v)[8], uint32_t top) {
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, bits_abs(v[j]));
  return top;
}

// WPR waves a row (4 of them are a workgroup's, otherwise it has 4 rows).  NV steps of 8
// values a lane stay in registers between the maximum and the codes; NV 0: any length, read
// twice.  Bound by memory for many rows (10,392 x 1536 f32: 16.6 us, 4.8 TB/s of what is read and
// written), by the chain row -> maximum -> codes for few.
template <typename XT, int NV, int WPR>
__global__ __launch_bounds__(256) void quantise_rows_kernel(const XT* __restrict__ x, int M, int K,
                                                            uint32_t pitch, char* codes,
                                                            float* scales) {
  constexpr int kStep = 512 * WPR;
  const int lane = threadIdx.x & (64 * WPR - 1);
  const int m = WPR == 4 ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= M) return;
  const XT* row = x + static_cast<size_t>(m) * K;
  char* to = codes + static_cast<size_t>(m) * pitch;
  const auto scale_of = [&](uint32_t top) {
    top = wave_umax(top);
    if constexpr (WPR == 4) {
      __shared__ uint32_t tops[4];
      if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
      __syncthreads();
      top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    }
    const RowScale s = row_scale(top);
    if (lane == 0) scales[m] = s.scale;
    return s;
  };
  const auto store = [&](int at, const float (&v)[8], const RowScale& s) {
    if (at < static_cast<int>(pitch))
      *reinterpret_cast<uint2*>(to + at) = make_uint2(codes_of(v, s), codes_of(v + 4, s));
  };
  if constexpr (NV > 0) {
    float v[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = i * kStep + lane * 8;
      load8(row, at, K - at, v[i]);
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) top = top_of(v[i], top);
    const RowScale s = scale_of(top);
#pragma unroll
    for (int i = 0; i < NV; ++i) store(i * kStep + lane * 8, v[i], s);
  } else {
    float v[8];
    uint32_t top = 0;
    for (int at = lane * 8; at < K; at += kStep) {
      load8(row, at, K - at, v);
      top = top_of(v, top);
    }
    const RowScale s = scale_of(top);
    for (int at = lane * 8; at < static_cast<int>(pitch); at += kStep) {
      load8(row, at, K - at, v);
      store(at, v, s);
    }
  }
}

// ---------------------------------------------------------------- what leaves
// (sum t) s + b.  FAR: a channel's scale of the linear may take the sum past f32 (kFar) where the
// row's brings it back: the sum is first multiplied by the largest power of two in a row's scale
// below 1, and stays a normal number whose product with t leaves f32 only where the result does.
// The bits are those of the other form wherever that does not leave f32; one more product a value,
// which costs 10,392 x 1536 -> 2 x 4096 gated 2.7 us of 164 (a linear without such a scale:
// nothing).
template <bool FAR>
struct RowScaleOf {
  float power = 1.0f, rest;
  __device__ __forceinline__ explicit RowScaleOf(float s) : rest(s) {
    if (FAR && s >= kLeastScale && s < 1.0f) {
      power = __uint_as_float(__float_as_uint(s) & 0x7f800000u);
      rest = __uint_as_float((__float_as_uint(s) & 0x007fffffu) | 0x3f800000u);
    }
  }
};
template <bool FAR>
__device__ __forceinline__ float linear_of(int acc, float channel, const RowScaleOf<FAR>& row,
                                           float bias) {
  const float sum = static_cast<float>(acc);
  return __builtin_fmaf((FAR ? sum * row.power : sum) * channel, row.rest, bias);
}

template <int END>
__device__ __forceinline__ float finish(float v, float ls) {
  if constexpr (END == kStore || END == kResidual) v = v * ls;  // 1 where there is none
  if constexpr (END == kGelu) v = vkd::gelu1<0>(v);
  return v;
}

// The tiles.  10,392 x 1536 -> 2 x 4096 gated: 142-150 us (1.8 POP/s); 10,392 x 768 -> 2304 in
// bf16: 29, six stages a tile whose beginning and end nothing covers; 866 x 4096 -> 1024 into the
// residual: 14, 224 tiles of 64 x 64 by two groups of waves (128 x 128: 30, by one group: 22).
template <int END, typename V, typename T>
__global__ __launch_bounds__(T::kThreads, T::kWavesASimd) void linear_i8_kernel(Args g) {
  VK_STAGES(T);
  __shared__ __align__(16) float cols[3][T::TN];  // scale, bias, LayerScale of the tile's columns
  int mt, nt;
  const int tiles = g.gm * g.gn, tile = blockIdx.x % tiles, part = blockIdx.x / tiles;
  vkp::tile_at(tile, g.gm, g.gn, g.group, &mt, &nt);
  const int m0 = mt * T::TM, n0 = nt * T::kHeld;
  for (int c = threadIdx.x; c < T::TN; c += T::kThreads) {
    const int n = n0 + c % T::kHeld;
    const int at = (n < g.N ? n : g.N - 1) + (c < T::kHeld ? 0 : g.N);
    cols[0][c] = g.sw[at];
    cols[1][c] = g.bias ? g.bias[at] : 0.0f;
    cols[2][c] = g.ls ? g.ls[at] : 1.0f;
  }
  const vkp::Place<T> place;
  vkp::i32x16 acc[T::MT][T::NT];
  if (!vkp::product_tile<kI8, T>(g.a, g.b, g.k_bytes, m0, n0, g.split, part, tile, tiles, place,
                                 stages_, acc))
    return;
  const int lane = place.lane, wave = place.wave, wm = place.wm, wn = place.wn;
  constexpr int kCols = T::PAIRED ? T::NT / 2 : T::NT;
  constexpr int J = sizeof(V) == 4 || kCols % 2 ? 1 : 2;
  typedef vkp::Chunk<V, J> C;
  static_assert(T::kWaves * C::kBytes <= T::kBytes, "the chunks fit a stage buffer");
  char* chunk = stages_[0] + wave * C::kBytes;
  V* out = static_cast<V*>(g.out);
  const auto leave = [&](auto act, auto far) {
#pragma unroll
    for (int i = 0; i < T::MT; ++i) {
      const int mb = m0 + (wm * T::MT + i) * 32, m = mb + (lane & 31);
      const RowScaleOf<far.value> row(g.sx[m < g.M ? m : g.M - 1]);
#pragma unroll
      for (int jg = 0; jg < kCols; jg += J) {
#pragma unroll
        for (int jj = 0; jj < J; ++jj)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int j = jg + jj, c = T::b_row(wn, j) + 8 * q + 4 * (lane >> 5);
            const auto at = [&](int p, int c_) {
              return *reinterpret_cast<const vkp::f32x4*>(&cols[p][c_]);
            };
            const vkp::f32x4 s = at(0, c), b = at(1, c);
            vkp::f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = linear_of(acc[i][j][4 * q + e], s[e], row, b[e]);
            if constexpr (T::PAIRED) {
              const vkp::f32x4 us = at(0, c + T::kHeld), ub = at(1, c + T::kHeld);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                v[e] = vkp::gate<act.value>(v[e]) *
                       linear_of(acc[i][j + kCols][4 * q + e], us[e], row, ub[e]);
            } else {
              const vkp::f32x4 l = at(2, c);
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = finish<END>(v[e], l[e]);
            }
            typename C::V4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = static_cast<V>(v[e]);
            *C::at(chunk, lane, jj, q) = w;
          }
        vkd::wave_lds_fence();
        C::template store<END == kResidual>(chunk, lane, out, g.N, mb, g.M, n0 + T::b_row(wn, jg),
                                            g.N);
        vkd::wave_lds_fence();
      }
    }
  };
  const auto leave_as = [&](auto far) {
    if constexpr (END == kGated)
      vkp::with_act(g.act, [&](auto act) { leave(act, far); });
    else
      leave(std::integral_constant<int, 0>{}, far);
  };
  if (g.far)
    leave_as(std::true_type{});
  else
    leave_as(std::false_type{});
}

// What leaves after the waves' sums are joined: thread by thread.
template <int END, typename V, int RT>
__device__ __forceinline__ void few_finish(const Args& g, const char* smem, int n0,
                                           const float* scales) {
  constexpr bool kPaired = END == kGated;
  for (int e = threadIdx.x; e < 256 * RT; e += vkp::kFewThreads) {
    const int m = e >> 4, n = n0 + (e & 15);
    if (m >= g.M || n >= g.N) continue;
    const RowScaleOf<true> row(scales[m]);
    V* to = static_cast<V*>(g.out) + static_cast<size_t>(m) * g.N + n;
    float v = linear_of(vkp::few_sum<kI8, RT, kPaired>(smem, 0, m, e & 15), g.sw[n], row,
                        g.bias ? g.bias[n] : 0.0f);
    if constexpr (kPaired) {
      const int p = g.N + n;
      const float u = linear_of(vkp::few_sum<kI8, RT, true>(smem, 1, m, e & 15), g.sw[p], row,
                                g.bias ? g.bias[p] : 0.0f);
      vkp::with_act(g.act, [&](auto act) { v = vkp::gate<act.value>(v) * u; });
    }
    if constexpr (!kPaired) v = finish<END>(v, g.ls ? g.ls[n] : 1.0f);
    if constexpr (END == kResidual) v = *to + v;
    *to = static_cast<V>(v);
  }
}

// At most 16 RT rows, their codes in memory.
template <int END, typename V, int RT>
__global__ __launch_bounds__(vkp::kFewThreads) void linear_i8_few_kernel(Args g) {
  constexpr bool kPaired = END == kGated;
  __shared__ __align__(16) char smem[vkp::few_bytes<kI8, RT, kPaired>()];
  const int n0 = blockIdx.x * 16;
  vkp::few_product<kI8, RT, kPaired>(g.a, g.b, g.k_bytes, n0, smem);
  few_finish<END, V, RT>(g, smem, n0, g.sx);
}

// Rows of at most kOwnBytes of codes in all: every workgroup quantises them for itself, in one
// launch, while its weights are on their way.  Thread by thread eight values; sixteen lanes are of
// one row, whose maximum meets in LDS.  1 x 1024 -> 4096 4.0 us, 1 x 1536 -> 2 x 4096 gated 5.7:
// the launch and the chain row -> maximum -> codes -> products -> sums.
template <typename XT>
__device__ __forceinline__ void load8_of(const Args& g, int m, int at, float (&v)[8]) {
  load8(static_cast<const XT*>(g.x) + static_cast<size_t>(m) * g.K, at, g.K - at, v);
}

template <int END, typename V>
__global__ __launch_bounds__(vkp::kFewThreads) void linear_i8_rows_kernel(Args g) {
  constexpr bool kPaired = END == kGated;
  constexpr int kEights = vkp::kOwnBytes / 8 / vkp::kFewThreads;  // of a thread
  __shared__ __align__(16) char smem[vkp::few_bytes<kI8, 1, kPaired>()];
  __shared__ __align__(16) char codes[vkp::kOwnBytes + 16 * vkp::kOwnRows];
  __shared__ uint32_t tops[vkp::kOwnRows];
  __shared__ float scales[vkp::kOwnRows];
  const int n0 = blockIdx.x * 16, tid = threadIdx.x, c = tid & 15;
  const int pitch = g.k_bytes + 16;  // rows start in different banks
  if (tid < vkp::kOwnRows) tops[tid] = 0;
  vkp::few_product<kI8, 1, kPaired>(
      g.b, g.k_bytes, n0, smem,
      [&] {
        float v[kEights][8];
        int m[kEights], at[kEights];
        const int eights = g.k_bytes / 8;
#pragma unroll
        for (int i = 0; i < kEights; ++i) {
          const int e = tid + i * vkp::kFewThreads;
          m[i] = e / eights;
          at[i] = (e - m[i] * eights) * 8;
          if (m[i] >= g.M) continue;
          if (g.x_type == VK_F32) load8_of<float>(g, m[i], at[i], v[i]);
          else if (g.x_type == VK_F16) load8_of<_Float16>(g, m[i], at[i], v[i]);
          else load8_of<__bf16>(g, m[i], at[i], v[i]);
        }
        __syncthreads();  // the maxima are cleared
#pragma unroll
        for (int i = 0; i < kEights; ++i) {
          if (m[i] >= g.M) continue;
          uint32_t top = top_of(v[i], 0);
#pragma unroll
          for (int d = 8; d > 0; d >>= 1) {
            const uint32_t o = static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d, 16));
            top = o > top ? o : top;
          }
          if (c == 0) atomicMax(&tops[m[i]], top);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEights; ++i) {
          if (m[i] >= g.M) continue;
          const RowScale s = row_scale(tops[m[i]]);
          *reinterpret_cast<uint2*>(codes + m[i] * pitch + at[i]) =
              make_uint2(codes_of(v[i], s), codes_of(v[i] + 4, s));
          if (at[i] == 0) scales[m[i]] = s.scale;
        }
        __syncthreads();
      },
      [&](int, int k) {
        vkp::i32x4 a = {0, 0, 0, 0};
        if (c < g.M && k < g.k_bytes)
          a = *reinterpret_cast<const vkp::i32x4*>(codes + c * pitch + k);
        return a;
      },
      [](int) { return vkp::i32x4{0, 0, 0, 0}; });
  few_finish<END, V, 1>(g, smem, n0, scales);
}

// ---------------------------------------------------------------- launches
// Four waves a row of more than 1024 codes: shorter chains, and up to 8192 stay in registers (f32,
// with a product of 64 columns behind it, us, one wave a row against four: 866 x 768 9.3 and 9.4,
// 10,392 x 768 14.8 and 17.5; 866 x 1536 10.9 and 10.7, 10,392 x 1536 21.5 and 21.2; 866 x 4096
// 15.0 and 14.5, 10,392 x 4096 44.0 and 42.1; 10,392 x 8192 146 and 102).
template <typename XT>
void quantise(const vk_runtime* rt, const XT* x, int M, int K, size_t pitch, char* codes,
              float* scales) {
  const bool wide = pitch > 1024;
  const dim3 grid(wide ? M : (M + 3) / 4), block(256);
  const auto p = static_cast<uint32_t>(pitch);
#define VK_LAUNCH(NV, WPR)                                                                     \
  hipLaunchKernelGGL((quantise_rows_kernel<XT, NV, WPR>), grid, block, 0, rt->stream, x, M, K, \
                     p, codes, scales)
  if (pitch <= 512) VK_LAUNCH(1, 1);
  else if (pitch <= 1024) VK_LAUNCH(2, 1);
  else if (pitch <= 2048) VK_LAUNCH(1, 4);
  else if (pitch <= 4096) VK_LAUNCH(2, 4);
  else if (pitch <= 8192) VK_LAUNCH(4, 4);
  else VK_LAUNCH(0, 4);
#undef VK_LAUNCH
}

template <int END, typename V>
int launch(vk_runtime* rt, Args& g, const vkp::Plan& p) {
  constexpr bool kPaired = END == kGated;
  if (g.x) {
    hipLaunchKernelGGL((linear_i8_rows_kernel<END, V>), dim3((g.N + 15) / 16),
                       dim3(vkp::kFewThreads), 0, rt->stream, g);
    return vk::check_launch("linear_i8_rows_kernel");
  }
  if (p.few) {
    const dim3 grid((g.N + 15) / 16), block(vkp::kFewThreads);
    if (g.M <= 16)
      hipLaunchKernelGGL((linear_i8_few_kernel<END, V, 1>), grid, block, 0, rt->stream, g);
    else
      hipLaunchKernelGGL((linear_i8_few_kernel<END, V, 2>), grid, block, 0, rt->stream, g);
    return vk::check_launch("linear_i8_few_kernel");
  }
  vkp::with_tile<kPaired>(p.tile, [&](auto tile) {
    typedef decltype(tile) T;
    g.gm = (g.M + T::TM - 1) / T::TM;
    g.gn = (g.N + T::kHeld - 1) / T::kHeld;
    g.group = vkp::kGroupRows / T::TM;
    g.split.count = p.splits;
    g.split.arrivals = rt->arrivals;
    hipLaunchKernelGGL((linear_i8_kernel<END, V, T>), dim3(g.gm * g.gn * p.splits),
                       dim3(T::kThreads), 0, rt->stream, g);
  });
  return vk::check_launch("linear_i8_kernel");
}

template <int END>
int launch_type(vk_runtime* rt, Args& g, const vkp::Plan& p, vk_dtype type) {
  if (type == VK_F32) return launch<END, float>(rt, g, p);
  return type == VK_F16 ? launch<END, _Float16>(rt, g, p) : launch<END, __bf16>(rt, g, p);
}

bool is_float(const vk_tensor* t) {
  return t->dtype == VK_F32 || t->dtype == VK_F16 || t->dtype == VK_BF16;
}

int check_tensor(const vk_runtime* rt, const vk_tensor* t, size_t rows, size_t cols,
                 const char* what) {
  VK_REQUIRE(t, "linear_i8: null %s", what);
  VK_REQUIRE(is_float(t) && t->len == rows * cols,
             "linear_i8: %s must be f32, f16 or bf16 [%zu x %zu] (holds %zu)", what, rows, cols,
             t->len);
  VK_REQUIRE(reinterpret_cast<uintptr_t>(t->ptr) % 16 == 0, "linear_i8: %s must be 16-byte aligned",
             what);
  return vk::check_device(rt, t, what);
}

int run(vk_runtime* rt, const vk_linear_i8* lin, const vk_tensor* x, size_t rows, vk_tensor* out,
        End end, int act) {
  VK_TRY(vk::bind(rt));
  VK_REQUIRE(lin, "linear_i8: null linear");
  VK_REQUIRE(lin->rt->device == rt->device, "linear_i8: a linear of another device");
  VK_UNSUPPORTED_IF(rows > kMostRows, "linear_i8: %zu rows (at most %zu)", rows, kMostRows);
  const size_t K = lin->in_features;
  if (end == kGated) {
    VK_REQUIRE(lin->out_features % 2 == 0, "linear_i8: gated over %zu columns", lin->out_features);
    VK_REQUIRE(act == VK_GATE_SILU || act == VK_GATE_GELU, "linear_i8: unknown activation %d", act);
  }
  VK_REQUIRE(!lin->ls_gamma || end == kStore || end == kResidual,
             "linear_i8: this call's linear carries no LayerScale");
  const size_t N = end == kGated ? lin->out_features / 2 : lin->out_features;
  VK_TRY(check_tensor(rt, x, rows, K, "x"));
  VK_TRY(check_tensor(rt, out, rows, N, end == kResidual ? "residual" : "out"));
  VK_REQUIRE(end != kResidual || out->dtype == VK_F32, "linear_i8: residual must be f32");
  VK_REQUIRE(!vk::overlap(x, out), "linear_i8: the output overlaps x");
  if (rows == 0) return VK_OK;
  VK_UNSUPPORTED_IF(((rows + 63) / 64) * ((N + 31) / 32) > 0x7fffffULL,
                    "linear_i8: %zu x %zu outputs", rows, N);

  const int M = static_cast<int>(rows);
  const vkp::Shape shape{M, static_cast<long long>(lin->out_features),
                         static_cast<long long>(lin->pitch), end == kGated};
  const vkp::Plan p = vkp::plan(rt->cu_count, shape);
  Args g{};
  if (vkp::own_rows(rows, lin->pitch)) {
    g.x = x->ptr;
    g.K = static_cast<int>(K);
    g.x_type = x->dtype;
  } else {
    const size_t code_bytes = rows * lin->pitch, scale_bytes = (rows * 4 + 255) / 256 * 256;
    const size_t sums = p.few ? 0 : vkp::split_bytes(p.tile, vkp::Job{shape, p.splits});
    VK_TRY(vk::ensure_work(rt, (code_bytes + scale_bytes + sums) / 4, "linear_i8"));
    char* codes = reinterpret_cast<char*>(rt->work);  // (code_bytes: a multiple of 128)
    float* scales = reinterpret_cast<float*>(codes + code_bytes);
    g.split.partial = codes + code_bytes + scale_bytes;
    if (x->dtype == VK_F32)
      quantise(rt, static_cast<const float*>(x->ptr), M, static_cast<int>(K), lin->pitch, codes,
               scales);
    else if (x->dtype == VK_F16)
      quantise(rt, static_cast<const _Float16*>(x->ptr), M, static_cast<int>(K), lin->pitch, codes,
               scales);
    else
      quantise(rt, static_cast<const __bf16*>(x->ptr), M, static_cast<int>(K), lin->pitch, codes,
               scales);
    VK_TRY(vk::check_launch("quantise_rows_kernel"));
    g.a = Operand{codes, M, static_cast<uint32_t>(lin->pitch)};
    g.sx = scales;
  }
  g.b = Operand{reinterpret_cast<const char*>(lin->codes), static_cast<int>(lin->out_features),
                static_cast<uint32_t>(lin->pitch)};
  g.sw = lin->scale;
  g.bias = lin->bias;
  g.ls = lin->ls_gamma;
  g.far = lin->far;
  g.out = out->ptr;
  g.M = M;
  g.N = static_cast<int>(N);
  g.k_bytes = static_cast<int>(lin->pitch);
  g.act = act;
  switch (end) {
    case kStore: return launch_type<kStore>(rt, g, p, out->dtype);
    case kGelu: return launch_type<kGelu>(rt, g, p, out->dtype);
    case kResidual: return launch<kResidual, float>(rt, g, p);
    default: return launch_type<kGated>(rt, g, p, out->dtype);
  }
}

// ---------------------------------------------------------------- weights
int check_prepare(size_t in, size_t out) {
  VK_REQUIRE(in > 0 && out > 0, "linear_i8: empty");
  VK_UNSUPPORTED_IF(in > kMostK, "linear_i8: in_features=%zu (at most %zu: the int32 sum)", in,
                    kMostK);
  VK_UNSUPPORTED_IF(out > 0x7fffff00ULL / ((in + 127) / 128 * 128), "linear_i8: %zu x %zu weights",
                    in, out);
  return VK_OK;
}

int upload(void** dev, const void* host, size_t bytes) {
  VK_HIP(hipMalloc(dev, bytes));
  VK_HIP(hipMemcpy(*dev, host, bytes, hipMemcpyHostToDevice));
  return VK_OK;
}

// codes [out, pitch]
int make(vk_runtime* rt, size_t in, size_t out, size_t pitch, const int8_t* codes,
         const float* scale, const float* bias, const float* ls, vk_linear_i8** res) {
  auto* lin = new (std::nothrow) vk_linear_i8;
  if (!lin) return vk::set_error(VK_ERR_OOM, "linear_i8: out of host memory");
  lin->rt = rt;
  vk::retain(rt);
  lin->in_features = in;
  lin->out_features = out;
  lin->pitch = pitch;
  for (size_t o = 0; o < out; ++o)
    if (std::isfinite(scale[o]) && std::fabs(scale[o]) >= kFar) lin->far = true;
  int s = upload(reinterpret_cast<void**>(&lin->codes), codes, out * pitch);
  if (s == VK_OK) s = upload(reinterpret_cast<void**>(&lin->scale), scale, out * 4);
  if (s == VK_OK && bias) s = upload(reinterpret_cast<void**>(&lin->bias), bias, out * 4);
  if (s == VK_OK && ls) s = upload(reinterpret_cast<void**>(&lin->ls_gamma), ls, out * 4);
  if (s != VK_OK) {
    vk_linear_i8_destroy(lin);
    return s;
  }
  *res = lin;
  return VK_OK;
}

}  // namespace

extern "C" {

int vk_linear_i8_prepare(vk_runtime* rt, size_t in_features, size_t out_features,
                         const int8_t* codes_out_in, const float* scale, const float* bias,
                         const float* ls_gamma, vk_linear_i8** out) try {
  VK_TRY(vk::bind(rt));
  VK_REQUIRE(out && codes_out_in && scale, "null argument");
  VK_TRY(check_prepare(in_features, out_features));
  const size_t pitch = (in_features + 127) / 128 * 128;
  if (pitch == in_features)
    return make(rt, in_features, out_features, pitch, codes_out_in, scale, bias, ls_gamma, out);
  std::vector<int8_t> w(pitch * out_features, 0);
  for (size_t o = 0; o < out_features; ++o)
    std::memcpy(&w[o * pitch], codes_out_in + o * in_features, in_features);
  return make(rt, in_features, out_features, pitch, w.data(), scale, bias, ls_gamma, out);
} catch (const std::bad_alloc&) {
  return vk::set_error(VK_ERR_OOM, "linear_i8: out of host memory");
}

int vk_linear_i8_prepare_f32(vk_runtime* rt, size_t in_features, size_t out_features,
                             const float* weight_in_out, const float* bias, const float* ls_gamma,
                             vk_linear_i8** out) try {
  // (on the host, once: 1536 -> 8192 in 21 ms, 4096 -> 1536 in 40; from codes 0.5 and 0.2)
  VK_TRY(vk::bind(rt));
  VK_REQUIRE(out && weight_in_out, "null argument");
  VK_TRY(check_prepare(in_features, out_features));
  const size_t pitch = (in_features + 127) / 128 * 128;
  std::vector<int8_t> w(pitch * out_features, 0);
  std::vector<float> scale(out_features, 0.0f);  // first each channel's largest |w|
  std::vector<char> odd(out_features, 0);
  for (size_t i = 0; i < in_features; ++i)
    for (size_t o = 0; o < out_features; ++o) {
      const float a = std::fabs(weight_in_out[i * out_features + o]);
      if (!std::isfinite(a)) odd[o] = 1;
      if (a > scale[o]) scale[o] = a;
    }
  for (size_t o = 0; o < out_features; ++o) {
    const float d = scale[o] / kTop;
    scale[o] = odd[o] ? std::nanf("") : (d < kLeastScale ? 0.0f : d);
  }
  for (size_t i = 0; i < in_features; ++i)
    for (size_t o = 0; o < out_features; ++o)
      if (scale[o] > 0.0f)
        w[o * pitch + i] =
            static_cast<int8_t>(std::nearbyint(weight_in_out[i * out_features + o] / scale[o]));
  return make(rt, in_features, out_features, pitch, w.data(), scale.data(), bias, ls_gamma, out);
} catch (const std::bad_alloc&) {
  return vk::set_error(VK_ERR_OOM, "linear_i8: out of host memory");
}

int vk_linear_i8_destroy(vk_linear_i8* lin) {
  if (!lin) return VK_OK;
  vk_runtime* rt = lin->rt;
  (void)vk::bind_device(rt);
  (void)hipStreamSynchronize(rt->stream);
  for (void* p : {static_cast<void*>(lin->codes), static_cast<void*>(lin->scale),
                  static_cast<void*>(lin->bias), static_cast<void*>(lin->ls_gamma)})
    if (p) (void)hipFree(p);
  delete lin;
  vk::release(rt);
  return VK_OK;
}

size_t vk_linear_i8_input_features(const vk_linear_i8* lin) { return lin ? lin->in_features : 0; }

int vk_linear_i8_run_into(vk_runtime* rt, const vk_linear_i8* lin, const vk_tensor* x, size_t rows,
                          vk_tensor* out) {
  return run(rt, lin, x, rows, out, kStore, 0);
}

int vk_linear_i8_run_gelu(vk_runtime* rt, const vk_linear_i8* lin, const vk_tensor* x, size_t rows,
                          vk_tensor* out) {
  return run(rt, lin, x, rows, out, kGelu, 0);
}

int vk_linear_i8_run_residual(vk_runtime* rt, const vk_linear_i8* lin, const vk_tensor* x,
                              size_t rows, vk_tensor* residual) {
  return run(rt, lin, x, rows, residual, kResidual, 0);
}

int vk_linear_i8_run_gated(vk_runtime* rt, const vk_linear_i8* lin, const vk_tensor* x, size_t rows,
                           int activation, vk_tensor* out) {
  return run(rt, lin, x, rows, out, kGated, activation);
}

}  // extern "C"
