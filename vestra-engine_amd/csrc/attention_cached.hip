// Attention over the 8-bit cache of K and V rows (kv_cache.h), with capped
// scores, a bias by distance, and causal, prefix and document masks.
//
// The mathematics.  A held value is code * scale, one scale a row, and both kinds of
// code (int8, e4m3) are exact in f16.  So the products run over codes: score_j = K's
// scale_j * (q . code_j), and out = sum_j (p_j * V's scale_j) code_j / sum_j p_j with
// p_j = 2^(score_j - m) in base 2, m a reference that follows the row's largest score.  An
// f32 factor (q; p times V's scale) is taken as two f16 parts of 11 bits each, so each of the
// two products is two on the f16 matrix cores, summed in f32: twice the time of
// one f16 product, where the f32 matrix cores take seven times that of one.
//
// Three kernels (plans.h says which, and over how many workgroups the keys are split), and one
// that joins the splits:
//   attention_row_kernel   one query: a lane a key, f32 on the vector units.  Bound by memory (16 x
//                          124,704 keys: 53.3 us called back to back, 47 in a graph, 5.1 and
//                          5.8 TB/s); a short cache by its CUs' vector units (12 x 866 keys:
//                          5.9 us).  It reads every key whatever the masks leave: 12 x 124,704
//                          keys 38 us, of which one document of 866 is seen 39.
//   attention_few_kernel   up to 32 queries of a cache head: a wave a block of 64 keys.  Bound
//                          by the latency of a block's chain (12 x 10,392 keys, 32 queries:
//                          14.2 us, 13.4 in a graph).
//   attention_tile_kernel  128 queries a workgroup, the blocks through LDS.  Bound by the vector
//                          units beside the matrix cores (softmax and the splitting of weights: 63% and
//                          41% of the time; 12 x 10,392 rows over the frames before theirs: 405 us,
//                          887 TFLOP/s of f16 products where a large library product reaches
//                          1,080).
// No atomics and no order that depends on timing: the same call gives the same bits, and a
// row's do not depend on the values of other queries.
#include <cmath>
#include <type_traits>
#include <utility>

#include "kv_cache.h"
#include "split_f16.h"

namespace {

constexpr int HD = 64;
constexpr float kLog2e = 1.44269504088896341f;
// V's scale in the single row's sums: room for weights up to 2^4 and 2^20 keys of the largest
// numbers.
constexpr float kRowDown = 0x1p-24f, kRowUp = 0x1p24f;

struct Rules {
  float scale, cap;
  const float* slopes;
  const int* prefix;  // with causal
  const int* q_docs;
  const int* k_docs;
  int causal, docs_ordered;
};

struct Shape {
  vkc::Cache cache;
  vkc::Rows rows;
  Rules rules;
  uint32_t heads, group;  // query heads, and how many of them share a cache head
  uint32_t limit;         // keys at or past it are not seen (capacity, max_length)
  uint32_t splits, tiles;
  uint32_t parts;         // workgroups a tile and split: 2 with documents apart (document_part)
  struct {
    uint32_t share, heads;
  } order;
};

// Keys of sequence s: those of slots 0 .. keys_of - 1.
__device__ __forceinline__ int keys_of(const Shape& a, uint32_t s) {
  const int c = vkc::count_of(a.rows, s);
  if (c <= 0) return 0;
  long long end = static_cast<long long>(vkc::start_of(a.rows, s)) + c;
  end = end < static_cast<long long>(a.limit) ? end : static_cast<long long>(a.limit);
  return end > 0 ? static_cast<int>(end) : 0;
}

// Position of row i; every key lies below the largest.
__device__ __forceinline__ int position(int start, uint32_t i) {
  const long long p = static_cast<long long>(start) + i;
  return p < 0x7ffffffe ? static_cast<int>(p) : 0x7ffffffe;
}

// Largest over the wave, without a round trip through LDS: rotations inside rows of
// 16 lanes, then swaps of rows and of halves.
__device__ __forceinline__ float wave_max(float v) {
#define VK_ROR(n)                                                                            \
  v = fmaxf(v, __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(               \
                   static_cast<int>(__float_as_uint(v)), 0x120 | n, 0xf, 0xf, true))));
  VK_ROR(8) VK_ROR(4) VK_ROR(2) VK_ROR(1)
#undef VK_ROR
  const auto a =
      __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  v = fmaxf(__uint_as_float(a0), __uint_as_float(a1));
  const auto b =
      __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return fmaxf(__uint_as_float(b0), __uint_as_float(b1));
}

template <int FORMAT, int N>
__device__ __forceinline__ void drop_nan(uint32_t (&w)[N]);

constexpr int kRowWaves = 8;
constexpr float kRoom = 4.0f;  // a lane's maximum follows scores that pass it by 2^kRoom

// One query a sequence and cache head: a workgroup a query and key split, a lane a key.  The
// lane's 64 products are F32 FMAs with the query uniform (scalar registers, and what they do not
// hold read back out of lanes of a vector register; four running sums), and it keeps a softmax
// of its own (maximum, sum and 64 sums of values) over the keys that it meets; the lanes are
// joined once, at the end, halving: lane d is left with d.  A short cache's few rows have four
// workgroups each (PARTS), which share V's columns and all take the scores: a CU has 60% of the
// vector work (12 x 866 keys 5.9 us, 7.1 in one).
template <int FORMAT, int PARTS>
__global__ __launch_bounds__(64 * kRowWaves) void attention_row_kernel(const float* __restrict__ q,
                                                                       float* __restrict__ out,
                                                                       float* __restrict__ part,
                                                                       Shape a) {
  constexpr int ND = HD / PARTS;
  __shared__ float so[kRowWaves][ND];
  __shared__ float sm[kRowWaves], sl[kRowWaves];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t all = a.rows.sequences * a.heads;
  const uint32_t split = PARTS > 1 ? 0 : blockIdx.x % a.splits;
  const uint32_t row = PARTS > 1 ? blockIdx.x % all : blockIdx.x / a.splits;
  const int d0 = PARTS > 1 ? static_cast<int>(blockIdx.x / all) * ND : 0;
  const uint32_t h = row % a.heads, s = row / a.heads;
  const Rules& ru = a.rules;
  // a scale below 1 comes before K's, one above 1 after it: neither product leaves f32's
  // range where the score is inside
  const bool less = fabsf(ru.scale) < 1.0f;
  const float before = less ? ru.scale : 1.0f, after = less ? 1.0f : ru.scale;
  // every scalar together: none waits for another
  const int count = vkc::count_of(a.rows, s), start = vkc::start_of(a.rows, s);
  const float slope = ru.slopes ? ru.slopes[h] : 0.0f;
  const int pre = ru.prefix ? ru.prefix[s] : 0;
  const int doc = ru.q_docs ? ru.q_docs[s] : 0;
  const float* qr = q + vkc::row_at(a.rows, a.heads, s, h, 0);
  if (count <= 0) return;
  const int keys = keys_of(a, s);
  const int p = position(start, 0);
  const size_t first = (static_cast<size_t>(s) * a.cache.heads + h) * a.cache.capacity;

  float m = -INFINITY, l = 0.0f, acc[ND];
  const int blocks = (keys + 63) / 64;
  const int b0 = static_cast<int>(static_cast<long long>(split) * blocks / a.splits);
  const int b1 = static_cast<int>(static_cast<long long>(split + 1) * blocks / a.splits);
  // The wave's blocks; whether q . code of a key that is seen went past f32's range, which K's
  // scale may bring it back into: `small` takes the codes times kDown.
  const auto run = [&](auto small) {
    constexpr bool kSmall = decltype(small)::value;
    constexpr float kDown = 0x1p-24f;
    uint32_t past = 0;
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = 0.0f;
    for (int b = b0 + wave; b < b1; b += kRowWaves) {
      const int j = b * 64 + lane;
      // the key's codes and scales, all at once (past the end the last key's)
      const size_t slot = first + (j < keys ? j : keys - 1);
      const uint4* kc = reinterpret_cast<const uint4*>(a.cache.k + slot * HD);
      const uint4* vc = reinterpret_cast<const uint4*>(a.cache.v + slot * HD + d0);
      uint4 kw[4], vw[ND / 16];
#pragma unroll
      for (int c = 0; c < 4; ++c) kw[c] = kc[c];
      const float ks = a.cache.ks[slot], vs = a.cache.vs[slot];
#pragma unroll
      for (int c = 0; c < ND / 16; ++c) vw[c] = vc[c];
      bool seen = j < keys;
      if (ru.causal) seen = seen && (j <= p || j < pre);
      if (ru.q_docs && seen) {
        const int kd = ru.k_docs[static_cast<size_t>(s) * a.cache.capacity + j];
        seen = ru.docs_ordered ? kd <= doc : kd == doc;
      }
      float u[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t ws[4] = {kw[c].x, kw[c].y, kw[c].z, kw[c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float4 x = vkc::decode4<FORMAT>(ws[e]);
          if constexpr (kSmall) x = make_float4(x.x * kDown, x.y * kDown, x.z * kDown, x.w * kDown);
          u[0] = __builtin_fmaf(qr[16 * c + 4 * e], x.x, u[0]);
          u[1] = __builtin_fmaf(qr[16 * c + 4 * e + 1], x.y, u[1]);
          u[2] = __builtin_fmaf(qr[16 * c + 4 * e + 2], x.z, u[2]);
          u[3] = __builtin_fmaf(qr[16 * c + 4 * e + 3], x.w, u[3]);
        }
      }
      const float dot = (u[0] + u[1]) + (u[2] + u[3]);
      float t = dot * before * ks * after;
      if constexpr (kSmall) t *= 1.0f / kDown;
      // (a hidden code may be no number)
      past = max(past, seen ? __float_as_uint(dot) & 0x7fffffffu : 0u);
      if (ru.cap > 0.0f) t = ru.cap * tanhf(t / ru.cap);
      if (ru.slopes) {
        const long long far = p > j ? static_cast<long long>(p) - j : static_cast<long long>(j) - p;
        t -= slope * static_cast<float>(far);
      }
      // (a scale that is infinite or a NaN, of K or of V, makes the score a NaN)
      t = t * kLog2e + ((ks - ks) + (vs - vs));
      seen = seen && !(t == -INFINITY);
      if (seen && t > m + kRoom) {
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - t);
        l *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] *= f;
        m = t;
      }
      const float w = seen ? __builtin_amdgcn_exp2f(t - m) : 0.0f;
      l += w;
      const float wv = seen ? w * (vs * kRowDown) : 0.0f;
#pragma unroll
      for (int c = 0; c < ND / 16; ++c) {
        uint32_t ws[4] = {vw[c].x, vw[c].y, vw[c].z, vw[c].w};
        drop_nan<FORMAT>(ws);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 x = vkc::decode4<FORMAT>(ws[e]);
          const int d = 16 * c + 4 * e;
          acc[d] = __builtin_fmaf(wv, x.x, acc[d]);
          acc[d + 1] = __builtin_fmaf(wv, x.y, acc[d + 1]);
          acc[d + 2] = __builtin_fmaf(wv, x.z, acc[d + 2]);
          acc[d + 3] = __builtin_fmaf(wv, x.w, acc[d + 3]);
        }
      }
    }
    return past >= 0x7f800000u;
  };
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(run(std::false_type{})) != 0, 0))
    run(std::true_type{});
  const float mw = wave_max(m);
  const float f = m == -INFINITY && l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - mw);
  l *= f;
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] *= f;
  // halving by swaps of halves and of rows of 16, then by exchanges inside them (sums of the
  // same element once each lane has but one): lane x is left with element x / PARTS
#pragma unroll
  for (int d = 0; d < ND / 2; ++d) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[d]),
                                                    __float_as_uint(acc[d + ND / 2]), false, false);
    const uint32_t x = r[0], y = r[1];
    acc[d] = __uint_as_float(x) + __uint_as_float(y);
  }
#pragma unroll
  for (int d = 0; d < ND / 4; ++d) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[d]),
                                                    __float_as_uint(acc[d + ND / 4]), false, false);
    const uint32_t x = r[0], y = r[1];
    acc[d] = __uint_as_float(x) + __uint_as_float(y);
  }
#pragma unroll
  for (int w = 8; w; w >>= 1) {
    const int half = w / PARTS;  // elements left after the step (0: one before it, too)
    const bool up = (lane & w) != 0;
    if (half == 0) {
      acc[0] += __shfl_xor(acc[0], w, 64);
      continue;
    }
#pragma unroll
    for (int d = 0; d < half; ++d) {
      const float send = up ? acc[d] : acc[d + half];
      acc[d] = (up ? acc[d + half] : acc[d]) + __shfl_xor(send, w, 64);
    }
  }
#pragma unroll
  for (int w = 32; w; w >>= 1) l += __shfl_xor(l, w, 64);
  if (lane % PARTS == 0) so[wave][lane / PARTS] = acc[0];
  if (lane == 0) {
    sm[wave] = mw;
    sl[wave] = l;
  }
  __syncthreads();
  if (wave != 0 || lane >= ND) return;
  float mg = sm[0];
#pragma unroll
  for (int w = 1; w < kRowWaves; ++w) mg = fmaxf(mg, sm[w]);
  float o = 0.0f, lg = 0.0f;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    const float g = sm[w] == -INFINITY && sl[w] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(sm[w] - mg);
    o += so[w][lane] * g;
    lg += sl[w] * g;
  }
  if (PARTS == 1 && part) {
    const size_t rows = static_cast<size_t>(a.rows.sequences) * a.heads;
    const size_t at = static_cast<size_t>(split) * rows + row;
    part[at * HD + lane] = o;
    if (lane == 0)
      *reinterpret_cast<float4*>(part + a.splits * rows * HD + 4 * at) =
          make_float4(mg, 0.0f, lg, 0.0f);
  } else {
    out[vkc::row_at(a.rows, a.heads, s, h, 0) + d0 + lane] = lg == 0.0f ? 0.0f : o / lg * kRowUp;
  }
}

// ---------------------------------------------------------------------------
// 32 queries a wave on the f16 matrix cores
// ---------------------------------------------------------------------------
// S^T = K Q^T by 32x32x16 products, a block of 64 keys x 32 queries in 32 registers: a lane
// holds one query (lane l and l ^ 32 query l % 32), so maxima, references and denominators stay
// in the lane, S^T's registers are O^T += V^T P^T's operand as they stand, and no weight goes
// through LDS.  What belongs to a key (scales, documents) is spread over the 16 lanes of a row and
// broadcast by the instruction that uses it.
//
// The reference does not follow the maximum at every block: weights may be up to 2^(kPBits +
// kSlack) = 2^15, f16's upper end, and it moves once a row's largest score * V's scale
// passes it by 2^kSlack.  It holds V's scale too, so that the weights that matter have all
// their bits in f16 however small V is: a row's largest is at least 2^kPBits, its second
// part's last place 2^-24, which is 2^-33 of it (a rounding 2^-34).
using vks::f32x16;
using vks::f32x4;
using vks::u32x4;

constexpr int KB = 64;          // keys of a block
constexpr int kKPitch = 144;    // bytes of a K row in LDS: 64 f16 + 16
constexpr int kVPitch = 192;    // of a V row: 64 f16 + 64
constexpr float kPBits = 9.0f, kSlack = 6.0f;
constexpr float kLowest = -3e38f;       // the running reference before any key
constexpr float kFar = 65536.0f;        // scores of this size are taken from the row's own base
constexpr float kLeastLsv = -88.0f;     // of a key's V in the choice of the reference
constexpr int kCap = 1, kBias = 2;      // what SCORE does to a product beside its scale
constexpr int kQUp = 10;                // binary digits that Q is scaled up by

// Lane R of each 16-lane row, to all of the row.
template <int R>
__device__ __forceinline__ float bcast(float v) {
  return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(
      static_cast<int>(__float_as_uint(v)), 0x150 | R, 0xf, 0xf, true)));
}

template <int I>
using Int = std::integral_constant<int, I>;

template <typename F, int... I>
__device__ __forceinline__ void each(F f, std::integer_sequence<int, I...>) {
  (f(Int<I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F f) {
  each(f, std::make_integer_sequence<int, N>{});
}

__device__ __forceinline__ float other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// Eight codes as f16 (exact).
template <int FORMAT>
__device__ __forceinline__ u32x4 decode8(uint2 w) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  u32x4 r;
  if constexpr (FORMAT == VK_CACHE_Q8) {
    // code + 128 in the low byte of 1024 + .., and 1152 taken off
    const uint32_t a = w.x ^ 0x80808080u, b = w.y ^ 0x80808080u;
    const f16x2 off = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    const uint32_t p[4] = {__builtin_amdgcn_perm(a, 0x64646464u, 0x00050004u),
                           __builtin_amdgcn_perm(a, 0x64646464u, 0x00070006u),
                           __builtin_amdgcn_perm(b, 0x64646464u, 0x00050004u),
                           __builtin_amdgcn_perm(b, 0x64646464u, 0x00070006u)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2 x = __builtin_bit_cast(f16x2, p[i]) - off;
      r[i] = __builtin_bit_cast(uint32_t, x);
    }
  } else {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w.x), 1.0f, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w.x), 1.0f, true);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w.y), 1.0f, false);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w.y), 1.0f, true);
    r = u32x4{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
              __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)};
  }
  return r;
}

// V's codes that are no number (e4m3's 0x7f and 0xff, which the cache's write never makes, but
// a slot that nothing wrote may hold) as zeros: a weight of 0 does not take them away.
template <int FORMAT, int N>
__device__ __forceinline__ void drop_nan(uint32_t (&w)[N]) {
  if constexpr (FORMAT == VK_CACHE_F8) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) any |= (w[i] & 0x7f7f7f7fu) + 0x01010101u;
    if (__builtin_expect((any & 0x80808080u) != 0, 0)) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t bad = ((w[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        w[i] &= ~((bad << 1) - (bad >> 7));  // all of a byte
      }
    }
  }
}

// Four keys' values of one d a lane, out of LDS rows [key][d] of f16: in each 16
// lanes, lane 4 r + c gives the address of key r's values d = 4 c .. 4 c + 3, and lane d
// receives its d of keys 0 .. 3.
__device__ __forceinline__ uint2 read_tr(const char* p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 lds_t;
  const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lds_t*)(const_cast<char*>(p)));
  return __builtin_bit_cast(uint2, v);
}

// What a block's keys bring beside their codes, in LDS: 64 of each, key 32 t + 8
// (r / 4) + 4 half + r % 4 at 32 t + 16 half + r.
struct KeyData {
  float ks[KB];   // K's scale / 2^kQUp (a NaN where a scale of the key is no finite number)
  float lsv[KB];  // log2 of V's scale, at least kLeastLsv
  float sv[KB];   // V's scale (0 there)
  int doc[KB];
};

// The same as a lane of a wave takes them: of the keys of its row of 16 lanes, its own.
struct KeyRegs {
  float ks[2], lsv[2], sv[2];  // of the 32 keys t
  int doc[2];
};

__device__ __forceinline__ KeyRegs key_regs(const KeyData& kd, bool docs) {
  const int lane = threadIdx.x & 63, at = 16 * (lane >> 5) + (lane & 15);
  KeyRegs k;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    k.ks[t] = kd.ks[32 * t + at];
    k.lsv[t] = kd.lsv[32 * t + at];
    k.sv[t] = kd.sv[32 * t + at];
    k.doc[t] = docs ? kd.doc[32 * t + at] : 0;
  }
  return k;
}

// ks, lsv and sv from the scales of a row of K and of V.
__device__ __forceinline__ void key_values(float k, float v, float* ks, float* lsv, float* sv) {
  const float odd = (k - k) + (v - v);  // 0, or a NaN
  *ks = __builtin_fmaf(k, 1.0f / (1 << kQUp), odd);
  *sv = odd == 0.0f ? v : 0.0f;
  *lsv = fmaxf(__builtin_amdgcn_logf(fmaxf(*sv, vkc::kLeastScale)), kLeastLsv);
}

__device__ __forceinline__ int key_slot(int key) {
  return (key & 32) | (key & 4) << 2 | (key & 24) >> 1 | (key & 3);
}

// tanh to a few units of the last place: the odd series to x^11 below kTanhSeries, (e - 1) /
// (e + 1) as 1 - 2 / (e + 1) from there.
constexpr float kTanhSeries = 0.35f;

__device__ __forceinline__ float tanh_series(float x) {
  const float y = x * x;
  float p = __builtin_fmaf(y, -0.008863236f, 0.021869488f);
  p = __builtin_fmaf(y, p, -0.053968254f);
  p = __builtin_fmaf(y, p, 0.13333334f);
  p = __builtin_fmaf(y, p, -0.33333334f);
  return __builtin_fmaf(x * y, p, x);
}

__device__ __forceinline__ float tanh1(float x) {
  const float e = __builtin_amdgcn_exp2f(x * 2.8853900817779268f);
  const float b = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
  return fabsf(x) < kTanhSeries ? tanh_series(x) : b;
}

// A wave's 32 queries: lane l and lane l ^ 32 hold query l % 32.
struct Queries {
  u32x4 q[4][2];         // two f16 parts of eight values, four steps of 16 d
  int undo;              // the power of two that undoes the row's own scale (usually 0)
  bool own_scale;        // uniform: some row has one
  bool far;              // uniform: some row has a base
  float slope, cap_up;   // per unit of distance and cap, in base 2
  int pos, doc;
  int seen;              // causal: keys below it are seen
  f32x16 o[2];
  float m, l;            // running reference, this lane's denominators
};

// 2^x, -126 <= x <= 127.
__device__ __forceinline__ float pow2(int x) {
  return __uint_as_float(static_cast<uint32_t>(127 + x) << 23);
}
__device__ __forceinline__ int exponent(float v) {
  return static_cast<int>(__float_as_uint(v) >> 23) - 127;
}

// q c, scaled by a power of two of its own where a row's largest is not of the usual size:
// neither q c nor what undoes the scale has to be in f32's range (c is within 2^41 of 1).
// The order of d: element j of step ks is d = DK ks + DH half + j.
template <int DK, int DH>
__device__ __forceinline__ void load_queries(Queries& w, const float* row, float c, int half) {
  f32x4 x[4][2];
  float m = 0.0f;
#pragma unroll
  for (int ks = 0; ks < 4; ++ks)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[ks][i] = *reinterpret_cast<const f32x4*>(row + DK * ks + DH * half + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(x[ks][i][e]));
    }
  m = fmaxf(m, other_half(m));
  const int eq = min(exponent(m), 126);
  const float down = pow2(-eq);
  const int e = eq + exponent(m * down * fabsf(c));  // of the largest |q c|
  const bool usual = m == 0.0f || (e >= -10 && e < 5);
  const int up = usual ? kQUp : 14 - e;
  const float f = c * pow2(eq + up);
  w.undo = kQUp - up;
  w.own_scale = __builtin_amdgcn_ballot_w64(up != kQUp) != 0;
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    uint32_t h[4], l[4];
    const f32x4 a = x[ks][0] * down * f, b = x[ks][1] * down * f;
    vks::split2_plain(a[0], a[1], &h[0], &l[0]);
    vks::split2_plain(a[2], a[3], &h[1], &l[1]);
    vks::split2_plain(b[0], b[1], &h[2], &l[2]);
    vks::split2_plain(b[2], b[3], &h[3], &l[3]);
    w.q[ks][0] = u32x4{h[0], h[1], h[2], h[3]};
    w.q[ks][1] = u32x4{l[0], l[1], l[2], l[3]};
  }
#pragma unroll
  for (int dt = 0; dt < 2; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) w.o[dt][r] = 0.0f;
  w.m = kLowest;
  w.l = 0.0f;
  w.far = false;
}

// A row's base in LDS, 0 at first: once a row's reference passes +-kFar its scores are taken as
// differences from the base (exact near it), and so are the references, which hold V's scales
// and kPBits: beside a score of 2^26 f32 has no bits for those.
__device__ __forceinline__ float& base_of(float* bases) { return bases[threadIdx.x & 31]; }

// The reference of a join: (reference, base) pairs by their exact difference.
__device__ __forceinline__ float apart(float2 a, float2 b) {
  return (a.y - b.y) + (a.x - b.x);
}

// That of the two that stands higher, by value: a choice between an LDS element and a local
// would be one of addresses, and the local be kept in scratch.
__device__ __forceinline__ float2 larger(float2 a, float2 m) {
  const bool more = apart(a, m) > 0.0f;
  return make_float2(more ? a.x : m.x, more ? a.y : m.y);
}

// Two weights as f16 parts, packed: the remainder by one mixed-precision FMA each.
// `one` is 1.0 that the compiler does not see through: it would take the FMA apart.
__device__ __forceinline__ void split_weights2(float a, float b, float one, uint32_t* p0,
                                               uint32_t* p1) {
  const vks::f16x2 h = __builtin_convertvector((vks::f32x2{a, b}), vks::f16x2);
  const vks::f16x2 l = {
      static_cast<_Float16>(__builtin_fmaf(a, one, -static_cast<float>(h[0]))),
      static_cast<_Float16>(__builtin_fmaf(b, one, -static_cast<float>(h[1])))};
  *p0 = __builtin_bit_cast(uint32_t, h);
  *p1 = __builtin_bit_cast(uint32_t, l);
}

// One step of 16 d of S^T = K Q^T for a block of 64 keys: the small products first.
__device__ __forceinline__ void score_step(f32x16 (&s)[2], const Queries& w, const char* k, int ks) {
  const int lane = threadIdx.x & 63;
  const char* kf = k + (lane & 31) * kKPitch + 16 * (lane >> 5) + 32 * ks;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const u32x4 f = *reinterpret_cast<const u32x4*>(kf + 32 * t * kKPitch);
    s[t] = vks::mfma32(f, w.q[ks][1], s[t]);
    s[t] = vks::mfma32(f, w.q[ks][0], s[t]);
  }
}

__device__ __forceinline__ void clear(f32x16 (&s)[2]) {
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[t][r] = 0.0f;
}

// Half (the second half: `rest` 1) of the undoing of a row's own scale.
__device__ __forceinline__ void unscale(f32x16 (&s)[2], int undo, int rest) {
  asm volatile("" : "+v"(undo));  // keeps the work in the branch around it
  const float f = pow2((undo + rest) >> 1);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[t][r] *= f;
}

// The scores of a block from the products: scales, cap, bias and masks, base 2;
// `left` keys of it are held, `masked` (uniform) says whether a query of the wave may
// not see some of them.  Moves the reference of queries whose weights would leave
// f16's upper end: it follows the largest of score + log2 of V's scale, the size of a key's
// part of the value sum, once that passes it by kSlack.
template <int SCORE, bool MASK>
__device__ __forceinline__ void score_block(f32x16 (&s)[2], Queries& w, const Rules& ru,
                                            const KeyRegs& key, int k0, int left, bool masked,
                                            float* bases) {
  const int half = (threadIdx.x & 63) >> 5;
  // a row's own scale is undone in two steps about K's: either alone may leave f32's range
  if (__builtin_expect(w.own_scale, 0)) unscale(s, w.undo, 0);
  each<32>([&](auto i) { s[i / 16][i % 16] *= bcast<i % 16>(key.ks[i / 16]); });
  if (__builtin_expect(w.own_scale, 0)) unscale(s, w.undo, 1);
  if constexpr (SCORE != 0) __builtin_amdgcn_sched_barrier(0);
  if constexpr ((SCORE & kCap) != 0) {
    // scores far below the cap, the usual case, are the series' alone (3 x 16 x 1,301 queries
    // over up to 2,600 keys: 110 us, 138 where they are not; both for every score 131)
    float top = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(s[t][r]));
    if (__builtin_amdgcn_ballot_w64(top >= kTanhSeries) == 0) {
      each<32>([&](auto i) {
        s[i / 16][i % 16] = tanh_series(s[i / 16][i % 16]) * w.cap_up;
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // four at a time: registers
      });
    } else {
      each<32>([&](auto i) {
        s[i / 16][i % 16] = tanh1(s[i / 16][i % 16]) * w.cap_up;
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      });
    }
  }
  if constexpr ((SCORE & kBias) != 0) {
    const float base = static_cast<float>(static_cast<long long>(w.pos) - (k0 + 4 * half));
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[t][r] = __builtin_fmaf(-w.slope, fabsf(base - (32 * t + 8 * (r / 4) + r % 4)), s[t][r]);
  }
  if (__builtin_expect(w.far, 0)) {
    const float base = base_of(bases);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[t][r] -= base;
  }
  // nothing of the rules' work is begun ahead of it, in registers that the tile has not
  if constexpr (SCORE != 0) __builtin_amdgcn_sched_barrier(0);
  const bool causal = MASK && masked && ru.causal;
  if (__builtin_expect(left < KB || causal, 0)) {
    int lim = left;
    if (causal) lim = min(lim, w.seen - k0);
    lim -= 4 * half;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[t][r] = 32 * t + 8 * (r / 4) + r % 4 < lim ? s[t][r] : -INFINITY;
  }
  if (MASK && masked && ru.q_docs) {
    // a later document, or any other
    const int least = ru.docs_ordered ? -0x7fffffff - 1 : w.doc;
    each<32>([&](auto i) {
      const int d = __float_as_int(bcast<i % 16>(__int_as_float(key.doc[i / 16])));
      s[i / 16][i % 16] = d <= w.doc && d >= least ? s[i / 16][i % 16] : -INFINITY;
    });
  }
  float lsv[2] = {key.lsv[0], key.lsv[1]};
  // the broadcasts stay here, part of the additions
  asm volatile("" : "+v"(lsv[0]), "+v"(lsv[1]));
  float mb = kLowest;
  each<32>([&](auto i) { mb = fmaxf(mb, s[i / 16][i % 16] + bcast<i % 16>(lsv[i / 16])); });
  if (__builtin_amdgcn_ballot_w64(mb > w.m + kSlack) != 0) {
    mb = fmaxf(mb, other_half(mb));
    bool moves = mb > w.m + kSlack;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(moves && fabsf(mb) >= kFar) != 0, 0)) {
      // the base moves there, and what V's scales add is seen again without the score's rounding
      const float by = moves && fabsf(mb) >= kFar ? mb : 0.0f, base = base_of(bases);
      const float to = base + by, shift = to - base;
      base_of(bases) = to;
      vkd::wave_lds_fence();
      w.far = true;
      w.m = fmaxf(w.m - shift, kLowest);
      float again = kLowest;
      each<32>([&](auto i) {
        s[i / 16][i % 16] -= shift;
        again = fmaxf(again, s[i / 16][i % 16] + bcast<i % 16>(lsv[i / 16]));
      });
      mb = fmaxf(again, other_half(again));
    }
    // in two steps: V's scales, which the references carry, may be far apart
    const float f = moves ? __builtin_amdgcn_exp2f(0.5f * (w.m - mb)) : 1.0f;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) w.o[dt][r] = w.o[dt][r] * f * f;
    w.l = w.l * f * f;
    w.m = moves ? mb : w.m;
  }
}

// The weights of a block's scores, p = 2^(score - reference), their sum, and O^T += V^T
// (p V's scale)^T.
__device__ __forceinline__ void value_block(const f32x16 (&s)[2], Queries& w, const char* v,
                                            const KeyRegs& key) {
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const float ref = w.m - kPBits;
  float one = 1.0f;
  asm("" : "+s"(one));
  float sum[2] = {0.0f, 0.0f};
  // the transposed reads: key 16 ch + 4 half + (l % 16) / 4 (+ 8), d 32 dt + 16 (l / 16 % 2) + 4 (l % 4)
  const char* vf =
      v + (4 * half + ((lane & 15) >> 2)) * kVPitch + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
  each<4>([&](auto ch) {
    constexpr int kStep = 8 * kVPitch, t = ch >> 1, r0 = 8 * (ch & 1);
    u32x4 vv[2];
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) {
      const uint2 a = read_tr(vf + 2 * ch * kStep + 64 * dt);
      const uint2 b = read_tr(vf + (2 * ch + 1) * kStep + 64 * dt);
      vv[dt] = u32x4{a.x, a.y, b.x, b.y};
    }
    u32x4 p0, p1;
    each<4>([&](auto j) {
      constexpr int r = r0 + 2 * j;
      const float a = __builtin_amdgcn_exp2f(s[t][r] - ref);
      const float b = __builtin_amdgcn_exp2f(s[t][r + 1] - ref);
      sum[0] += a;
      sum[1] += b;
      uint32_t x, y;
      split_weights2(a * bcast<r>(key.sv[t]), b * bcast<r + 1>(key.sv[t]), one, &x, &y);
      p0[j()] = x;
      p1[j()] = y;
    });
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) w.o[dt] = vks::mfma32(vv[dt], p1, w.o[dt]);
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) w.o[dt] = vks::mfma32(vv[dt], p0, w.o[dt]);
  });
  w.l += sum[0] + sum[1];
}

// The queries of a wave: row `row` of cache head kh's, whose query heads lie side by side.
template <int SCORE, bool MASK, int DK, int DH>
__device__ __forceinline__ void take_queries(Queries& w, const float* __restrict__ q, const Shape& a,
                                             uint32_t s, uint32_t kh, uint32_t row, uint32_t* i,
                                             uint32_t* h) {
  const Rules& ru = a.rules;
  *i = row / a.group;
  *h = kh * a.group + (row - *i * a.group);
  load_queries<DK, DH>(w, q + vkc::row_at(a.rows, a.heads, s, *h, *i),
                       ru.cap > 0.0f ? ru.scale / ru.cap : ru.scale * kLog2e,
                       (threadIdx.x & 63) >> 5);
  w.cap_up = ru.cap * kLog2e;
  w.slope = (SCORE & kBias) != 0 ? ru.slopes[*h] * kLog2e : 0.0f;
  w.pos = position(vkc::start_of(a.rows, s), *i);
  const int pre = MASK && ru.prefix ? ru.prefix[s] : 0;
  w.seen = max(max(w.pos + 1, pre), 0);
  w.doc = MASK && ru.q_docs ? ru.q_docs[static_cast<size_t>(s) * a.rows.n + *i] : 0;
}

// What a tile's queries may see, as a whole, and a wave's of them.
struct Span {
  int p_low, p_high, pre;  // positions and prefix
  int q_low, q_high;       // documents
  int w_high, w_doc_low, w_doc_high;  // the wave's last position, its documents
};

// Whether some query of the wave may see a key of the block of keys k0 ..
__device__ __forceinline__ bool wave_sees(const Span& p, const Rules& ru, const KeyData& kd,
                                          int k0) {
  if (ru.causal && k0 > p.w_high && k0 >= p.pre) return false;
  if (!ru.q_docs) return true;
  const int d = kd.doc[threadIdx.x & 63];
  return __builtin_amdgcn_ballot_w64(d <= p.w_doc_high && (ru.docs_ordered || d >= p.w_doc_low)) != 0;
}

// Of rows row_first .. row_last of a workgroup of WAVES waves; `range` is LDS.
template <int WAVES>
__device__ __forceinline__ Span tile_span(const Queries& w, const Shape& a, uint32_t s,
                                          int row_first, int row_last, bool live, int* range) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int start = vkc::start_of(a.rows, s);
  Span p{position(start, row_first / a.group), position(start, row_last / a.group),
         a.rules.prefix ? a.rules.prefix[s] : 0, 0, 0, 0, 0, 0};
  p.w_high = position(start, min(row_first + 32 * wave + 31, row_last) / a.group);
  if (a.rules.q_docs) {
    int lo = w.doc, hi = w.doc;
#pragma unroll
    for (int m = 16; m; m >>= 1) {
      lo = min(lo, __shfl_xor(lo, m, 64));
      hi = max(hi, __shfl_xor(hi, m, 64));
    }
    p.w_doc_low = __builtin_amdgcn_readfirstlane(lo);
    p.w_doc_high = __builtin_amdgcn_readfirstlane(hi);
    if (lane == 0) {
      range[wave] = live ? lo : 0x7fffffff;
      range[WAVES + wave] = live ? hi : -0x7fffffff - 1;
    }
    __syncthreads();
    p.q_low = range[0];
    p.q_high = range[WAVES];
#pragma unroll
    for (int x = 1; x < WAVES; ++x) {
      p.q_low = min(p.q_low, range[x]);
      p.q_high = max(p.q_high, range[WAVES + x]);
    }
  }
  return p;
}

// A tile across the border of two documents would take the blocks of both, one after the
// other, for half of its queries each (10,392 queries over documents of 866, most tiles in one
// of them: 143 us, so 100).  It has two workgroups, and where its first rows have a document that
// no later row has, the first takes those and the second the rest; else the second has nothing
// (documents of 8 x 128: 89 us, so 91).  Ordered documents hold the earlier ones' keys too and
// gain nothing (407 us, 480 so).  Row bounds in, and out; false: no row.
__device__ __forceinline__ bool document_part(const Shape& a, uint32_t s, uint32_t part, int* row0,
                                              int* row_end) {
  static_assert(vk::kTileRows == 128, "two rows a lane");
  const int lane = threadIdx.x & 63, rows = *row_end - *row0;
  const int* docs = a.rules.q_docs + static_cast<size_t>(s) * a.rows.n;
  const auto doc_of = [&](int i) {
    return docs[static_cast<uint32_t>(*row0 + min(i, rows - 1)) / a.group];
  };
  const int d0 = doc_of(0), x = doc_of(lane), y = doc_of(64 + lane);
  const uint64_t e0 = __builtin_amdgcn_ballot_w64(x == d0 && lane < rows);
  const uint64_t e1 = __builtin_amdgcn_ballot_w64(y == d0 && lane + 64 < rows);
  const int same = __popcll(e0) + __popcll(e1);
  // the same rows are the first ones
  const bool first = ~e0 ? __builtin_ctzll(~e0) == same : !~e1 || 64 + __builtin_ctzll(~e1) == same;
  if (!first || same == rows) return part == 0;
  if (part == 0)
    *row_end = *row0 + same;
  else
    *row0 += same;
  return true;
}

constexpr int kList = 2048;  // blocks whose visibility is worked out at a time

// Smallest and largest of a 16-lane row.
__device__ __forceinline__ void row16_range(int* lo, int* hi) {
#define VK_ROR(n)                                                              \
  *lo = min(*lo, __builtin_amdgcn_mov_dpp(*lo, 0x120 | n, 0xf, 0xf, true));    \
  *hi = max(*hi, __builtin_amdgcn_mov_dpp(*hi, 0x120 | n, 0xf, 0xf, true));
  VK_ROR(8) VK_ROR(4) VK_ROR(2) VK_ROR(1)
#undef VK_ROR
}

// Lists the blocks of seg .. seg_end - 1 that some query of the tile may see, in order: the
// block less seg, times two, plus one where not every query sees all of it.  First the documents'
// part, 16 lanes a block and 16 blocks a wave in flight (1,000 workgroups over 163 blocks,
// with the attention: a thread a block 157 us, so 131), as 2 (some) + 1 (not all) in the block's
// place; then a thread a block takes the order in and closes the gaps.  `count` is LDS.
template <int WAVES>
__device__ __forceinline__ int list_blocks(uint16_t* list, int* count, const Shape& a,
                                           const Span& p, int seg, int seg_end, int keys,
                                           size_t doc_first) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Rules& ru = a.rules;
  if (ru.causal) {  // blocks with a key that is not behind every query
    const int top = max(max(p.p_high + 1, p.pre), 0);
    seg_end = min(seg_end, top / KB + (top % KB != 0));
  }
  if (ru.q_docs) {
    const int* d = ru.k_docs + doc_first;
    for (int base = seg; base < seg_end; base += 16 * WAVES) {
      int x[4][4];
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const int b = base + 4 * WAVES * y + 4 * wave + (lane >> 4);
          x[y][z] = d[min(b * KB + 16 * z + (lane & 15), keys - 1)];
        }
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int b = base + 4 * WAVES * y + 4 * wave + (lane >> 4);
        int lo = min(min(x[y][0], x[y][1]), min(x[y][2], x[y][3]));
        int hi = max(max(x[y][0], x[y][1]), max(x[y][2], x[y][3]));
        row16_range(&lo, &hi);
        const bool any = lo <= p.q_high && (ru.docs_ordered || hi >= p.q_low);
        const bool full = ru.docs_ordered
                              ? hi <= p.q_low
                              : lo == hi && p.q_low == p.q_high && lo == p.q_low;
        if ((lane & 15) == 0 && b < seg_end)
          list[b - seg] = static_cast<uint16_t>((any ? 2 : 0) | (full ? 0 : 1));
      }
    }
    __syncthreads();
  }
  int filled = 0;
  for (int b0 = seg; b0 < seg_end; b0 += 64 * WAVES) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    bool any = b < seg_end, full = true;
    if (any) {
      if (ru.causal) {
        const int k1 = min(b * KB + KB, keys) - 1;  // last key
        full = k1 <= p.p_low || k1 < p.pre;
      }
      if (ru.q_docs) {
        const int x = list[b - seg];
        any = (x & 2) != 0;
        full = full && (x & 1) == 0;
      }
    }
    const uint64_t m = __builtin_amdgcn_ballot_w64(any);
    __syncthreads();  // the counts of the run before are read, and the marks of this one
    if (lane == 0) count[wave] = __popcll(m);
    __syncthreads();
    int at = filled;
#pragma unroll
    for (int x = 0; x < WAVES; ++x) {
      if (x < wave) at += count[x];
      filled += count[x];
    }
    if (any)
      list[at + __popcll(m & ((1ull << lane) - 1))] =
          static_cast<uint16_t>((b - seg) << 1 | (full ? 0 : 1));
  }
  __syncthreads();
  return filled;
}

// A query's share of the result: its sums and their denominators to `part` (and the
// reference they stand in), or their quotient to `out`.
__device__ __forceinline__ void store_part(float* part, const Shape& a, uint32_t split, uint32_t s,
                                           uint32_t h, uint32_t i, int d, const f32x4& o) {
  const size_t rows = static_cast<size_t>(a.rows.sequences) * a.heads * a.rows.n;
  const size_t at = static_cast<size_t>(split) * rows +
                    (static_cast<size_t>(s) * a.heads + h) * a.rows.n + i;
  *reinterpret_cast<f32x4*>(part + at * HD + d) = o;
}

__device__ __forceinline__ void store_ml(float* part, const Shape& a, uint32_t split, uint32_t s,
                                         uint32_t h, uint32_t i, float m, float l, float base) {
  const size_t rows = static_cast<size_t>(a.rows.sequences) * a.heads * a.rows.n;
  const size_t at = static_cast<size_t>(split) * rows +
                    (static_cast<size_t>(s) * a.heads + h) * a.rows.n + i;
  *reinterpret_cast<float4*>(part + a.splits * rows * HD + 4 * at) = make_float4(m, base, l, 0.0f);
}

__device__ __forceinline__ f32x4 quotient(const f32x4& o, float l) {
  if (l == 0.0f) return f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  return f32x4{o[0] / l, o[1] / l, o[2] / l, o[3] / l};
}

// A lane's offset into a buffer, so that what a load adds to it is added there, as the
// instruction's own offset, and not ahead of the loop in a register each.
__device__ __forceinline__ int here(int offset) {
  asm volatile("" : "+v"(offset));
  return offset;
}

// Staging by all threads: eight codes of K (or V) a thread and row.  The block's
// rows are a buffer of their own (its base and the bytes left of it in scalar registers), so
// a load has no address arithmetic and keys past the end read zeros (every offset is part of
// the lane's, constants in the instruction: the uniform offset is left out of bounds checks).
template <int FORMAT, int THREADS>
struct StageRows {
  static constexpr int kPer = KB * 8 / THREADS;
  uint2 w[kPer];

  __device__ __forceinline__ void load(const uint8_t* codes, size_t first, int k0, int keys) {
    typedef int i32x2_t __attribute__((ext_vector_type(2)));
    const int left = keys - k0 < KB ? keys - k0 : KB;
    const __amdgpu_buffer_rsrc_t r =
        vkd::buffer_rsrc(codes + (first + k0) * HD, static_cast<uint32_t>(left * HD));
    const int at = here(8 * static_cast<int>(threadIdx.x));
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const i32x2_t x = __builtin_amdgcn_raw_buffer_load_b64(
          r, at + 8 * THREADS * i, 0, 0);
      w[i] = make_uint2(static_cast<uint32_t>(x[0]), static_cast<uint32_t>(x[1]));
    }
  }

  template <int PITCH, bool V = false>
  __device__ __forceinline__ void store(char* to) {
    const int tid = threadIdx.x;
    if constexpr (V) {
      uint32_t x[2 * kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[2 * i] = w[i].x, x[2 * i + 1] = w[i].y;
      drop_nan<FORMAT>(x);
#pragma unroll
      for (int i = 0; i < kPer; ++i) w[i] = make_uint2(x[2 * i], x[2 * i + 1]);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      *reinterpret_cast<u32x4*>(to + ((tid >> 3) + i * (THREADS / 8)) * PITCH + 16 * (tid & 7)) =
          decode8<FORMAT>(w[i]);
  }
};

// A key's scales and document, one a thread of the first wave.
struct StageKeys {
  float ks, vs;
  int doc;

  __device__ __forceinline__ void load(const Shape& a, size_t first, size_t doc_first, int k0,
                                       int keys) {
    const int left = keys - k0 < KB ? keys - k0 : KB;
    const int at = 4 * static_cast<int>(threadIdx.x), bytes = 4 * left;
    ks = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
        vkd::buffer_rsrc(a.cache.ks + first + k0, bytes), at, 0, 0));
    vs = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
        vkd::buffer_rsrc(a.cache.vs + first + k0, bytes), at, 0, 0));
    if (a.rules.k_docs)
      doc = static_cast<int>(__builtin_amdgcn_raw_buffer_load_b32(
          vkd::buffer_rsrc(a.rules.k_docs + doc_first + k0, bytes), at, 0, 0));
  }

  __device__ __forceinline__ void store(const Shape& a, KeyData& kd) const {
    const int at = key_slot(threadIdx.x);
    key_values(ks, vs, &kd.ks[at], &kd.lsv[at], &kd.sv[at]);
    if (a.rules.k_docs) kd.doc[at] = doc;
  }
};

// Three workgroups a CU; two with a cap, whose work a score wants the registers (in 168 of
// them it spills: 122 us for 110).  A masked bias spills 8 to 11 of the 168, a plain mask one at
// most; two workgroups are slower there (12 x 10,392 queries, documents of 866: 173 us for 109).
template <int FORMAT, int SCORE, bool MASK, int QW>
__global__ __launch_bounds__(64 * QW, SCORE & kCap ? 2 : 3) void attention_tile_kernel(const float* __restrict__ q,
                                                                    float* __restrict__ out,
                                                                    float* __restrict__ part,
                                                                    Shape a) {
  constexpr int kThreads = 64 * QW, kRows = 32 * QW;
  static_assert(kRows == vk::kTileRows, "the plan's tiles");
  __shared__ __align__(16) char kl[2][KB * kKPitch];
  __shared__ __align__(16) char vl[2][KB * kVPitch];
  __shared__ KeyData kd[2];
  __shared__ uint16_t list[MASK ? kList : 1];
  __shared__ int wave_count[QW], doc_range[2 * QW];
  __shared__ float base[QW][32];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  __builtin_assume(tid < kThreads);
  const Rules& ru = a.rules;

  // Workgroups go round the 8 XCDs.  `order.share` of them take a group of `order.heads`
  // (sequence, cache head) pairs between them, so that a pair's K and V stay in few L2s; a
  // group's pairs are a head's of every sequence, whose lengths differ (3 sequences of 16 heads:
  // 107 us with a group's of one sequence, 98 so).  In a group the last tiles come first: with a
  // causal mask they take longest.
  const uint32_t xcd = blockIdx.x & 7;
  const uint32_t in = (blockIdx.x >> 3) * a.order.share + xcd % a.order.share;
  if (in >= a.order.heads * a.splits * a.tiles * a.parts) return;
  const uint32_t pair = in % a.order.heads, u = in / a.order.heads;
  const uint32_t split = u % a.splits, v = u / a.splits;
  // (the second parts first: most of them end at once)
  const uint32_t tile = a.tiles - 1 - v % a.tiles, piece = a.parts - 1 - v / a.tiles;
  const uint32_t sh = xcd / a.order.share * a.order.heads + pair;
  const uint32_t s = sh % a.rows.sequences, kh = sh / a.rows.sequences;
  const int count = vkc::count_of(a.rows, s);
  const int rows = count > 0 ? count * static_cast<int>(a.group) : 0;  // query i's heads side by side
  int row0 = static_cast<int>(tile) * kRows;
  if (row0 >= rows) return;
  int row_end = row0 + kRows < rows ? row0 + kRows : rows;
  if (MASK && a.parts > 1 && !document_part(a, s, piece, &row0, &row_end)) return;
  const int keys = keys_of(a, s);
  const size_t first = (static_cast<size_t>(s) * a.cache.heads + kh) * a.cache.capacity;
  const size_t doc_first = static_cast<size_t>(s) * a.cache.capacity;
  const bool live = row0 + 32 * wave < row_end;  // uniform over the wave
  const int row = row0 + 32 * wave + (lane & 31);
  uint32_t i, h;
  Queries w;
  take_queries<SCORE, MASK, 16, 8>(w, q, a, s, kh, row < row_end ? row : row_end - 1, &i, &h);

  base_of(base[wave]) = 0.0f;  // (both lanes of a query, the same)
  const int blocks = (keys + KB - 1) / KB;
  Span span;
  if constexpr (MASK)
    span = tile_span<QW>(w, a, s, row0, row_end - 1, live, doc_range);
  StageRows<FORMAT, kThreads> rows_k, rows_v;
  StageKeys keys_d;
  // blocks listed (MASK) or all of them, a run of kList at a time
  for (int seg = 0; seg < blocks; seg += kList) {
    int listed = blocks - seg < kList ? blocks - seg : kList;
    if constexpr (MASK)
      listed = list_blocks<QW>(list, wave_count, a, span, seg, seg + listed, keys, doc_first);
    const int b_begin = static_cast<int>(split * static_cast<uint32_t>(listed) / a.splits);
    const int b_end = static_cast<int>((split + 1) * static_cast<uint32_t>(listed) / a.splits);
    if (b_begin == b_end) continue;  // uniform over the workgroup
    auto entry = [&](int x) { return MASK ? static_cast<int>(list[x]) : x << 1; };
    auto key_of = [&](int e) { return (seg + (e >> 1)) * KB; };
    int e = entry(b_begin);
    rows_k.load(a.cache.k, first, key_of(e), keys);
    rows_v.load(a.cache.v, first, key_of(e), keys);
    if (wave == 0) keys_d.load(a, first, doc_first, key_of(e), keys);
    rows_k.template store<kKPitch>(kl[0]);
    rows_v.template store<kVPitch, true>(vl[0]);
    if (wave == 0) keys_d.store(a, kd[0]);
    __syncthreads();
    for (int x = b_begin; x < b_end; ++x) {
      const int buf = (x - b_begin) & 1;
      const int e1 = entry(x + 1 < b_end ? x + 1 : x);
      const int k0 = key_of(e);
      rows_k.load(a.cache.k, first, key_of(e1), keys);
      rows_v.load(a.cache.v, first, key_of(e1), keys);
      if (wave == 0) keys_d.load(a, first, doc_first, key_of(e1), keys);
      __builtin_amdgcn_sched_barrier(0);
      if (live && !(MASK && (e & 1) && !wave_sees(span, ru, kd[buf], k0))) {
        f32x16 sc[2];
        clear(sc);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) score_step(sc, w, kl[buf], ks);
        const KeyRegs key = key_regs(kd[buf], MASK && ru.q_docs);
        score_block<SCORE, MASK>(sc, w, ru, key, k0, keys - k0, (e & 1) != 0, base[wave]);
        // ahead of the CU's other waves while it feeds the matrix cores (12 x 866 queries over
        // 10,392 keys 79.7 us without, 76.3 so; masked 413 and 408), and up to the barrier where
        // its blocks go by in step with theirs (73.4; masked 413)
        __builtin_amdgcn_s_setprio(1);
        value_block(sc, w, vl[buf], key);
        if constexpr (MASK) __builtin_amdgcn_s_setprio(0);
      }
      rows_k.template store<kKPitch>(kl[buf ^ 1]);
      rows_v.template store<kVPitch, true>(vl[buf ^ 1]);
      if (wave == 0) keys_d.store(a, kd[buf ^ 1]);
      e = e1;
      if constexpr (!MASK) __builtin_amdgcn_s_setprio(0);
      __syncthreads();
    }
  }
  const int half = lane >> 5;
  const float l = w.l + other_half(w.l);
  if (!live || row >= row_end) return;
#pragma unroll
  for (int dt = 0; dt < 2; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const f32x4 o = {w.o[dt][4 * r], w.o[dt][4 * r + 1], w.o[dt][4 * r + 2], w.o[dt][4 * r + 3]};
      const int d = 32 * dt + 8 * r + 4 * half;
      if (part)
        store_part(part, a, split, s, h, i, d, o);
      else
        *reinterpret_cast<f32x4*>(out + vkc::row_at(a.rows, a.heads, s, h, i) + d) = quotient(o, l);
    }
  if (part && half == 0) store_ml(part, a, split, s, h, i, w.m, l, base_of(base[wave]));
}

// 32 rows or fewer of a cache head: the waves of a workgroup hold the same queries and
// take blocks of keys in turn, each for itself: K straight from memory as the products' operand
// (d = 32 half + 8 ks + j: a lane's 32 codes of a key lie side by side), V through 12
// KiB of LDS of the wave's own for the transposed reads, a block ahead in registers.  No
// barrier until the waves are joined at the end.
constexpr int kFewWaves = 4;

template <int FORMAT, int SCORE, bool MASK>
__global__ __launch_bounds__(64 * kFewWaves, 2) void attention_few_kernel(
    const float* __restrict__ q, float* __restrict__ out, float* __restrict__ part, Shape a) {
  __shared__ __align__(16) char vl[kFewWaves][KB * kVPitch];
  __shared__ float2 sm[kFewWaves][32];  // reference, base
  __shared__ float sl[kFewWaves][32], base[kFewWaves][32];
  __shared__ uint16_t list[MASK ? kList : 1];
  __shared__ int wave_count[kFewWaves], doc_range[2 * kFewWaves];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5;
  __builtin_assume(tid < 64 * kFewWaves);
  const Rules& ru = a.rules;
  const uint32_t split = blockIdx.x % a.splits, sh = blockIdx.x / a.splits;
  const uint32_t kh = sh % a.cache.heads, s = sh / a.cache.heads;
  const int count = vkc::count_of(a.rows, s);
  if (count <= 0) return;
  const int rows = count * static_cast<int>(a.group);
  const int keys = keys_of(a, s);
  const size_t first = (static_cast<size_t>(s) * a.cache.heads + kh) * a.cache.capacity;
  const size_t doc_first = static_cast<size_t>(s) * a.cache.capacity;
  const int row = lane & 31;
  uint32_t i, h;
  Queries w;
  take_queries<SCORE, MASK, 8, 32>(w, q, a, s, kh, row < rows ? row : rows - 1, &i, &h);
  base_of(base[wave]) = 0.0f;
  const int blocks = (keys + KB - 1) / KB;
  Span span;
  if constexpr (MASK) span = tile_span<kFewWaves>(w, a, s, 0, rows - 1, true, doc_range);

  // a block's codes and scales in registers: K rows 32 t + l % 32, bytes 32 half ..; V rows
  // 16 x + l / 4, 16 bytes at l % 4; scales of keys 32 t + 8 (i / 4) + 4 half + i % 4, i = l % 16
  typedef int i32x4_t __attribute__((ext_vector_type(4)));
  i32x4_t kr[2][2], vr[4];
  float kss[2], vss[2];
  int docs[2];
  auto load = [&](int k0) {
    const int left = keys - k0 < KB ? keys - k0 : KB;
    const __amdgpu_buffer_rsrc_t kb =
        vkd::buffer_rsrc(a.cache.k + (first + k0) * HD, static_cast<uint32_t>(left * HD));
    const __amdgpu_buffer_rsrc_t vb =
        vkd::buffer_rsrc(a.cache.v + (first + k0) * HD, static_cast<uint32_t>(left * HD));
    const int k_off = here((lane & 31) * HD + 32 * half), v_off = here(16 * lane);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        kr[t][x] = __builtin_amdgcn_raw_buffer_load_b128(kb, k_off + 32 * HD * t + 16 * x, 0, 0);
#pragma unroll
    for (int x = 0; x < 4; ++x)
      vr[x] = __builtin_amdgcn_raw_buffer_load_b128(vb, v_off + 1024 * x, 0, 0);
    const __amdgpu_buffer_rsrc_t ksb = vkd::buffer_rsrc(a.cache.ks + first + k0, 4 * left);
    const __amdgpu_buffer_rsrc_t vsb = vkd::buffer_rsrc(a.cache.vs + first + k0, 4 * left);
    const int at = here(4 * (8 * ((lane & 15) >> 2) + 4 * half + (lane & 3)));
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      kss[t] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(ksb, at + 128 * t, 0, 0));
      vss[t] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(vsb, at + 128 * t, 0, 0));
    }
    if (MASK && ru.q_docs) {
      const __amdgpu_buffer_rsrc_t db =
          vkd::buffer_rsrc(ru.k_docs + doc_first + k0, 4 * left);
#pragma unroll
      for (int t = 0; t < 2; ++t)
        docs[t] = static_cast<int>(__builtin_amdgcn_raw_buffer_load_b32(db, at + 128 * t, 0, 0));
    }
  };
  char* vw = vl[wave];

  for (int seg = 0; seg < blocks; seg += kList) {
    int listed = blocks - seg < kList ? blocks - seg : kList;
    if constexpr (MASK)
      listed = list_blocks<kFewWaves>(list, wave_count, a, span, seg, seg + listed, keys, doc_first);
    const int b_begin = static_cast<int>(split * static_cast<uint32_t>(listed) / a.splits) + wave;
    const int b_end = static_cast<int>((split + 1) * static_cast<uint32_t>(listed) / a.splits);
    auto entry = [&](int x) {
      return MASK ? __builtin_amdgcn_readfirstlane(static_cast<int>(list[x])) : x << 1;
    };
    auto key_of = [&](int e) { return (seg + (e >> 1)) * KB; };
    int e = 0;
    if (b_begin < b_end) {
      e = entry(b_begin);
      load(key_of(e));
    }
    for (int x = b_begin; x < b_end; x += kFewWaves) {
      // this block's operands out of the loads' registers
      const int k0 = key_of(e);
      KeyRegs key;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        key_values(kss[t], vss[t], &key.ks[t], &key.lsv[t], &key.sv[t]);
        key.doc[t] = MASK && ru.q_docs ? docs[t] : 0;
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        char* to = vw + (16 * y + (lane >> 2)) * kVPitch + 32 * (lane & 3);
        const int c0 = vr[y][0], c1 = vr[y][1], c2 = vr[y][2], c3 = vr[y][3];
        uint32_t c[4] = {static_cast<uint32_t>(c0), static_cast<uint32_t>(c1),
                         static_cast<uint32_t>(c2), static_cast<uint32_t>(c3)};
        drop_nan<FORMAT>(c);
        *reinterpret_cast<u32x4*>(to) = decode8<FORMAT>(make_uint2(c[0], c[1]));
        *reinterpret_cast<u32x4*>(to + 16) = decode8<FORMAT>(make_uint2(c[2], c[3]));
      }
      f32x16 sc[2];
      clear(sc);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const i32x4_t c = kr[t][ks >> 1];
          const u32x4 f = decode8<FORMAT>(ks & 1 ? make_uint2(c[2], c[3]) : make_uint2(c[0], c[1]));
          sc[t] = vks::mfma32(f, w.q[ks][1], sc[t]);
          sc[t] = vks::mfma32(f, w.q[ks][0], sc[t]);
        }
      const int e1 = entry(x + kFewWaves < b_end ? x + kFewWaves : x);
      load(key_of(e1));
      vkd::wave_lds_fence();
      score_block<SCORE, MASK>(sc, w, ru, key, k0, keys - k0, (e & 1) != 0, base[wave]);
      value_block(sc, w, vw, key);
      vkd::wave_lds_fence();
      e = e1;
    }
    if constexpr (MASK) __syncthreads();  // the list is read
  }
  // the waves together, in their order: o through each wave's LDS as [query][d]
  w.l += other_half(w.l);
  float* so = reinterpret_cast<float*>(vw);
  constexpr int kOPitch = 68;
  static_assert(32 * kOPitch * 4 <= KB * kVPitch, "a wave's sums fit its LDS");
#pragma unroll
  for (int dt = 0; dt < 2; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<f32x4*>(so + row * kOPitch + 32 * dt + 8 * r + 4 * half) =
          f32x4{w.o[dt][4 * r], w.o[dt][4 * r + 1], w.o[dt][4 * r + 2], w.o[dt][4 * r + 3]};
  if (half == 0) {
    sm[wave][row] = make_float2(w.m, base_of(base[wave]));
    sl[wave][row] = w.l;
  }
  __syncthreads();
  for (int x = tid; x < 16 * rows; x += 64 * kFewWaves) {
    const int r = x >> 4, d = 4 * (x & 15);
    float2 m = sm[0][r];
#pragma unroll
    for (int y = 1; y < kFewWaves; ++y) m = larger(sm[y][r], m);
    float l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int y = 0; y < kFewWaves; ++y) {
      // in two steps: V's scales, which the references carry, may be far apart
      const float f = sl[y][r] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(0.5f * apart(sm[y][r], m));
      l += sl[y][r] * f * f;
      o += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(vl[y]) + r * kOPitch + d) *
           f * f;
    }
    const uint32_t ri = r / a.group, rh = kh * a.group + (r - ri * a.group);
    if (part) {
      store_part(part, a, split, s, rh, ri, d, o);
      if (d == 0) store_ml(part, a, split, s, rh, ri, m.x, l, m.y);
    } else {
      *reinterpret_cast<f32x4*>(out + vkc::row_at(a.rows, a.heads, s, rh, ri) + d) = quotient(o, l);
    }
  }
}

// Joins the key splits of a row: a wave a row, its 16-lane rows g taking splits g, g + 4, ..
// in order (every load before the first sum), and then the four together.
template <int PER>
__global__ __launch_bounds__(256) void attention_join_kernel(const float* __restrict__ part,
                                                             float* __restrict__ out, float up,
                                                             Shape a) {
  const size_t row = static_cast<size_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int g = (threadIdx.x & 63) >> 4, c = static_cast<int>(threadIdx.x & 15);
  const size_t rows = static_cast<size_t>(a.rows.sequences) * a.heads * a.rows.n;
  if (row >= rows) return;
  const uint32_t i = static_cast<uint32_t>(row % a.rows.n);
  const uint32_t sh = static_cast<uint32_t>(row / a.rows.n);
  const uint32_t h = sh % a.heads, s = sh / a.heads;
  if (static_cast<int>(i) >= vkc::count_of(a.rows, s)) return;
  const float4* ml = reinterpret_cast<const float4*>(part + a.splits * rows * HD);
  float4 x[PER];  // reference, base, denominator
  f32x4 y[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint32_t sp = g + 4 * j;
    const size_t at = (sp < a.splits ? sp : 0) * rows + row;
    x[j] = ml[at];
    y[j] = *reinterpret_cast<const f32x4*>(part + at * HD + 4 * c);
    if (sp >= a.splits) x[j].z = 0.0f;
  }
  float2 m = make_float2(x[0].x, x[0].y);  // again the first past the last
#pragma unroll
  for (int j = 1; j < PER; ++j) m = larger(make_float2(x[j].x, x[j].y), m);
#pragma unroll
  for (int w = 16; w <= 32; w <<= 1)
    m = larger(make_float2(__shfl_xor(m.x, w, 64), __shfl_xor(m.y, w, 64)), m);
  float l = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    // in two steps: V's scales, which the references carry, may be far apart
    const float w = x[j].z != 0.0f
                        ? __builtin_amdgcn_exp2f(0.5f * apart(make_float2(x[j].x, x[j].y), m))
                        : 0.0f;
    l += x[j].z * w * w;
    o += y[j] * w * w;
  }
#pragma unroll
  for (int w = 16; w <= 32; w <<= 1) {
    l += __shfl_xor(l, w, 64);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], w, 64);
  }
  if (g == 0)
    *reinterpret_cast<f32x4*>(out + vkc::row_at(a.rows, a.heads, s, h, i) + 4 * c) =
        quotient(o, l) * up;
}

int check_i32(const vk_runtime* rt, const vk_tensor* t, size_t len, const char* what) {
  VK_REQUIRE(t->dtype == VK_I32 && t->len == len, "%s must be i32 [%zu] (holds %zu)", what, len,
             t->len);
  return vk::check_device(rt, t, what);
}

}  // namespace

extern "C" {

int vk_attention_cached_f32(vk_runtime* rt, const vk_kv_cache* cache, const vk_tensor* q,
                            size_t heads, size_t n, const vk_tensor* starts,
                            const vk_tensor* counts, size_t max_length,
                            const vk_attention_rules* rules, vk_qk_layout layout, vk_tensor* out) {
  VK_TRY(vk::bind(rt));
  VK_TRY(vk::check_cache(rt, cache));
  VK_REQUIRE(layout == VK_QK_HEADS_OUTER || layout == VK_QK_VIEWS_OUTER, "unknown layout %d",
             static_cast<int>(layout));
  VK_REQUIRE(heads > 0 && heads % cache->heads == 0,
             "attention_cached: %zu heads over a cache of %zu", heads, cache->heads);
  VK_UNSUPPORTED_IF(heads > 0xffff || n > 0x7fffffffULL ||
                        (n > 0 && cache->sequences * heads > 0x7fffffffULL / n),
                    "attention_cached: %zu x %zu x %zu queries", cache->sequences, heads, n);
  const size_t rows = cache->sequences * heads * n;
  VK_TRY(vk::check_f32(rt, q, rows * HD, "q"));
  VK_TRY(vk::check_f32(rt, out, rows * HD, "out"));
  VK_TRY(vk::check_spans(rt, starts, counts, cache->sequences));
  static const vk_attention_rules kNone = {};
  const vk_attention_rules& ru = rules ? *rules : kNone;
  VK_REQUIRE(std::isfinite(ru.scale), "attention_cached: scale %g", static_cast<double>(ru.scale));
  VK_REQUIRE(std::isfinite(ru.cap) && ru.cap >= 0.0f, "attention_cached: cap %g",
             static_cast<double>(ru.cap));
  // so that what a query is multiplied by, and what undoes a row's own scale, are normal numbers
  const float scale = ru.scale == 0.0f ? 0.125f : ru.scale;
  const float by = std::fabs(ru.cap > 0.0f ? scale / ru.cap : scale);
  VK_UNSUPPORTED_IF(!(by >= 0x1p-40f && by <= 0x1p40f && std::fabs(scale) >= 0x1p-40f &&
                      std::fabs(scale) <= 0x1p40f),
                    "attention_cached: scale %g with cap %g (scale and scale / cap: 2^-40 to 2^40)",
                    static_cast<double>(ru.scale), static_cast<double>(ru.cap));
  if (ru.slopes) {
    VK_REQUIRE(ru.slopes->dtype == VK_F32 && ru.slopes->len == heads,
               "slopes must be f32 [%zu] (holds %zu)", heads, ru.slopes->len);
    VK_TRY(vk::check_device(rt, ru.slopes, "slopes"));
  }
  VK_REQUIRE(!ru.prefix || ru.causal, "attention_cached: prefix without causal");
  VK_REQUIRE((ru.q_docs != nullptr) == (ru.k_docs != nullptr),
             "attention_cached: q_docs and k_docs go together");
  VK_REQUIRE(!ru.docs_ordered || ru.q_docs, "attention_cached: docs_ordered without documents");
  if (ru.prefix) VK_TRY(check_i32(rt, ru.prefix, cache->sequences, "prefix"));
  if (ru.q_docs) {
    VK_TRY(check_i32(rt, ru.q_docs, cache->sequences * n, "q_docs"));
    VK_TRY(check_i32(rt, ru.k_docs, cache->sequences * cache->capacity, "k_docs"));
  }
  for (const vk_tensor* t : {q, static_cast<const vk_tensor*>(cache->k),
                             static_cast<const vk_tensor*>(cache->v),
                             static_cast<const vk_tensor*>(cache->k_scale),
                             static_cast<const vk_tensor*>(cache->v_scale), starts, counts,
                             ru.slopes, ru.prefix, ru.q_docs, ru.k_docs})
    VK_REQUIRE(!vk::overlap(out, t), "attention_cached: out overlaps an input");
  if (rows == 0) return VK_OK;

  const auto ints = [](const vk_tensor* t) {
    return t ? static_cast<const int*>(t->ptr) : nullptr;
  };
  Shape a;
  a.cache = vk::cache_args(cache);
  a.rows = vk::rows_args(starts, counts, cache->sequences, n, layout);
  a.rules.scale = scale;
  a.rules.cap = ru.cap;
  a.rules.slopes = ru.slopes ? static_cast<const float*>(ru.slopes->ptr) : nullptr;
  a.rules.prefix = ints(ru.prefix);
  a.rules.q_docs = ints(ru.q_docs);
  a.rules.k_docs = ints(ru.k_docs);
  a.rules.causal = ru.causal != 0;
  a.rules.docs_ordered = ru.docs_ordered != 0;
  a.heads = static_cast<uint32_t>(heads);
  a.group = static_cast<uint32_t>(heads / cache->heads);
  const size_t limit =
      max_length > 0 && max_length < cache->capacity ? max_length : cache->capacity;
  a.limit = static_cast<uint32_t>(limit);

  const auto* Q = static_cast<const float*>(q->ptr);
  auto* O = static_cast<float*>(out->ptr);
  const size_t blocks = (limit + KB - 1) / KB;
  const size_t pairs = cache->sequences * cache->heads;
  const size_t cus = rt->cu_count > 0 ? rt->cu_count : 256;
  const vk::CachedPlan plan = vk::cached_plan(cus, pairs, a.group * n, rows, blocks);
  const size_t tiles = (a.group * n + vk::kTileRows - 1) / vk::kTileRows;
  const size_t units = plan.form == vk::kTile ? pairs * tiles : pairs;
  const size_t splits = plan.splits;
  a.splits = static_cast<uint32_t>(splits);
  a.tiles = static_cast<uint32_t>(tiles);
  float* part = nullptr;
  if (splits > 1) {
    static_assert(vk::kCachedPart == HD + 4, "store_part's sums and store_ml's four");
    VK_TRY(vk::ensure_work(rt, splits * rows * vk::kCachedPart, "attention_cached"));
    part = rt->work;
  }
  // 8 / share groups of `heads` pairs each
  const uint32_t groups = pairs % 8 == 0 ? 8 : pairs % 4 == 0 ? 4 : pairs % 2 == 0 ? 2 : 1;
  a.order.share = 8 / groups;
  a.order.heads = static_cast<uint32_t>(pairs / groups);
  a.parts = a.rules.q_docs && !a.rules.docs_ordered ? 2 : 1;
  const size_t slots =
      (a.order.heads * tiles * splits * a.parts + a.order.share - 1) / a.order.share;
  const size_t wgs = plan.form == vk::kTile ? 8 * slots : units * splits;
  VK_UNSUPPORTED_IF(wgs * (plan.form == vk::kRow ? 64 * kRowWaves : 256) > 0xffffffffULL,
                    "attention_cached: %zu workgroups", wgs);
  const dim3 grid(static_cast<unsigned>(wgs));
  const bool q8 = cache->format == VK_CACHE_Q8;
  const int score = (ru.cap > 0.0f ? kCap : 0) | (ru.slopes ? kBias : 0);
  const bool mask = ru.causal || ru.q_docs;
#define VK_FORM(F, S, M)                                                                       \
  if (plan.form == vk::kFew)                                                                   \
    hipLaunchKernelGGL((attention_few_kernel<F, S, M>), grid, dim3(64 * kFewWaves), 0,         \
                       rt->stream, Q, O, part, a);                                             \
  else                                                                                         \
    hipLaunchKernelGGL((attention_tile_kernel<F, S, M, 4>), grid, dim3(256), 0, rt->stream, Q, \
                       O, part, a)
#define VK_RULE(F, S)                      \
  case S:                                  \
    if (mask) { VK_FORM(F, S, true); }     \
    else { VK_FORM(F, S, false); }         \
    break;
#define VK_RULES(F) \
  switch (score) { VK_RULE(F, 0) VK_RULE(F, kCap) VK_RULE(F, kBias) VK_RULE(F, (kCap | kBias)) }
  if (plan.form == vk::kRow) {
#define VK_ROW(F, P)                                                                        \
  hipLaunchKernelGGL((attention_row_kernel<F, P>), dim3(grid.x * P), dim3(64 * kRowWaves), 0, \
                     rt->stream, Q, O, part, a)
    const bool parts = splits == 1 && 4 * rows <= cus;  // where the card has the CUs
    if (q8) {
      if (parts) VK_ROW(VK_CACHE_Q8, 4);
      else VK_ROW(VK_CACHE_Q8, 1);
    } else {
      if (parts) VK_ROW(VK_CACHE_F8, 4);
      else VK_ROW(VK_CACHE_F8, 1);
    }
#undef VK_ROW
  } else if (q8) {
    VK_RULES(VK_CACHE_Q8)
  } else {
    VK_RULES(VK_CACHE_F8)
  }
#undef VK_RULES
#undef VK_RULE
#undef VK_FORM
  VK_TRY(vk::check_launch("attention_cached"));
  if (splits == 1) return VK_OK;
  const dim3 jgrid(static_cast<unsigned>((rows + 3) / 4));
#define VK_JOIN(N)                                                                          \
  hipLaunchKernelGGL(attention_join_kernel<N>, jgrid, dim3(256), 0, rt->stream, part, O, up, a)
  const float up = plan.form == vk::kRow ? kRowUp : 1.0f;
  if (splits <= 4) VK_JOIN(1);
  else if (splits <= 8) VK_JOIN(2);
  else if (splits <= 16) VK_JOIN(4);
  else if (splits <= 32) VK_JOIN(8);
  else VK_JOIN(16);
#undef VK_JOIN
  return vk::check_launch("attention_join_kernel");
}

}  // extern "C"
