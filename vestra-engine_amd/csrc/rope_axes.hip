// Q/K LayerNorm and rotary positions of several axes (time, height, width).
//
// A row of 64 values is 32 pairs; pair j belongs to an axis and turns by
// position[axis] * f_j: (u, w) -> (u cos - w sin, w cos + u sin).  Where the
// pairs lie in the row and which axis each takes is a table of 64 entries that
// the host makes from vk_rope_axes, so one kernel serves every convention.
//
// A row is one float4 a lane of a 16-lane DPP row; a 16-lane group takes
// kHeads heads of one token, so the cosines and sines of the token are worked
// out once for them.  A lane's partners of its four elements
// lie wherever the convention puts them: the normalised row goes through LDS (a
// row is its group's alone: no barrier, the lanes of a wave are in step).
//
// Bound by HBM for many tokens (10,392 of 24 heads: 24.2 us, 5.3 TB/s, of a copy's 5.0) and by
// the chain of loads (table, position, angle) for few (866: 4.0 us in a graph).  In the
// sequential LayerNorm order by its two chains of 64 sums: 30.5 and 5.1 us.
//
// The angle: turns = position * f_j / (2 pi) in 64 bits, reduced there to an
// eighth of a turn either side of a quarter, then single precision; a position
// of 2^31 is held to 2^-22 of a turn.
#include <cmath>
#include <cstring>

#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kGroups = kThreads / 16;  // tokens of a workgroup
// Rows of a group.  866 tokens of 24 heads: 4.1 us; 4.7 with four rows (half the
// workgroups), 5.3 with one (a token's angles for one row).  10,392: 24.2, 24.7, 34.
constexpr int kHeads = 2;
constexpr int kPitch = 68;              // floats of a row in LDS

struct alignas(16) AxesTable {
  double turns[64];     // f / (2 pi) of the element's pair
  uint8_t axis[64];     // its axis
  uint8_t partner[64];  // the pair's other element
  uint8_t second[64];   // 1: the element is the pair's second
};

struct AxesShape {
  uint32_t heads, kv_heads, n, axes, eps_bits;
  uint32_t rows;   // sequences * n
  uint32_t outer;  // vk_qk_layout
  vkd::FastDivU32 by_n;
};

// 1 / std of a row from the sum of its squared deviations, as each LayerNorm
// order of the Q/K rows takes it.
template <bool SEQ>
__device__ __forceinline__ float row_inv(float q, float eps) {
  const float var = q / 64.0f;
  return SEQ ? 1.0f / sqrtf(var + eps) : __builtin_amdgcn_rsqf(var + eps);
}

// A row's 64 values left to right, from LDS.
__device__ __forceinline__ float row_chain(const float* r) {
  float s = 0.0f;
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    const float4 w = reinterpret_cast<const float4*>(r)[c];
    s += w.x;
    s += w.y;
    s += w.z;
    s += w.w;
  }
  return s;
}

template <typename PT, typename POS, bool NORM, bool SEQ>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_axes_kernel(
    const float* q, const float* k, float* q_out, float* k_out, const PT* __restrict__ qg,
    const PT* __restrict__ qb, const PT* __restrict__ kg, const PT* __restrict__ kb,
    const void* __restrict__ pos, AxesTable tab, AxesShape sh) {
  __shared__ __align__(16) float lds[kGroups * kHeads * kPitch];
  const int l = threadIdx.x & 15, grp = threadIdx.x >> 4;
  float* mine = lds + grp * kHeads * kPitch;
  const uint32_t token = blockIdx.x * kGroups + grp;
  // groups past the last token work on it and store nothing
  const bool live = token < sh.rows;
  const uint32_t t = live ? token : sh.rows - 1;
  const uint32_t s = vkd::fdiv(t, sh.by_n), i = t - s * sh.n;
  const uint32_t all = sh.heads + sh.kv_heads;
  const uint32_t h = blockIdx.y * kHeads;  // the first head: of Q, then of K
  const float eps = __uint_as_float(sh.eps_bits);
  // first element of head h's row of this token
  auto row = [&](uint32_t h, uint32_t count) {
    const size_t r = sh.outer == VK_QK_HEADS_OUTER
                         ? static_cast<size_t>(h) * sh.rows + t
                         : (static_cast<size_t>(s) * count + h) * sh.n + i;
    return r * 64 + 4 * l;
  };
  auto at = [&](uint32_t h) -> size_t {
    return h < sh.heads ? row(h, sh.heads) : row(h - sh.heads, sh.kv_heads);
  };

  // the table's and the positions' loads first: the angles hang on both, one after the other
  float c[4], sn[4];
  const uint32_t axis4 = reinterpret_cast<const uint32_t*>(tab.axis)[l];
  const uint32_t partner4 = reinterpret_cast<const uint32_t*>(tab.partner)[l];
  const uint32_t second4 = reinterpret_cast<const uint32_t*>(tab.second)[l];
  double f[4];
  POS at_axis[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[e] = tab.turns[4 * l + e];
    at_axis[e] = static_cast<const POS*>(pos)[static_cast<size_t>(t) * sh.axes +
                                              (axis4 >> 8 * e & 0xff)];
  }
  float4 v[kHeads];
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    const uint32_t hh = h + j < all ? h + j : all - 1;
    v[j] = vkd::ld_stream(
        reinterpret_cast<const float4*>((hh < sh.heads ? q : k) + at(hh)));
  }
  // while the rows are on their way
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const double turns = static_cast<double>(at_axis[e]) * f[e];
    const double quarter = rint(4.0 * turns);
    const float r = static_cast<float>(turns - 0.25 * quarter);  // within 1/8
    float sr, cr;
    sincospif(2.0f * r, &sr, &cr);
    const int quad = static_cast<int>(quarter - 4.0 * floor(0.25 * quarter));
    float ca = quad & 1 ? sr : cr, sa = quad & 1 ? cr : sr;
    if (quad == 1 || quad == 2) ca = -ca;
    if (quad >= 2) sa = -sa;
    c[e] = ca;
    sn[e] = second4 >> 8 * e & 1 ? sa : -sa;
  }
  if constexpr (NORM) {
    float mean[kHeads], inv[kHeads];
    if constexpr (SEQ) {
#pragma unroll
      for (int j = 0; j < kHeads; ++j) *reinterpret_cast<float4*>(mine + j * kPitch + 4 * l) = v[j];
      vkd::wave_lds_fence();
      float st = l < kHeads ? row_chain(mine + l * kPitch) / 64.0f : 0.0f;
      vkd::wave_lds_fence();
#pragma unroll
      for (int j = 0; j < kHeads; ++j) {
        mean[j] = __shfl(st, j, 16);
        float4 d;
        d.x = v[j].x - mean[j]; d.x = d.x * d.x;
        d.y = v[j].y - mean[j]; d.y = d.y * d.y;
        d.z = v[j].z - mean[j]; d.z = d.z * d.z;
        d.w = v[j].w - mean[j]; d.w = d.w * d.w;
        *reinterpret_cast<float4*>(mine + j * kPitch + 4 * l) = d;
      }
      vkd::wave_lds_fence();
      st = l < kHeads ? row_inv<true>(row_chain(mine + l * kPitch), eps) : 0.0f;
      vkd::wave_lds_fence();
#pragma unroll
      for (int j = 0; j < kHeads; ++j) inv[j] = __shfl(st, j, 16);
    } else {
#pragma unroll
      for (int j = 0; j < kHeads; ++j) {
        float a = v[j].x;
        a += v[j].y;
        a += v[j].z;
        a += v[j].w;
        mean[j] = vkd::row16_sum(a) / 64.0f;
        float d, sq;
        d = v[j].x - mean[j]; sq = d * d;
        d = v[j].y - mean[j]; sq += d * d;
        d = v[j].z - mean[j]; sq += d * d;
        d = v[j].w - mean[j]; sq += d * d;
        inv[j] = row_inv<false>(vkd::row16_sum(sq), eps);
      }
    }
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const bool is_q = (h + j < all ? h + j : all - 1) < sh.heads;
      const float4 g = vkd::Param<PT>::load4(is_q ? qg : kg, l);
      const float4 b = vkd::Param<PT>::load4(is_q ? qb : kb, l);
      v[j] = vkd::ln_apply4(v[j], mean[j], inv[j], g, b);
    }
  }
#pragma unroll
  for (int j = 0; j < kHeads; ++j) *reinterpret_cast<float4*>(mine + j * kPitch + 4 * l) = v[j];
  vkd::wave_lds_fence();
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    const float* r = mine + j * kPitch;
    float4 o;
    o.x = v[j].x * c[0] + r[partner4 >> 0 & 0xff] * sn[0];
    o.y = v[j].y * c[1] + r[partner4 >> 8 & 0xff] * sn[1];
    o.z = v[j].z * c[2] + r[partner4 >> 16 & 0xff] * sn[2];
    o.w = v[j].w * c[3] + r[partner4 >> 24 & 0xff] * sn[3];
    v[j] = o;
  }
#pragma unroll
  for (int j = 0; j < kHeads; ++j)
    if (live && h + j < all)
      vkd::st_stream(reinterpret_cast<float4*>((h + j < sh.heads ? q_out : k_out) + at(h + j)),
                     v[j]);
}

// The host's table: vk_rope_axes laid out element by element.
AxesTable make_table(const vk_rope_axes& a) {
  AxesTable t;
  const bool inter = (a.mode & VK_ROPE_INTERLEAVED) != 0;
  const bool sections = (a.mode & VK_ROPE_SECTIONS) != 0;
  const bool head = sections || (a.mode & VK_ROPE_EXP_HEAD) != 0;
  unsigned pair = 0;
  for (size_t ax = 0; ax < a.count; ++ax) {
    const unsigned first = pair;
    for (unsigned i = 0; i < a.pairs[ax]; ++i, ++pair) {
      const unsigned in = sections ? pair : i;           // index among its pairs
      const unsigned half = sections ? 32 : a.pairs[ax];  // pairs there
      const unsigned base = sections ? 0 : 2 * first;
      const unsigned e0 = base + (inter ? 2 * in : in), e1 = inter ? e0 + 1 : e0 + half;
      const double f = std::pow(static_cast<double>(a.freq),
                                -2.0 * in / (head ? 64.0 : 2.0 * half));
      for (const unsigned e : {e0, e1}) {
        t.turns[e] = f / 6.283185307179586476925286766559;
        t.axis[e] = static_cast<uint8_t>(ax);
        t.partner[e] = static_cast<uint8_t>(e == e0 ? e1 : e0);
        t.second[e] = e == e1;
      }
    }
  }
  return t;
}

struct Launch {
  vk_runtime* rt;
  dim3 grid;
  const float *q, *k;
  float *q_out, *k_out;
  const vk_tensor *qg, *qb, *kg, *kb;
  const void* pos;
  AxesTable table;
  AxesShape shape;
};

const void* ptr(const vk_tensor* t) { return t ? t->ptr : nullptr; }

template <typename PT, typename POS, bool NORM, bool SEQ>
int launch(const Launch& a) {
  hipLaunchKernelGGL((qk_norm_rope_axes_kernel<PT, POS, NORM, SEQ>), a.grid, dim3(kThreads), 0,
                     a.rt->stream, a.q, a.k, a.q_out, a.k_out, static_cast<const PT*>(ptr(a.qg)),
                     static_cast<const PT*>(ptr(a.qb)), static_cast<const PT*>(ptr(a.kg)),
                     static_cast<const PT*>(ptr(a.kb)), a.pos, a.table, a.shape);
  return vk::check_launch("qk_norm_rope_axes_kernel");
}

template <typename POS>
int dispatch(const Launch& a) {
  if (!a.qg) return launch<float, POS, false, false>(a);
  const bool seq = a.rt->ln_order == VK_LN_ORDER_SEQUENTIAL;
  if (a.qg->dtype == VK_F16)
    return seq ? launch<uint16_t, POS, true, true>(a) : launch<uint16_t, POS, true, false>(a);
  return seq ? launch<float, POS, true, true>(a) : launch<float, POS, true, false>(a);
}

int check_param(const vk_runtime* rt, const vk_tensor* t, const vk_tensor* like, const char* what) {
  VK_REQUIRE(t && t->len == 64 && (t->dtype == VK_F32 || t->dtype == VK_F16),
             "qk_norm_rope_axes: %s must be f32 or f16 [64]", what);
  VK_REQUIRE(t->dtype == like->dtype, "qk_norm_rope_axes: norm parameters must share one dtype");
  VK_REQUIRE(reinterpret_cast<uintptr_t>(t->ptr) % 16 == 0,
             "qk_norm_rope_axes: %s must be 16-byte aligned", what);
  return vk::check_device(rt, t, what);
}

}  // namespace

extern "C" {

int vk_qk_norm_rope_axes_f32(vk_runtime* rt, const vk_tensor* q, const vk_tensor* k,
                             const vk_tensor* q_gamma, const vk_tensor* q_beta,
                             const vk_tensor* k_gamma, const vk_tensor* k_beta,
                             const vk_tensor* positions, size_t sequences, size_t heads,
                             size_t kv_heads, size_t n, size_t head_dim, const vk_rope_axes* axes,
                             vk_qk_layout layout, float eps, vk_tensor* q_out, vk_tensor* k_out) {
  VK_TRY(vk::bind(rt));
  VK_REQUIRE(q && q_out && positions && axes, "null argument");
  VK_REQUIRE((k != nullptr) == (k_out != nullptr) && (k != nullptr) == (kv_heads > 0),
             "qk_norm_rope_axes: k, k_out and kv_heads go together");
  VK_UNSUPPORTED_IF(head_dim != 64, "qk_norm_rope_axes: head_dim=%zu (qualified: 64)", head_dim);
  VK_REQUIRE(layout == VK_QK_HEADS_OUTER || layout == VK_QK_VIEWS_OUTER, "unknown layout %d",
             static_cast<int>(layout));
  VK_REQUIRE(axes->count >= 1 && axes->count <= VK_ROPE_MAX_AXES,
             "qk_norm_rope_axes: %zu axes (1 to %d)", axes->count, VK_ROPE_MAX_AXES);
  VK_REQUIRE((axes->mode & ~(VK_ROPE_INTERLEAVED | VK_ROPE_EXP_HEAD | VK_ROPE_SECTIONS)) == 0,
             "unknown RoPE convention flags 0x%x", axes->mode);
  VK_REQUIRE(std::isfinite(axes->freq) && axes->freq > 0.0f,
             "qk_norm_rope_axes: frequency base %g", static_cast<double>(axes->freq));
  unsigned long long pairs = 0;
  for (size_t a = 0; a < axes->count; ++a) pairs += axes->pairs[a];
  VK_REQUIRE(pairs == 32, "qk_norm_rope_axes: the axes have %llu pairs (32)", pairs);
  VK_REQUIRE(heads > 0, "qk_norm_rope_axes: no heads");
  VK_UNSUPPORTED_IF(sequences > 0x7fffffffULL || n > 0x7fffffffULL || heads > 0xffff ||
                        kv_heads > 0xffff || sequences * n > 0xffffff0ULL,
                    "qk_norm_rope_axes: too large");  // 16 threads a token, 2^32 a launch
  const size_t rows = sequences * n;
  VK_TRY(vk::check_f32(rt, q, heads * rows * 64, "q"));
  VK_TRY(vk::check_f32(rt, q_out, heads * rows * 64, "q_out"));
  if (k) {
    VK_TRY(vk::check_f32(rt, k, kv_heads * rows * 64, "k"));
    VK_TRY(vk::check_f32(rt, k_out, kv_heads * rows * 64, "k_out"));
  }
  VK_REQUIRE(positions->dtype == VK_F32 || positions->dtype == VK_I32 || positions->dtype == VK_I64,
             "positions must be f32, i32 or i64");
  VK_REQUIRE(positions->len == rows * axes->count,
             "positions must hold rows*axes = %zu (got %zu)", rows * axes->count, positions->len);
  VK_TRY(vk::check_device(rt, positions, "positions"));
  const bool any = q_gamma || q_beta || k_gamma || k_beta;
  if (any) {
    VK_REQUIRE(q_gamma, "q/k norm parameters must be all present or all null");
    VK_TRY(check_param(rt, q_gamma, q_gamma, "q_gamma"));
    VK_TRY(check_param(rt, q_beta, q_gamma, "q_beta"));
    if (k) {
      VK_TRY(check_param(rt, k_gamma, q_gamma, "k_gamma"));
      VK_TRY(check_param(rt, k_beta, q_gamma, "k_beta"));
    }
  }
  // each output in place of its own input, or apart from everything
  const vk_tensor* all_t[] = {q, k, q_out, k_out, positions, q_gamma, q_beta, k_gamma, k_beta};
  for (int o = 2; o < 4; ++o)
    for (int t = 0; t < 9; ++t) {
      const bool in_place = t == o - 2 && all_t[o] && all_t[t]->ptr == all_t[o]->ptr;
      VK_REQUIRE(t == o || in_place || !vk::overlap(all_t[o], all_t[t]),
                 "qk_norm_rope_axes: an output overlaps another tensor");
    }
  if (rows == 0) return VK_OK;
  Launch a;
  a.rt = rt;
  a.q = static_cast<const float*>(q->ptr);
  a.k = static_cast<const float*>(ptr(k));
  a.q_out = static_cast<float*>(q_out->ptr);
  a.k_out = k_out ? static_cast<float*>(k_out->ptr) : nullptr;
  a.qg = q_gamma;
  a.qb = q_beta;
  a.kg = k_gamma;
  a.kb = k_beta;
  a.pos = positions->ptr;
  a.table = make_table(*axes);
  AxesShape& sh = a.shape;
  sh.heads = static_cast<uint32_t>(heads);
  sh.kv_heads = static_cast<uint32_t>(kv_heads);
  sh.n = static_cast<uint32_t>(n);
  sh.rows = static_cast<uint32_t>(rows);
  sh.axes = static_cast<uint32_t>(axes->count);
  sh.outer = static_cast<uint32_t>(layout);
  sh.by_n = vkd::make_fastdiv(static_cast<uint32_t>(n));
  memcpy(&sh.eps_bits, &eps, sizeof eps);
  const size_t all = heads + kv_heads;
  a.grid = dim3(static_cast<unsigned>((rows + kGroups - 1) / kGroups),
                static_cast<unsigned>((all + kHeads - 1) / kHeads));
  switch (positions->dtype) {
    case VK_I32: return dispatch<int32_t>(a);
    case VK_I64: return dispatch<int64_t>(a);
    default: return dispatch<float>(a);
  }
}

}  // extern "C"
