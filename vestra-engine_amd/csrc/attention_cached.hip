// Attention over the 8-bit cache of K and V rows (kv_cache.h), with capped
// scores, a bias by distance, and causal, prefix and document masks.
//
// attention_row_kernel: a query a workgroup.  A lane takes a key, its 64 values
// and scores in F32, and keeps a softmax of its own (running maximum, sum and 64
// sums of values) over the keys that it meets; the lanes are joined once, at the
// end.
#include <cmath>

#include "kv_cache.h"

namespace {

constexpr int HD = 64;
constexpr float kLog2e = 1.44269504088896341f;

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
  uint32_t splits;
};

// Keys of sequence s: those of slots 0 .. keys_of - 1.
__device__ __forceinline__ int keys_of(const Shape& a, uint32_t s) {
  const int c = vkc::count_of(a.rows, s);
  if (c <= 0) return 0;
  long long end = static_cast<long long>(vkc::start_of(a.rows, s)) + c;
  end = end < static_cast<long long>(a.limit) ? end : static_cast<long long>(a.limit);
  return end > 0 ? static_cast<int>(end) : 0;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}

constexpr int kRowWaves = 4;
constexpr float kRoom = 4.0f;  // a lane's maximum follows scores that pass it by 2^kRoom

template <int FORMAT>
__global__ __launch_bounds__(64 * kRowWaves) void attention_row_kernel(const float* __restrict__ q,
                                                                       float* __restrict__ out,
                                                                       float* __restrict__ part,
                                                                       Shape a) {
  __shared__ float so[kRowWaves][HD];
  __shared__ float sm[kRowWaves], sl[kRowWaves];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t split = blockIdx.x % a.splits, row = blockIdx.x / a.splits;
  const uint32_t i = row % a.rows.n, sh = row / a.rows.n;
  const uint32_t h = sh % a.heads, s = sh / a.heads;
  if (static_cast<int>(i) >= vkc::count_of(a.rows, s)) return;
  const uint32_t kh = h / a.group;
  const int keys = keys_of(a, s);
  const long long p = static_cast<long long>(vkc::start_of(a.rows, s)) + i;
  const size_t first = (static_cast<size_t>(s) * a.cache.heads + kh) * a.cache.capacity;
  const float* qr = q + vkc::row_at(a.rows, a.heads, s, h, i);
  const Rules& ru = a.rules;
  const float slope = ru.slopes ? ru.slopes[h] : 0.0f;
  const int pre = ru.prefix ? ru.prefix[s] : 0;
  const int doc = ru.q_docs ? ru.q_docs[static_cast<size_t>(s) * a.rows.n + i] : 0;

  float m = -INFINITY, l = 0.0f, acc[HD];
#pragma unroll
  for (int d = 0; d < HD; ++d) acc[d] = 0.0f;
  const int blocks = (keys + 63) / 64;
  const int b0 = static_cast<int>(static_cast<long long>(split) * blocks / a.splits);
  const int b1 = static_cast<int>(static_cast<long long>(split + 1) * blocks / a.splits);
  for (int b = b0 + wave; b < b1; b += kRowWaves) {
    const int j = b * 64 + lane;
    bool seen = j < keys;
    if (ru.causal) seen = seen && (j <= p || j < pre);
    if (seen && ru.q_docs) {
      const int kd = ru.k_docs[static_cast<size_t>(s) * a.cache.capacity + j];
      seen = ru.docs_ordered ? kd <= doc : kd == doc;
    }
    if (!seen) continue;
    const size_t slot = first + j;
    float u[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint4* kc = reinterpret_cast<const uint4*>(a.cache.k + slot * HD);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint4 w = kc[c];
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4 x = vkc::decode4<FORMAT>(ws[e]);
        u[0] = __builtin_fmaf(qr[16 * c + 4 * e], x.x, u[0]);
        u[1] = __builtin_fmaf(qr[16 * c + 4 * e + 1], x.y, u[1]);
        u[2] = __builtin_fmaf(qr[16 * c + 4 * e + 2], x.z, u[2]);
        u[3] = __builtin_fmaf(qr[16 * c + 4 * e + 3], x.w, u[3]);
      }
    }
    float t = ((u[0] + u[1]) + (u[2] + u[3])) * a.cache.ks[slot] * ru.scale;
    if (ru.cap > 0.0f) t = ru.cap * tanhf(t / ru.cap);
    if (ru.slopes) {
      const long long far = p > j ? p - j : j - p;
      t -= slope * static_cast<float>(far);
    }
    t *= kLog2e;
    if (t == -INFINITY) continue;
    if (t > m + kRoom) {
      const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - t);
      l *= f;
#pragma unroll
      for (int d = 0; d < HD; ++d) acc[d] *= f;
      m = t;
    }
    const float w = __builtin_amdgcn_exp2f(t - m);
    l += w;
    const float wv = w * (a.cache.vs[slot] * 0x1p-24f);
    const uint4* vc = reinterpret_cast<const uint4*>(a.cache.v + slot * HD);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint4 x4 = vc[c];
      const uint32_t ws[4] = {x4.x, x4.y, x4.z, x4.w};
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
  // the wave: one maximum, the sums halved over the lanes, lane d left with d
  const float mw = wave_max(m);
  const float f = m == -INFINITY && l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - mw);
  l *= f;
#pragma unroll
  for (int d = 0; d < HD; ++d) acc[d] *= f;
#pragma unroll
  for (int w = 32; w; w >>= 1) {
    const bool up = (lane & w) != 0;
#pragma unroll
    for (int d = 0; d < w; ++d) {
      const float send = up ? acc[d] : acc[d + w];
      acc[d] = (up ? acc[d + w] : acc[d]) + __shfl_xor(send, w, 64);
    }
    l += __shfl_xor(l, w, 64);
  }
  so[wave][lane] = acc[0];
  if (lane == 0) {
    sm[wave] = mw;
    sl[wave] = l;
  }
  __syncthreads();
  if (wave != 0) return;
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
  if (part) {
    const size_t rows = static_cast<size_t>(a.rows.sequences) * a.heads * a.rows.n;
    const size_t at = static_cast<size_t>(split) * rows + row;
    part[at * HD + lane] = o;
    if (lane == 0)
      *reinterpret_cast<float2*>(part + a.splits * rows * HD + 2 * at) = make_float2(mg, lg);
  } else {
    out[vkc::row_at(a.rows, a.heads, s, h, i) + lane] = lg == 0.0f ? 0.0f : o / lg * 0x1p24f;
  }
}

// Joins the key splits of a row, in split order: 16 threads a row.
__global__ __launch_bounds__(256) void attention_join_kernel(const float* __restrict__ part,
                                                             float* __restrict__ out, float up,
                                                             Shape a) {
  const size_t idx = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  const size_t row = idx >> 4;
  const int c = static_cast<int>(idx & 15);
  const size_t rows = static_cast<size_t>(a.rows.sequences) * a.heads * a.rows.n;
  if (row >= rows) return;
  const uint32_t i = static_cast<uint32_t>(row % a.rows.n);
  const uint32_t sh = static_cast<uint32_t>(row / a.rows.n);
  const uint32_t h = sh % a.heads, s = sh / a.heads;
  if (static_cast<int>(i) >= vkc::count_of(a.rows, s)) return;
  const float2* ml = reinterpret_cast<const float2*>(part + a.splits * rows * HD);
  float m = -INFINITY;
  for (uint32_t sp = 0; sp < a.splits; ++sp) m = fmaxf(m, ml[sp * rows + row].x);
  float l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (uint32_t sp = 0; sp < a.splits; ++sp) {
    const float2 x = ml[sp * rows + row];
    const float w = x.x == -INFINITY && x.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(x.x - m);
    const float4 y = *reinterpret_cast<const float4*>(part + (sp * rows + row) * HD + 4 * c);
    l += x.y * w;
    o.x += y.x * w;
    o.y += y.y * w;
    o.z += y.z * w;
    o.w += y.w * w;
  }
  if (l == 0.0f)
    o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  else
    o = make_float4(o.x / l * up, o.y / l * up, o.z / l * up, o.w / l * up);
  *reinterpret_cast<float4*>(out + vkc::row_at(a.rows, a.heads, s, h, i) + 4 * c) = o;
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
  a.rules.scale = ru.scale == 0.0f ? 0.125f : ru.scale;
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

  const int cus = rt->cu_count > 0 ? rt->cu_count : 256;
  const size_t blocks = (limit + 63) / 64;
  size_t splits = 1;
  while (splits < 64 && rows * splits < 4 * static_cast<size_t>(cus) &&
         blocks / (2 * splits) >= 2 * kRowWaves)
    splits *= 2;
  VK_UNSUPPORTED_IF(rows * splits > 0x7fffffffULL, "attention_cached: %zu queries", rows);
  a.splits = static_cast<uint32_t>(splits);
  float* part = nullptr;
  if (splits > 1) {
    VK_TRY(vk::ensure_work(rt, splits * rows * (HD + 2), "attention_cached"));
    part = rt->work;
  }
  const auto* Q = static_cast<const float*>(q->ptr);
  auto* O = static_cast<float*>(out->ptr);
  const dim3 grid(static_cast<unsigned>(rows * splits));
  if (cache->format == VK_CACHE_Q8)
    hipLaunchKernelGGL(attention_row_kernel<VK_CACHE_Q8>, grid, dim3(64 * kRowWaves), 0, rt->stream,
                       Q, O, part, a);
  else
    hipLaunchKernelGGL(attention_row_kernel<VK_CACHE_F8>, grid, dim3(64 * kRowWaves), 0, rt->stream,
                       Q, O, part, a);
  VK_TRY(vk::check_launch("attention_row_kernel"));
  if (splits == 1) return VK_OK;
  hipLaunchKernelGGL(attention_join_kernel, dim3(static_cast<unsigned>((rows * 16 + 255) / 256)),
                     dim3(256), 0, rt->stream, part, O, 0x1p24f, a);
  return vk::check_launch("attention_join_kernel");
}

}  // extern "C"
