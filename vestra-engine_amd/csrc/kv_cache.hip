// A cache of K and V rows in 8 bits a value: quantised as it is written, and
// read back to f32.
//
// A row of 64 is one float4 a lane of a 16-lane DPP row, a K row and the V row
// of the same token to a group.  The scale is the row's largest |x| / 127 (448),
// a code the quotient rounded to f32 and then to the code: both divisions are
// the correctly rounded ones, so a program that quantises on the host gets the
// same codes.  Streams of one pass, bound by HBM from some hundred thousand rows on
// (12 heads of 10,392 read back: 13.5 us, 6.0 TB/s; 16 x 8 x 866 written 14.5, 5.0 TB/s) and by
// the launch and one chain of loads below (10,392 rows: written 3.8 us, read 2.9, in a graph).
#include "kv_cache.h"

namespace {

constexpr int kThreads = 256;
constexpr int kGroups = kThreads / 16;

// Largest of a 16-lane row, as unsigned bits: of |x|, a NaN is above an
// infinity is above every number.
__device__ __forceinline__ uint32_t row16_umax(uint32_t v) {
#define VK_ROR(n)                                                                            \
  {                                                                                          \
    const uint32_t o = static_cast<uint32_t>(                                                \
        __builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x120 | n, 0xf, 0xf, true));           \
    v = o > v ? o : v;                                                                       \
  }
  VK_ROR(8) VK_ROR(4) VK_ROR(2) VK_ROR(1)
#undef VK_ROR
  return v;
}

__device__ __forceinline__ uint32_t bits_abs(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Four codes (little-endian) of a lane and the row's scale.
template <int FORMAT>
__device__ __forceinline__ uint32_t quantise(const float4& x, float* scale) {
  constexpr float kTop = FORMAT == VK_CACHE_Q8 ? 127.0f : 448.0f;
  constexpr float kMost = FORMAT == VK_CACHE_Q8 ? 0x1.020406p+121f : 0x1.249248p+119f;
  uint32_t m = bits_abs(x.x);
  m = max(m, bits_abs(x.y));
  m = max(m, bits_abs(x.z));
  m = row16_umax(max(m, bits_abs(x.w)));
  // (at most the scale whose largest code is still finite)
  float d = fminf(__uint_as_float(m) / kTop, kMost);
  const bool odd = m >= 0x7f800000u;  // an infinity or a NaN
  const bool none = odd || d < vkc::kLeastScale;
  const float by = none ? 1.0f : d;
  *scale = odd ? __uint_as_float(0x7fc00000u) : (none ? 0.0f : d);
  const float a = x.x / by, b = x.y / by, c = x.z / by, e = x.w / by;
  uint32_t w;
  if constexpr (FORMAT == VK_CACHE_Q8) {
    const auto code = [](float y) { return static_cast<uint32_t>(static_cast<int>(rintf(y))) & 0xffu; };
    w = none ? 0u : code(a) | code(b) << 8 | code(c) << 16 | code(e) << 24;
  } else {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(c, e, p, true);
    w = none ? 0u : static_cast<uint32_t>(p);
  }
  return w;
}

// Row group -> (sequence, head, row), rows innermost.
struct Split {
  vkd::FastDivU32 by_n, by_heads;
  uint32_t groups;
};

__device__ __forceinline__ uint32_t group_id() {
  return (blockIdx.y * gridDim.x + blockIdx.x) * kGroups + (threadIdx.x >> 4);
}

__device__ __forceinline__ bool place(const Split& sp, const vkc::Rows& r, const vkc::Cache& c,
                                      uint32_t g, size_t* f32_at, size_t* slot) {
  if (g >= sp.groups) return false;
  const uint32_t sh = vkd::fdiv(g, sp.by_n), i = g - sh * r.n;
  const uint32_t s = vkd::fdiv(sh, sp.by_heads), h = sh - s * c.heads;
  const int count = vkc::count_of(r, s), start = vkc::start_of(r, s);  // one wait for both
  const long long at = static_cast<long long>(start) + i;
  if (static_cast<int>(i) >= count || at < 0 || at >= static_cast<long long>(c.capacity))
    return false;
  *f32_at = vkc::row_at(r, c.heads, s, h, i);
  *slot = (static_cast<size_t>(s) * c.heads + h) * c.capacity + static_cast<size_t>(at);
  return true;
}

template <int FORMAT>
__global__ __launch_bounds__(kThreads) void kv_cache_write_kernel(const float* __restrict__ k,
                                                                  const float* __restrict__ v,
                                                                  vkc::Cache c, vkc::Rows r,
                                                                  Split sp) {
  const int l = threadIdx.x & 15;
  size_t from, slot;
  if (!place(sp, r, c, group_id(), &from, &slot)) return;
  const float4 a = vkd::ld_stream(reinterpret_cast<const float4*>(k + from) + l);
  const float4 b = vkd::ld_stream(reinterpret_cast<const float4*>(v + from) + l);
  float da, db;
  const uint32_t wa = quantise<FORMAT>(a, &da), wb = quantise<FORMAT>(b, &db);
  reinterpret_cast<uint32_t*>(c.k + slot * 64)[l] = wa;
  reinterpret_cast<uint32_t*>(c.v + slot * 64)[l] = wb;
  if (l == 0) {
    c.ks[slot] = da;
    c.vs[slot] = db;
  }
}

template <int FORMAT>
__device__ __forceinline__ float4 values(uint32_t w, float d) {
  const float4 x = vkc::decode4<FORMAT>(w);
  return make_float4(x.x * d, x.y * d, x.z * d, x.w * d);
}

template <int FORMAT>
__global__ __launch_bounds__(kThreads) void kv_cache_read_kernel(float* __restrict__ k,
                                                                 float* __restrict__ v,
                                                                 vkc::Cache c, vkc::Rows r,
                                                                 Split sp) {
  const int l = threadIdx.x & 15;
  size_t to, slot;
  if (!place(sp, r, c, group_id(), &to, &slot)) return;
  uint32_t wa = 0, wb = 0;
  float da = 0.0f, db = 0.0f;
  if (k) {
    wa = reinterpret_cast<const uint32_t*>(c.k + slot * 64)[l];
    da = c.ks[slot];
  }
  if (v) {
    wb = reinterpret_cast<const uint32_t*>(c.v + slot * 64)[l];
    db = c.vs[slot];
  }
  if (k) vkd::st_stream(reinterpret_cast<float4*>(k + to) + l, values<FORMAT>(wa, da));
  if (v) vkd::st_stream(reinterpret_cast<float4*>(v + to) + l, values<FORMAT>(wb, db));
}

int make_split(const vk_kv_cache* c, size_t n, Split* sp) {
  const size_t groups = c->sequences * c->heads * n;
  VK_UNSUPPORTED_IF(groups > 0x7fffffffULL, "kv_cache: %zu rows", groups);
  sp->by_n = vkd::make_fastdiv(static_cast<uint32_t>(n));
  sp->by_heads = vkd::make_fastdiv(static_cast<uint32_t>(c->heads));
  sp->groups = static_cast<uint32_t>(groups);
  return VK_OK;
}

// 2^20 workgroups a row of the grid: a launch holds at most 2^32 threads a dimension.
dim3 make_grid(const Split& sp) {
  const uint32_t wgs = (sp.groups + kGroups - 1) / kGroups, x = wgs < (1u << 20) ? wgs : 1u << 20;
  return dim3(x, (wgs + x - 1) / x);
}

int check_rows(const vk_kv_cache* c, size_t n, vk_qk_layout layout) {
  VK_REQUIRE(layout == VK_QK_HEADS_OUTER || layout == VK_QK_VIEWS_OUTER, "unknown layout %d",
             static_cast<int>(layout));
  VK_UNSUPPORTED_IF(n > 0x7fffffffULL, "kv_cache: %zu rows a sequence", n);
  VK_UNSUPPORTED_IF(n > 0 && c->sequences * c->heads > 0x7fffffffULL / n,
                    "kv_cache: %zu x %zu x %zu rows", c->sequences, c->heads, n);
  return VK_OK;
}

}  // namespace

namespace vk {

int check_cache(const vk_runtime* rt, const vk_kv_cache* c) {
  VK_REQUIRE(c, "null cache");
  VK_UNSUPPORTED_IF(c->head_dim != 64, "kv_cache: head_dim=%zu (qualified: 64)", c->head_dim);
  VK_REQUIRE(c->format == VK_CACHE_Q8 || c->format == VK_CACHE_F8, "kv_cache: unknown format %d",
             c->format);
  VK_REQUIRE(c->heads > 0, "kv_cache: no heads");
  VK_UNSUPPORTED_IF(c->capacity > 0x7fff0000ULL || c->sequences > 0xffffff || c->heads > 0xffff,
                    "kv_cache: %zu sequences of %zu heads and %zu slots", c->sequences, c->heads,
                    c->capacity);
  VK_UNSUPPORTED_IF(c->capacity > 0 && c->sequences * c->heads > (size_t{1} << 48) / c->capacity,
                    "kv_cache: %zu x %zu x %zu rows", c->sequences, c->heads, c->capacity);
  const size_t rows = c->sequences * c->heads * c->capacity;
  const vk_tensor* t[] = {c->k, c->v, c->k_scale, c->v_scale};
  static const char* const name[] = {"cache k", "cache v", "cache k_scale", "cache v_scale"};
  for (int i = 0; i < 4; ++i) {
    const vk_dtype want = i < 2 ? VK_U8 : VK_F32;
    const size_t len = i < 2 ? rows * 64 : rows;
    VK_REQUIRE(t[i] && t[i]->dtype == want && t[i]->len == len, "%s must be %s [%zu] (holds %zu)",
               name[i], i < 2 ? "u8" : "f32", len, t[i] ? t[i]->len : 0);
    VK_REQUIRE(reinterpret_cast<uintptr_t>(t[i]->ptr) % 16 == 0, "%s must be 16-byte aligned",
               name[i]);
    VK_TRY(check_device(rt, t[i], name[i]));
    for (int j = 0; j < i; ++j)
      VK_REQUIRE(!overlap(t[i], t[j]), "%s overlaps %s", name[i], name[j]);
  }
  return VK_OK;
}

int check_spans(const vk_runtime* rt, const vk_tensor* starts, const vk_tensor* counts,
                size_t sequences) {
  const vk_tensor* t[] = {starts, counts};
  for (int i = 0; i < 2; ++i) {
    if (!t[i]) continue;
    const char* what = i ? "counts" : "starts";
    VK_REQUIRE(t[i]->dtype == VK_I32 && t[i]->len == sequences, "%s must be i32 [%zu] (holds %zu)",
               what, sequences, t[i]->len);
    VK_TRY(check_device(rt, t[i], what));
  }
  return VK_OK;
}

}  // namespace vk

extern "C" {

int vk_kv_cache_write_f32(vk_runtime* rt, const vk_kv_cache* cache, const vk_tensor* k,
                          const vk_tensor* v, size_t n, const vk_tensor* starts,
                          const vk_tensor* counts, vk_qk_layout layout) {
  VK_TRY(vk::bind(rt));
  VK_TRY(vk::check_cache(rt, cache));
  VK_TRY(check_rows(cache, n, layout));
  const size_t len = cache->sequences * cache->heads * n * 64;
  VK_TRY(vk::check_f32(rt, k, len, "k"));
  VK_TRY(vk::check_f32(rt, v, len, "v"));
  VK_TRY(vk::check_spans(rt, starts, counts, cache->sequences));
  for (const vk_tensor* out : {cache->k, cache->v, cache->k_scale, cache->v_scale})
    for (const vk_tensor* t : {k, v, starts, counts})
      VK_REQUIRE(!vk::overlap(out, t), "kv_cache: the cache overlaps an input");
  if (len == 0 || cache->capacity == 0) return VK_OK;
  Split sp;
  VK_TRY(make_split(cache, n, &sp));
  const dim3 grid = make_grid(sp);
  const auto* K = static_cast<const float*>(k->ptr);
  const auto* V = static_cast<const float*>(v->ptr);
  const vkc::Cache c = vk::cache_args(cache);
  const vkc::Rows r = vk::rows_args(starts, counts, cache->sequences, n, layout);
  if (cache->format == VK_CACHE_Q8)
    hipLaunchKernelGGL(kv_cache_write_kernel<VK_CACHE_Q8>, grid, dim3(kThreads), 0, rt->stream, K,
                       V, c, r, sp);
  else
    hipLaunchKernelGGL(kv_cache_write_kernel<VK_CACHE_F8>, grid, dim3(kThreads), 0, rt->stream, K,
                       V, c, r, sp);
  return vk::check_launch("kv_cache_write_kernel");
}

int vk_kv_cache_read_f32(vk_runtime* rt, const vk_kv_cache* cache, size_t n,
                         const vk_tensor* starts, const vk_tensor* counts, vk_tensor* k,
                         vk_tensor* v, vk_qk_layout layout) {
  VK_TRY(vk::bind(rt));
  VK_TRY(vk::check_cache(rt, cache));
  VK_TRY(check_rows(cache, n, layout));
  VK_REQUIRE(k || v, "kv_cache: neither k nor v to read");
  const size_t len = cache->sequences * cache->heads * n * 64;
  if (k) VK_TRY(vk::check_f32(rt, k, len, "k"));
  if (v) VK_TRY(vk::check_f32(rt, v, len, "v"));
  VK_TRY(vk::check_spans(rt, starts, counts, cache->sequences));
  VK_REQUIRE(!vk::overlap(k, v), "kv_cache: k overlaps v");
  for (const vk_tensor* out : {k, v})
    for (const vk_tensor* t : {static_cast<const vk_tensor*>(cache->k),
                               static_cast<const vk_tensor*>(cache->v),
                               static_cast<const vk_tensor*>(cache->k_scale),
                               static_cast<const vk_tensor*>(cache->v_scale), starts, counts})
      VK_REQUIRE(!vk::overlap(out, t), "kv_cache: an output overlaps an input");
  if (len == 0 || cache->capacity == 0) return VK_OK;
  Split sp;
  VK_TRY(make_split(cache, n, &sp));
  const dim3 grid = make_grid(sp);
  float* K = k ? static_cast<float*>(k->ptr) : nullptr;
  float* V = v ? static_cast<float*>(v->ptr) : nullptr;
  const vkc::Cache c = vk::cache_args(cache);
  const vkc::Rows r = vk::rows_args(starts, counts, cache->sequences, n, layout);
  if (cache->format == VK_CACHE_Q8)
    hipLaunchKernelGGL(kv_cache_read_kernel<VK_CACHE_Q8>, grid, dim3(kThreads), 0, rt->stream, K, V,
                       c, r, sp);
  else
    hipLaunchKernelGGL(kv_cache_read_kernel<VK_CACHE_F8>, grid, dim3(kThreads), 0, rt->stream, K, V,
                       c, r, sp);
  return vk::check_launch("kv_cache_read_kernel");
}

}  // extern "C"
