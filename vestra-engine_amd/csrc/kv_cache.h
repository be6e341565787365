// The 8-bit cache of K and V rows as its kernels see it: codes [sequences,
// heads, capacity, 64], one scale a row.
#pragma once

#include "common.h"

namespace vkc {

struct Cache {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  uint32_t heads, capacity;
};

// Rows of a call: row i < count of sequence s is slot start + i.
struct Rows {
  const int* starts;  // null: 0
  const int* counts;  // null: n
  uint32_t sequences, n;
  uint32_t outer;  // vk_qk_layout of the f32 side
};

__device__ __forceinline__ int start_of(const Rows& r, uint32_t s) {
  return r.starts ? r.starts[s] : 0;
}

__device__ __forceinline__ int count_of(const Rows& r, uint32_t s) {
  const int n = static_cast<int>(r.n);
  if (!r.counts) return n;
  const int c = r.counts[s];
  return c < n ? c : n;
}

// First element of (sequence s, head h, row i) on the f32 side, of `heads` heads.
__device__ __forceinline__ size_t row_at(const Rows& r, uint32_t heads, uint32_t s, uint32_t h,
                                         uint32_t i) {
  const size_t row =
      r.outer == VK_QK_HEADS_OUTER
          ? (static_cast<size_t>(h) * r.sequences + s) * r.n + i
          : (static_cast<size_t>(s) * heads + h) * r.n + i;
  return row * 64;
}

// A scale below this is held as 0 (its row as zeros): the attention takes the
// scales' inverses and products with weights, which stay normal numbers then.
constexpr float kLeastScale = 0x1p-100f;

// The four values of four codes.
template <int FORMAT>
__device__ __forceinline__ float4 decode4(uint32_t w) {
  if constexpr (FORMAT == VK_CACHE_Q8) {
    return make_float4(static_cast<float>(static_cast<int8_t>(w)),
                       static_cast<float>(static_cast<int8_t>(w >> 8)),
                       static_cast<float>(static_cast<int8_t>(w >> 16)),
                       static_cast<float>(static_cast<int8_t>(w >> 24)));
  } else {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    return make_float4(a[0], a[1], b[0], b[1]);
  }
}

}  // namespace vkc

namespace vk {
// VK_ERR_* unless the cache's tensors are of its sizes, aligned and on the
// runtime's device.
int check_cache(const vk_runtime* rt, const vk_kv_cache* c);
// The same for starts and counts (either may be null) of `sequences` i32.
int check_spans(const vk_runtime* rt, const vk_tensor* starts, const vk_tensor* counts,
                size_t sequences);
inline vkc::Cache cache_args(const vk_kv_cache* c) {
  return vkc::Cache{static_cast<uint8_t*>(c->k->ptr), static_cast<uint8_t*>(c->v->ptr),
                    static_cast<float*>(c->k_scale->ptr), static_cast<float*>(c->v_scale->ptr),
                    static_cast<uint32_t>(c->heads), static_cast<uint32_t>(c->capacity)};
}
inline vkc::Rows rows_args(const vk_tensor* starts, const vk_tensor* counts, size_t sequences,
                           size_t n, vk_qk_layout layout) {
  return vkc::Rows{starts ? static_cast<const int*>(starts->ptr) : nullptr,
                   counts ? static_cast<const int*>(counts->ptr) : nullptr,
                   static_cast<uint32_t>(sequences), static_cast<uint32_t>(n),
                   static_cast<uint32_t>(layout)};
}
}  // namespace vk
