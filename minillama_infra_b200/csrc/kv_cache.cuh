// kv_cache.cuh -- what the paged key-value cache's kernels share: element
// types, the cache as kernels see it, and the checks of a caller's struct.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mli_common.cuh"
#include "mli_internal.h"

namespace mli {

constexpr int kMaxHeadDim = 256;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// One layer of a cache.
template <typename T>
struct CacheLayer {
  T* k;
  T* v;
  long long page_stride, head_stride, slot_stride;
  int pages, page_size, kv_heads, head_dim;
};

template <typename T>
CacheLayer<T> cache_layer(const mli_kv_cache& c, int layer) {
  const long long off = c.layer_stride * layer;
  return CacheLayer<T>{static_cast<T*>(c.k) + off, static_cast<T*>(c.v) + off, c.page_stride, c.head_stride,
                       c.slot_stride, c.pages, c.page_size, c.kv_heads, c.head_dim};
}

inline int cache_element_bytes(int dtype) { return dtype == MLI_KV_F32 ? 4 : 2; }

// The status of a caller's cache struct (MLI_OK: every kernel can use it).
inline int check_cache(const mli_kv_cache* c) {
  if (!c || !c->k || !c->v || c->dtype < MLI_KV_F32 || c->dtype > MLI_KV_BF16 || c->layers <= 0 || c->pages <= 0 ||
      c->page_size <= 0 || c->kv_heads <= 0 || c->head_dim <= 0 || c->layer_stride < 0 || c->page_stride < 0 ||
      c->head_stride < 0 || c->slot_stride < 0)
    return MLI_ERR_INVALID_ARG;
  const long long vec = 16 / cache_element_bytes(c->dtype);
  if (c->head_dim > kMaxHeadDim || c->head_dim % vec || c->layer_stride % vec || c->page_stride % vec ||
      c->head_stride % vec || c->slot_stride % vec || !aligned(c->k, 16) || !aligned(c->v, 16))
    return MLI_ERR_UNSUPPORTED;
  // heads that lie on one another (an expanded tensor's): tokens written at once would race
  if ((c->layers > 1 && c->layer_stride < c->head_dim) || (c->pages > 1 && c->page_stride < c->head_dim) ||
      (c->kv_heads > 1 && c->head_stride < c->head_dim) || (c->page_size > 1 && c->slot_stride < c->head_dim))
    return MLI_ERR_INVALID_ARG;
  return MLI_OK;
}

// Rows of a float matrix that kernels read or write 16 bytes at a time.
inline bool aligned_rows(const void* p, long long stride) { return aligned(p, 16) && stride % 4 == 0; }

}  // namespace mli
