// paged_attention.cu -- attention of one new token a row over a paged
// key-value cache (sm_100a).
//
//   out = sum_t p_t v_t / sum_t p_t,   p_t = exp(scale q.k_t - max)
//
// One pass over the cache with the running maximum and sum of the softmax.
// The reference's fused_attention_kernel (src/model_cuda_v2_shared.cu:291-365)
// holds a head's scores of a contiguous cache in shared memory.
#include <math.h>

#include "kv_cache.cuh"

namespace mli {
namespace {

constexpr int kWarps = 4;

// One CTA per (query head, row); its warps take every fourth token.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) paged_attention_kernel(const mli_attention_op op, const CacheLayer<T> c) {
  __shared__ float s_acc[kWarps][kMaxHeadDim], s_m[kWarps], s_l[kWarps];
  constexpr int kPer = kMaxHeadDim / 32;
  griddep_wait();
  griddep_launch_dependents();
  const int h = blockIdx.x, r = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seq = op.seq ? op.seq[r] : r;
  int len = op.lengths[r];
  bool bad = false;
  if (len > 0 && (seq < 0 || seq >= op.table_rows)) {
    len = 0;
    bad = true;
  }
  const long long room = static_cast<long long>(op.table_cols) * c.page_size;
  if (len > room) {
    len = static_cast<int>(room);
    bad = true;
  }
  const int dim = c.head_dim;
  const long long head = (h / (op.heads / c.kv_heads)) * c.head_stride;
  float q[kPer], acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = lane + 32 * i;
    q[i] = e < dim ? op.q[r * op.q_stride + static_cast<long long>(h) * dim + e] * op.scale : 0.f;
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int t = warp; t < len; t += kWarps) {
    const int page = op.page_table[seq * op.table_stride + t / c.page_size];
    if (page < 0 || page >= c.pages) {
      bad = true;
      continue;
    }
    const long long off = page * c.page_stride + head + (t % c.page_size) * c.slot_stride;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane + 32 * i < dim) s = fmaf(q[i], to_float(c.k[off + lane + 32 * i]), s);
    s = warp_sum(s);
    const float top = fmaxf(m, s);
    const float keep = m == top ? 1.f : expf(m - top), p = expf(s - top);
    m = top;
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane + 32 * i < dim) acc[i] = fmaf(p, to_float(c.v[off + lane + 32 * i]), acc[i] * keep);
  }
  if (bad && lane == 0) record_device_error(kDevPageRange);
#pragma unroll
  for (int i = 0; i < kPer; ++i) s_acc[warp][lane + 32 * i] = acc[i];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  float top = -INFINITY, total = 0.f, weight[kWarps];
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w]);
  for (int w = 0; w < kWarps; ++w) {
    weight[w] = s_l[w] == 0.f ? 0.f : expf(s_m[w] - top);
    total += weight[w] * s_l[w];
  }
  for (int e = threadIdx.x; e < dim; e += kWarps * 32) {
    float y = 0.f;
    for (int w = 0; w < kWarps; ++w) y += weight[w] * s_acc[w][e];
    op.out[r * op.out_stride + static_cast<long long>(h) * dim + e] = total == 0.f ? 0.f : y / total;
  }
}

template <typename T>
int launch_attention(const mli_attention_op& op, const mli_kv_cache& cache, int layer, cudaStream_t stream) {
  return check_cuda(launch(paged_attention_kernel<T>, dim3(op.heads, op.rows), dim3(kWarps * 32), 0, stream, true, op,
                           cache_layer<T>(cache, layer)));
}

}  // namespace
}  // namespace mli

using namespace mli;

extern "C" {

size_t mli_paged_attention_workspace_bytes(int rows, int heads, int kv_heads, int head_dim) {
  if (rows <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || head_dim <= 0 || head_dim > kMaxHeadDim) return 0;
  return 16;
}

int mli_paged_attention(const mli_attention_op* op, const mli_kv_cache* cache, int layer, void* stream) {
  const int bad = check_cache(cache);
  if (bad == MLI_ERR_INVALID_ARG || !op || layer < 0 || layer >= cache->layers) return set_status(MLI_ERR_INVALID_ARG);
  if (!op->out || !op->q || !op->lengths || !op->page_table || !op->workspace || op->rows <= 0 || op->heads <= 0 ||
      op->heads % cache->kv_heads || !(op->scale > 0.f) || !isfinite(op->scale) || op->table_rows <= 0 ||
      op->table_cols <= 0 || op->table_stride < op->table_cols || (!op->seq && op->rows > op->table_rows))
    return set_status(MLI_ERR_INVALID_ARG);
  const long long row = static_cast<long long>(op->heads) * cache->head_dim;
  if (op->q_stride < row || op->out_stride < row ||
      op->workspace_bytes <
          mli_paged_attention_workspace_bytes(op->rows, op->heads, cache->kv_heads, cache->head_dim))
    return set_status(MLI_ERR_INVALID_ARG);
  if (bad != MLI_OK || !aligned_rows(op->q, op->q_stride) || !aligned_rows(op->out, op->out_stride) ||
      !aligned(op->workspace, 16) || op->rows > 65535)
    return set_status(MLI_ERR_UNSUPPORTED);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (cache->dtype) {
    case MLI_KV_F32: return launch_attention<float>(*op, *cache, layer, s);
    case MLI_KV_F16: return launch_attention<__half>(*op, *cache, layer, s);
    default: return launch_attention<__nv_bfloat16>(*op, *cache, layer, s);
  }
}

}  // extern "C"
