// kv_cache.cu -- what goes into a paged key-value cache (sm_100a): rotary
// positions (with the norms of queries and keys), the append of keys and
// values, and copies of pages.
//
// The reference does these one token at a time: rope_kernel
// (src/model_cuda_v2_shared.cu:233-281) and two device copies into a
// contiguous cache (:391-392).
#include <math.h>

#include "kv_cache.cuh"

namespace mli {
namespace {

constexpr int kAppendThreads = 128;

// One CTA per token: cosine and sine of the token's pairs go to shared memory,
// then each warp takes heads of q, k and v in turn.
template <typename T>
__global__ void __launch_bounds__(kAppendThreads) rope_append_kernel(const mli_rope_op op, const CacheLayer<T> c) {
  __shared__ float s_cos[kMaxHeadDim / 2], s_sin[kMaxHeadDim / 2];
  griddep_wait();
  griddep_launch_dependents();
  const int t = blockIdx.x;
  const int pos = op.pos[t];
  if (pos < 0) return;  // padding
  const int half = op.rot_dim / 2;
  for (int i = threadIdx.x; i < half; i += kAppendThreads) {
    // the angle's whole turns are dropped in 64 bits: 2^31 positions leave 22 bits of a turn's fraction
    const double turn = pos * op.turns[i];
    float s, co;
    sincospif(static_cast<float>(2.0 * (turn - rint(turn))), &s, &co);
    s_cos[i] = op.amplitude * co;
    s_sin[i] = op.amplitude * s;
  }
  // the token's slot, or -1
  long long slot = -1;
  const int seq = op.seq ? op.seq[t] : t;
  if (seq >= 0 && seq < op.table_rows && pos / c.page_size < op.table_cols) {
    const int page = op.page_table[seq * op.table_stride + pos / c.page_size];
    if (page >= 0 && page < c.pages) slot = page * c.page_stride + (pos % c.page_size) * c.slot_stride;
  }
  if (slot < 0 && threadIdx.x == 0) record_device_error(kDevPageRange);
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int dim = c.head_dim;
  for (int h = threadIdx.x >> 5; h < op.heads + 2 * c.kv_heads; h += kAppendThreads / 32) {
    const bool is_q = h < op.heads;
    const int hk = is_q ? 0 : (h - op.heads) % c.kv_heads;
    const bool is_v = h >= op.heads + c.kv_heads;
    if (!is_q && slot < 0) break;
    const float* x = is_q ? op.q + t * op.q_stride + static_cast<long long>(h) * dim
                          : (is_v ? op.v + t * op.v_stride : op.k + t * op.k_stride) + hk * dim;
    T* to = is_q ? nullptr : (is_v ? c.v : c.k) + slot + hk * c.head_stride;
    float* qo = op.q_out + t * op.q_out_stride + static_cast<long long>(h) * dim;
    if (is_v) {
      for (int e = lane; e < dim; e += 32) to[e] = from_float<T>(x[e]);
      continue;
    }
    const float* w = is_q ? op.q_norm : op.k_norm;
    float inv = 1.f;
    if (w) {
      float ss = 0.f;
      for (int e = lane; e < dim; e += 32) ss += x[e] * x[e];
      inv = 1.f / sqrtf(warp_sum(ss) / dim + op.eps);
    }
    float y[kMaxHeadDim / 32];
#pragma unroll
    for (int k = 0; k < kMaxHeadDim / 32; ++k) {
      const int e = lane + 32 * k;
      if (e >= dim) break;
      float a = x[e] * inv;
      if (w) a *= w[e];
      if (e < op.rot_dim) {
        const int i = op.interleaved ? e >> 1 : (e < half ? e : e - half);
        const bool second = op.interleaved ? (e & 1) : e >= half;
        const int o = op.interleaved ? e ^ 1 : (second ? e - half : e + half);
        float b = x[o] * inv;
        if (w) b *= w[o];
        a = second ? a * s_cos[i] + b * s_sin[i] : a * s_cos[i] - b * s_sin[i];
      }
      y[k] = a;
    }
    __syncwarp();  // q_out may be q
#pragma unroll
    for (int k = 0; k < kMaxHeadDim / 32; ++k) {
      const int e = lane + 32 * k;
      if (e >= dim) break;
      if (is_q)
        qo[e] = y[k];
      else
        to[e] = from_float<T>(y[k]);
    }
  }
}

template <typename T>
int launch_append(const mli_rope_op& op, const mli_kv_cache& cache, int layer, cudaStream_t stream) {
  return check_cuda(launch(rope_append_kernel<T>, dim3(static_cast<unsigned>(op.m)), dim3(kAppendThreads), 0, stream,
                           true, op, cache_layer<T>(cache, layer)));
}

constexpr int kCopyThreads = 256;

struct CopyArgs {
  uint4* k;
  uint4* v;
  // in 16-byte units
  long long layer_stride, page_stride, head_stride, slot_stride;
  int pages, heads, slots, vecs;  // vecs: 16-byte pieces of one head's slot
};

// One CTA per (pair, layer, keys or values).
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const CopyArgs a, const int* src, const int* dst) {
  griddep_wait();
  griddep_launch_dependents();
  const int from = src[blockIdx.x], to = dst[blockIdx.x];
  if (from < 0 || to < 0) return;
  if (from >= a.pages || to >= a.pages) {
    if (threadIdx.x == 0) record_device_error(kDevPageRange);
    return;
  }
  uint4* base = (blockIdx.z ? a.v : a.k) + blockIdx.y * a.layer_stride;
  const uint4* p = base + from * a.page_stride;
  uint4* q = base + to * a.page_stride;
  const int rows = a.slots * a.vecs;
  for (int h = 0; h < a.heads; ++h)
    for (int i = threadIdx.x; i < rows; i += kCopyThreads) {
      const long long off = h * a.head_stride + (i / a.vecs) * a.slot_stride + i % a.vecs;
      q[off] = p[off];
    }
}

}  // namespace
}  // namespace mli

using namespace mli;

extern "C" {

int mli_rope_turns(double* turns, int rot_dim, double theta, int scaling, double factor, double low, double high,
                   int original_len) {
  const double two_pi = 6.283185307179586476925286766559;
  if (!turns || rot_dim <= 0 || rot_dim % 2 || !(theta > 0.0) || !isfinite(theta) || scaling < MLI_ROPE_PLAIN ||
      scaling > MLI_ROPE_YARN)
    return set_status(MLI_ERR_INVALID_ARG);
  if (scaling != MLI_ROPE_PLAIN && (!(factor > 0.0) || !isfinite(factor))) return set_status(MLI_ERR_INVALID_ARG);
  if (scaling >= MLI_ROPE_LLAMA3 && (!(low > 0.0) || !(high > low) || !isfinite(high) || original_len <= 0))
    return set_status(MLI_ERR_INVALID_ARG);
  if (scaling == MLI_ROPE_YARN && theta == 1.0) return set_status(MLI_ERR_INVALID_ARG);
  // YaRN: the pair that turns `r` times over original_len, as a real index
  const auto pair_of = [&](double r) { return rot_dim * log(original_len / (r * two_pi)) / (2.0 * log(theta)); };
  for (int i = 0; i < rot_dim / 2; ++i) {
    const double f = pow(theta, -2.0 * i / rot_dim);  // radians per position
    double keep = 1.0;                                // share of the unscaled frequency
    if (scaling == MLI_ROPE_LINEAR) {
      keep = 0.0;
    } else if (scaling == MLI_ROPE_LLAMA3) {
      const double times = original_len * f / two_pi;  // turns over the original context
      keep = fmin(1.0, fmax(0.0, (times - low) / (high - low)));
    } else if (scaling == MLI_ROPE_YARN) {
      const double first = fmax(0.0, floor(pair_of(high)));
      const double last = fmin(rot_dim - 1.0, ceil(pair_of(low)));
      const double ramp = (i - first) / fmax(last - first, 1e-3);
      keep = 1.0 - fmin(1.0, fmax(0.0, ramp));
    }
    turns[i] = f * (keep + (scaling == MLI_ROPE_PLAIN ? 0.0 : (1.0 - keep) / factor)) / two_pi;
  }
  return set_status(MLI_OK);
}

int mli_rope_append(const mli_rope_op* op, const mli_kv_cache* cache, int layer, void* stream) {
  const int bad = check_cache(cache);
  if (bad == MLI_ERR_INVALID_ARG || !op || layer < 0 || layer >= cache->layers) return set_status(MLI_ERR_INVALID_ARG);
  if (!op->q_out || !op->q || !op->k || !op->v || !op->pos || !op->page_table || op->m <= 0 || op->heads <= 0 ||
      op->heads % cache->kv_heads || op->rot_dim < 0 || op->rot_dim % 2 || op->rot_dim > cache->head_dim ||
      (op->rot_dim > 0 && !op->turns) || op->table_rows <= 0 || op->table_cols <= 0 ||
      op->table_stride < op->table_cols || (!op->seq && op->m > op->table_rows) || !isfinite(op->amplitude) ||
      ((op->q_norm || op->k_norm) && !(op->eps >= 0.f && isfinite(op->eps))))
    return set_status(MLI_ERR_INVALID_ARG);
  const long long q_row = static_cast<long long>(op->heads) * cache->head_dim;
  const long long kv_row = static_cast<long long>(cache->kv_heads) * cache->head_dim;
  if (op->q_stride < q_row || op->q_out_stride < q_row || op->k_stride < kv_row || op->v_stride < kv_row ||
      (op->q_out == op->q && op->q_stride != op->q_out_stride))
    return set_status(MLI_ERR_INVALID_ARG);
  if (bad != MLI_OK || !aligned_rows(op->q, op->q_stride) || !aligned_rows(op->q_out, op->q_out_stride) ||
      !aligned_rows(op->k, op->k_stride) || !aligned_rows(op->v, op->v_stride) ||
      (op->q_norm && !aligned(op->q_norm, 16)) || (op->k_norm && !aligned(op->k_norm, 16)))
    return set_status(MLI_ERR_UNSUPPORTED);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (cache->dtype) {
    case MLI_KV_F32: return launch_append<float>(*op, *cache, layer, s);
    case MLI_KV_F16: return launch_append<__half>(*op, *cache, layer, s);
    default: return launch_append<__nv_bfloat16>(*op, *cache, layer, s);
  }
}

int mli_kv_copy_pages(const mli_kv_cache* cache, const int* src, const int* dst, int n, void* stream) {
  const int bad = check_cache(cache);
  if (bad == MLI_ERR_INVALID_ARG || !src || !dst || n <= 0) return set_status(MLI_ERR_INVALID_ARG);
  if (bad != MLI_OK || cache->layers > 65535) return set_status(MLI_ERR_UNSUPPORTED);
  const int per = 16 / cache_element_bytes(cache->dtype);
  const CopyArgs a{static_cast<uint4*>(cache->k), static_cast<uint4*>(cache->v),
                   cache->layer_stride / per, cache->page_stride / per, cache->head_stride / per,
                   cache->slot_stride / per, cache->pages, cache->kv_heads, cache->page_size, cache->head_dim / per};
  return check_cuda(launch(copy_pages_kernel, dim3(static_cast<unsigned>(n), cache->layers, 2), dim3(kCopyThreads), 0,
                           static_cast<cudaStream_t>(stream), true, a, src, dst));
}

}  // extern "C"
