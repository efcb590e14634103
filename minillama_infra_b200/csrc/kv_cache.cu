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

// Two warps: each repeats a token's set-up, so 8192 tokens of 24 / 8 heads of 128 take 54 us with four and 51 with two;
// with one (50 us) 1999 tokens of 35 / 5 heads of 80 take 24 us instead of 18, 500 of 32 / 8 heads of 128 11 instead of 7.
constexpr int kAppendWarps = 2;
constexpr int kAppendThreads = kAppendWarps * 32;

// Where the other value of a rotated pair comes from.
enum Partner {
  kSameQuad,   // interleaved pairs: the same four values
  kOtherLane,  // halves of whole quads, both within 32 lanes' first quads
  kOtherQuad,  // halves of 32 quads, two quads a lane
  kExchange,   // any other half: through shared memory
};

__device__ __forceinline__ void store4(float* p, const float (&y)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[2], y[3]);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&y)[4]) {
  __align__(8) T v[4] = {from_float<T>(y[0]), from_float<T>(y[1]), from_float<T>(y[2]), from_float<T>(y[3])};
  *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(v);
}

// A pass over memory: a token's heads are read once, 16 bytes a lane, and written once.  kLanes lanes hold a head,
// kQuads times four values each; a warp's heads go in batches whose reads are all under way while the CTA computes
// its token's cosines and sines (one pair a thread, in shared memory; from there each lane keeps those of its own
// values for all heads).  blockIdx.x is the token; blockIdx.y shares out the heads of few tokens.
// 8192 tokens of 24 / 8 heads of 128 into a bf16 cache: 51 us, 5.90 TB/s of 302 MB (copies run at 6.48); 64 tokens with
// norms 3.7 us, one token 2.5 us.  With norms the instructions bind: 4096 tokens of 32 / 8 heads of 128 38 us, 4.81 TB/s;
// 1999 tokens of 35 / 5 heads of 80, 20 of 32 lanes in use, 18 us, 3.0 TB/s.
template <typename T, int kLanes, int kQuads, Partner kPartner, bool kNorms>
__global__ void __launch_bounds__(kAppendThreads, 12) rope_append_kernel(const mli_rope_op op, const CacheLayer<T> c) {
  constexpr int kAtOnce = 32 / kLanes, kBatch = 4 / kQuads;  // heads of a warp side by side, and after one another
  __shared__ float s_cos[kMaxHeadDim / 2], s_sin[kMaxHeadDim / 2];
  __shared__ float4 s_heads[kPartner == kExchange ? kAppendWarps : 1][kPartner == kExchange ? kBatch : 1][kQuads][32];
  griddep_wait();
  griddep_launch_dependents();
  const int t = blockIdx.x;
  const int pos = op.pos[t];
  if (pos < 0) return;  // padding
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int l = lane % kLanes, sub = lane / kLanes;
  const int dim = c.head_dim, half = op.rot_dim / 2, keys = op.heads, values = op.heads + c.kv_heads;
  const int total = values + c.kv_heads, step = gridDim.y * kAppendWarps * kAtOnce;
  // value 0 of a head, were the keys' and values' heads counted on from the queries'
  const float* const q_row = op.q + t * op.q_stride;
  const float* const k_row = op.k + (t * op.k_stride - static_cast<long long>(keys) * dim);
  const float* const v_row = op.v + (t * op.v_stride - static_cast<long long>(values) * dim);
  const auto source = [&](int h) {
    return (h < keys ? q_row : h < values ? k_row : v_row) + static_cast<long long>(h) * dim;
  };
  float4 x[kBatch][kQuads];
  const auto read = [&](int first) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = first + b * step + sub;
      const float* p = source(h) + 4 * l;
#pragma unroll
      for (int i = 0; i < kQuads; ++i)
        x[b][i] = h < total && 4 * (l + 32 * i) < dim ? *reinterpret_cast<const float4*>(p + 128 * i)
                                                      : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  int first = (blockIdx.y * kAppendWarps + warp) * kAtOnce;
  read(first);

  // the token's slot, or -1
  long long slot = -1;
  const int seq = op.seq ? op.seq[t] : t, col = pos / c.page_size;
  if (seq >= 0 && seq < op.table_rows && col < op.table_cols) {
    const int page = op.page_table[seq * op.table_stride + col];
    if (page >= 0 && page < c.pages) slot = page * c.page_stride + (pos - col * c.page_size) * c.slot_stride;
  }
  if (slot < 0 && threadIdx.x == 0 && blockIdx.y == 0) record_device_error(kDevPageRange);

  for (int i = threadIdx.x; i < half; i += kAppendThreads) {
    // pos * turns in two numbers, its whole turns dropped in 64 bits: far positions lose nothing.  The half turns that are
    // left go to sincospi in fp32; what fp32 does not hold of them (up to pi 2^-25 as an angle: many units of a cosine or
    // sine near zero) turns its results by that much more.
    const double turn = __dmul_rn(pos, op.turns[i]), rest = fma(static_cast<double>(pos), op.turns[i], -turn);
    const double angle = 2.0 * (turn - rint(turn) + rest);
    const float near = static_cast<float>(angle), more = static_cast<float>(3.14159265358979324 * (angle - near));
    float s, co;
    sincospif(near, &s, &co);
    s_cos[i] = op.amplitude * fmaf(-more, s, co);
    s_sin[i] = op.amplitude * fmaf(more, co, s);
  }
  __syncthreads();
  // a value y of a pair becomes y cs + (the other) sn; values behind rot_dim: y 1 + 0 0
  float cs[kQuads][4], sn[kQuads][4];
#pragma unroll
  for (int i = 0; i < kQuads; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = 4 * (l + 32 * i) + j;
      const bool on = e < op.rot_dim;
      const bool second = kPartner == kSameQuad ? (j & 1) : e >= half;
      const int pair = !on ? 0 : kPartner == kSameQuad ? e >> 1 : second ? e - half : e;
      cs[i][j] = on ? s_cos[pair] : 1.f;
      sn[i][j] = on ? (second ? s_sin[pair] : -s_sin[pair]) : 0.f;
    }
  const float per_dim = 1.f / dim;
  float* const q_to = op.q_out + t * op.q_out_stride + 4 * l;
  T* const k_to = c.k + slot + 4 * l;
  T* const v_to = c.v + slot + 4 * l;

  for (; first < total; first += kBatch * step, read(first)) {
    float inv[kBatch];
    if constexpr (kNorms) {
      // the batch's sums of squares together: an exchange adds another lane's to half of the heads and gives away the
      // other half, until a lane has one head's, whose root it takes for all
      float ss[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        ss[b] = 0.f;
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
          const float4 v = x[b][i];
          ss[b] += (v.x * v.x + v.y * v.y) + (v.z * v.z + v.w * v.w);
        }
      }
#pragma unroll
      for (int off = kLanes / 2, n = kBatch / 2; off > 0; off /= 2, n /= 2) {
        if (n > 0) {
          const bool upper = l & off;
#pragma unroll
          for (int b = 0; b < n; ++b) {
            const float kept = upper ? ss[b + n] : ss[b], sent = upper ? ss[b] : ss[b + n];
            ss[b] = kept + __shfl_xor_sync(0xffffffffu, sent, off);
          }
        } else {
          ss[0] += __shfl_xor_sync(0xffffffffu, ss[0], off);
        }
      }
      const float root = rsqrtf(ss[0] * per_dim + op.eps);
#pragma unroll
      for (int b = 0; b < kBatch; ++b) inv[b] = __shfl_sync(0xffffffffu, root, b * (kLanes / kBatch), kLanes);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = first + b * step + sub;
      float y[kQuads][4];
#pragma unroll
      for (int i = 0; i < kQuads; ++i) {
        y[i][0] = x[b][i].x;
        y[i][1] = x[b][i].y;
        y[i][2] = x[b][i].z;
        y[i][3] = x[b][i].w;
      }
      const float* w = h < keys ? op.q_norm : h < values ? op.k_norm : nullptr;
      if (kNorms && w) {
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
          const int e = 4 * (l + 32 * i);
          const float4 u = e < dim ? *reinterpret_cast<const float4*>(w + e) : make_float4(1.f, 1.f, 1.f, 1.f);
          y[i][0] *= inv[b] * u.x;
          y[i][1] *= inv[b] * u.y;
          y[i][2] *= inv[b] * u.z;
          y[i][3] *= inv[b] * u.w;
        }
      }
      if constexpr (kPartner == kExchange) {
        static_assert(kBatch > 1, "a head's buffer comes round again after the barrier of another");
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
          s_heads[warp][b][i][lane] = make_float4(y[i][0], y[i][1], y[i][2], y[i][3]);
        __syncwarp();
      }
      float z[kQuads][4];
#pragma unroll
      for (int i = 0; i < kQuads; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = 4 * (l + 32 * i) + j;
          float other = 0.f;
          if constexpr (kPartner == kSameQuad) {
            other = y[i][j ^ 1];
          } else if constexpr (kPartner == kOtherLane) {
            if (i == 0) other = __shfl_sync(0xffffffffu, y[i][j], l < half / 4 ? l + half / 4 : l - half / 4, kLanes);
          } else if constexpr (kPartner == kOtherQuad) {
            other = y[i ^ 1][j];
          } else {
            const float* head = reinterpret_cast<const float*>(s_heads[warp][b]) + 4 * kLanes * sub;
            if (e < op.rot_dim) other = head[e < half ? e + half : e - half];
          }
          // behind rot_dim the other value, whatever it is, is not part of the result
          z[i][j] = h >= values ? y[i][j] : fmaf(y[i][j], cs[i][j], (e < op.rot_dim ? other : 0.f) * sn[i][j]);
        }
#pragma unroll
      for (int i = 0; i < kQuads; ++i) {
        if (4 * (l + 32 * i) >= dim) continue;
        if (h < keys)
          store4(q_to + static_cast<long long>(h) * dim + 128 * i, z[i]);
        else if (h < total && slot >= 0)
          store4((h < values ? k_to + (h - keys) * c.head_stride : v_to + (h - values) * c.head_stride) + 128 * i, z[i]);
      }
    }
  }
}

template <typename T, int kLanes, int kQuads, bool kNorms>
auto append_kernel(Partner partner) {
  switch (partner) {
    case kSameQuad: return rope_append_kernel<T, kLanes, kQuads, kSameQuad, kNorms>;
    case kOtherLane: return rope_append_kernel<T, kLanes, kQuads, kOtherLane, kNorms>;
    case kOtherQuad:
      if constexpr (kQuads == 2) return rope_append_kernel<T, kLanes, kQuads, kOtherQuad, kNorms>;
    default: return rope_append_kernel<T, kLanes, kQuads, kExchange, kNorms>;
  }
}
template <typename T, bool kNorms>
auto append_kernel(int dim, Partner partner) {
  return dim <= 64    ? append_kernel<T, 16, 1, kNorms>(partner)
         : dim <= 128 ? append_kernel<T, 32, 1, kNorms>(partner)
                      : append_kernel<T, 32, 2, kNorms>(partner);
}

template <typename T>
int launch_append(const mli_rope_op& op, const mli_kv_cache& cache, int layer, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  const DeviceInfo& dev = current_device(&e);
  if (e != cudaSuccess) return check_cuda(e);
  const int half = op.rot_dim / 2, dim = cache.head_dim;
  const Partner partner = op.interleaved || half == 0       ? kSameQuad
                          : half % 4 == 0 && half <= 64     ? kOtherLane
                          : half == 128                     ? kOtherQuad
                                                            : kExchange;
  // (a kernel without the norms' code moves 4096 tokens of 32 / 8 heads of 128 in 33.7 us, one with it in 34.7)
  const auto kernel = op.q_norm || op.k_norm ? append_kernel<T, true>(dim, partner) : append_kernel<T, false>(dim, partner);
  // Few tokens: their heads over as many CTAs as put eight on an SM, of four turns a warp at least (500 tokens of 32 / 8
  // heads of 128 with norms 7.9 us, with four on an SM 11.0; 64 tokens 4.0 us, with one turn a warp 5.9).
  const int turn = kAppendWarps * (dim <= 64 ? 2 : 1), heads = op.heads + 2 * cache.kv_heads;
  const int most = (heads + 4 * turn - 1) / (4 * turn), fill = 8 * dev.sm_count / op.m;
  const int share = fill < 1 ? 1 : fill < most ? fill : most;
  const dim3 grid(static_cast<unsigned>(op.m), static_cast<unsigned>(share));
  return check_cuda(launch(kernel, grid, dim3(kAppendThreads), 0, stream, true, op, cache_layer<T>(cache, layer)));
}

constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 8;  // reads of a thread under way at once: 32 KB a CTA

// A page as rows of contiguous 16-byte pieces: row r of `outer` x `inner` begins at (r / inner) * outer_stride +
// (r % inner) * inner_stride.
struct CopyArgs {
  uint4* k;
  uint4* v;
  long long layer_stride, page_stride, outer_stride, inner_stride;  // in 16-byte pieces
  int pages, inner, row, total;                                     // pieces of a row, of a page
};

// One CTA per (pair, layer, keys or values); bound by HBM, reads and writes alike: 256 pages of 16 tokens, 28 layers of
// 8 heads of 128 in bf16 (470 MB), 143 us, 6.57 TB/s read and written; 4 pages of 16 layers of 8 heads of 64, 2.2 us.
template <bool kWhole>  // a page is one row
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
  for (int i0 = threadIdx.x; i0 < a.total; i0 += kCopyUnroll * kCopyThreads) {
    uint4 x[kCopyUnroll];
    long long off[kCopyUnroll];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u) {
      const int i = i0 + u * kCopyThreads;
      if (i >= a.total) break;
      const int r = kWhole ? 0 : i / a.row;
      off[u] = kWhole ? i : (r / a.inner) * a.outer_stride + (r % a.inner) * a.inner_stride + i % a.row;
      x[u] = __ldcs(p + off[u]);
    }
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u) {
      if (i0 + u * kCopyThreads >= a.total) break;
      __stcs(q + off[u], x[u]);
    }
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
  // pieces of a page are counted in 32 bits
  if (bad != MLI_OK || cache->layers > 65535 ||
      static_cast<long long>(cache->kv_heads) * cache->page_size > (1 << 24))
    return set_status(MLI_ERR_UNSUPPORTED);
  const int per = 16 / cache_element_bytes(cache->dtype), vecs = cache->head_dim / per;
  const long long head = cache->head_stride / per, slot = cache->slot_stride / per;
  CopyArgs a{static_cast<uint4*>(cache->k), static_cast<uint4*>(cache->v), cache->layer_stride / per,
             cache->page_stride / per, head, slot, cache->pages, cache->page_size, vecs,
             cache->kv_heads * cache->page_size * vecs};
  // contiguous slots of a head, or heads of a slot, are one row; and all of them together, where they follow one another
  if (slot == vecs || cache->page_size == 1) {
    a.row *= cache->page_size;
    a.inner = 1;
    a.inner_stride = 0;
    if (head == a.row || cache->kv_heads == 1) a.row = a.total;
  } else if (head == vecs || cache->kv_heads == 1) {
    a.row *= cache->kv_heads;
    a.inner = 1;
    a.inner_stride = 0;
    a.outer_stride = slot;
    if (slot == a.row) a.row = a.total;
  }
  return check_cuda(launch(a.row == a.total ? copy_pages_kernel<true> : copy_pages_kernel<false>,
                           dim3(static_cast<unsigned>(n), cache->layers, 2), dim3(kCopyThreads), 0,
                           static_cast<cudaStream_t>(stream), true, a, src, dst));
}

}  // extern "C"
