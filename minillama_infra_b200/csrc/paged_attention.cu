// paged_attention.cu -- attention of one new token a row over a paged
// key-value cache (sm_100a).
//
//   out = sum_t p_t v_t / sum_t p_t,   p_t = 2^(c (s_t - m)),  s_t = q.k_t,
//   c = scale log2(e),  m = max_t s_t
//
// One pass over the cache with the running maximum and sum of the softmax.
// The reference's fused_attention_kernel (src/model_cuda_v2_shared.cu:291-365)
// holds a head's scores of a contiguous cache in shared memory.
//
// Split over the length.  A row's keys and values of one key-value head are a
// segment, cut into tiles of kTok tokens; all tiles of all segments, in order,
// are dealt out to the warps of one CTA per SM in equal contiguous ranges, so
// ragged batches and single long rows load the GPU alike.  Lengths live on the
// device (a captured step replays with others), so every CTA derives the ranges
// from them itself.  A warp that holds a whole segment writes its output; pieces
// of a segment are joined in shared memory within a CTA, and by the last CTA to
// finish where a segment spans several, in CTA order: results do not depend on
// timing.
//
// Each warp streams its tiles through a ring of its own in shared memory
// (16-byte cp.async, chunks of a row permuted by its number so that column reads
// do not collide); warps never wait for one another before the join.
#include <float.h>
#include <math.h>

#include <type_traits>

#include "kv_cache.cuh"

namespace mli {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kGroup = 8;          // query heads that share a pass over a segment
constexpr int kStageBytes = 16384;  // one tile of keys and of values
constexpr int kMaxCtas = 160;       // CTAs with partial results in the workspace

// ---- division of n < 2^31 by a number known at launch ------------------------
struct FastDiv {
  unsigned mul, shift, by;
};
FastDiv fast_div(unsigned by) {
  unsigned s = 0;
  while ((1ull << s) < by) ++s;
  // ceil(2^(31+s) / by) < 2^32: off by less than 2^s in 2^(31+s), so n < 2^31 divides exactly
  return FastDiv{static_cast<unsigned>(((1ull << (31 + s)) + by - 1) / by), 31 + s, by};
}
__device__ __forceinline__ unsigned divide(unsigned n, const FastDiv& d) {
  return static_cast<unsigned>((static_cast<unsigned long long>(n) * d.mul) >> d.shift);
}

__device__ __forceinline__ void cp_async16(void* smem, const void* src, bool live) {
  // a chunk that is not live is filled with zeros, its source not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(src), "r"(live ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

struct Args {
  const float* q;
  float* out;
  long long q_stride, out_stride;
  const int* lengths;
  const int* seq;
  const int* page_table;
  long long table_stride;
  int rows, heads, table_rows;
  long long room;  // tokens a page-table row can name
  int group;       // query heads of a key-value head
  int chunks;      // passes of up to kGroup of them
  float scale;     // times log2(e)
  FastDiv page_div;
  float* partials;     // [kMaxCtas][2] pieces
  unsigned* arrivals;  // [rows * kv_heads * chunks], zero between calls
};

// A piece of a segment: the unnormalised output, the maximum, the sum and c of each head.
template <int kDim>
struct Piece {
  float o[kGroup][kDim];
  float m[kGroup], l[kGroup], c[kGroup];
};
// What a piece of maximum m counts beside one of maximum top (no piece: 1, and its sums are zero).
__device__ __forceinline__ float piece_weight(float m, float top, float c) {
  return m == top ? 1.f : exp2f((m - top) * c);
}

// ---- the products on the tensor cores, 16-bit caches --------------------------
//
// S = q K^T and O = p V as m16n8k16 products with fp32 accumulation.  q and p
// keep all their fp32 bits: each is the sum of three 16-bit numbers (8 bits
// each in bf16, 11 in fp16), and the rows of the left operand that a decode
// step would leave empty carry the parts: rows 0-7 the first of 8 heads, 8-15
// the second, and a second product the third.  With up to 4 heads rows 0-3, 8-11
// and 12-15 take all three in one product.  fp16's range is kept
// by powers of two: q scaled so that its largest value has exponent 14, p by 2^15.
template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ unsigned pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(unsigned u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3,
                                             unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <>
struct Pair<__half> {
  static __device__ __forceinline__ unsigned pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(unsigned u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3,
                                             unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// The three 16-bit parts of two floats.
template <typename T>
__device__ __forceinline__ void split3(float x, float y, unsigned& hi, unsigned& mid, unsigned& lo) {
  hi = Pair<T>::pack(x, y);
  float2 f = Pair<T>::unpack(hi);
  x -= f.x;
  y -= f.y;
  mid = Pair<T>::pack(x, y);
  f = Pair<T>::unpack(mid);
  lo = Pair<T>::pack(x - f.x, y - f.y);
}

__device__ __forceinline__ void ldmatrix4(unsigned (&r)[4], unsigned addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(unsigned (&r)[4], unsigned addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// kDim: the head dimension's room in shared memory (64, 128 or 256).  kFew: at most 4 heads.
template <typename T, int kDim, bool kFew>
struct TensorMath {
  static constexpr int kTok = kStageBytes / (2 * kDim * 2);  // 64, 32 or 16 tokens a tile
  static constexpr int kSteps = kDim / 16;
  static constexpr float kUp = std::is_same<T, __half>::value ? 32768.f : 1.f;

  unsigned q[kSteps][kFew ? 4 : 6];
  float o[kDim / 8][2];
  float m, l, c;
  int head;  // this lane's head within the pass
  bool third;

  __device__ __forceinline__ void begin(const Args& a, const float* qp, int heads, int dim, float*) {
    const int lane = threadIdx.x & 31, g = lane >> 2, col = 2 * (lane & 3);
    head = kFew ? g & 3 : g;
    third = kFew && g >= 4;
    const float* row = qp + head * dim;
    const bool live = head < heads;
    float2 x[kSteps][2];
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int e = 16 * k + 8 * j + col;
        x[k][j] = live && e < dim ? *reinterpret_cast<const float2*>(row + e) : make_float2(0.f, 0.f);
        if (kUp != 1.f) top = fmaxf(top, fmaxf(fabsf(x[k][j].x), fabsf(x[k][j].y)));
      }
    c = a.scale;
    float up = 1.f;
    if (kUp != 1.f) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int exponent = (__float_as_int(top) >> 23) & 255;
      const int f = exponent == 255 ? 127 : min(127 + 60, 268 - exponent);
      up = __int_as_float(f << 23);
      c = fmaxf(c * __int_as_float((254 - f) << 23), FLT_MIN);  // c = 0 would make c s of -inf a NaN
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        unsigned hi, mid, lo;
        split3<T>(x[k][j].x * up, x[k][j].y * up, hi, mid, lo);
        q[k][2 * j] = third ? 0u : hi;
        q[k][2 * j + 1] = third ? lo : mid;
        if (!kFew) q[k][4 + j] = lo;
      }
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < kDim / 8; ++i) o[i][0] = o[i][1] = 0.f;
  }

  // live: bit t for token t of the tile
  __device__ __forceinline__ void tile(const unsigned char* slot, unsigned long long live, float*) {
    const int lane = threadIdx.x & 31;
    const unsigned keys = smem_u32(slot), values = keys + kTok * kDim * 2;
    const int mat = lane >> 3, in = lane & 7;
    float s[kTok / 8][4];
#pragma unroll
    for (int n = 0; n < kTok / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
    {
      // matrices (tokens 0-7, 8-15) x (dims 0-7, 8-15) of a 16-token block
      const unsigned row = keys + ((mat >> 1) * 8 + in) * (kDim * 2);
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const unsigned chunk = ((2 * k + (mat & 1)) ^ in) * 16;
#pragma unroll
        for (int n = 0; n < kTok / 16; ++n) {
          unsigned b[4];
          ldmatrix4(b, row + n * 16 * (kDim * 2) + chunk);
          Pair<T>::mma(s[2 * n], q[k][0], q[k][1], q[k][2], q[k][3], b[0], b[1]);
          Pair<T>::mma(s[2 * n + 1], q[k][0], q[k][1], q[k][2], q[k][3], b[2], b[3]);
          if (!kFew) {
            Pair<T>::mma(s[2 * n], q[k][4], 0u, q[k][5], 0u, b[0], b[1]);
            Pair<T>::mma(s[2 * n + 1], q[k][4], 0u, q[k][5], 0u, b[2], b[3]);
          }
        }
      }
    }
    float top = m;
#pragma unroll
    for (int n = 0; n < kTok / 8; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x = s[n][j] + s[n][j + 2];
        if (kFew) x += __shfl_xor_sync(0xffffffffu, x, 16);
        x = (live >> (8 * n + 2 * (lane & 3) + j)) & 1 ? x : -INFINITY;
        s[n][j] = x;
        top = fmaxf(top, x);
      }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float base = top == -INFINITY ? 0.f : top;
    const float keep = exp2f((m - base) * c);  // m = -inf: 0
    m = top;
    l *= keep;
    unsigned p[kTok / 8][3];
#pragma unroll
    for (int n = 0; n < kTok / 8; ++n) {
      const float x = exp2f((s[n][0] - base) * c), y = exp2f((s[n][1] - base) * c);
      l += x + y;
      unsigned hi, mid, lo;
      split3<T>(x * kUp, y * kUp, hi, mid, lo);
      p[n][0] = third ? 0u : hi;
      p[n][1] = third ? lo : mid;
      p[n][2] = lo;
    }
    const unsigned row = values + ((mat & 1) * 8 + in) * (kDim * 2);
#pragma unroll
    for (int d = 0; d < kDim / 16; ++d) {
      float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      const unsigned chunk = ((2 * d + (mat >> 1)) ^ in) * 16;
#pragma unroll
      for (int n = 0; n < kTok / 16; ++n) {
        unsigned b[4];
        ldmatrix4_trans(b, row + n * 16 * (kDim * 2) + chunk);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          Pair<T>::mma(acc[h], p[2 * n][0], p[2 * n][1], p[2 * n + 1][0], p[2 * n + 1][1], b[2 * h], b[2 * h + 1]);
          if (!kFew) Pair<T>::mma(acc[h], p[2 * n][2], 0u, p[2 * n + 1][2], 0u, b[2 * h], b[2 * h + 1]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 2; ++j) o[2 * d + h][j] = fmaf(o[2 * d + h][j], keep, acc[h][j] + acc[h][j + 2]);
    }
  }

  // The sums over lanes; after it lane (head, col) of the first parts holds dims 8 i + col, + 1.
  __device__ __forceinline__ void finish() {
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (kFew) {
#pragma unroll
      for (int i = 0; i < kDim / 8; ++i) {
        o[i][0] += __shfl_xor_sync(0xffffffffu, o[i][0], 16);
        o[i][1] += __shfl_xor_sync(0xffffffffu, o[i][1], 16);
      }
    }
  }
  __device__ __forceinline__ void store(float* out, int heads, int dim) {
    finish();
    if (third || head >= heads) return;
    const float inv = l == 0.f ? 0.f : 1.f / (l * kUp);
    float* row = out + head * dim + 2 * (threadIdx.x & 3);
#pragma unroll
    for (int i = 0; i < kDim / 8; ++i)
      if (8 * i < dim) *reinterpret_cast<float2*>(row + 8 * i) = make_float2(o[i][0] * inv, o[i][1] * inv);
  }
  __device__ __forceinline__ void store(Piece<kDim>& to) {
    finish();
    if (third) return;
    const int col = 2 * (threadIdx.x & 3);
#pragma unroll
    for (int i = 0; i < kDim / 8; ++i)
      *reinterpret_cast<float2*>(&to.o[head][8 * i + col]) = make_float2(o[i][0], o[i][1]);
    if (col == 0) {
      to.m[head] = m;
      to.l[head] = l * kUp;
      to.c[head] = c;
    }
  }
};

// ---- the products in fp32, fp32 caches ----------------------------------------
//
// A lane takes one token of the tile (or a part of its dims) for the scores
// and four dims of a token (or eight) for the outputs; q and p come from shared memory
// as broadcasts.
template <int kDim, bool kFew>
struct FloatMath {
  static constexpr int kTok = kStageBytes / (2 * kDim * 4);  // 32, 16 or 8 tokens a tile
  static constexpr int kHeads = kFew ? 4 : 8;
  static constexpr int kParts = 32 / kTok;   // lanes of a token's score
  static constexpr int kChunks = kDim / 4;   // 16-byte pieces of a token
  static constexpr int kRows = kChunks < 32 ? 32 / kChunks : 1;  // tokens side by side in the outputs' sum
  static constexpr int kOwn = kChunks < 32 ? 1 : kChunks / 32;   // pieces of a token a lane sums

  float2 o[kHeads][kOwn][2];
  float m[kHeads], l[kHeads], c;

  __device__ __forceinline__ void begin(const Args& a, const float* qp, int heads, int dim, float* scratch) {
    const int lane = threadIdx.x & 31;
    float4* qs = reinterpret_cast<float4*>(scratch);
    __syncwarp();
    for (int i = lane; i < kHeads * kChunks; i += 32) {
      const int h = i / kChunks, e = 4 * (i % kChunks);
      qs[i] = h < heads && e < dim ? *reinterpret_cast<const float4*>(qp + h * dim + e)
                                   : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncwarp();
    c = a.scale;
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) o[h][i][0] = o[h][i][1] = make_float2(0.f, 0.f);
    }
  }

  __device__ __forceinline__ void tile(const unsigned char* slot, unsigned long long live, float* scratch) {
    const int lane = threadIdx.x & 31;
    const float4* keys = reinterpret_cast<const float4*>(slot);
    const float4* values = keys + kTok * kChunks;
    const float4* qs = reinterpret_cast<const float4*>(scratch);
    float* ps = scratch + kHeads * kDim;  // [kTok][kHeads]
    const int t = lane % kTok, part = lane / kTok;
    float2 acc[kHeads][2];
#pragma unroll
    for (int h = 0; h < kHeads; ++h) acc[h][0] = acc[h][1] = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int k = part; k < kChunks; k += kParts) {
      const float4 x = keys[t * kChunks + (k ^ (t & 7))];
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        const float4 y = qs[h * kChunks + k];
        acc[h][0] = fma2(make_float2(x.x, x.y), make_float2(y.x, y.y), acc[h][0]);
        acc[h][1] = fma2(make_float2(x.z, x.w), make_float2(y.z, y.w), acc[h][1]);
      }
    }
    float keep[kHeads];
    const bool on = (live >> t) & 1;
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      float s = (acc[h][0].x + acc[h][0].y) + (acc[h][1].x + acc[h][1].y);
#pragma unroll
      for (int off = kTok; off < 32; off *= 2) s += __shfl_xor_sync(0xffffffffu, s, off);
      s = on ? s : -INFINITY;
      float top = s;
#pragma unroll
      for (int off = kTok / 2; off > 0; off /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      top = fmaxf(top, m[h]);
      const float base = top == -INFINITY ? 0.f : top;
      keep[h] = exp2f((m[h] - base) * c);
      m[h] = top;
      const float p = exp2f((s - base) * c);
      l[h] = fmaf(l[h], keep[h], part == 0 ? p : 0.f);
      if (part == 0) ps[t * kHeads + h] = p;
    }
    __syncwarp();
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) o[h][i][j] = mul2(o[h][i][j], make_float2(keep[h], keep[h]));
    const int first = kRows > 1 ? lane / kChunks : 0, piece = kRows > 1 ? lane % kChunks : lane;
#pragma unroll 4
    for (int r = first; r < kTok; r += kRows) {
      float4 x[kOwn];
#pragma unroll
      for (int i = 0; i < kOwn; ++i) x[i] = values[r * kChunks + ((piece + 32 * i) ^ (r & 7))];
#pragma unroll
      for (int h4 = 0; h4 < kHeads / 4; ++h4) {
        const float4 p4 = *reinterpret_cast<const float4*>(ps + r * kHeads + 4 * h4);
        const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
          for (int i = 0; i < kOwn; ++i) {
            o[4 * h4 + h][i][0] = fma2(make_float2(p[h], p[h]), make_float2(x[i].x, x[i].y), o[4 * h4 + h][i][0]);
            o[4 * h4 + h][i][1] = fma2(make_float2(p[h], p[h]), make_float2(x[i].z, x[i].w), o[4 * h4 + h][i][1]);
          }
      }
    }
    __syncwarp();  // ps is written again by the next tile
  }

  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      l[h] = warp_sum(l[h]);
      if (kRows > 1) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int off = kChunks; off < 32; off *= 2) {
            o[h][0][j].x += __shfl_xor_sync(0xffffffffu, o[h][0][j].x, off);
            o[h][0][j].y += __shfl_xor_sync(0xffffffffu, o[h][0][j].y, off);
          }
      }
    }
  }
  __device__ __forceinline__ void store(float* out, int heads, int dim) {
    finish();
    const int lane = threadIdx.x & 31;
    if (kRows > 1 && lane >= kChunks) return;
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const float inv = l[h] == 0.f ? 0.f : 1.f / l[h];
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int e = 4 * (lane + 32 * i);
        if (h < heads && e < dim)
          *reinterpret_cast<float4*>(out + h * dim + e) = make_float4(o[h][i][0].x * inv, o[h][i][0].y * inv,
                                                                      o[h][i][1].x * inv, o[h][i][1].y * inv);
      }
    }
  }
  __device__ __forceinline__ void store(Piece<kDim>& to) {
    finish();
    const int lane = threadIdx.x & 31;
    if (kRows > 1 && lane >= kChunks) return;
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
        *reinterpret_cast<float4*>(&to.o[h][4 * (lane + 32 * i)]) =
            make_float4(o[h][i][0].x, o[h][i][0].y, o[h][i][1].x, o[h][i][1].y);
      if (lane == 0) {
        to.m[h] = m[h];
        to.l[h] = l[h];
        to.c[h] = c;
      }
    }
  }
};

// ---- the tiles of a call ---------------------------------------------------------
// Tokens that row r attends to: its length, cut to the page table; 0 for a row led outside it.
__device__ __forceinline__ int row_tokens(const Args& a, int r, bool* bad) {
  const int len = a.lengths[r];
  if (len <= 0) return 0;
  if (a.seq != nullptr) {
    const int s = a.seq[r];
    if (s < 0 || s >= a.table_rows) {
      *bad = true;
      return 0;
    }
  }
  if (len > a.room) *bad = true;
  return len > a.room ? static_cast<int>(a.room) : len;
}

// A segment's place among all tiles.
struct Segment {
  int row, item;      // item: key-value head * chunks + chunk
  long long start;    // first tile
  int tiles, tokens;
};

// A warp's walk over the tiles [at, end).
template <int kTok>
struct Walk {
  Segment s;
  long long at, end;

  __device__ __forceinline__ void advance(const Args& a, int items) {
    if (++at < s.start + s.tiles || at >= end) return;
    s.start += s.tiles;
    if (++s.item < items) return;
    s.item = 0;
    bool bad;
    do {
      s.tokens = row_tokens(a, ++s.row, &bad);
    } while (s.tokens == 0 && s.row + 1 < a.rows);
    s.tiles = (s.tokens + kTok - 1) / kTok;
  }
};

enum : int { kFirst = 1, kLast = 2, kWhole = 4 };  // a tile's place in its piece; the piece is a whole segment

struct TileInfo {
  unsigned long long live;
  long long start;  // the segment's first tile
  int row, item, tiles, flags;
};

// What a CTA knows of a piece it holds in shared memory.
struct Held {
  long long start;  // the segment's first tile
  int row, item, tiles, used;
};

template <typename Math, typename T, int kDim, int kStages>
__global__ void __launch_bounds__(kThreads, 1) paged_attention_kernel(const Args a, const CacheLayer<T> cache) {
  constexpr int kTok = Math::kTok;
  constexpr int kChunks = kDim * sizeof(T) / 16;  // 16-byte pieces of a token's keys
  constexpr int kPer = kTok > 32 ? kTok / 32 : 1;  // tokens whose place a lane looks up
  constexpr bool kFloat = sizeof(T) == 4;
  constexpr int kScratch = kFloat ? kGroup * kDim + kTok * kGroup : 0;  // floats of FloatMath's q and p

  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long s_scan[kThreads / 32];
  __shared__ Segment s_first[kWarps];
  __shared__ TileInfo s_info[kWarps][kStages];
  __shared__ Held s_held[2 * kWarps];
  __shared__ int s_last;
  // rings, then two pieces of each warp, then FloatMath's scratch
  Piece<kDim>* pieces = reinterpret_cast<Piece<kDim>*>(smem + kWarps * kStages * kStageBytes);
  float* scratch_all = reinterpret_cast<float*>(pieces + 2 * kWarps);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned char* ring = smem + warp * (kStages * kStageBytes);
  float* scratch = scratch_all + warp * kScratch;
  const int dim = cache.head_dim, items = cache.kv_heads * a.chunks;
  const int live_chunks = dim * static_cast<int>(sizeof(T)) / 16;
  if (live_chunks < kChunks) {  // the columns that no token fills
    for (int i = lane; i < kStages * kStageBytes / 16; i += 32)
      reinterpret_cast<uint4*>(ring)[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  if (lane == 0) {
    s_held[2 * warp].used = s_held[2 * warp + 1].used = 0;
    s_first[warp] = Segment{0, 0, 0, 0, 0};
  }
  griddep_wait();
  griddep_launch_dependents();

  // Where each warp starts: thread i sums the tiles of rows [i n, (i + 1) n).
  const int n = (a.rows + kThreads - 1) / kThreads;
  const int r0 = min(a.rows, tid * n), r1 = min(a.rows, r0 + n);
  long long mine = 0;
  bool bad = false;
  for (int r = r0; r < r1; ++r) mine += (row_tokens(a, r, &bad) + kTok - 1) / kTok;
  if (bad && blockIdx.x == 0) record_device_error(kDevPageRange);
  long long sum = mine;
#pragma unroll
  for (int off = 1; off < 32; off *= 2) {
    const long long x = __shfl_up_sync(0xffffffffu, sum, off);
    if (lane >= off) sum += x;
  }
  if (lane == 31) s_scan[warp] = sum;
  __syncthreads();
  long long before = sum - mine, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += s_scan[w];
    all += s_scan[w];
  }
  const long long total = all * items, workers = static_cast<long long>(gridDim.x) * kWarps;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const long long from = total * (static_cast<long long>(blockIdx.x) * kWarps + w) / workers;
    if (mine > 0 && from >= before * items && from < (before + mine) * items) {
      long long at = before;
      for (int r = r0; r < r1; ++r) {
        bool b;
        const int tokens = row_tokens(a, r, &b), tiles = (tokens + kTok - 1) / kTok;
        if (from < (at + tiles) * items) {
          const int item = static_cast<int>((from - at * items) / tiles);
          s_first[w] = Segment{r, item, at * items + static_cast<long long>(item) * tiles, tiles, tokens};
          break;
        }
        at += tiles;
      }
    }
  }
  // rows without tokens
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
    bool b;
    if (row_tokens(a, r, &b) == 0)
      for (int i = tid; i < a.heads * dim / 4; i += kThreads)
        reinterpret_cast<float4*>(a.out + r * a.out_stride)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __syncthreads();

  const long long worker = static_cast<long long>(blockIdx.x) * kWarps + warp;
  const long long begin = total * worker / workers, end = total * (worker + 1) / workers;
  const auto heads_of = [&](int item) { return min(kGroup, a.group - item % a.chunks * kGroup); };
  const auto head_of = [&](int item) { return item / a.chunks * a.group + item % a.chunks * kGroup; };

  if (begin < end) {
    Walk<kTok> load;
    load.s = s_first[warp];
    load.at = begin;
    load.end = end;
    // places of the next tile's tokens: 16-byte units from the layer's first element, -1: none
    long long place[kPer];
    const auto look_up = [&]() {
      const Segment& s = load.s;
      const int t0 = static_cast<int>(load.at - s.start) * kTok;
      const int seq = a.seq ? a.seq[s.row] : s.row;
      const int* table = a.page_table + seq * a.table_stride;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int t = t0 + lane + 32 * i;
        place[i] = -1;
        if (lane + 32 * i < kTok && t < s.tokens) {
          const unsigned col = divide(t, a.page_div);
          const int page = table[col];
          if (page >= 0 && page < cache.pages)
            place[i] = page * cache.page_stride + (t - col * a.page_div.by) * cache.slot_stride;
          else
            record_device_error(kDevPageRange);
        }
      }
    };
    const auto issue = [&](int slot) {
      const Segment& s = load.s;
      unsigned long long live = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        live |= static_cast<unsigned long long>(__ballot_sync(0xffffffffu, place[i] >= 0)) << (32 * i);
      if (lane == 0) {
        int flags = 0;
        if (load.at == s.start || load.at == begin) flags |= kFirst;
        if (load.at + 1 == s.start + s.tiles || load.at + 1 == end) flags |= kLast;
        if (s.start >= begin && s.start + s.tiles <= end) flags |= kWhole;
        s_info[warp][slot] = TileInfo{live, s.start, s.row, s.item, s.tiles, flags};
      }
      const long long head = s.item / a.chunks * cache.head_stride;
      unsigned char* to = ring + slot * kStageBytes;
      constexpr int kRowsAtOnce = 32 / kChunks > 0 ? 32 / kChunks : 1;
      constexpr int kWide = kChunks > 32 ? kChunks / 32 : 1;
      const int chunk = lane % kChunks;
      constexpr int kVec = 16 / sizeof(T);
#pragma unroll
      for (int i = 0; i < kTok / kRowsAtOnce; ++i) {
        const int t = i * kRowsAtOnce + (kChunks < 32 ? lane / kChunks : 0);
        const long long at = __shfl_sync(0xffffffffu, place[i * kRowsAtOnce / 32], t & 31);
        const bool on = at >= 0;
        const long long off = on ? at + head : 0;
#pragma unroll
        for (int j = 0; j < kWide; ++j) {
          const int k = chunk + 32 * j;
          if (k < live_chunks) {
            unsigned char* p = to + (t * kChunks + (k ^ (t & 7))) * 16;
            cp_async16(p, cache.k + off + k * kVec, on);
            cp_async16(p + kTok * kChunks * 16, cache.v + off + k * kVec, on);
          }
        }
      }
    };
    const auto next = [&](int slot) {
      if (load.at < end) {
        issue(slot);
        load.advance(a, items);
        if (load.at < end) look_up();
      }
      cp_async_commit();
    };
    look_up();
    for (int i = 0; i < kStages - 1; ++i) next(i);
    Math math;
    int slot = 0, ahead = kStages - 1;
    bool one_held = false;
    for (long long at = begin; at < end; ++at) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      const TileInfo info = s_info[warp][slot];
      next(ahead);
      const int heads = heads_of(info.item);
      const long long first = static_cast<long long>(head_of(info.item)) * dim;
      if (info.flags & kFirst) math.begin(a, a.q + info.row * a.q_stride + first, heads, dim, scratch);
      math.tile(ring + slot * kStageBytes, info.live, scratch);
      if (info.flags & kLast) {
        if (info.flags & kWhole) {
          math.store(a.out + info.row * a.out_stride + first, heads, dim);
        } else {
          const int h = 2 * warp + one_held;
          one_held = true;
          math.store(pieces[h]);
          if (lane == 0) s_held[h] = Held{info.start, info.row, info.item, info.tiles, 1};
        }
      }
      slot = slot + 1 == kStages ? 0 : slot + 1;
      ahead = ahead + 1 == kStages ? 0 : ahead + 1;
    }
    cp_async_wait<0>();
  }
  __syncthreads();

  // ---- the join -------------------------------------------------------------------
  const long long cta_begin = total * blockIdx.x / gridDim.x, cta_end = total * (blockIdx.x + 1) / gridDim.x;
  int p = 0;
  while (p < 2 * kWarps) {
    if (!s_held[p].used) {
      ++p;
      continue;
    }
    const Held held = s_held[p];
    unsigned members = 0;  // this CTA's pieces of the segment
    for (; p < 2 * kWarps && (!s_held[p].used || s_held[p].start == held.start); ++p)
      if (s_held[p].used) members |= 1u << p;
    const int heads = heads_of(held.item);
    float* out = a.out + held.row * a.out_stride + static_cast<long long>(head_of(held.item)) * dim;
    const bool whole = held.start >= cta_begin && held.start + held.tiles <= cta_end;
    Piece<kDim>* mine_out =
        reinterpret_cast<Piece<kDim>*>(a.partials) + 2 * blockIdx.x + (held.start >= cta_begin && held.start != cta_begin ? 1 : 0);
    for (int i = tid; i < heads * (kDim / 4); i += kThreads) {
      const int h = i / (kDim / 4), e = 4 * (i % (kDim / 4));
      float top = -INFINITY, sum_l = 0.f;
      for (unsigned b = members; b; b &= b - 1) top = fmaxf(top, pieces[__ffs(b) - 1].m[h]);
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      for (unsigned b = members; b; b &= b - 1) {
        const Piece<kDim>& x = pieces[__ffs(b) - 1];
        const float w = piece_weight(x.m[h], top, x.c[h]);
        const float4 v = *reinterpret_cast<const float4*>(&x.o[h][e]);
        sum_l = fmaf(w, x.l[h], sum_l);
        y = make_float4(fmaf(w, v.x, y.x), fmaf(w, v.y, y.y), fmaf(w, v.z, y.z), fmaf(w, v.w, y.w));
      }
      if (whole) {
        const float inv = sum_l == 0.f ? 0.f : 1.f / sum_l;
        if (e < dim)
          *reinterpret_cast<float4*>(out + h * dim + e) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
      } else {
        *reinterpret_cast<float4*>(&mine_out->o[h][e]) = y;
        if (e == 0) {
          mine_out->m[h] = top;
          mine_out->l[h] = sum_l;
          mine_out->c[h] = pieces[__ffs(members) - 1].c[h];
        }
      }
    }
    if (whole) continue;
    // the CTAs that hold tiles of the segment: all from the first to the last, or one a tile when there are
    // more CTAs than tiles
    const auto cta_of = [&](long long tile) { return ((tile + 1) * gridDim.x - 1) / total; };
    const long long first_cta = cta_of(held.start);
    const bool sparse = total < gridDim.x;
    const int parts = sparse ? held.tiles : static_cast<int>(cta_of(held.start + held.tiles - 1) - first_cta) + 1;
    __syncthreads();
    if (tid == 0) {
      __threadfence();
      // wraps to zero at the last arrival: ready for the next call
      s_last = atomicInc(a.arrivals + static_cast<long long>(held.row) * items + held.item, parts - 1) ==
               static_cast<unsigned>(parts - 1);
      __threadfence();
    }
    __syncthreads();
    if (s_last) {
      const Piece<kDim>* from = reinterpret_cast<const Piece<kDim>*>(a.partials);
      const auto part = [&](int i) {
        const long long cta = sparse ? cta_of(held.start + i) : first_cta + i;
        const long long b = total * cta / gridDim.x;
        return from + 2 * cta + (held.start > b ? 1 : 0);
      };
      for (int i = tid; i < heads * (kDim / 4); i += kThreads) {
        const int h = i / (kDim / 4), e = 4 * (i % (kDim / 4));
        if (e >= dim) continue;
        float top = -INFINITY, sum_l = 0.f;
        for (int k = 0; k < parts; ++k) top = fmaxf(top, __ldcg(&part(k)->m[h]));
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < parts; ++k) {
          const Piece<kDim>* x = part(k);
          const float w = piece_weight(__ldcg(&x->m[h]), top, __ldcg(&x->c[h]));
          const float4 v = __ldcg(reinterpret_cast<const float4*>(&x->o[h][e]));
          sum_l = fmaf(w, __ldcg(&x->l[h]), sum_l);
          y = make_float4(fmaf(w, v.x, y.x), fmaf(w, v.y, y.y), fmaf(w, v.z, y.z), fmaf(w, v.w, y.w));
        }
        const float inv = sum_l == 0.f ? 0.f : 1.f / sum_l;
        *reinterpret_cast<float4*>(out + h * dim + e) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
      }
    }
    __syncthreads();
  }
}

template <typename Math, typename T, int kDim, int kStages>
int launch_math(Args a, const mli_attention_op& op, const mli_kv_cache& cache, int layer, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  const DeviceInfo& dev = current_device(&e);
  if (e != cudaSuccess) return check_cuda(e);
  const size_t smem = static_cast<size_t>(kWarps) * kStages * kStageBytes + 2 * kWarps * sizeof(Piece<kDim>) +
                      (sizeof(T) == 4 ? kWarps * (kGroup * kDim + Math::kTok * kGroup) * sizeof(float) : 0);
  auto kernel = paged_attention_kernel<Math, T, kDim, kStages>;
  e = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return check_cuda(e);
  // no more CTAs than tiles can be
  const long long most = static_cast<long long>(op.rows) * cache.kv_heads * a.chunks;
  const long long tiles = (a.room + Math::kTok - 1) / Math::kTok;
  int grid = dev.sm_count < kMaxCtas ? dev.sm_count : kMaxCtas;
  if (most < grid && most * tiles < grid) grid = static_cast<int>(most * tiles);
  return check_cuda(launch(kernel, dim3(grid), dim3(kThreads), smem, stream, true, a, cache_layer<T>(cache, layer)));
}

template <typename T, int kDim>
int launch_dim(const Args& a, const mli_attention_op& op, const mli_kv_cache& cache, int layer, cudaStream_t s) {
  // stages: what is left of 227 KB beside the pieces, at most 3
  constexpr int kStages = kDim == 256 ? 2 : 3;
  const bool few = a.group <= 4;
  if constexpr (sizeof(T) == 4) {
    constexpr int kFloatStages = 2;
    return few ? launch_math<FloatMath<kDim, true>, T, kDim, kFloatStages>(a, op, cache, layer, s)
               : launch_math<FloatMath<kDim, false>, T, kDim, kFloatStages>(a, op, cache, layer, s);
  } else {
    return few ? launch_math<TensorMath<T, kDim, true>, T, kDim, kStages>(a, op, cache, layer, s)
               : launch_math<TensorMath<T, kDim, false>, T, kDim, kStages>(a, op, cache, layer, s);
  }
}

template <typename T>
int launch_attention(const Args& a, const mli_attention_op& op, const mli_kv_cache& cache, int layer, cudaStream_t s) {
  return cache.head_dim <= 64    ? launch_dim<T, 64>(a, op, cache, layer, s)
         : cache.head_dim <= 128 ? launch_dim<T, 128>(a, op, cache, layer, s)
                                 : launch_dim<T, 256>(a, op, cache, layer, s);
}

// The same for every head size, so that the arrivals' place does not depend on it: what one call leaves
// in the partial results is never another's counter.
constexpr size_t kPartialBytes = 2 * kMaxCtas * sizeof(Piece<kMaxHeadDim>);

}  // namespace
}  // namespace mli

using namespace mli;

extern "C" {

size_t mli_paged_attention_workspace_bytes(int rows, int heads, int kv_heads, int head_dim) {
  if (rows <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || head_dim <= 0 || head_dim > kMaxHeadDim) return 0;
  const size_t items = static_cast<size_t>(kv_heads) * ((heads / kv_heads + kGroup - 1) / kGroup);
  return kPartialBytes + (items * rows * sizeof(unsigned) + 15) / 16 * 16;
}

int mli_paged_attention(const mli_attention_op* op, const mli_kv_cache* cache, int layer, void* stream) {
  const int bad = check_cache(cache);
  if (bad == MLI_ERR_INVALID_ARG || !op || layer < 0 || layer >= cache->layers) return set_status(MLI_ERR_INVALID_ARG);
  if (!op->out || !op->q || !op->lengths || !op->page_table || !op->workspace || op->rows <= 0 || op->heads <= 0 ||
      op->heads % cache->kv_heads || !(op->scale > 0.f) || !isfinite(op->scale) || op->table_rows <= 0 ||
      op->table_cols <= 0 || op->table_stride < op->table_cols || (!op->seq && op->rows > op->table_rows))
    return set_status(MLI_ERR_INVALID_ARG);
  const long long row = static_cast<long long>(op->heads) * cache->head_dim;
  if (op->q_stride < row || op->out_stride < row) return set_status(MLI_ERR_INVALID_ARG);
  if (bad != MLI_OK || !aligned_rows(op->q, op->q_stride) || !aligned_rows(op->out, op->out_stride) ||
      !aligned(op->workspace, 16))
    return set_status(MLI_ERR_UNSUPPORTED);
  if (op->workspace_bytes <
      mli_paged_attention_workspace_bytes(op->rows, op->heads, cache->kv_heads, cache->head_dim))
    return set_status(MLI_ERR_INVALID_ARG);
  Args a = {};
  a.q = op->q;
  a.out = op->out;
  a.q_stride = op->q_stride;
  a.out_stride = op->out_stride;
  a.lengths = op->lengths;
  a.seq = op->seq;
  a.page_table = op->page_table;
  a.table_stride = op->table_stride;
  a.rows = op->rows;
  a.heads = op->heads;
  a.table_rows = op->table_rows;
  a.room = static_cast<long long>(op->table_cols) * cache->page_size;
  a.group = op->heads / cache->kv_heads;
  a.chunks = (a.group + kGroup - 1) / kGroup;
  a.scale = fmaxf(op->scale * 1.4426950408889634f, FLT_MIN);  // log2(e)
  a.page_div = fast_div(cache->page_size);
  a.partials = static_cast<float*>(op->workspace);
  a.arrivals = reinterpret_cast<unsigned*>(static_cast<char*>(op->workspace) + kPartialBytes);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (cache->dtype) {
    case MLI_KV_F32: return launch_attention<float>(a, *op, *cache, layer, s);
    case MLI_KV_F16: return launch_attention<__half>(a, *op, *cache, layer, s);
    default: return launch_attention<__nv_bfloat16>(a, *op, *cache, layer, s);
  }
}

}  // extern "C"
