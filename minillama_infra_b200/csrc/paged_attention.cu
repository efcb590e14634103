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
// Each warp streams its tiles through a ring of its own in shared memory, a
// slot for a tile's keys, the next for its values (16-byte cp.async, chunks of a
// row permuted by its number so that column reads do not collide); warps never
// wait for one another before the join.  Slots of 8 KB with three to a warp and
// eight warps keep up to 192 KB a SM under way; four warps with 16 KB tiles of keys and
// values together reached 3.4 TB/s on the first line below.
//
// Bound by HBM: 4 products a 16-bit value read with 4 query heads a key-value
// head.  Measured on one B200 whose copies run at 6.48 TB/s, calls captured one after
// another, data not in L2:
//   1 row of 131072 tokens, 24 / 8 heads of 128, bf16         91 us   5.90 TB/s
//   64 rows of 0..8192 tokens, same heads                     174 us   6.15 TB/s
//   64 rows of 4096, 64 / 8 heads of 128, bf16                175 us   6.14 TB/s
//   32 rows of 4096, 32 / 4 heads of 256, bf16                115 us   4.67 TB/s
//   64 rows of 2048, 32 / 8 heads of 128, fp32                174 us   6.17 TB/s
//   64 rows of 2048, 64 / 8 heads of 128, fp32                218 us   4.93 TB/s
//   64 rows of 2048, 128 / 8 heads of 128, bf16 (two passes)  168 us   3.20 TB/s of the bytes of one
//   16 rows of 1..4096, 32 / 8 heads of 64, bf16               19 us   3.69 TB/s
//   1 row of 53, 32 / 8 heads of 64, fp32                       6 us
// A call's first bytes are asked for after 2 us (lengths, the search of each warp's place, the page
// table: one after another), its joins take 1 to 3 us; equal shares do not end at once (63 to 89 us for the
// first line: SMs get unequal bandwidth).  Eight heads of 256, and of fp32, have fewer warps: their queries
// and pieces take the shared memory.
#include <float.h>
#include <math.h>

#include <type_traits>

#include "kv_cache.cuh"

namespace mli {
namespace {

constexpr int kGroup = 8;         // query heads that share a pass over a segment
constexpr int kSlotBytes = 8192;  // one tile's keys, or its values
constexpr int kSlots = 3;         // of a warp's ring
constexpr int kMaxCtas = 160;     // CTAs with partial results in the workspace
// Of a row, so that the numbers of a last tile's tokens (64 at most), counted on from here, are ints.
constexpr long long kMaxTokens = (1ll << 31) - 64;

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

// Keys and values pass through L2 once a step: marked to be evicted first, they leave the page table, the queries,
// the partial results and the kernel's own code there.
__device__ __forceinline__ unsigned long long stream_policy() {
  unsigned long long p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void cp_async16(unsigned smem, const void* src, unsigned long long policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(smem), "l"(src), "l"(policy)
               : "memory");
}
// The same where `live`, else zeros, the source not read.
__device__ __forceinline__ void cp_async16(unsigned smem, const void* src, unsigned long long policy, bool live) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(smem), "l"(src),
               "r"(live ? 16 : 0), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// atomicInc that publishes what the CTA wrote before a barrier, and sees what earlier arrivals published.
__device__ __forceinline__ unsigned arrive(unsigned* p, unsigned most) {
  unsigned old;
  asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(most) : "memory");
  return old;
}

// Reads of another CTA's part from L2.
__device__ __forceinline__ float read_l2(const float* p) {
  float x;
  asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(x) : "l"(p) : "memory");
  return x;
}
__device__ __forceinline__ float4 read_l2_4(const float* p) {
  float4 x;
  asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "l"(p)
               : "memory");
  return x;
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
  long long room;  // tokens a page-table row can name, kMaxTokens at most
  int group;       // query heads of a key-value head
  int chunks;      // passes of up to kGroup of them
  float scale;     // times log2(e)
  FastDiv page_div;
  void* partials;      // [kMaxCtas][2] pieces
  unsigned* arrivals;  // [rows * kv_heads * chunks], zero between calls
};

// A piece of a segment: of each head the unnormalised output, the maximum, the sum and c.
template <int kDim, int kHeads>
struct Piece {
  float o[kHeads][kDim];
  float m[kHeads], l[kHeads], c[kHeads];
  float weight[kHeads], top[kHeads];  // beside the other pieces of its CTA, and their maximum
};
// What a piece of maximum m counts beside one of maximum top (no piece: 1, and its sums are zero).
__device__ __forceinline__ float piece_weight(float m, float top, float c) {
  return exp2_approx(m == top ? 0.f : (m - top) * c);
}

// ---- the products on the tensor cores, 16-bit caches --------------------------
//
// S = q K^T and O = p V as m16n8k16 products with fp32 accumulation.  q and p
// keep all their fp32 bits: each is the sum of three 16-bit numbers (8 bits
// each in bf16, 11 in fp16), and the rows of the left operand that a decode
// step would leave empty carry the parts: rows 0-7 the first of 8 heads, 8-15
// the second, and a second product the third.  With up to 4 heads rows 0-3, 8-11
// and 12-15 take all three in one product (128 -> 64 products a tile of 32 tokens of 128).  Powers of two keep the parts
// in range: a head's q is scaled so that its largest value has exponent 14 (fp16) or 0 (bf16), p in fp16 by 2^15.  What the
// third part cannot hold then lies below 2^-39 or 2^-133 of the largest query, and 2^-40 or 2^-134 of the largest weight.
// The tensor pipe is busy a fifth of the time: the fifth-generation instruction's 128-row tiles would hold at most 8
// queries here, and have the values' tile transposed.
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
};
// d = a b, or d += a b
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                    unsigned b1, bool fresh) {
  const float c[4] = {fresh ? 0.f : d[0], fresh ? 0.f : d[1], fresh ? 0.f : d[2], fresh ? 0.f : d[3]};
  if constexpr (std::is_same<T, __half>::value)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

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
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(unsigned (&r)[4], unsigned addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// Shared address of chunk `chunk ^ row & 7` given that of chunk `x` of the same row, x < 8 (rows begin on 128 bytes).
__device__ __forceinline__ unsigned swizzled(unsigned first, int chunk) {
  return (first ^ ((chunk & 7) << 4)) + ((chunk >> 3) << 7);
}

// kDim: the head dimension's room in shared memory (64, 128 or 256), the first kUsed of it multiplied.  kFew: at most
// 4 heads.
template <typename T, int kDim, int kUsed, bool kFew>
struct TensorMath {
  static constexpr int kTok = kSlotBytes / (kDim * 2);  // 64, 32 or 16 tokens a tile
  static constexpr int kHeads = kFew ? 4 : 8;
  static constexpr int kSteps = kUsed / 16;
  // The third parts of 8 heads' queries of 128 dims and more do not fit in registers beside the rest: they are in shared
  // memory, which costs a warp (64 rows of 4096, 64 / 8 heads of 128: 175 us, spilling them 181; 32 rows, 32 / 4 heads
  // of 256: 116 and 130; 256 rows of 100, 64 / 8 heads of 128: 37.7 and 36.4).  The kernels for 256 dims but that of 8 heads
  // in fp16 still spill 20 bytes.
  static constexpr bool kThirdShared = kUsed >= 128 && !kFew;
  static constexpr int kScratch = kThirdShared ? kSteps * 64 : 0;
  static constexpr int kReadBytes = kUsed * 2;  // of a token
  static constexpr float kUp = std::is_same<T, __half>::value ? 32768.f : 1.f;
  static constexpr int kTop = std::is_same<T, __half>::value ? 14 : 0;
  using Part = Piece<kDim, kHeads>;

  unsigned q[kSteps][kFew || kThirdShared ? 4 : 6];
  unsigned p[kTok / 8][kFew ? 2 : 3];
  float2 o[kUsed / 8];
  float m, l, c, keep;
  int head;  // this lane's head within the pass
  bool third;

  // A pass begins: its queries are read and taken apart.
  __device__ __forceinline__ void begin(const float* qp, int heads, int dim, float scale, float* scratch) {
    const int lane = threadIdx.x & 31, g = lane >> 2, col = 2 * (lane & 3);
    head = kFew ? g & 3 : g;
    third = kFew && g >= 4;
    const float* row = qp + head * dim;
    const bool live = head < heads;
    constexpr int kBatch = kSteps < 8 ? kSteps : 8;  // steps whose reads are under way at once
    float2 x[kBatch][2];
    const auto read = [&](int k0) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int e = 16 * (k0 + k) + 8 * j + col;
          x[k][j] = live && e < dim ? *reinterpret_cast<const float2*>(row + e) : make_float2(0.f, 0.f);
        }
    };
    float top = 0.f;
#pragma unroll
    for (int k0 = kSteps - kBatch; k0 >= 0; k0 -= kBatch) {
      read(k0);
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) top = fmaxf(top, fmaxf(fabsf(x[k][j].x), fabsf(x[k][j].y)));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // A power of two, of exponent f - 127, that takes the largest query to exponent kTop; c is divided by it and stays a
    // normal number: where that holds f back, what the parts lose changes a score times c by less than 2^-100.
    const int exponent = (__float_as_int(top) >> 23) & 255;
    const int f = exponent == 255 ? 127
                                  : max(1, min(min(254 + kTop - exponent, 253), 126 + (__float_as_int(scale) >> 23)));
    const float up = __int_as_float(f << 23);
    c = fminf(scale * __int_as_float((254 - f) << 23), FLT_MAX);
#pragma unroll
    for (int k0 = 0; k0 < kSteps; k0 += kBatch) {
      if (k0 > 0) read(k0);  // the maximum's last batch is the first
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          unsigned hi, mid, lo;
          split3<T>(x[k][j].x * up, x[k][j].y * up, hi, mid, lo);
          q[k0 + k][2 * j] = third ? 0u : hi;
          q[k0 + k][2 * j + 1] = third ? lo : mid;
          if constexpr (kThirdShared)
            reinterpret_cast<unsigned*>(scratch)[(k0 + k) * 64 + 2 * lane + j] = lo;
          else if constexpr (!kFew)
            q[k0 + k][4 + j] = lo;
        }
    }
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < kUsed / 8; ++i) o[i] = make_float2(0.f, 0.f);
  }

  // The tile's weights from its keys.  live: bit t for token t.  A score runs through 4 to 32 products one after another,
  // whose fp32 sums the tensor cores truncate.  That is left so: at its worst, values of one sign in 256 dims, a score is
  // off by 2.1 u of sum |q k| in the root mean square (u = 2^-24), the fp32 product of the plain form by 5.7 u.
  __device__ __forceinline__ void scores(unsigned keys, unsigned long long live, const float* scratch) {
    const int lane = threadIdx.x & 31, mat = lane >> 3, in = lane & 7;
    float s[kTok / 8][4];
    // matrices (tokens 0-7, 8-15) x (dims 0-7, 8-15) of a 16-token block
    const unsigned row = keys + ((mat >> 1) * 8 + in) * (kDim * 2) + (((mat & 1) ^ in) << 4);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const unsigned at = swizzled(row, 2 * k);
      uint2 third_part = make_uint2(0u, 0u);
      if constexpr (kThirdShared)
        third_part = reinterpret_cast<const uint2*>(scratch)[k * 32 + lane];
      else if constexpr (!kFew)
        third_part = make_uint2(q[k][4], q[k][5]);
#pragma unroll
      for (int n = 0; n < kTok / 16; ++n) {
        unsigned b[4];
        ldmatrix4(b, at + n * 16 * (kDim * 2));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float(&d)[4] = s[2 * n + h];
          mma<T>(d, q[k][0], q[k][1], q[k][2], q[k][3], b[2 * h], b[2 * h + 1], k == 0);
          if (!kFew) mma<T>(d, third_part.x, 0u, third_part.y, 0u, b[2 * h], b[2 * h + 1], false);
        }
      }
    }
    constexpr unsigned long long kAll = ~0ull >> (64 - kTok);
    float top = m;
#pragma unroll
    for (int n = 0; n < kTok / 8; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x = s[n][j] + s[n][j + 2];
        if (kFew) x += __shfl_xor_sync(0xffffffffu, x, 16);
        s[n][j] = x;
      }
    if (live != kAll) {
      const unsigned long long mine = live >> (2 * (lane & 3));
#pragma unroll
      for (int n = 0; n < kTok / 8; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) s[n][j] = (mine >> (8 * n + j)) & 1 ? s[n][j] : -INFINITY;
    }
#pragma unroll
    for (int n = 0; n < kTok / 8; ++n) top = fmaxf(top, fmaxf(s[n][0], s[n][1]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float base = top == -INFINITY ? 0.f : top;
    keep = exp2_approx((m - base) * c);  // m = -inf: 0
    m = top;
    l *= keep;
#pragma unroll
    for (int n = 0; n < kTok / 8; ++n) {
      const float x = exp2_approx((s[n][0] - base) * c), y = exp2_approx((s[n][1] - base) * c);
      l += x + y;
      unsigned hi, mid, lo;
      split3<T>(x * kUp, y * kUp, hi, mid, lo);
      p[n][0] = third ? 0u : hi;
      p[n][1] = third ? lo : mid;
      if (!kFew) p[n][2] = lo;
    }
  }

  // The tile's outputs from its values.  A tile's sum starts from zero, so that the tensor cores' accumulation
  // (which truncates) never runs over more than a tile.
  __device__ __forceinline__ void outputs(unsigned values, const float*) {
    const int lane = threadIdx.x & 31, mat = lane >> 3, in = lane & 7;
    const unsigned row = values + ((mat & 1) * 8 + in) * (kDim * 2) + (((mat >> 1) ^ in) << 4);
    const float2 keep2 = make_float2(keep, keep);
#pragma unroll
    for (int d = 0; d < kSteps; ++d) {
      float acc[2][4];
      const unsigned at = swizzled(row, 2 * d);
#pragma unroll
      for (int n = 0; n < kTok / 16; ++n) {
        unsigned b[4];
        ldmatrix4_trans(b, at + n * 16 * (kDim * 2));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mma<T>(acc[h], p[2 * n][0], p[2 * n][1], p[2 * n + 1][0], p[2 * n + 1][1], b[2 * h], b[2 * h + 1],
                 n == 0);
          if (!kFew) mma<T>(acc[h], p[2 * n][2], 0u, p[2 * n + 1][2], 0u, b[2 * h], b[2 * h + 1], false);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
        o[2 * d + h] = fma2(o[2 * d + h], keep2,
                            add2(make_float2(acc[h][0], acc[h][1]), make_float2(acc[h][2], acc[h][3])));
    }
  }

  // The sums over lanes; after it lane (head, col) of the first parts holds dims 8 i + col, + 1.
  __device__ __forceinline__ void finish() {
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (kFew) {
#pragma unroll
      for (int i = 0; i < kUsed / 8; ++i) {
        o[i].x += __shfl_xor_sync(0xffffffffu, o[i].x, 16);
        o[i].y += __shfl_xor_sync(0xffffffffu, o[i].y, 16);
      }
    }
  }
  __device__ __forceinline__ void store(float* out, int heads, int dim) {
    finish();
    if (third || head >= heads) return;
    const float inv = l == 0.f ? 0.f : 1.f / (l * kUp);
    float* row = out + head * dim + 2 * (threadIdx.x & 3);
#pragma unroll
    for (int i = 0; i < kUsed / 8; ++i)
      if (8 * i < dim) *reinterpret_cast<float2*>(row + 8 * i) = make_float2(o[i].x * inv, o[i].y * inv);
  }
  __device__ __forceinline__ void store(Part& to) {
    finish();
    if (third) return;
    const int col = 2 * (threadIdx.x & 3);
#pragma unroll
    for (int i = 0; i < kUsed / 8; ++i) *reinterpret_cast<float2*>(&to.o[head][8 * i + col]) = o[i];
    if (col == 0) {
      to.m[head] = m;
      to.l[head] = l * kUp;
      to.c[head] = c;
    }
  }
};

__device__ __forceinline__ const float4* shared_float4(unsigned addr) {
  return reinterpret_cast<const float4*>(__cvta_shared_to_generic(addr));
}

// ---- the products in fp32, fp32 caches ----------------------------------------
//
// A lane takes a part of the dims of two tokens for the scores; the lanes that share a token then share out its heads,
// each adding up and weighing its own.  For the outputs a lane takes four dims of a token (or eight) of all heads; q, p and
// the factor of the earlier outputs come from shared memory as broadcasts, p of 8 heads twice over, as the packed
// products take it.
template <int kDim, bool kFew>
struct FloatMath {
  static constexpr int kTok = kSlotBytes / (kDim * 4);  // 32, 16 or 8 tokens a tile
  static constexpr int kHeads = kFew ? 4 : 8;
  static constexpr int kCopies = kFew ? 1 : 2;  // of p
  static constexpr int kScratch = kHeads * (kDim + kTok * kCopies + 1);  // floats: q, the tile's p, a number a head
  static constexpr int kReadBytes = kDim * 4;  // of a token
  static constexpr int kLanes = kTok / 2;      // side by side in the scores, two tokens each
  static constexpr int kParts = 32 / kLanes;   // lanes that share a token's dims, then its heads
  static constexpr int kMine = kHeads > kParts ? kHeads / kParts : 1;  // heads of a lane
  static constexpr int kChunks = kDim / 4;     // 16-byte pieces of a token
  static constexpr int kRows = kChunks < 32 ? 32 / kChunks : 1;  // tokens side by side in the outputs' sum
  static constexpr int kOwn = kChunks < 32 ? 1 : kChunks / 32;   // pieces of a token a lane sums

  using Part = Piece<kDim, kHeads>;

  float2 o[kHeads][kOwn][2];
  float m[kMine], l[kMine], c;
  float* per_head;  // kHeads numbers in shared memory
  int base_head;    // this lane's first head
  bool owner;       // of its heads among lanes with the same tokens and heads

  __device__ __forceinline__ void begin(const float* qp, int heads, int dim, float scale, float* scratch) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kHeads * kChunks / 32; ++k) {
      const int i = lane + 32 * k, h = i / kChunks, e = 4 * (i % kChunks);
      reinterpret_cast<float4*>(scratch)[i] = h < heads && e < dim
                                                  ? *reinterpret_cast<const float4*>(qp + h * dim + e)
                                                  : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncwarp();
    c = scale;
    per_head = scratch + kHeads * (kDim + kTok * kCopies);
    base_head = 0;
    owner = true;
#pragma unroll
    for (int off = 16, half = kHeads / 2; off >= kLanes; off /= 2, half /= 2) {
      if (half > 0)
        base_head += lane & off ? half : 0;
      else
        owner = owner && !(lane & off);
    }
#pragma unroll
    for (int h = 0; h < kMine; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
    }
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
#pragma unroll
      for (int i = 0; i < kOwn; ++i) o[h][i][0] = o[h][i][1] = make_float2(0.f, 0.f);
  }

  __device__ __forceinline__ void scores(unsigned slot, unsigned long long live, float* scratch) {
    const int lane = threadIdx.x & 31;
    const float4* keys = shared_float4(slot);
    const float4* qs = reinterpret_cast<const float4*>(scratch);
    float* ps = scratch + kHeads * kDim;  // [kTok][kHeads][kCopies]
    const int t = lane % kLanes, part = lane / kLanes;
    float2 acc[2][kHeads][2];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int h = 0; h < kHeads; ++h) acc[r][h][0] = acc[r][h][1] = make_float2(0.f, 0.f);
    // of 8 neighbouring lanes with 4 tokens the two parts read pieces 4 apart: other banks
    const int first = kLanes < 8 ? (part & 1) * 4 + (part >> 1) : part;
#pragma unroll 2
    for (int k = first; k < kChunks; k += kParts) {
      const float4 x0 = keys[t * kChunks + (k ^ (t & 7))];
      const float4 x1 = keys[(t + kLanes) * kChunks + (k ^ ((t + kLanes) & 7))];
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        const float4 y = qs[h * kChunks + k];
        acc[0][h][0] = fma2(make_float2(x0.x, x0.y), make_float2(y.x, y.y), acc[0][h][0]);
        acc[0][h][1] = fma2(make_float2(x0.z, x0.w), make_float2(y.z, y.w), acc[0][h][1]);
        acc[1][h][0] = fma2(make_float2(x1.x, x1.y), make_float2(y.x, y.y), acc[1][h][0]);
        acc[1][h][1] = fma2(make_float2(x1.z, x1.w), make_float2(y.z, y.w), acc[1][h][1]);
      }
    }
    float s[2][kHeads];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        const float2 x = add2(acc[r][h][0], acc[r][h][1]);
        s[r][h] = x.x + x.y;
      }
    // each exchange adds another lane's part to half of the heads and gives away the other half
#pragma unroll
    for (int off = 16, half = kHeads / 2; off >= kLanes; off /= 2, half /= 2) {
      const bool upper = lane & off;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (half > 0) {
#pragma unroll
          for (int h = 0; h < half; ++h) {
            const float kept = upper ? s[r][h + half] : s[r][h], sent = upper ? s[r][h] : s[r][h + half];
            s[r][h] = kept + __shfl_xor_sync(0xffffffffu, sent, off);
          }
        } else {
          s[r][0] += __shfl_xor_sync(0xffffffffu, s[r][0], off);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < kMine; ++h) {
#pragma unroll
      for (int r = 0; r < 2; ++r) s[r][h] = (live >> (t + r * kLanes)) & 1 ? s[r][h] : -INFINITY;
      float top = fmaxf(s[0][h], s[1][h]);
#pragma unroll
      for (int off = kLanes / 2; off > 0; off /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      top = fmaxf(top, m[h]);
      const float base = top == -INFINITY ? 0.f : top;
      const float keep = exp2_approx((m[h] - base) * c);
      m[h] = top;
#pragma unroll
      for (int r = 0; r < 2; ++r) s[r][h] = exp2_approx((s[r][h] - base) * c);
      l[h] = fmaf(l[h], keep, s[0][h] + s[1][h]);
      if (owner) {
        if (t == 0) per_head[base_head + h] = keep;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float* to = ps + ((t + r * kLanes) * kHeads + base_head + h) * kCopies;
          if constexpr (kCopies == 2)
            *reinterpret_cast<float2*>(to) = make_float2(s[r][h], s[r][h]);
          else
            *to = s[r][h];
        }
      }
    }
    __syncwarp();
  }

  // The tile's outputs from its values.  Its sum starts from zero, so that a long share adds up tiles, not tokens.
  __device__ __forceinline__ void outputs(unsigned slot, float* scratch) {
    const int lane = threadIdx.x & 31;
    const float4* values = shared_float4(slot);
    const float4* ps = reinterpret_cast<const float4*>(scratch + kHeads * kDim);
    float2 acc[kHeads][kOwn][2];
    const int first = kRows > 1 ? lane / kChunks : 0, piece = kRows > 1 ? lane % kChunks : lane;
    const auto add = [&](int r, auto fresh) {  // token r's values
      const auto plus = [](float2 a, float2 b, float2 c) { return decltype(fresh)::value ? mul2(a, b) : fma2(a, b, c); };
      float4 x[kOwn];
#pragma unroll
      for (int i = 0; i < kOwn; ++i) x[i] = values[r * kChunks + ((piece + 32 * i) ^ (r & 7))];
      constexpr int kReads = kHeads * kCopies / 4, kEach = 4 / kCopies;  // of p, and heads of a read
#pragma unroll
      for (int g = 0; g < kReads; ++g) {
        const float4 p4 = ps[r * kReads + g];
        const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
        for (int h = 0; h < kEach; ++h)
#pragma unroll
          for (int i = 0; i < kOwn; ++i) {
            const float2 w = make_float2(p[h * kCopies], p[h * kCopies + kCopies - 1]);
            float2(&to)[2] = acc[g * kEach + h][i];
            to[0] = plus(w, make_float2(x[i].x, x[i].y), to[0]);
            to[1] = plus(w, make_float2(x[i].z, x[i].w), to[1]);
          }
      }
    };
    // Without an addition to zero first, and all the way unrolled (64 rows of 2048, 64 / 8 heads of 128: 218 us; zeroed sums
    // and four tokens a turn, 231).
    add(first, std::true_type());
#pragma unroll
    for (int r = kRows; r < kTok; r += kRows) add(first + r, std::false_type());
#pragma unroll
    for (int h4 = 0; h4 < kHeads / 4; ++h4) {
      const float4 k4 = reinterpret_cast<const float4*>(per_head)[h4];
      const float keep[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            o[4 * h4 + h][i][j] = fma2(o[4 * h4 + h][i][j], make_float2(keep[h], keep[h]), acc[4 * h4 + h][i][j]);
    }
    __syncwarp();  // ps and per_head are written again by the next tile
  }

  // The sums over lanes; after it every lane finds all heads' in per_head.
  __device__ __forceinline__ void finish() {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int h = 0; h < kMine; ++h) {
#pragma unroll
      for (int off = kLanes / 2; off > 0; off /= 2) l[h] += __shfl_xor_sync(0xffffffffu, l[h], off);
      if (owner && lane % kLanes == 0) per_head[base_head + h] = l[h];
    }
    if (kRows > 1) {
#pragma unroll
      for (int h = 0; h < kHeads; ++h)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int off = kChunks; off < 32; off *= 2) {
            o[h][0][j].x += __shfl_xor_sync(0xffffffffu, o[h][0][j].x, off);
            o[h][0][j].y += __shfl_xor_sync(0xffffffffu, o[h][0][j].y, off);
          }
    }
    __syncwarp();
  }
  __device__ __forceinline__ void store(float* out, int heads, int dim) {
    finish();
    const int lane = threadIdx.x & 31;
    if (kRows > 1 && lane >= kChunks) return;
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const float sum = per_head[h], inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int e = 4 * (lane + 32 * i);
        if (h < heads && e < dim)
          *reinterpret_cast<float4*>(out + h * dim + e) = make_float4(o[h][i][0].x * inv, o[h][i][0].y * inv,
                                                                      o[h][i][1].x * inv, o[h][i][1].y * inv);
      }
    }
  }
  __device__ __forceinline__ void store(Part& to) {
    finish();
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int h = 0; h < kMine; ++h)
      if (owner && lane % kLanes == 0) {
        to.m[base_head + h] = m[h];
        to.l[base_head + h] = l[h];
        to.c[base_head + h] = c;
      }
    if (kRows > 1 && lane >= kChunks) return;
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
        *reinterpret_cast<float4*>(&to.o[h][4 * (lane + 32 * i)]) =
            make_float4(o[h][i][0].x, o[h][i][0].y, o[h][i][1].x, o[h][i][1].y);
  }
};

// ---- the tiles of a call ---------------------------------------------------------
struct Row {
  int tokens;  // that it attends to: its length, cut to the page table; 0 if its sequence lies outside it
  int seq;     // its row of the page table
  bool bad;    // led outside the page table
};
__device__ __forceinline__ Row row_of(const Args& a, int r) {
  const int len = a.lengths[r], seq = a.seq ? a.seq[r] : r;
  if (len <= 0) return Row{0, 0, false};
  if (seq < 0 || seq >= a.table_rows) return Row{0, 0, true};
  return Row{len > a.room ? static_cast<int>(a.room) : len, seq, len > a.room};
}

// A segment's place among all tiles.
struct Segment {
  int start;      // first tile
  int row, item;  // item: key-value head * chunks + chunk
  int seq, tiles, tokens;
};

// Tiles [first, to) in equal shares: the first `more` of `among` take one more than the others.
struct Shares {
  int first, each, more;
  __device__ __forceinline__ Shares(int from, int to, int among) : first(from) {
    each = (to - from) / among;
    more = to - from - each * among;
  }
  __device__ __forceinline__ int begin(int i) const { return first + i * each + min(i, more); }
  __device__ __forceinline__ int owner(int tile) const {
    const int longer = more * (each + 1);
    tile -= first;
    return tile < longer ? tile / (each + 1) : more + (tile - longer) / each;
  }
};

// A piece that a CTA holds in shared memory.
struct Held {
  int start;  // the segment's first tile
  int row, item, tiles, used;
};

// Bytes of a warp, and how many of them an SM's 227 KB hold beside the static arrays and 128 bytes for alignment.
constexpr int kStaticBytes = 1408;
constexpr int kSmemRoom = 232448 - kStaticBytes - 128;
template <typename Math>
constexpr int kWarpBytes = kSlots * kSlotBytes + sizeof(typename Math::Part) + Math::kScratch * 4;
template <typename Math>
constexpr int kWarpsOf = kSmemRoom / kWarpBytes<Math> < 8 ? kSmemRoom / kWarpBytes<Math> : 8;

template <typename Math, typename T, int kDim>
__global__ void __launch_bounds__(kWarpsOf<Math> * 32, 1) paged_attention_kernel(const Args a,
                                                                                 const CacheLayer<T> cache) {
  using Part = typename Math::Part;
  constexpr int kWarps = kWarpsOf<Math>, kThreads = kWarps * 32;
  constexpr int kTok = Math::kTok;
  constexpr int kRowBytes = kDim * sizeof(T);
  constexpr int kChunks = kRowBytes / 16;          // 16-byte pieces of a token's keys
  constexpr int kPer = kTok > 32 ? kTok / 32 : 1;  // tokens whose place a lane looks up
  constexpr unsigned long long kAll = ~0ull >> (64 - kTok);

  extern __shared__ unsigned char smem_any[];
  __shared__ int s_scan[kWarps], s_before[kThreads];
  __shared__ Held s_held[2 * kWarps];
  __shared__ int s_last[2];
  static_assert(sizeof(s_scan) + sizeof(s_before) + sizeof(s_held) + sizeof(s_last) <= kStaticBytes, "static arrays");
  // the swizzle's exclusive-or works on addresses whose rows begin on 128 bytes
  unsigned char* smem = smem_any + (-smem_u32(smem_any) & 127u);
  // rings, then a piece of each warp, then its scratch.  A warp's second piece takes its ring, which is empty by then.
  Part* first_pieces = reinterpret_cast<Part*>(smem + kWarps * kSlots * kSlotBytes);
  const auto piece_at = [&](int i) {
    return i & 1 ? reinterpret_cast<Part*>(smem + (i >> 1) * (kSlots * kSlotBytes)) : first_pieces + (i >> 1);
  };

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned char* ring = smem + warp * (kSlots * kSlotBytes);
  float* scratch = reinterpret_cast<float*>(first_pieces + kWarps) + warp * Math::kScratch;
  const int dim = cache.head_dim, items = cache.kv_heads * a.chunks;
  const int live_chunks = dim * static_cast<int>(sizeof(T)) / 16;
  if (live_chunks * 16 < Math::kReadBytes) {  // columns that are multiplied, but that no token fills
    for (int i = lane; i < kSlots * kSlotBytes / 16; i += 32)
      reinterpret_cast<uint4*>(ring)[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  if (lane == 0) s_held[2 * warp].used = s_held[2 * warp + 1].used = 0;
  griddep_wait();
  griddep_launch_dependents();

  // Where each warp starts: thread i sums the tiles of rows [i n, (i + 1) n).
  const int n = (a.rows + kThreads - 1) / kThreads;
  int mine = 0;
  {
    bool bad = false;
    for (int r = tid * n; r < min(a.rows, (tid + 1) * n); ++r) {
      const Row row = row_of(a, r);
      mine += (row.tokens + kTok - 1) / kTok;
      bad |= row.bad;
    }
    if (bad && blockIdx.x == 0) record_device_error(kDevPageRange);
  }
  int sum = mine;
#pragma unroll
  for (int off = 1; off < 32; off *= 2) {
    const int x = __shfl_up_sync(0xffffffffu, sum, off);
    if (lane >= off) sum += x;
  }
  if (lane == 31) s_scan[warp] = sum;
  __syncthreads();
  int before = sum - mine, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += s_scan[w];
    all += s_scan[w];
  }
  s_before[tid] = before;
  const int total = all * items;
  // CTAs in use: no more than have four tiles each, so that short rows are joined within a CTA (16 rows of 64 tokens, 8
  // key-value heads of 128: 6.6 us, with eight tiles each 8.2, with one 8.5)
  const int ctas = min(static_cast<int>(gridDim.x), (total + 3) / 4);
  const int cta = blockIdx.x;
  const auto clear_empty_rows = [&]() {
    for (int r = cta; r < a.rows; r += gridDim.x)
      if (row_of(a, r).tokens == 0)
        for (int i = tid; i < a.heads * dim / 4; i += kThreads)
          reinterpret_cast<float4*>(a.out + r * a.out_stride)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  };
  if (cta >= ctas) {
    clear_empty_rows();
    return;
  }
  const Shares shares(0, total, ctas);
  const int cta_begin = shares.begin(cta), cta_end = shares.begin(cta + 1);
  const Shares warp_shares(cta_begin, cta_end, kWarps);
  const int begin = warp_shares.begin(warp), end = warp_shares.begin(warp + 1);
  // an item's key-value head, its first query head, and how many it has
  const auto kv_head_of = [&](int item) { return a.chunks == 1 ? item : item / a.chunks; };
  const auto head_of = [&](int item) {
    const int kv = kv_head_of(item);
    return kv * a.group + (item - kv * a.chunks) * kGroup;
  };
  const auto heads_of = [&](int item) { return min(kGroup, a.group - (item - kv_head_of(item) * a.chunks) * kGroup); };
  __syncthreads();

  if (begin < end) {
    // the segment of the warp's first tile: in the rows of the last thread that has no more tiles than that before it
    Segment load;  // of the tile to be loaded next
    {
      const int row_tile = begin / items;  // were every row one item
      int owner = -1;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) owner += __popc(__ballot_sync(0xffffffffu, s_before[32 * k + lane] <= row_tile));
      int before_row = s_before[owner], r = owner * n;
      Row row = row_of(a, r);
      int tiles = (row.tokens + kTok - 1) / kTok;
      while (row_tile >= before_row + tiles && r + 1 < a.rows) {
        before_row += tiles;
        row = row_of(a, ++r);
        tiles = (row.tokens + kTok - 1) / kTok;
      }
      const int start = before_row * items, item = min(items - 1, (begin - start) / max(1, tiles));
      load = Segment{start + item * tiles, r, item, row.seq, tiles, row.tokens};
    }
    int load_at = begin;
    long long place[kPer];  // bytes from the layer's first element to the lane's tokens of that tile; -1: none
    unsigned long long live = 0;
    const auto look_up = [&]() {
      const int t0 = (load_at - load.start) * kTok;
      const int* table = a.page_table + load.seq * a.table_stride;
      const long long head = kv_head_of(load.item) * cache.head_stride;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int t = t0 + lane + 32 * i;
        place[i] = -1;
        if (lane + 32 * i < kTok && t < load.tokens) {
          const unsigned col = divide(t, a.page_div);
          const int page = table[col];
          if (page >= 0 && page < cache.pages)
            place[i] = (page * cache.page_stride + (t - col * a.page_div.by) * cache.slot_stride + head) *
                       static_cast<long long>(sizeof(T));
          else
            record_device_error(kDevPageRange);
        }
      }
    };
    const auto advance = [&]() {
      if (++load_at < load.start + load.tiles || load_at >= end) return;
      load.start += load.tiles;
      if (++load.item < items) return;
      load.item = 0;
      Row row;
      do {
        row = row_of(a, ++load.row);
      } while (row.tokens == 0 && load.row + 1 < a.rows);
      load.tokens = row.tokens;
      load.seq = row.seq;
      load.tiles = (load.tokens + kTok - 1) / kTok;
    };
    // One tile's keys or values into a slot: each lane a 16-byte chunk of one row in kAtOnce.
    constexpr int kAtOnce = kChunks < 32 ? 32 / kChunks : 1, kWide = kChunks > 32 ? kChunks / 32 : 1;
    const int sub = kChunks < 32 ? lane / kChunks : 0, chunk = lane % kChunks;
    const unsigned lane_to = sub * kRowBytes + (((chunk & 7) ^ sub) << 4) + ((chunk >> 3) << 7);
    const unsigned long long policy = stream_policy();
    const auto fill = [&](int slot, const T* from) {
      const unsigned to = smem_u32(ring) + slot * kSlotBytes + lane_to;
      const char* src = reinterpret_cast<const char*>(from) + chunk * 16;
      const auto copy = [&](auto whole) {
#pragma unroll
        for (int i = 0; i < kTok / kAtOnce; ++i) {
          const long long at = __shfl_sync(0xffffffffu, place[i * kAtOnce / 32], (i * kAtOnce + sub) & 31);
          const unsigned p = swizzled(to, i * kAtOnce & 7) + i * kAtOnce * kRowBytes;
#pragma unroll
          for (int j = 0; j < kWide; ++j) {
            if (chunk + 32 * j >= live_chunks) continue;
            if constexpr (decltype(whole)::value)
              cp_async16(p + 512 * j, src + at + 512 * j, policy);
            else
              cp_async16(p + 512 * j, src + (at >= 0 ? at : 0) + 512 * j, policy, at >= 0);
          }
        }
      };
      if (live == kAll)
        copy(std::true_type());
      else
        copy(std::false_type());
    };
    const auto find_live = [&]() {
      live = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        live |= static_cast<unsigned long long>(__ballot_sync(0xffffffffu, place[i] >= 0)) << (32 * i);
    };
    const auto next_slot = [](int s) { return s + 1 == kSlots ? 0 : s + 1; };

    Math math;
    look_up();
    find_live();
    fill(0, cache.k);
    cp_async_commit();
    fill(1, cache.v);
    cp_async_commit();
    Segment now = load;
    unsigned long long now_live = live;
    advance();
    if (load_at < end) look_up();
    int slot = 0;
    for (int at = begin; at < end; ++at) {
      // a slot is filled again as soon as all lanes are done with it: two tiles' halves are under way while a third
      // is worked on
      __syncwarp();
      const int value_slot = next_slot(slot), free_slot = next_slot(value_slot);
      const bool more = load_at < end;
      if (more) {
        find_live();
        fill(free_slot, cache.k);
      }
      cp_async_commit();
      // the queries come while the keys do
      if (at == begin || at == now.start)
        math.begin(a.q + now.row * a.q_stride + static_cast<long long>(head_of(now.item)) * dim, heads_of(now.item), dim,
                   a.scale, scratch);
      cp_async_wait<2>();
      __syncwarp();
      math.scores(smem_u32(ring) + slot * kSlotBytes, now_live, scratch);
      __syncwarp();
      const Segment next = load;
      if (more) fill(slot, cache.v);
      cp_async_commit();
      const unsigned long long next_live = live;
      if (more) {
        advance();
        if (load_at < end) look_up();
      }
      cp_async_wait<2>();
      __syncwarp();
      math.outputs(smem_u32(ring) + value_slot * kSlotBytes, scratch);
      const int after = now.start + now.tiles;
      if (at + 1 == after || at + 1 == end) {
        if (now.start >= begin && after <= end) {
          math.store(a.out + now.row * a.out_stride + static_cast<long long>(head_of(now.item)) * dim,
                     heads_of(now.item), dim);
        } else {
          const int h = 2 * warp + (at + 1 == end);
          __syncwarp();  // every lane has read its last values
          math.store(*piece_at(h));
          if (lane == 0) s_held[h] = Held{now.start, now.row, now.item, now.tiles, 1};
        }
      }
      now = next;
      now_live = next_live;
      slot = free_slot;
    }
    cp_async_wait<0>();
  }
  clear_empty_rows();
  __syncthreads();

  // ---- the join -------------------------------------------------------------------
  // Every warp lists the segments that the CTA holds pieces of: lane i looks at piece i, and a group begins at each
  // piece whose segment is not that of the piece before.
  Held held = Held{0, 0, 0, 0, 0};
  if (lane < 2 * kWarps) held = s_held[lane];
  const unsigned used = __ballot_sync(0xffffffffu, held.used != 0);
  const unsigned below = used & ((1u << lane) - 1);
  const int left = __shfl_sync(0xffffffffu, held.start, below ? 31 - __clz(below) : lane);
  const unsigned firsts = __ballot_sync(0xffffffffu, held.used != 0 && (below == 0 || left != held.start));
  const int groups = __popc(firsts);
  const auto members_of = [&](int from) {  // of the group that begins at piece `from`
    const unsigned later = firsts & ~((2u << from) - 1);
    return used & ~((1u << from) - 1) & (later ? (later & -later) - 1 : ~0u);
  };
  // a thread a piece and head: what it weighs beside the others of its group
  for (int i = tid; i < 2 * kWarps * Math::kHeads; i += kThreads) {
    const int j = i / Math::kHeads, h = i % Math::kHeads;
    if (!((used >> j) & 1)) continue;
    const unsigned members = members_of(31 - __clz(firsts & ((2u << j) - 1)));
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < 2 * kWarps; ++k) top = fmaxf(top, (members >> k) & 1 ? piece_at(k)->m[h] : -INFINITY);
    piece_at(j)->weight[h] = piece_weight(piece_at(j)->m[h], top, piece_at(j)->c[h]);
    piece_at(j)->top[h] = top;
  }
  __syncthreads();
  const auto group_lane = [&](int g) {
    unsigned rest = firsts;
    for (; g > 0; --g) rest &= rest - 1;
    return __ffs(rest) - 1;
  };
  const auto group_held = [&](int from) {
    return Held{__shfl_sync(0xffffffffu, held.start, from), __shfl_sync(0xffffffffu, held.row, from),
                __shfl_sync(0xffffffffu, held.item, from), __shfl_sync(0xffffffffu, held.tiles, from), 1};
  };
  const auto out_of = [&](const Held& g) {
    return a.out + g.row * a.out_stride + static_cast<long long>(head_of(g.item)) * dim;
  };
  Part* parts = static_cast<Part*>(a.partials);
  constexpr int kQuads = kDim / 4, kItems = Math::kHeads * kQuads;  // a group's float4, a multiple of 32
  for (int i = tid; i < groups * kItems; i += kThreads) {
    const int from = group_lane(i / kItems);
    const Held g = group_held(from);
    const unsigned members = members_of(from);
    const int h = i % kItems / kQuads, e = 4 * (i % kQuads);
    if (h >= heads_of(g.item)) continue;
    float sum_l = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (unsigned rest = members; rest;) {  // four at a time
      float w[4], l[4];
      float4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool on = rest != 0;
        const Part& x = *piece_at(on ? __ffs(rest) - 1 : from);
        w[u] = x.weight[h];
        l[u] = x.l[h];
        v[u] = *reinterpret_cast<const float4*>(&x.o[h][e]);
        // one too many adds nothing, and no NaN
        if (!on) w[u] = l[u] = v[u].x = v[u].y = v[u].z = v[u].w = 0.f;
        rest &= rest - 1;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        sum_l = fmaf(w[u], l[u], sum_l);
        y = make_float4(fmaf(w[u], v[u].x, y.x), fmaf(w[u], v[u].y, y.y), fmaf(w[u], v[u].z, y.z),
                        fmaf(w[u], v[u].w, y.w));
      }
    }
    if (g.start >= cta_begin && g.start + g.tiles <= cta_end) {
      const float inv = sum_l == 0.f ? 0.f : 1.f / sum_l;
      if (e < dim)
        *reinterpret_cast<float4*>(out_of(g) + h * dim + e) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
    } else {
      // a CTA's first segment may have begun before it (slot 0), its last may go on behind it (slot 1)
      Part* to = parts + 2 * cta + (g.start > cta_begin ? 1 : 0);
      *reinterpret_cast<float4*>(&to->o[h][e]) = y;
      if (e == 0) {
        to->m[h] = piece_at(from)->top[h];
        to->l[h] = sum_l;
        to->c[h] = piece_at(from)->c[h];
      }
    }
  }
  // Only the first and the last segment can go beyond the CTA; of each, every CTA from that of its first tile to that
  // of its last holds a part.  The last of them to get here joins them, in order.
  const auto end_group = [&](int k) { return group_held(group_lane(k == 0 ? 0 : groups - 1)); };
  const auto beyond = [&](const Held& g) { return g.start < cta_begin || g.start + g.tiles > cta_end; };
  const Held ends[2] = {end_group(0), end_group(1)};
  const bool shared[2] = {groups > 0 && beyond(ends[0]), groups > 1 && beyond(ends[1])};
  if (!shared[0] && !shared[1]) return;
  int first_ctas[2], counts[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    first_ctas[k] = shared[k] ? shares.owner(ends[k].start) : 0;
    counts[k] = shared[k] ? shares.owner(ends[k].start + ends[k].tiles - 1) - first_ctas[k] + 1 : 0;
  }
  __syncthreads();
  if (tid < 2) {
    const Held g = tid == 0 ? ends[0] : ends[1];
    bool last = false;
    if (tid == 0 ? shared[0] : shared[1]) {
      const unsigned most = (tid == 0 ? counts[0] : counts[1]) - 1;
      // wraps to zero at the last arrival: ready for the next call
      last = arrive(a.arrivals + static_cast<long long>(g.row) * items + g.item, most) == most;
    }
    s_last[tid] = last;
  }
  __syncthreads();
  for (int i = tid; i < 2 * kItems; i += kThreads) {
    const int k = i / kItems, h = i % kItems / kQuads, e = 4 * (i % kQuads);
    const Held& g = k == 0 ? ends[0] : ends[1];
    if (!s_last[k] || h >= heads_of(g.item) || e >= dim) continue;
    const int first_cta = k == 0 ? first_ctas[0] : first_ctas[1], count = k == 0 ? counts[0] : counts[1];
    // slot 0 of all CTAs but the first, in which the segment may be the last one
    const Part* other = parts + 2 * first_cta;
    const Part* first_part = other + (g.start > shares.begin(first_cta) ? 1 : 0);
    const float c = read_l2(&first_part->c[h]);
    float top = -INFINITY, sum_l = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    int done = 0;
    const auto join = [&](auto batch) {  // parts whose reads are under way at once
      constexpr int kBatch = decltype(batch)::value;
      float m[kBatch], l[kBatch];
      float4 v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const Part* x = done + j == 0 ? first_part : other + 2 * min(done + j, count - 1);
        m[j] = read_l2(&x->m[h]);
        l[j] = read_l2(&x->l[h]);
        v[j] = read_l2_4(&x->o[h][e]);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        // one too many adds nothing, and no NaN; without a branch, behind which its reads would be moved
        const bool on = done + j < count;
        m[j] = on ? m[j] : -INFINITY;
        l[j] = on ? l[j] : 0.f;
        v[j] = make_float4(on ? v[j].x : 0.f, on ? v[j].y : 0.f, on ? v[j].z : 0.f, on ? v[j].w : 0.f);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const float both = fmaxf(top, m[j]);
        const float keep = piece_weight(top, both, c), w = piece_weight(m[j], both, c);
        top = both;
        sum_l = fmaf(sum_l, keep, w * l[j]);
        y = make_float4(fmaf(y.x, keep, w * v[j].x), fmaf(y.y, keep, w * v[j].y), fmaf(y.z, keep, w * v[j].z),
                        fmaf(y.w, keep, w * v[j].w));
      }
      done += kBatch;
    };
    while (done < count) {
      if (count - done > 4)
        join(std::integral_constant<int, 16>());
      else
        join(std::integral_constant<int, 4>());
    }
    const float inv = sum_l == 0.f ? 0.f : 1.f / sum_l;
    *reinterpret_cast<float4*>(out_of(g) + h * dim + e) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
  }
}

template <typename Math, typename T, int kDim>
int launch_math(const Args& a, const mli_attention_op& op, const mli_kv_cache& cache, int layer, cudaStream_t stream) {
  // tiles, were every row as long as its page table; they are counted in ints
  const double most = static_cast<double>(op.rows) * cache.kv_heads * a.chunks *
                      static_cast<double>((a.room + Math::kTok - 1) / Math::kTok);
  if (most > 2e9) return set_status(MLI_ERR_UNSUPPORTED);
  cudaError_t e = cudaSuccess;
  const DeviceInfo& dev = current_device(&e);
  if (e != cudaSuccess) return check_cuda(e);
  constexpr int kWarps = kWarpsOf<Math>;
  constexpr size_t kSmem = static_cast<size_t>(kWarps) * kWarpBytes<Math> + 128;
  auto kernel = paged_attention_kernel<Math, T, kDim>;
  e = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), kSmem);
  if (e != cudaSuccess) return check_cuda(e);
  const int sms = dev.sm_count < kMaxCtas ? dev.sm_count : kMaxCtas;
  const int grid = most < sms ? static_cast<int>(most) : sms;
  return check_cuda(
      launch(kernel, dim3(grid), dim3(kWarps * 32), kSmem, stream, true, a, cache_layer<T>(cache, layer)));
}

template <typename T, int kDim, int kUsed>
int launch_dim(const Args& a, const mli_attention_op& op, const mli_kv_cache& cache, int layer, cudaStream_t s) {
  // Half of the products where all heads of a pass fit beside their parts.  With the kernel for 4 heads and with the one
  // for 8, bf16: 256 rows of 100 tokens, 32 / 8 heads of 128, 27.8 and 34.2 us; 64 rows of 2048, 16 / 4 heads of 256, 96
  // and 111; 16 rows to 4096, 32 / 8 of 64, 18.5 and 20.2; bound by HBM, 64 rows of 4096, 32 / 8 of 128, 175 and 174, of
  // 2048 92.7 and 91.6.  fp32: 16 rows to 1024, 32 / 8 of 64, 13.3 and 18.1; 64 rows of 2048, 32 / 8 of 128, 174 and 213.
  const bool few = a.group <= 4;
  if constexpr (sizeof(T) == 4)
    return few ? launch_math<FloatMath<kDim, true>, T, kDim>(a, op, cache, layer, s)
               : launch_math<FloatMath<kDim, false>, T, kDim>(a, op, cache, layer, s);
  else
    return few ? launch_math<TensorMath<T, kDim, kUsed, true>, T, kDim>(a, op, cache, layer, s)
               : launch_math<TensorMath<T, kDim, kUsed, false>, T, kDim>(a, op, cache, layer, s);
}

template <typename T>
int launch_attention(const Args& a, const mli_attention_op& op, const mli_kv_cache& cache, int layer, cudaStream_t s) {
  const int dim = cache.head_dim;
  if (dim <= 64) return launch_dim<T, 64, 64>(a, op, cache, layer, s);
  // The tensor cores' share of a call goes by the dims they multiply: 80 and 96 have kernels of their own.  With them and
  // with the one for 128, bf16: 64 rows of 2048, 64 / 8 heads, 66 and 88 us of 80, 75 and 89 of 96; 256 rows of 100, 32 / 8
  // heads, 23.6 and 26.0 of 80, 25.2 and 26.6 of 96; bound by HBM, 64 rows of 4096, 32 / 8 heads, 118 and 117 of 80, 138
  // and 137 of 96.
  if constexpr (sizeof(T) == 2) {
    if (dim <= 80) return launch_dim<T, 128, 80>(a, op, cache, layer, s);
    if (dim <= 96) return launch_dim<T, 128, 96>(a, op, cache, layer, s);
  }
  if (dim <= 128) return launch_dim<T, 128, 128>(a, op, cache, layer, s);
  return launch_dim<T, 256, 256>(a, op, cache, layer, s);
}

// The same for every head size, so that the arrivals' place does not depend on it: what one call leaves
// in the partial results is never another's counter.
constexpr size_t kPartialBytes = 2 * kMaxCtas * sizeof(Piece<kMaxHeadDim, kGroup>);

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
  // in place with another stride, a row's output would land on queries that others still read
  if (op->out == op->q && op->out_stride != op->q_stride && op->rows > 1) return set_status(MLI_ERR_INVALID_ARG);
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
  if (a.room > kMaxTokens) a.room = kMaxTokens;
  a.group = op->heads / cache->kv_heads;
  a.chunks = (a.group + kGroup - 1) / kGroup;
  a.scale = fminf(fmaxf(op->scale * 1.4426950408889634f, FLT_MIN), FLT_MAX);  // log2(e)
  a.page_div = fast_div(cache->page_size);
  a.partials = op->workspace;
  a.arrivals = reinterpret_cast<unsigned*>(static_cast<char*>(op->workspace) + kPartialBytes);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (cache->dtype) {
    case MLI_KV_F32: return launch_attention<float>(a, *op, *cache, layer, s);
    case MLI_KV_F16: return launch_attention<__half>(a, *op, *cache, layer, s);
    default: return launch_attention<__nv_bfloat16>(a, *op, *cache, layer, s);
  }
}

}  // extern "C"
