// The walk through a tree of drafted tokens by rejection sampling from given random numbers.
//
// At a node with p = softmax(logits / T) its children are tried in order: child c with token x is taken if
// u[c] q(x) < p(x), else p becomes max(p - q, 0) / sum (q: the draft's probabilities, or 1 at x).  Behind the last
// child the next token is the first x whose cumulative sum of p is above u_draw times the total.
//
// A cumulative sum over a vocabulary of 1.5e5 tokens has tokens narrower than fp32's rounding next to every border,
// so decisions rest on 64-bit weights and sums, or on fp32 ones where their error cannot matter.  exp2 in 64 bits costs 9
// fp64 instructions here (an SM does 64 a clock) of some 30 in all: the argument is taken apart into a multiple of 1/32
// (a table entry, and an exponent by integer addition) and a rest |r| <= 1/64, and 2^r = exp(t), t = r ln 2, |t| <= h, is
// 1 + t + .. + t^4/24 with t^5/120 spread over t and t^3 as (h^5/120) (20 (t/h)^3 - 5 t/h) / 16, off by Chebyshev's
// h^5/1920 = 7.9e-14 at most (left out it would be 1.3e-12), and by nothing at t = 0.  The table's halves are read as
// words: 32 entries, a bank each.  A weight w is within 8e-14 + 2^-52 |ln w| + 2^-53 |m| / T of itself (m: the chunk's
// largest logit, whose product with 1 / T is rounded), p within 1e-13 with the roundings of sums and products (|m| / T up to
// 50, weights above 2^-40 of the largest).  So the decisions are those of exact arithmetic but for random numbers that
// close to a border; behind rejections 1e-13 over the product of the masses that they left, since max(p - q, 0) keeps p's
// error and loses most of p where q is near it.  They do not depend on how many CTAs share a row.
//
// One cluster of CTAs walks one tree, so only the rows of visited nodes are read.  A row is cut into chunks of
// 512 tokens; a warp sums a chunk relative to the chunk's maximum and sends (sum, maximum) to every CTA of the
// cluster, whose first warps then take the same decisions from the same numbers: one cluster barrier per row, and one
// ahead of the first, since a CTA's shared memory may be written to from outside only once it has started.
#include "common.cuh"
#include "tcgen05.cuh"
#include "tree.h"

namespace nvb {
namespace {

constexpr int BLOCK = 512;         // tokens of a warp's step: 16 per lane
constexpr int MAX_CHUNKS = 512;    // longer vocabularies have longer chunks
constexpr float NEG = -INFINITY;
constexpr double SLACK = 1.0 / 262144.0;  // 2^-18: bounds the fp32 sums' relative error (sum_block_fast)
constexpr unsigned SPAN = 0xC0DC2000u;  // upper word of -28800 = -32 x 900: weights below 2^-900 of the largest are none

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct ChunkSum {
  double sum;  // relative to max (walk over the logits), or as it is (residuals)
  float max;
  int first;   // token of the first maximum
};

// exp(A r), |r| <= 1/2: coefficients of r .. r^4 (above: A = ln 2 / 32, h = A / 2)
constexpr double A = 0.69314718055994530942 / 32.0, H2 = A * A / 4.0;
constexpr double E1 = A * (1.0 - H2 * H2 / 384.0), E2 = A * A / 2.0, E3 = A * A * A * (1.0 / 6.0 + H2 / 96.0), E4 = A * A * A * A / 24.0;

// 2^(z / 32) for z <= 0 (or a rounding above it) from a table of 2^(j / 32), possibly times a factor, as words;
// z below -28800 counts as that.  The two factors of the result.
struct Power {
  double scale, poly;
};
__device__ __forceinline__ Power power(double z, const uint32_t* hi32, const uint32_t* lo32) {
  z = __hiloint2double((int)min((unsigned)__double2hiint(z), SPAN), __double2loint(z));
  const double t = z + 6755399441055744.0;  // 1.5 * 2^52: the low word is the nearest integer
  const int j = __double2loint(t);
  const double r = z - (t - 6755399441055744.0);
  Power p;
  p.poly = fma(fma(fma(fma(E4, r, E3), r, E2), r, E1), r, 1.0);
  p.scale = __hiloint2double((int)hi32[j & 31] + (j >> 5) * (1 << 20), (int)lo32[j & 31]);
  return p;
}

// The same for four at a time, step by step: one alone waits for its own last instruction most of the time.
__device__ __forceinline__ void power4(double (&z)[4], const uint32_t* hi32, const uint32_t* lo32, double (&scale)[4],
                                       double (&poly)[4]) {
  double t[4];
  int j[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) z[i] = __hiloint2double((int)min((unsigned)__double2hiint(z[i]), SPAN), __double2loint(z[i]));
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = z[i] + 6755399441055744.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    j[i] = __double2loint(t[i]);
    t[i] -= 6755399441055744.0;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) z[i] -= t[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    scale[i] = __hiloint2double((int)hi32[j[i] & 31] + (j[i] >> 5) * (1 << 20), (int)lo32[j[i] & 31]);
    poly[i] = fma(E4, z[i], E3);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) poly[i] = fma(poly[i], z[i], E2);
#pragma unroll
  for (int i = 0; i < 4; ++i) poly[i] = fma(poly[i], z[i], E1);
#pragma unroll
  for (int i = 0; i < 4; ++i) poly[i] = fma(poly[i], z[i], 1.0);
}

// The 64-bit value of an fp32 one by its bits (no conversion instruction: those are a quarter as many a clock).
// 0 and subnormals become about 2^-127, infinities 2^128.
__device__ __forceinline__ double wide(uint32_t f) {
  return __hiloint2double((int)((((int)f >> 3) & 0x8fffffff) + 0x38000000), (int)(f << 29));
}

// What a token's weight is made of, at the node at hand.
struct Dist {
  double c;        // 32 log2(e) / T
  double inv_sum;  // 1 / sum of the weights
  float max;       // the row's maximum (a NaN counts as -inf)
  float cf;        // log2(e) / T
  bool greedy;
  // Whether fp32's range holds log2(e) / T, with room.
  __device__ __forceinline__ bool moderate() const { return cf > 1e-6f && cf < 1e6f; }
  // Whether l c - top c in one instruction, with top c rounded, is exact enough (2^-35 of 1/32), and -inf far enough off.
  __device__ __forceinline__ bool plain(float top) const { return c > 1e-9 && fabs((double)top) * c < 262144.0; }
};

struct Tables {
  const uint32_t *hi, *lo;  // 2^(j / 32)
};

template <bool BF16>
__device__ __forceinline__ float logit_at(const void* row, int64_t x) {
  float v;
  if constexpr (BF16)
    v = __bfloat162float(static_cast<const __nv_bfloat16*>(row)[x]);
  else
    v = static_cast<const float*>(row)[x];
  return fmaxf(v, NEG);  // a NaN counts as -inf
}

template <bool BF16>
__device__ __forceinline__ float raw_logit(uint32_t raw) {
  return fmaxf(__uint_as_float(BF16 ? raw << 16 : raw), NEG);
}

// exp((l - top) / T), 0 for -inf and below 2^-900; an infinite maximum leaves its own tokens alone.
__device__ __forceinline__ double weight(float l, float top, double c, const Tables& tb) {
  if (l == NEG) return 0.0;
  if (top == INFINITY) return l == INFINITY ? 1.0 : 0.0;
  const double z = ((double)l - (double)top) * c;
  if ((unsigned)__double2hiint(z) > SPAN) return 0.0;
  const Power p = power(z, tb.hi, tb.lo);
  return p.scale * p.poly;
}

// 16 logits of a lane in a block of 512: fp32 bits.
template <bool BF16>
struct Lane {
  static constexpr int VECS = BF16 ? 2 : 4;
  uint4 v[VECS];
  // Tokens s .. s + 511 of the row (row + s: on 16 bytes), -inf outside 0 .. V - 1.
  __device__ __forceinline__ void load(const void* row, int s, int V, int lane) {
    constexpr int E = BF16 ? 2 : 4, N = 16 / E;
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(row) + (int64_t)s * E) + lane;
    if (s >= 0 && s + BLOCK <= V) {
#pragma unroll
      for (int i = 0; i < VECS; ++i) v[i] = __ldg(p + i * 32);
      return;
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int t = s + (i * 32 + lane) * N;
      if (t >= 0 && t + N <= V) {
        v[i] = __ldg(p + i * 32);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (BF16) {
            const unsigned short* h = static_cast<const unsigned short*>(row) + t + 2 * e;
            const uint32_t lo = (unsigned)(t + 2 * e) < (unsigned)V ? __ldg(h) : 0xff80;
            const uint32_t hi = (unsigned)(t + 2 * e + 1) < (unsigned)V ? __ldg(h + 1) : 0xff80;
            w[e] = hi << 16 | lo;
          } else {
            w[e] = (unsigned)(t + e) < (unsigned)V ? __ldg(static_cast<const uint32_t*>(row) + t + e) : 0xff800000u;
          }
        }
        v[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  // fp32 bits of value i
  __device__ __forceinline__ uint32_t bits(int i) const {
    if constexpr (BF16) {
      const uint4& q = v[i >> 3];
      const uint32_t w = (i & 7) < 2 ? q.x : (i & 7) < 4 ? q.y : (i & 7) < 6 ? q.z : q.w;
      return i & 1 ? w & 0xffff0000u : w << 16;
    } else {
      const uint4& q = v[i >> 2];
      return (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
    }
  }
  __device__ __forceinline__ static int place(int i, int lane) {  // token of value i in the block
    return BF16 ? ((i >> 3) * 32 + lane) * 8 + (i & 7) : ((i >> 2) * 32 + lane) * 4 + (i & 3);
  }
  // NaN to -inf
  __device__ __forceinline__ void clean() {
#pragma unroll
    for (int k = 0; k < VECS; ++k) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&v[k]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (BF16) {
          const uint32_t neg = 0xff80ff80u;
          __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&w[e]), *reinterpret_cast<const __nv_bfloat162*>(&neg));
          w[e] = *reinterpret_cast<uint32_t*>(&m);
        } else {
          w[e] = __float_as_uint(fmaxf(__uint_as_float(w[e]), NEG));
        }
      }
    }
  }
  __device__ __forceinline__ float max() const {
    if constexpr (BF16) {
      __nv_bfloat162 m[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        m[e] = __hmax2(reinterpret_cast<const __nv_bfloat162*>(&v[0])[e], reinterpret_cast<const __nv_bfloat162*>(&v[1])[e]);
      m[0] = __hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3]));
      return fmaxf(__low2float(m[0]), __high2float(m[0]));
    } else {
      float m = NEG;
#pragma unroll
      for (int i = 0; i < 16; ++i) m = fmaxf(m, __uint_as_float(bits(i)));
      return m;
    }
  }
};

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
  return v;
}

// The row's chunks: every `len` tokens from the 16-byte boundary at or before it, `shift` tokens ahead of it.
struct Cut {
  int shift, len, count, V;
  __device__ __forceinline__ int start(int k) const { return k * len - shift; }  // of the first: may be below 0
  __device__ __forceinline__ int begin(int k) const { return max(0, start(k)); }
  __device__ __forceinline__ int end(int k) const { return min(V, start(k + 1)); }
};

// 16 draft probabilities of a lane in a block of 512 tokens, 0 outside 0 .. V - 1.
template <bool BF16>
__device__ __forceinline__ void load_draft(float (&q)[16], const float* draft, int s, int V, int lane) {
  const float* at = draft + s;
  if (s >= 0 && s + BLOCK <= V && (reinterpret_cast<uintptr_t>(at) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(at + Lane<BF16>::place(i, lane)));
      q[i] = f.x;
      q[i + 1] = f.y;
      q[i + 2] = f.z;
      q[i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int t = Lane<BF16>::place(i, lane);
      q[i] = (unsigned)(s + t) < (unsigned)V ? __ldg(at + t) : 0.f;
    }
  }
}

// Sum over a block of exp((l - m) / T) and m, its maximum; at T <= 0 the first maximum alone.
template <bool BF16>
__device__ __forceinline__ ChunkSum sum_block(Lane<BF16>& x, int s, const Dist& d, const Tables& tb, int lane) {
  x.clean();
  ChunkSum out;
  out.max = warp_max(x.max());
  out.sum = 0.0;
  out.first = 0x7fffffff;
  if (out.max == NEG) return out;
  if (d.greedy) {
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 15; i >= 0; --i)
      if (__uint_as_float(x.bits(i)) == out.max) at = s + Lane<BF16>::place(i, lane);
    out.first = __reduce_min_sync(FULL_MASK, at);
    return out;
  }
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  if (out.max < INFINITY && d.plain(out.max)) {
    const double mc = -(double)out.max * d.c;
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      double z[4], scale[4], poly[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = fma(wide(x.bits(i + e)), d.c, mc);
      power4(z, tb.hi, tb.lo, scale, poly);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = fma(scale[e], poly[e], sum[e]);
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < 16; ++i) {
      uint32_t b = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (k == i) b = x.bits(k);
      sum[0] += weight(__uint_as_float(b), out.max, d.c, tb);
    }
  }
  out.sum = warp_sum64((sum[0] + sum[1]) + (sum[2] + sum[3]));
  return out;
}

// The same in fp32.  y = (l - m) log2(e) / T has a relative error of 3 x 2^-24 (cf, difference, product), exp2 one of
// 2^-22; the sum of w |y| over a block is at most 9 times that of w (the entropy of 512 values is at most 9 bits), so
// the weights' errors come to 9 ln 2 x 3 x 2^-24 + 2^-22 = 23 x 2^-24 of the sum; with 11 roundings in the sum it is
// within 34 x 2^-24, about half of SLACK.  (What exp2 flushes to 0 is below 2^-126 of the maximum.)
template <bool BF16>
__device__ __forceinline__ ChunkSum sum_block_fast(Lane<BF16>& x, int s, const Dist& d, const Tables& tb, int lane) {
  if (d.greedy) return sum_block<BF16>(x, s, d, tb, lane);
  x.clean();
  ChunkSum out;
  out.max = warp_max(x.max());
  out.sum = 0.0;
  out.first = 0x7fffffff;
  if (out.max == NEG) return out;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (out.max < INFINITY) {
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i & 3] += ex2((__uint_as_float(x.bits(i)) - out.max) * d.cf);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i & 3] += __uint_as_float(x.bits(i)) == INFINITY ? 1.f : 0.f;
  }
  out.sum = (double)warp_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
  return out;
}

// The same for a chunk of any length, token by token.
template <bool BF16>
__device__ ChunkSum sum_tokens(const void* row, int s, int end, const Dist& d, const Tables& tb, int lane) {
  ChunkSum out;
  float m = NEG;
  for (int x = s + lane; x < end; x += 32) m = fmaxf(m, logit_at<BF16>(row, x));
  out.max = m = warp_max(m);
  int at = 0x7fffffff;
  double sum = 0.0;
  if (m > NEG)
    for (int x = s + lane; x < end; x += 32) {
      const float l = logit_at<BF16>(row, x);
      if (d.greedy) {
        if (l == m) at = min(at, x);
      } else {
        sum += weight(l, m, d.c, tb);
      }
    }
  out.first = __reduce_min_sync(FULL_MASK, at);
  out.sum = warp_sum64(sum);
  return out;
}

// The distribution at a node after `k` rejected children, up to its normalisation.
struct Residual {
  const float* draft;       // the node's row, or null: rejected tokens are gone
  const double* inv_mass;   // of the residuals before the last
  int k;
  const int* gone;          // without a draft: rejected tokens
};

__device__ __forceinline__ double draft_at(const Residual& r, int64_t x) {
  const float q = r.draft[x];
  return q > 0.f ? (double)q : 0.0;
}

__device__ __forceinline__ double left_of(double p, double q, const Residual& r) {
  for (int i = 0; i < r.k; ++i) {
    p = fmax(p - q, 0.0);
    if (i + 1 < r.k) p *= r.inv_mass[i];
  }
  return p;
}

template <bool BF16>
__device__ double left_at(const void* row, int x, const Dist& d, const Tables& tb, const Residual& r) {
  const double p = weight(logit_at<BF16>(row, x), d.max, d.c, tb) * d.inv_sum;
  if (!r.draft) {
    for (int i = 0; i < r.k; ++i)
      if (r.gone[i] == x) return 0.0;
    return p;
  }
  return r.k ? left_of(p, draft_at(r, x), r) : p;
}

template <bool BF16>
__device__ double left_tokens(const void* row, int s, int end, const Dist& d, const Tables& tb, const Residual& r, int lane) {
  double sum = 0.0;
  for (int x = s + lane; x < end; x += 32) sum += left_at<BF16>(row, x, d, tb, r);
  return warp_sum64(sum);
}

// Mass of the residual over a block; tb: the table times 1 / sum.
template <bool BF16>
__device__ __forceinline__ double left_block(Lane<BF16>& x, const float (&q)[16], const Dist& d, const Tables& tb,
                                             const Residual& r) {
  x.clean();
  const double mc = -(double)d.max * d.c;
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    double z[4], scale[4], poly[4], qd[4];
    bool none[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      z[e] = fma(wide(x.bits(i + e)), d.c, mc);
      none[e] = (unsigned)__double2hiint(z[e]) > SPAN;
      qd[e] = q[i + e] > 0.f ? wide(__float_as_uint(q[i + e])) : 0.0;
    }
    power4(z, tb.hi, tb.lo, scale, poly);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      scale[e] = fma(scale[e], poly[e], -qd[e]);
      scale[e] = __double2hiint(scale[e]) < 0 || none[e] ? 0.0 : scale[e];
    }
    for (int k = 1; k < r.k; ++k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        scale[e] = fma(scale[e], r.inv_mass[k - 1], -qd[e]);
        scale[e] = __double2hiint(scale[e]) < 0 ? 0.0 : scale[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += scale[e];
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// REDO: fp32's roundings could have decided.
enum Action { DRAW = 0, GO = 1, RESIDUAL = 2, REDO = 3 };

struct Shared {
  ChunkSum chunk[2][MAX_CHUNKS];
  uint32_t hi[32], lo[32];      // 2^(j / 32)
  uint32_t r_hi[32], r_lo[32];  // times 1 / sum
  double mass[TREE_MAX_NODES];      // of the residual after i rejections (0: the distribution itself, 1)
  double inv_mass[TREE_MAX_NODES];  // [i]: 1 / mass[i + 1]
  double scan[16];
  double now;    // mass at hand
  double share, ahead;  // of the draw: what the cumulative sum has to pass, and the sum ahead of the chunk
  float wmax[16];
  int wfirst[16];
  int parent[TREE_MAX_NODES], token[TREE_MAX_NODES], gone[TREE_MAX_NODES], kid[TREE_MAX_NODES];
  float u[TREE_MAX_NODES];
  int action, child, rejected;
  int at;        // the next child to try
  int summed;  // rejections that the chunk sums at hand stand for
  int best;    // first maximum of the row
  int found, held, drawn_chunk, sure;
};

// Sum of a chunk in units of the row's maximum.
__device__ __forceinline__ double scaled(const ChunkSum& c, const Dist& d, const Tables& tb) {
  if (c.max == d.max) return c.sum;  // (an empty row's, too)
  return weight(c.max, d.max, d.c, tb) * c.sum;
}

__device__ __forceinline__ void send(ChunkSum* to, const ChunkSum& c, int ctas, int lane) {
  if (lane < ctas)
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(tc::cluster_map(smem_u32(to), lane)),
                 "r"(__double2loint(c.sum)), "r"(__double2hiint(c.sum)), "r"(__float_as_int(c.max)), "r"(c.first)
                 : "memory");
}

// A warp's chunks in 64 bits behind an fp32 walk: few nodes come to it, and its registers are not that walk's.
template <bool BF16>
__device__ __noinline__ void sum_again(const void* row, const Cut& cut, const Dist& d, const Tables& tb, ChunkSum* to, int k,
                                       int stride, int ctas) {
  const int lane = threadIdx.x & 31;
  for (; k < cut.count; k += stride) {
    ChunkSum c;
    if (cut.len == BLOCK) {
      Lane<BF16> x;
      x.load(row, cut.start(k), cut.V, lane);
      c = sum_block<BF16>(x, cut.start(k), d, tb, lane);
    } else {
      c = sum_tokens<BF16>(row, cut.begin(k), cut.end(k), d, tb, lane);
    }
    send(to + k, c, ctas, lane);
  }
}

// 512 threads and one CTA per SM while there are SMs for all, else 256 threads and two or three CTAs.
// FAST (no draft): nodes are summed in fp32 first, and again in 64 bits where its roundings could decide: a draw of a
// token of less than some 1e-5, a number that close to a border.  In 64 bits a token costs some 30 instructions, which
// bound a call of many trees, in fp32 8 (256 trees of 8 nodes, 151936 tokens: 174 us all in 64 bits, 127 so).
// Few trees wait for their longest walk, where a node walked twice costs more than fp32 gains (17 of up to 64: 64 -> 102),
// and with a draft a rejection's chain of residuals multiplies the error (64 of 16: 171 -> 204).
template <bool BF16, int VT, bool FAST>
__global__ void __launch_bounds__(VT, VT == 512 ? 1 : FAST || BF16 ? 3 : 2) tree_verify_kernel(TreeVerify a, int len) {
  constexpr int VWARPS = VT / 32;
  tc::cluster_arrive();  // this CTA has started; waited for below, ahead of the first store to another CTA
  pdl_wait();     // inputs come from the previous kernel in the stream
  pdl_trigger();  // the next kernel may start its prologue
  extern __shared__ __align__(16) uint8_t vsm[];
  Shared& sh = *reinterpret_cast<Shared*>(vsm);
  uint32_t cta, ctas;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(cta));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  const int b = blockIdx.x / ctas;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = min(max(a.cu_q[b], 0), a.T), n = min(min(a.cu_q[b + 1], a.T) - t0, a.max_nodes);
  int* path = a.path + (int64_t)b * a.max_nodes;
  if (n <= 0) {  // every CTA of the cluster
    if (cta == 0) {
      for (int i = threadIdx.x; i < a.max_nodes; i += VT) path[i] = -1;
      if (threadIdx.x == 0) {
        a.length[b] = 0;
        a.next_token[b] = -1;
      }
    }
    tc::cluster_wait();
    return;
  }
  for (int i = threadIdx.x; i < n; i += VT) {
    sh.parent[i] = a.parents[t0 + i];
    sh.token[i] = a.tokens[t0 + i];
    sh.u[i] = a.u[t0 + i];
  }
  if (threadIdx.x < 32) {
    const double e = exp2(threadIdx.x / 32.0);
    sh.hi[threadIdx.x] = (uint32_t)__double2hiint(e);
    sh.lo[threadIdx.x] = (uint32_t)__double2loint(e);
  }
  const Tables tb{sh.hi, sh.lo}, scaled_tb{sh.r_hi, sh.r_lo};
  const float temp = a.temps[b];
  Dist d;
  d.greedy = !(temp > 0.f);
  // above 0 at an infinite temperature too, where -inf still has no weight
  d.c = d.greedy ? 0.0 : fmax(32.0 * 1.4426950408889634074 / (double)temp, 1e-300);
  d.cf = (float)(d.c / 32.0);
  d.inv_sum = 0.0;
  d.max = NEG;
  Residual left;
  left.draft = nullptr;
  left.inv_mass = sh.inv_mass;
  left.gone = sh.gone;
  left.k = 0;
  int node = 0, length = 1;
  const bool slow = !FAST || d.greedy || !d.moderate();
  bool exact = slow;  // this node in 64 bits
  uint32_t phase = 0;
  const void* row = nullptr;
  Cut cut;
  cut.V = a.V;
  cut.len = len;

  // First warp: the children of `node` in sh.kid; lane i holds child i's logit and draft probability, whose loads run
  // beside the pass over the row, and later its probability.
  int kids = 0;
  uint32_t kid_raw = 0;  // as loaded: nothing waits for it before it is used
  float kid_draft = 0.f;
  bool kid_in = false;
  double kid_p = 0.0;
  auto find_children = [&]() {
    kids = 0;
    for (int i = (node + 1) & ~31; i < n; i += 32) {
      const bool hit = i + lane > node && i + lane < n && sh.parent[i + lane] == node;
      const unsigned all = __ballot_sync(FULL_MASK, hit);
      if (hit) sh.kid[kids + __popc(all & ((1u << lane) - 1))] = i + lane;
      kids += __popc(all);
    }
    __syncwarp();
    kid_draft = 0.f;
    const int x = lane < kids ? sh.token[sh.kid[lane]] : -1;
    kid_in = x >= 0 && x < a.V;
    if (kid_in) {
      kid_raw = BF16 ? __ldg(static_cast<const unsigned short*>(row) + x) : __ldg(static_cast<const unsigned*>(row) + x);
      if (left.draft) kid_draft = __ldg(left.draft + x);
    }
  };
  // The chunk sums, in the shared memory of every CTA.  A warp's next block is on its way while it works on one.
  auto pass = [&](bool residual) -> ChunkSum* {
    ChunkSum* to = sh.chunk[phase & 1];
    const int stride = ctas * VWARPS;
    const bool blocks = len == BLOCK && (!residual || (d.plain(d.max) && d.max < INFINITY));
    Lane<BF16> x, nx;
    int k = cta * VWARPS + warp;
    if (FAST && exact && !d.greedy) {
      if (warp == 0) find_children();
      sum_again<BF16>(row, cut, d, tb, to, k, stride, ctas);
      k = cut.count;
    }
    if (blocks && k < cut.count) x.load(row, cut.start(k), cut.V, lane);
    if (!residual && warp == 0) find_children();
    for (; k < cut.count; k += stride) {
      const int s = cut.start(k), nk = k + stride;
      if (blocks && nk < cut.count) nx.load(row, cut.start(nk), cut.V, lane);
      ChunkSum c;
      if (!residual) {
        c = blocks ? (FAST ? sum_block_fast<BF16>(x, s, d, tb, lane) : sum_block<BF16>(x, s, d, tb, lane))
                   : sum_tokens<BF16>(row, cut.begin(k), cut.end(k), d, tb, lane);
      } else {
        if (blocks) {
          float q[16];
          load_draft<BF16>(q, left.draft, s, cut.V, lane);
          c.sum = warp_sum64(left_block<BF16>(x, q, d, scaled_tb, left));
        } else {
          c.sum = left_tokens<BF16>(row, cut.begin(k), cut.end(k), d, tb, left, lane);
        }
        c.max = 0.f;
        c.first = 0;
      }
      send(to + k, c, ctas, lane);
      x = nx;
    }
    // the other buffer is written from here on, which every CTA has read before it came to this barrier
    tc::cluster_arrive();
    tc::cluster_wait();
    ++phase;
    return to;
  };
  // First warp: tries children from sh.at on until one is taken, a residual is needed or none is left (with the same
  // numbers in every lane and every CTA).
  auto try_children = [&]() {
    int at = sh.at, rejected = sh.rejected, action = DRAW;
    double mass = sh.now;
    __syncwarp();
    for (; at < kids; ++at) {
      const int child = sh.kid[at], x = sh.token[child];
      const bool in = x >= 0 && x < a.V;
      if (d.greedy) {
        if (in && x == sh.best) {
          action = GO;
          break;
        }
        continue;
      }
      double p = 0.0, q = 1.0;
      if (at < 32) {
        p = __shfl_sync(FULL_MASK, kid_p, at);
        const float f = __shfl_sync(FULL_MASK, kid_draft, at);
        if (left.draft) q = f > 0.f ? (double)f : 0.0;
      } else if (in) {
        p = weight(logit_at<BF16>(row, x), d.max, d.c, tb) * d.inv_sum;
        if (left.draft) q = draft_at(left, x);
      }
      left.k = rejected;
      if (left.draft)
        p = left_of(p, q, left);
      else
        for (int i = 0; i < rejected; ++i)
          if (sh.gone[i] == x) p = 0.0;
      // p is within SLACK of itself, the mass (1 less the rejected tokens) within SLACK
      if (FAST && !exact && in && p > 0.0 &&
          (!(fabs(p - (double)sh.u[child] * mass) > SLACK * (p + fabs((double)sh.u[child]))) || mass - p < 8.0 * SLACK)) {
        action = REDO;
        break;
      }
      if (in && (double)sh.u[child] * q * mass < p) {
        action = GO;
        break;
      }
      if (left.draft) {
        if (mass > 0.0) {  // nothing is left to take q from otherwise
          ++rejected;
          ++at;
          action = RESIDUAL;
          break;
        }
      } else if (p > 0.0 && mass - p > 0.0) {
        if (lane == 0) sh.gone[rejected] = x;
        __syncwarp();
        ++rejected;
        mass -= p;
      }
    }
    if (lane == 0) {
      sh.at = at;
      sh.child = action == GO ? sh.kid[at] : -1;
      sh.rejected = rejected;
      sh.now = mass;
      sh.action = action;
    }
  };

  // The draw: the chunk in which the cumulative sum passes the share, then the token in it.  False where fp32's
  // roundings could have decided: with every chunk within SLACK of its sum, so is the cumulative sum's share of the
  // total.  (At most one thread is sure of its token.)  FAST: in every CTA of the cluster, which all learn by it
  // whether the node is walked again.
  int next = 0;
  auto draw = [&](ChunkSum* sums) -> bool {
    if (d.greedy) {
      next = max(sh.best, 0);
      return true;
    }
    if (!left.draft || left.k == 0)
      for (int k = threadIdx.x; k < cut.count; k += VT) sums[k].sum = scaled(sums[k], d, tb) * d.inv_sum;
    __syncthreads();
    if (!left.draft) {
      for (int i = warp; i < left.k; i += VWARPS) {  // a rejected token's chunk is summed again without it
        const int k = (sh.gone[i] + cut.shift) / len;
        const double part = left_tokens<BF16>(row, cut.begin(k), cut.end(k), d, tb, left, lane);
        if (lane == 0) sums[k].sum = part;
      }
      __syncthreads();
    }
    if (warp == 0) {
      // a lane takes consecutive chunks
      const int per = (cut.count + 31) / 32, k0 = min(cut.count, lane * per), k1 = min(cut.count, k0 + per);
      double mine = 0.0;
      for (int k = k0; k < k1; ++k) mine += sums[k].sum;
      double upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(FULL_MASK, upto, o);
        if (lane >= o) upto += up;
      }
      const double total = __shfl_sync(FULL_MASK, upto, 31);
      const float u = a.u_draw[b];
      const double share = (double)(u > 0.f ? fminf(u, 1.f) : 0.f) * total;
      const unsigned above = __ballot_sync(FULL_MASK, mine > 0.0 && upto > share), any = __ballot_sync(FULL_MASK, mine > 0.0);
      if (lane == 0) {
        sh.found = 0x7fffffff;
        sh.sure = 0;
        sh.held = -1;
        if (!any) sh.drawn_chunk = -1;  // no logit above -inf
      }
      if (any && lane == (above ? __ffs(above) - 1 : 31 - __clz(any))) {
        double sum = upto - mine;
        int at = -1;
        double ahead = 0.0;
        for (int k = k0; k < k1; ++k) {
          if (sums[k].sum > 0.0) {
            at = k;  // the last one with any mass where rounding leaves none above the share
            ahead = sum;
          }
          sum += sums[k].sum;
          if (above && sums[k].sum > 0.0 && sum > share) break;
        }
        sh.drawn_chunk = at;
        sh.ahead = ahead;
        sh.share = share;
      }
    }
    __syncthreads();
    const int k = sh.drawn_chunk;
    if (k < 0) {
      next = 0;
      return true;
    }
    double before = sh.ahead;
    const double share = sh.share;
    for (int s = cut.begin(k); s < cut.end(k); s += VT) {
      const int x = s + threadIdx.x;
      const double v = x < cut.end(k) ? left_at<BF16>(row, x, d, tb, left) : 0.0;
      double sum = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(FULL_MASK, sum, o);
        if (lane >= o) sum += up;
      }
      if (lane == 31) sh.scan[warp] = sum;
      __syncthreads();
      double ahead = before;
      for (int w = 0; w < VWARPS; ++w) {
        if (w < warp) ahead += sh.scan[w];
        before += sh.scan[w];
      }
      const int at = __reduce_min_sync(FULL_MASK, v > 0.0 && ahead + sum > share ? x : 0x7fffffff);
      if (FAST && !exact && v > 0.0 && ahead + sum - v + 2.0 * SLACK <= share && share <= ahead + sum - 2.0 * SLACK) sh.sure = 1;
      const int held = __reduce_max_sync(FULL_MASK, v > 0.0 ? x : -1);
      if (lane == 0) {
        atomicMin(&sh.found, at);
        atomicMax(&sh.held, held);
      }
      __syncthreads();
      if (sh.found != 0x7fffffff) break;  // the same in every thread: written ahead of the barrier only
      __syncthreads();
    }
    // the chunk's sum may have been a rounding above that of its tokens
    next = sh.found != 0x7fffffff ? sh.found : max(sh.held, 0);
    return exact || sh.sure != 0;
  };

  ChunkSum* sums = nullptr;
  tc::cluster_wait();  // every CTA of the cluster has started
  while (true) {
    const int64_t r = (int64_t)t0 + node;
    constexpr int E = BF16 ? 2 : 4;
    row = static_cast<const uint8_t*>(a.logits) + r * a.ld * E;
    left.draft = !FAST && a.draft && !d.greedy ? a.draft + r * a.ld_draft : nullptr;
    left.k = 0;
    cut.shift = (int)(reinterpret_cast<uintptr_t>(row) & 15) / E;
    cut.count = (a.V + cut.shift + len - 1) / len;
    __syncthreads();  // the table (first node); every thread has read the last node's decision
    sums = pass(false);
    // the row's maximum and sum, by all threads, the same numbers in each
    float m = NEG;
    for (int k = threadIdx.x; k < cut.count; k += VT) m = fmaxf(m, sums[k].max);
    m = warp_max(m);
    if (lane == 0) sh.wmax[warp] = m;
    __syncthreads();
    d.max = NEG;
#pragma unroll
    for (int w = 0; w < VWARPS; ++w) d.max = fmaxf(d.max, sh.wmax[w]);
    double total = 0.0;
    int first = 0x7fffffff;
    for (int k = threadIdx.x; k < cut.count; k += VT) {
      total += scaled(sums[k], d, tb);
      if (sums[k].max == d.max) first = min(first, sums[k].first);
    }
    total = warp_sum64(total);
    first = __reduce_min_sync(FULL_MASK, first);
    if (lane == 0) {
      sh.scan[warp] = total;
      sh.wfirst[warp] = first;
    }
    __syncthreads();
    total = 0.0;
#pragma unroll
    for (int w = 0; w < VWARPS; ++w) {
      total += sh.scan[w];
      first = min(first, sh.wfirst[w]);
    }
    d.inv_sum = total > 0.0 ? 1.0 / total : 0.0;
    if (warp == 0) {
      if (lane == 0) {
        sh.best = d.max == NEG ? -1 : first;
        sh.now = sh.mass[0] = total > 0.0 ? 1.0 : 0.0;
        sh.rejected = sh.summed = sh.at = 0;
      }
      if (!d.greedy) kid_p = weight(kid_in ? raw_logit<BF16>(kid_raw) : NEG, d.max, d.c, tb) * d.inv_sum;
      if (left.draft) {
        const double e = __hiloint2double((int)tb.hi[lane], (int)tb.lo[lane]) * d.inv_sum;
        sh.r_hi[lane] = (uint32_t)__double2hiint(e);
        sh.r_lo[lane] = (uint32_t)__double2loint(e);
      }
      __syncwarp();
      try_children();
    }
    __syncthreads();
    while (!FAST && sh.action == RESIDUAL) {
      left.k = sh.rejected;
      sums = pass(true);
      double part = 0.0;
      for (int k = threadIdx.x; k < cut.count; k += VT) part += sums[k].sum;
      part = warp_sum64(part);
      if (lane == 0) sh.scan[warp] = part;
      __syncthreads();
      if (warp == 0) {
        double m = 0.0;
#pragma unroll
        for (int w = 0; w < VWARPS; ++w) m += sh.scan[w];
        if (lane == 0) {
          const int k = left.k;
          if (m > 0.0) {
            sh.now = sh.mass[k] = m;
            sh.inv_mass[k - 1] = 1.0 / m;
            sh.summed = k;
          } else {  // nothing would be left: p stays
            sh.rejected = k - 1;
            sh.now = sh.mass[k - 1];
            sh.summed = -1;
          }
        }
        __syncwarp();
        try_children();
      }
      __syncthreads();
    }
    if (FAST && sh.action == REDO) {
      exact = true;
      continue;
    }
    if (sh.action != GO) {
      left.k = sh.rejected;
      if (left.draft && sh.summed != left.k) sums = pass(left.k > 0);
      if ((!FAST && cta != 0) || draw(sums)) break;
      exact = true;
      continue;
    }
    exact = slow;
    node = sh.child;
    if (cta == 0 && threadIdx.x == 0) path[length] = node;
    ++length;
  }

  if (cta != 0) return;
  for (int i = threadIdx.x; i < a.max_nodes; i += VT)
    if (i == 0 || i >= length) path[i] = i ? -1 : 0;
  if (threadIdx.x == 0) {
    a.length[b] = length;
    a.next_token[b] = next;
  }
}

}  // namespace

cudaError_t launch_tree_verify(const TreeVerify& a, cudaStream_t stream) {
  if (a.num_seqs <= 0 || a.V <= 0 || a.max_nodes < 1 || a.max_nodes > TREE_MAX_NODES) return cudaErrorInvalidValue;
  int len = BLOCK;
  while ((int64_t)len * (MAX_CHUNKS - 1) < a.V) len *= 2;  // (one chunk more for a row off a 16-byte boundary)
  // CTAs per tree.  Few trees: all SMs, one CTA of 512 threads on each, no more than have a chunk per warp.  More:
  // smaller CTAs, three to an SM.  Behind some 32 trees eight of them, no more than have two chunks per warp, although
  // that takes several rounds of clusters: walks differ in length, and the longest one of 256 trees on a CTA each was
  // what the call took.  In fp32 four are enough for many.  Measured (us, 256 threads unless noted) at 1, 4, 8, 16 CTAs:
  //   256 trees of 8 nodes, 151936 tokens, fp32 first        199  127  168  293   (all in 64 bits 362, 178, 178, 252)
  //   64 of 16, fp32 first                                   236   91   74   99
  //   120 of 8, 32000 tokens, fp32 first                      55   43   58  108
  //   64 of 16, 151936 tokens, with a draft                  485  184  134  149
  //   120 of 8, 32000 tokens, with a draft                    95   55   66  121
  //   32 of 16, 151936 tokens                                325  110   79   69   (512 threads: 236, 84, 73, 93)
  //   20 of 16, with a draft                                 339  109   79   64   (237, 81, 68, 85)
  //   8 of 8, with a draft; 1 of 8: 512 threads              188, 63;  65, 28;  47, 23;  43, 20
  const bool few = a.num_seqs * 16 <= 148, crowded = a.num_seqs > 32, fast = crowded && !a.draft;
  const int vt = few ? 512 : 256, most = !crowded ? 16 : fast && a.num_seqs > 128 ? 4 : 8;
  const int chunks = (a.V + len - 1) / len;
  int ctas = 1;
  while (ctas < most && (crowded ? 2 * ctas * (vt / 32) <= chunks : ctas * (vt / 32) < chunks)) ctas *= 2;
  auto kern = fast ? (a.logits_bf16 ? tree_verify_kernel<true, 256, true> : tree_verify_kernel<false, 256, true>)
              : few ? (a.logits_bf16 ? tree_verify_kernel<true, 512, false> : tree_verify_kernel<false, 512, false>)
                    : (a.logits_bf16 ? tree_verify_kernel<true, 256, false> : tree_verify_kernel<false, 256, false>);
  static std::atomic<uint64_t> done[6] = {{0}, {0}, {0}, {0}, {0}, {0}};
  cudaError_t e = smem_opt_in(done[(a.logits_bf16 ? 1 : 0) + (fast ? 4 : few ? 2 : 0)], kern, (int)sizeof(Shared), true);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.num_seqs * ctas);
  cfg.blockDim = dim3(vt);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, a, len);
}

}  // namespace nvb
