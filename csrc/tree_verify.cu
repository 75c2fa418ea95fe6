// The walk through a tree of drafted tokens by rejection sampling from given random numbers.
//
// At a node with p = softmax(logits / T) its children are tried in order: child c with token x is taken if
// u[c] q(x) < p(x), else p becomes max(p - q, 0) / sum (q: the draft's probabilities, or 1 at x).  Behind the last
// child the next token is the first x whose cumulative sum of p is above u_draw times the total.
//
// A cumulative sum over a vocabulary of 1.5e5 tokens has tokens narrower than fp32's rounding next to every border,
// so weights and sums are 64-bit: decisions are those of exact arithmetic but for random numbers within some 1e-12 of
// a border, and do not depend on how many CTAs share a row.  exp2 in 64 bits costs 9 fp64 instructions here: the
// argument is taken apart into a multiple of 1/256 (a table entry, and an exponent by integer addition) and a rest
// |r| <= 1/512 with 2^r = 1 + t + t^2/2 + t^3/6, t = r ln 2 (next term: 1.4e-13).
//
// One cluster of CTAs walks one tree, so only the rows of visited nodes are read.  A row is cut into chunks of
// 1024 tokens; a warp sums a chunk relative to the chunk's maximum and sends (sum, maximum) to every CTA of the
// cluster, whose first warps then take the same decisions from the same numbers: one cluster barrier per row.
#include "common.cuh"
#include "tcgen05.cuh"
#include "tree.h"

namespace nvb {
namespace {

constexpr int VT = 512;            // threads per CTA
constexpr int VWARPS = VT / 32;
constexpr int BLOCK = 1024;        // tokens of a warp's step: 32 per lane
constexpr int MAX_CHUNKS = 512;    // longer vocabularies have longer chunks
constexpr float NEG = -INFINITY;

struct ChunkSum {
  double sum;  // relative to max (walk over the logits), or as it is (residuals)
  float max;
  int first;   // token of the first maximum
};

struct Exp2 {
  const double* table;  // 2^(j / 256)
  // 2^(z / 256) p + acc for z <= 0 (or a rounding above it); z below -256000 counts as that
  __device__ __forceinline__ double fma_to(double z, double acc) const {
    const unsigned hi = min((unsigned)__double2hiint(z), 0xC10F4000u);  // -256000 and its low word's worth
    z = __hiloint2double((int)hi, __double2loint(z));
    const double t = z + 6755399441055744.0;  // 1.5 * 2^52: the low word is the nearest integer
    const int j = __double2loint(t);
    const double r = z - (t - 6755399441055744.0);
    constexpr double A = 0.69314718055994530942 / 256.0;
    const double p = fma(fma(fma(A * A * A / 6.0, r, A * A / 2.0), r, A), r, 1.0);
    const double e = table[j & 255];
    const double s = __hiloint2double(__double2hiint(e) + (j >> 8) * (1 << 20), __double2loint(e));
    return fma(s, p, acc);
  }
};

// What a token's weight is made of, at the node at hand.
struct Dist {
  double c256;     // 256 log2(e) / T
  double inv_sum;  // 1 / sum of the weights
  float max;       // the row's maximum (a NaN counts as -inf)
  bool greedy;
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

// exp((l - max) / T), 0 for -inf and below 2^-1000; an infinite maximum leaves its own tokens alone.
__device__ __forceinline__ double weight(float l, const Dist& d, const Exp2& ex) {
  if (l == NEG) return 0.0;
  if (d.max == INFINITY) return l == INFINITY ? 1.0 : 0.0;
  const double z = ((double)l - (double)d.max) * d.c256;
  return z < -256000.0 ? 0.0 : ex.fma_to(z, 0.0);
}

// Token of value i of a lane's 32 in a block.
template <bool BF16>
__device__ __forceinline__ int place(int i, int lane) {
  return BF16 ? ((i >> 3) * 32 + lane) * 8 + (i & 7) : ((i >> 2) * 32 + lane) * 4 + (i & 3);
}

// 32 logits of the block [s, s + BLOCK) per lane; tokens from `end` on are -inf.
template <bool BF16>
__device__ __forceinline__ void load_block(const void* row, int s, int end, bool aligned, int lane, float (&v)[32]) {
  if (aligned && s + BLOCK <= end) {
    if constexpr (BF16) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(row) + s) + lane;
      uint4 x[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] = __ldg(p + q * 32);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float f[8];
        bf16x8_to_f32(x[q], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[q * 8 + e] = fmaxf(f[e], NEG);
      }
    } else {
      const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(row) + s) + lane;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float4 x = __ldg(p + q * 32);
        v[q * 4] = fmaxf(x.x, NEG);
        v[q * 4 + 1] = fmaxf(x.y, NEG);
        v[q * 4 + 2] = fmaxf(x.z, NEG);
        v[q * 4 + 3] = fmaxf(x.w, NEG);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int x = s + place<BF16>(i, lane);
      v[i] = x < end ? logit_at<BF16>(row, x) : NEG;
    }
  }
}

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
  return v;
}

// The row's chunks: the first ends at a 16-byte boundary (`head` tokens in) plus `len`, the others have `len` tokens.
struct Cut {
  int head, len, count, V;
  __device__ __forceinline__ int begin(int k) const { return k ? head + k * len : 0; }
  __device__ __forceinline__ int end(int k) const { return min(V, head + (k + 1) * len); }
};

// f(block start, block end, aligned) over the blocks of chunk k.
template <typename F>
__device__ __forceinline__ void blocks_of(const Cut& cut, int k, F&& f) {
  int s = cut.begin(k);
  const int end = cut.end(k);
  if (k == 0 && cut.head) {
    f(0, min(cut.head, end), false);
    s = cut.head;
  }
  for (; s < end; s += BLOCK) f(s, end, true);
}

// Sum over chunk k of exp((l - m) / T) and m, its maximum; at T <= 0 the first maximum alone.
template <bool BF16>
__device__ ChunkSum sum_chunk(const void* row, const Cut& cut, int k, const Dist& d, const Exp2& ex, int lane) {
  float m = NEG;
  double sum = 0.0;
  int first = 0x7fffffff;
  blocks_of(cut, k, [&](int s, int end, bool aligned) {
    float v[32];
    load_block<BF16>(row, s, end, aligned, lane, v);
    float bm = v[0];
#pragma unroll
    for (int i = 1; i < 32; ++i) bm = fmaxf(bm, v[i]);
    bm = warp_max(bm);
    const float nm = fmaxf(m, bm);
    if (nm == NEG) return;
    if (d.greedy) {
      if (bm > m) {  // an earlier block keeps an equal maximum
        int at = 0x7fffffff;
#pragma unroll
        for (int i = 31; i >= 0; --i)
          if (v[i] == bm) at = s + place<BF16>(i, lane);
        first = __reduce_min_sync(FULL_MASK, at);
      }
      m = nm;
      return;
    }
    if (nm == INFINITY) {
      if (m < nm) sum = 0.0;
#pragma unroll
      for (int i = 0; i < 32; ++i) sum += v[i] == INFINITY ? 1.0 : 0.0;
      m = nm;
      return;
    }
    const double top = (double)nm;
    if (m != NEG && nm > m) sum = ex.fma_to(((double)m - top) * d.c256, 0.0) * sum;
    double part = 0.0;
#pragma unroll
    for (int i = 0; i < 32; ++i) part = ex.fma_to(((double)v[i] - top) * d.c256, part);
    sum += part;
    m = nm;
  });
  ChunkSum out;
  out.sum = d.greedy ? 0.0 : warp_sum64(sum);
  out.max = m;
  out.first = first;
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
__device__ double left_at(const void* row, int x, const Dist& d, const Exp2& ex, const Residual& r) {
  const double p = weight(logit_at<BF16>(row, x), d, ex) * d.inv_sum;
  if (!r.draft) {
    for (int i = 0; i < r.k; ++i)
      if (r.gone[i] == x) return 0.0;
    return p;
  }
  return r.k ? left_of(p, draft_at(r, x), r) : p;
}

template <bool BF16>
__device__ ChunkSum sum_residual(const void* row, const Cut& cut, int k, const Dist& d, const Exp2& ex,
                                 const Residual& r, int lane) {
  double sum = 0.0;
  blocks_of(cut, k, [&](int s, int end, bool aligned) {
    float v[32];
    load_block<BF16>(row, s, end, aligned, lane, v);
#pragma unroll 8
    for (int i = 0; i < 32; ++i) {
      const int x = s + place<BF16>(i, lane);
      if (x < end) sum += left_of(weight(v[i], d, ex) * d.inv_sum, draft_at(r, x), r);
    }
  });
  ChunkSum out;
  out.sum = warp_sum64(sum);
  out.max = 0.f;
  out.first = 0;
  return out;
}

enum Action { DRAW = 0, GO = 1, RESIDUAL = 2 };

struct Shared {
  ChunkSum chunk[2][MAX_CHUNKS];
  double table[256];
  double mass[TREE_MAX_NODES];      // of the residual after i rejections (0: the distribution itself, 1)
  double inv_mass[TREE_MAX_NODES];  // [i]: 1 / mass[i + 1]
  double scan[VWARPS];
  double now;    // mass at hand
  double share;  // of the draw: what the cumulative sum has to pass
  Dist dist;
  int parent[TREE_MAX_NODES], token[TREE_MAX_NODES], gone[TREE_MAX_NODES];
  float u[TREE_MAX_NODES];
  int action, child, rejected;
  int summed;  // rejections that the chunk sums at hand stand for
  int best;    // first maximum of the row
  int found, held, drawn_chunk;
};

// Sum of a chunk in units of the row's maximum.
__device__ __forceinline__ double scaled(const ChunkSum& c, const Dist& d, const Exp2& ex) {
  if (c.max == NEG) return 0.0;
  if (c.max == d.max) return c.sum;
  if (d.max == INFINITY) return 0.0;
  return ex.fma_to(((double)c.max - (double)d.max) * d.c256, 0.0) * c.sum;
}

template <bool BF16>
__global__ void __launch_bounds__(VT, 2) tree_verify_kernel(TreeVerify a, int len) {
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
    return;
  }
  for (int i = threadIdx.x; i < n; i += VT) {
    sh.parent[i] = a.parents[t0 + i];
    sh.token[i] = a.tokens[t0 + i];
    sh.u[i] = a.u[t0 + i];
  }
  for (int i = threadIdx.x; i < 256; i += VT) sh.table[i] = exp2(i / 256.0);
  const Exp2 ex{sh.table};
  const float temp = a.temps[b];
  Dist d;
  d.greedy = !(temp > 0.f);
  // above 0 at an infinite temperature too, where -inf still has no weight
  d.c256 = d.greedy ? 0.0 : fmax(256.0 * 1.4426950408889634074 / (double)temp, 1e-300);
  d.inv_sum = 0.0;
  d.max = NEG;
  Residual left;
  left.draft = nullptr;
  left.inv_mass = sh.inv_mass;
  left.gone = sh.gone;
  left.k = 0;
  int node = 0, length = 1;
  uint32_t phase = 0;
  const void* row = nullptr;
  Cut cut;
  cut.V = a.V;
  cut.len = len;

  // The chunk sums, in the shared memory of every CTA.
  auto pass = [&](bool residual) -> ChunkSum* {
    ChunkSum* to = sh.chunk[phase & 1];
    for (int k = cta * VWARPS + warp; k < cut.count; k += ctas * VWARPS) {
      const ChunkSum c =
          residual ? sum_residual<BF16>(row, cut, k, d, ex, left, lane) : sum_chunk<BF16>(row, cut, k, d, ex, lane);
      if (lane < (int)ctas)
        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(tc::cluster_map(smem_u32(to + k), lane)),
                     "r"(__double2loint(c.sum)), "r"(__double2hiint(c.sum)), "r"(__float_as_int(c.max)), "r"(c.first)
                     : "memory");
    }
    // the other buffer is written from here on, which every CTA has read before it came to this barrier
    tc::cluster_arrive();
    tc::cluster_wait();
    ++phase;
    return to;
  };
  // The first child of `node` from index `from` on, or n.  All lanes of a warp.
  auto next_child = [&](int from) {
    for (int i = from; i < n; i += 32) {
      const unsigned hit = __ballot_sync(FULL_MASK, i + lane < n && sh.parent[i + lane] == node);
      if (hit) return i + __ffs(hit) - 1;
    }
    return n;
  };
  // Tries children from sh.child on until one is taken, a residual is needed or none is left (first warp, with
  // the same numbers in every lane and every CTA).
  auto try_children = [&]() {
    int child = sh.child, rejected = sh.rejected, action = DRAW;
    double mass = sh.now;
    __syncwarp();
    for (child = next_child(child); child < n; child = next_child(child + 1)) {
      const int x = sh.token[child];
      const bool in = x >= 0 && x < a.V;
      if (d.greedy) {
        if (in && x == sh.best) {
          action = GO;
          break;
        }
        continue;
      }
      left.k = rejected;
      const double p = in ? left_at<BF16>(row, x, d, ex, left) : 0.0;
      const double q = !left.draft ? 1.0 : in ? draft_at(left, x) : 0.0;
      if (in && (double)sh.u[child] * q * mass < p) {
        action = GO;
        break;
      }
      if (left.draft) {
        if (mass > 0.0) {  // nothing is left to take q from otherwise
          ++rejected;
          ++child;
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
      sh.child = child;
      sh.rejected = rejected;
      sh.now = mass;
      sh.action = action;
    }
  };

  ChunkSum* sums = nullptr;
  while (true) {
    const int64_t r = (int64_t)t0 + node;
    constexpr int E = BF16 ? 2 : 4;
    row = static_cast<const uint8_t*>(a.logits) + r * a.ld * E;
    left.draft = a.draft && !d.greedy ? a.draft + r * a.ld_draft : nullptr;
    left.k = 0;
    cut.head = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / E;
    cut.count = a.V <= cut.head + len ? 1 : (a.V - cut.head + len - 1) / len;
    __syncthreads();  // the table (first node); every thread has read the last node's decision
    sums = pass(false);
    if (warp == 0) {
      float m = NEG;
      int first = 0x7fffffff;
      for (int k = lane; k < cut.count; k += 32) {
        const ChunkSum c = sums[k];
        if (c.max > m) {
          m = c.max;
          first = c.first;
        }
      }
      d.max = warp_max(m);
      first = __reduce_min_sync(FULL_MASK, m == d.max ? first : 0x7fffffff);
      double total = 0.0;
      for (int k = lane; k < cut.count; k += 32) total += scaled(sums[k], d, ex);
      total = warp_sum64(total);
      d.inv_sum = total > 0.0 ? 1.0 / total : 0.0;
      if (lane == 0) {
        sh.dist = d;
        sh.best = d.max == NEG ? -1 : first;
        sh.now = sh.mass[0] = total > 0.0 ? 1.0 : 0.0;
        sh.rejected = sh.summed = 0;
        sh.child = node + 1;
      }
      __syncwarp();
      try_children();
    }
    __syncthreads();
    d = sh.dist;
    while (sh.action == RESIDUAL) {
      left.k = sh.rejected;
      sums = pass(true);
      if (warp == 0) {
        double m = 0.0;
        for (int k = lane; k < cut.count; k += 32) m += sums[k].sum;
        m = warp_sum64(m);
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
    if (sh.action != GO) break;
    node = sh.child;
    if (cta == 0 && threadIdx.x == 0) path[length] = node;
    ++length;
  }

  left.k = sh.rejected;
  if (left.draft && sh.summed != left.k) sums = pass(left.k > 0);
  if (cta != 0) return;
  for (int i = threadIdx.x; i < a.max_nodes; i += VT)
    if (i == 0 || i >= length) path[i] = i ? -1 : 0;
  if (threadIdx.x == 0) a.length[b] = length;
  if (d.greedy) {
    if (threadIdx.x == 0) a.next_token[b] = max(sh.best, 0);
    return;
  }
  // ---- the draw: the chunk in which the cumulative sum passes the share, then the token in it
  if (warp == 0) {
    if (!left.draft || left.k == 0)
      for (int k = lane; k < cut.count; k += 32) sums[k].sum = scaled(sums[k], d, ex) * d.inv_sum;
    __syncwarp();
    if (!left.draft)
      for (int i = 0; i < left.k; ++i) {  // a rejected token's chunk is summed again without it
        const int k = sh.gone[i] < cut.head ? 0 : (sh.gone[i] - cut.head) / len;
        double part = 0.0;
        for (int x = cut.begin(k) + lane; x < cut.end(k); x += 32) part += left_at<BF16>(row, x, d, ex, left);
        part = warp_sum64(part);
        if (lane == 0) sums[k].sum = part;
        __syncwarp();
      }
    double carry = 0.0;
    for (int k0 = 0; k0 < cut.count; k0 += 32) {
      double v = k0 + lane < cut.count ? sums[k0 + lane].sum : 0.0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(FULL_MASK, v, o);
        if (lane >= o) v += up;
      }
      v += carry;
      if (k0 + lane < cut.count) sums[k0 + lane].sum = v;
      carry = __shfl_sync(FULL_MASK, v, 31);
    }
    __syncwarp();
    const float u = a.u_draw[b];
    const double share = (double)(u > 0.f ? fminf(u, 1.f) : 0.f) * carry;
    int at = -1, held = -1;
    for (int k0 = 0; k0 < cut.count && at < 0; k0 += 32) {
      const int k = k0 + lane;
      const double v = k < cut.count ? sums[k].sum : 0.0, before = k && k < cut.count ? sums[k - 1].sum : 0.0;
      const unsigned above = __ballot_sync(FULL_MASK, k < cut.count && v > share);
      const unsigned any = __ballot_sync(FULL_MASK, k < cut.count && v > before);
      if (any) held = k0 + 31 - __clz(any);
      if (above) at = k0 + __ffs(above) - 1;
    }
    if (lane == 0) {
      sh.share = share;
      sh.drawn_chunk = at >= 0 ? at : held;
      sh.found = 0x7fffffff;
      sh.held = -1;
    }
  }
  __syncthreads();
  const int k = sh.drawn_chunk;
  if (k < 0) {  // no logit above -inf
    if (threadIdx.x == 0) a.next_token[b] = 0;
    return;
  }
  double before = k ? sums[k - 1].sum : 0.0;
  const double share = sh.share;
  for (int s = cut.begin(k); s < cut.end(k); s += 2 * VT) {
    const int x = s + 2 * threadIdx.x, end = cut.end(k);
    const double v0 = x < end ? left_at<BF16>(row, x, d, ex, left) : 0.0;
    const double v1 = x + 1 < end ? left_at<BF16>(row, x + 1, d, ex, left) : 0.0;
    double sum = v0 + v1;
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
    const double c1 = ahead + sum, c0 = c1 - v1;
    int at = 0x7fffffff, held = -1;
    if (v1 > 0.0 && c1 > share) at = x + 1;
    if (v0 > 0.0 && c0 > share) at = x;
    if (v0 > 0.0) held = x;
    if (v1 > 0.0) held = x + 1;
    at = __reduce_min_sync(FULL_MASK, at);
    held = __reduce_max_sync(FULL_MASK, held);
    if (lane == 0) {
      atomicMin(&sh.found, at);
      atomicMax(&sh.held, held);
    }
    __syncthreads();
    if (sh.found != 0x7fffffff) break;  // the same in every thread: written ahead of the barrier only
    __syncthreads();
  }
  // the sums of the whole chunk may have been a rounding above those of its tokens
  if (threadIdx.x == 0) a.next_token[b] = sh.found != 0x7fffffff ? sh.found : max(sh.held, 0);
}

}  // namespace

cudaError_t launch_tree_verify(const TreeVerify& a, cudaStream_t stream) {
  if (a.num_seqs <= 0 || a.V <= 0 || a.max_nodes < 1 || a.max_nodes > TREE_MAX_NODES) return cudaErrorInvalidValue;
  int len = BLOCK;
  while ((int64_t)len * (MAX_CHUNKS - 1) < a.V) len *= 2;
  // CTAs per tree: as many as keep every cluster resident at two CTAs per SM, at least eight chunks for each
  const int chunks = (a.V + len - 1) / len;
  int ctas = 1;
  while (ctas < 16 && (int64_t)a.num_seqs * ctas * 2 <= 2 * 148 && ctas * 2 * 8 <= chunks) ctas *= 2;
  auto kern = a.logits_bf16 ? tree_verify_kernel<true> : tree_verify_kernel<false>;
  static std::atomic<uint64_t> done[2] = {{0}, {0}};
  cudaError_t e = smem_opt_in(done[a.logits_bf16 ? 1 : 0], kern, (int)sizeof(Shared), true);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.num_seqs * ctas);
  cfg.blockDim = dim3(VT);
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
