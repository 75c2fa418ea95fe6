// Trees of drafted tokens: ancestor masks, and the accepted nodes' K/V moved to consecutive positions.
#include "common.cuh"
#include "tree.h"

namespace nvb {
namespace {

// ------------------------------------------------------------------------------ masks
// See[i] = {i} u See[parent(i)].  One CTA per sequence, one node per thread: each round joins a node's set with the
// set of the node it jumps to and doubles the jump, so a chain of n nodes takes log2(n) rounds.  The work is a few
// hundred bytes per sequence; the launch bounds it.
template <int WORDS>
__global__ void tree_mask_kernel(const int* __restrict__ parents, const int* __restrict__ cu_q, int T, int max_nodes,
                                 int64_t* __restrict__ mask, int words, int* __restrict__ depth) {
  pdl_wait();     // inputs come from the previous kernel in the stream
  pdl_trigger();  // the next kernel may start its prologue
  __shared__ uint64_t see[WORDS * 64][WORDS];
  __shared__ int jump[WORDS * 64];
  const int b = blockIdx.x, i = threadIdx.x;
  const int t0 = min(max(cu_q[b], 0), T), t1 = min(max(cu_q[b + 1], t0), T);
  const int n = min(t1 - t0, max_nodes);
  uint64_t mine[WORDS];
#pragma unroll
  for (int w = 0; w < WORDS; ++w) mine[w] = (i >> 6) == w ? 1ull << (i & 63) : 0ull;
  int to = -1;
  if (i < n) {
    to = parents[t0 + i];
    if (to >= i) to = -1;
  }
  while (__syncthreads_or(to >= 0)) {
    // every thread has read its sources of the round before
#pragma unroll
    for (int w = 0; w < WORDS; ++w) see[i][w] = mine[w];
    jump[i] = to;
    __syncthreads();
    if (to >= 0) {
#pragma unroll
      for (int w = 0; w < WORDS; ++w) mine[w] |= see[to][w];
      to = jump[to];
    }
  }
  if (i < t1 - t0) {
    int d = -1;
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      if (w < words) mask[(int64_t)(t0 + i) * words + w] = i < n ? (int64_t)mine[w] : 0;
      d += __popcll(mine[w]);
    }
    depth[t0 + i] = i < n ? d : 0;
  }
  // nodes past the sizes that the thread block covers, and rows behind the last sequence
  int64_t z0 = t0 + blockDim.x, z1 = t1;
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t t = z0 + i; t < z1; t += blockDim.x) {
      for (int w = 0; w < words; ++w) mask[t * words + w] = 0;
      depth[t] = 0;
    }
    z0 = t1;
    z1 = b == (int)gridDim.x - 1 ? T : 0;
  }
}

// ----------------------------------------------------------------------------- commit
// Row base + path[j] -> base + j for every (K or V, layer, head).  path increases, so path[j] >= j: in the order of
// j no destination lies above a source that is still to be read, and one group of lanes that reads rows in batches
// before it writes them needs no other order.  Every byte is read and written once; a call for one sequence is
// bound by the launch and two dependent reads (path, then rows).
constexpr int CT = 256;   // threads per CTA
constexpr int BATCH = 4;  // rows in flight per group: four CTAs per SM, with eight three

template <bool FP8>
__global__ void __launch_bounds__(CT, 4) tree_commit_kernel(TreeCommit a) {
  pdl_wait();     // inputs come from the previous kernel in the stream
  pdl_trigger();  // the next kernel may start its prologue
  constexpr int LANES = FP8 ? 8 : 16;  // lanes of 16 bytes per row
  constexpr int UNITS = CT / LANES;
  constexpr int ROW = FP8 ? 128 : 256;  // bytes
  // The rows to move, in the order of their destinations, and the tree's blocks (ids; -1: none).
  __shared__ int s_block[TREE_MAX_NODES + 1];
  __shared__ uint32_t s_src[TREE_MAX_NODES], s_dst[TREE_MAX_NODES];  // (block of the tree) << 24 | offset in it
  __shared__ int s_first, s_len;
  extern __shared__ float s_scale[];  // e4m3: [UNITS][blocks of the tree]
  const int b = blockIdx.y, bs = a.block_size;
  const int n = min(a.cu_q[b + 1] - a.cu_q[b], a.max_nodes), base = a.ctx_lens[b] - (a.cu_q[b + 1] - a.cu_q[b]);
  const int want = min(min(a.length[b], a.max_path), TREE_MAX_NODES);
  if (base < 0 || want <= 1) return;
  const int* path = a.path + (int64_t)b * a.path_stride;
  const int block0 = base / bs, blocks = (base + n - 1) / bs - block0 + 1;
  if (threadIdx.x == 0) s_first = s_len = want;
  for (int i = threadIdx.x; i < blocks; i += CT) {
    const int id = block0 + i < a.W ? a.block_tables[(int64_t)b * a.bt_stride + block0 + i] : -1;
    s_block[i] = id >= 0 && id < a.num_blocks ? id : -1;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < want; j += CT) {
    const int node = path[j], before = j ? path[j - 1] : -1;
    if (!(node > before && node < n)) {
      atomicMin(&s_len, j);  // the path ends where it does not increase, or leaves the tree
    } else {
      const int src = base + node, dst = base + j;
      s_src[j] = (uint32_t)(src / bs - block0) << 24 | src % bs;
      s_dst[j] = (uint32_t)(dst / bs - block0) << 24 | dst % bs;
      if (node != j) atomicMin(&s_first, j);
    }
  }
  __syncthreads();
  const int first = s_first, len = s_len;
  const int lane = threadIdx.x % LANES;
  for (int unit = blockIdx.x * UNITS + threadIdx.x / LANES; unit < 2 * a.layers * a.nkv && first < len; unit += gridDim.x * UNITS) {
    const int h = unit % a.nkv, layer = unit / a.nkv % a.layers, kv = unit / a.nkv / a.layers;
    uint8_t* pool = static_cast<uint8_t*>(a.kv) + kv * a.stride_kv + layer * a.stride_layer + lane * 16;
    auto at = [&](uint32_t where) {
      return reinterpret_cast<uint4*>(pool + (((int64_t)s_block[where >> 24] * a.nkv + h) * bs + (where & 0xffffff)) * ROW);
    };
    auto moves = [&](int j) { return j < len && s_block[s_src[j] >> 24] >= 0 && s_block[s_dst[j] >> 24] >= 0; };
    if constexpr (!FP8) {
      for (int j0 = first; j0 < len; j0 += BATCH) {
        uint4 x[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
          if (moves(j0 + u)) x[u] = *at(s_src[j0 + u]);
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
          if (moves(j0 + u)) *at(s_dst[j0 + u]) = x[u];
      }
    } else {
      float* scales = a.scale + kv * a.scale_stride_kv + layer * a.scale_stride_layer + h;
      const unsigned group = 0xffu << (threadIdx.x & 24);
      // the scales of the tree's blocks as they were: a moved first row replaces its block's
      float* old = s_scale + threadIdx.x / LANES * ((a.max_nodes - 1) / bs + 2);
      for (int i = lane; i < blocks; i += LANES) old[i] = s_block[i] >= 0 ? scales[(int64_t)s_block[i] * a.nkv] : 1.f;
      __syncwarp(group);
      float now = 1.f;  // of the destination's block
      int now_block = -1;
      for (int j0 = first; j0 < len; j0 += BATCH) {
        uint4 x[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
          if (moves(j0 + u)) x[u] = *at(s_src[j0 + u]);
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          if (!moves(j0 + u)) continue;
          const uint32_t dst = s_dst[j0 + u];
          const float from = old[s_src[j0 + u] >> 24];
          if ((int)(dst >> 24) != now_block) now = old[dst >> 24];
          now_block = dst >> 24;
          float f[16];
          const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) e4m3x4_to_f32(w[k], f + 4 * k);
#pragma unroll
          for (int k = 0; k < 16; ++k) f[k] = __fmul_rn(f[k], from);
          if ((dst & 0xffffff) == 0) {
            // the block begins with this row: its scale, as the store of a first token sets it
            float amax = 0.f;
#pragma unroll
            for (int k = 0; k < 16; ++k) amax = fmaxf(amax, fabsf(f[k]));
#pragma unroll
            for (int o = 4; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(group, amax, o, 8));
            now = fmaxf(__fmul_rn(amax, 4.0f / 448.0f), 1e-8f);
            if (lane == 0) scales[(int64_t)s_block[now_block] * a.nkv] = now;
          }
          if (now != from) {  // rounded to 8 bits again, to within half a step of e4m3
            uint32_t y[4];
            // (|f| <= 448 from: with from <= 1e30 now the quotient is far from fp32's largest)
            if (fminf(now, from) > 1e-20f && fmaxf(now, from) < 1e20f && from <= __fmul_rn(1e30f, now)) {
              // f / now, correctly rounded, from the correctly rounded reciprocal: the remainder of f * r is exact
              // and corrects it (P. Markstein, 1990); the bounds keep the remainder above fp32's smallest
              const float r = __frcp_rn(now);
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const float q = __fmul_rn(f[k], r);
                f[k] = q == 0.f ? q : fmaf(fmaf(-q, now, f[k]), r, q);  // (a zero keeps its sign)
              }
            } else {
#pragma unroll
              for (int k = 0; k < 16; ++k) f[k] = __fdiv_rn(f[k], now);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = f32x4_to_e4m3(f + 4 * k);
            x[u] = make_uint4(y[0], y[1], y[2], y[3]);
          }
          *at(dst) = x[u];
        }
      }
      __syncwarp(group);  // `old` is filled anew
    }
  }
}

}  // namespace

cudaError_t launch_tree_mask(const int* parents, const int* cu_q, int num_seqs, int T, int max_nodes, int64_t* mask,
                             int words, int* depth, cudaStream_t stream) {
  if (num_seqs <= 0 || max_nodes < 1 || max_nodes > TREE_MAX_NODES || words != (max_nodes + 63) / 64)
    return cudaErrorInvalidValue;
  const dim3 grid(num_seqs);
  if (words == 1)
    launch_pdl(tree_mask_kernel<1>, grid, dim3(64), 0, stream, parents, cu_q, T, max_nodes, mask, words, depth);
  else if (words == 2)
    launch_pdl(tree_mask_kernel<2>, grid, dim3(128), 0, stream, parents, cu_q, T, max_nodes, mask, words, depth);
  else
    launch_pdl(tree_mask_kernel<4>, grid, dim3(256), 0, stream, parents, cu_q, T, max_nodes, mask, words, depth);
  NVB_LAUNCH_CHECK();
  return cudaSuccess;
}

cudaError_t launch_tree_commit(const TreeCommit& a, cudaStream_t stream) {
  if (a.num_seqs <= 0 || a.num_seqs > 65535 || a.layers <= 0 || a.nkv <= 0 || a.block_size <= 0 || a.max_path <= 0 ||
      a.max_nodes <= 0 || a.max_nodes > TREE_MAX_NODES)
    return cudaErrorInvalidValue;
  // CTAs per sequence: in all as many as four rounds of four per SM, since paths differ in length; a group of lanes
  // then has a few units, and a CTA's way to its first row is paid a few times only.  128 trees of 16 nodes, 64
  // layers, e4m3, at 1, 2, 4, 8, 16, 32 CTAs each: 183, 106, 66, 49, 44, 46 us (115 MB in rows of 128 bytes on one pair of
  // caches, most of which stays in the L2: 2.6 TB/s; on caches in turn, as in a step, 60 us at 16: 1.9 TB/s).
  const int units = CT / (a.kv_fp8 ? 8 : 16), most = (2 * a.layers * a.nkv + units - 1) / units;
  const int share = (16 * 148 + a.num_seqs - 1) / a.num_seqs;
  const dim3 grid(share < most ? share : most, a.num_seqs);
  if (a.kv_fp8)
    launch_pdl(tree_commit_kernel<true>, grid, dim3(CT), units * ((a.max_nodes - 1) / a.block_size + 2) * sizeof(float),
               stream, a);
  else
    launch_pdl(tree_commit_kernel<false>, grid, dim3(CT), 0, stream, a);
  NVB_LAUNCH_CHECK();
  return cudaSuccess;
}

}  // namespace nvb
