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
constexpr int BATCH = 8;  // rows in flight per group

__device__ __forceinline__ int64_t page_row(const TreeCommit& a, int b, int pos) {
  const int bi = pos / a.block_size;
  if (bi >= a.W) return -1;
  const int blk = a.block_tables[(int64_t)b * a.bt_stride + bi];
  if (blk < 0 || blk >= a.num_blocks) return -1;
  return (int64_t)blk * a.nkv * a.block_size + pos % a.block_size;
}

template <bool FP8>
__global__ void __launch_bounds__(CT) tree_commit_kernel(TreeCommit a) {
  pdl_wait();     // inputs come from the previous kernel in the stream
  pdl_trigger();  // the next kernel may start its prologue
  constexpr int LANES = FP8 ? 8 : 16;  // lanes of 16 bytes per row
  constexpr int UNITS = CT / LANES;
  __shared__ int64_t s_src[TREE_MAX_NODES], s_dst[TREE_MAX_NODES];
  __shared__ int s_off[TREE_MAX_NODES];  // destination's offset in its block; -1: nothing moves
  __shared__ int s_first, s_len;
  extern __shared__ float s_scale[];     // e4m3: [UNITS][blocks of the tree]
  const int b = blockIdx.y;
  const int n = a.cu_q[b + 1] - a.cu_q[b], base = a.ctx_lens[b] - n;
  const int want = min(min(a.length[b], a.max_path), TREE_MAX_NODES);
  if (base < 0 || want <= 1) return;
  const int* path = a.path + (int64_t)b * a.path_stride;
  if (threadIdx.x == 0) {
    s_first = want;
    s_len = want;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < want; j += CT) {
    const int node = path[j], before = j ? path[j - 1] : -1;
    if (!(node > before && node < min(n, a.max_nodes))) atomicMin(&s_len, j);
  }
  __syncthreads();
  const int len = s_len;
  for (int j = threadIdx.x; j < len; j += CT) {
    const int node = path[j];
    const int64_t src = page_row(a, b, base + node), dst = page_row(a, b, base + j);
    const bool moves = node != j && src >= 0 && dst >= 0;
    s_src[j] = src;
    s_dst[j] = dst;
    s_off[j] = moves ? (base + j) % a.block_size : -1;
    if (node != j) atomicMin(&s_first, j);
  }
  __syncthreads();
  const int first = s_first;
  if (first >= len) return;
  const int unit = blockIdx.x * UNITS + threadIdx.x / LANES, lane = threadIdx.x % LANES;
  if (unit >= 2 * a.layers * a.nkv) return;
  const int h = unit % a.nkv, layer = unit / a.nkv % a.layers, kv = unit / a.nkv / a.layers;
  const int row_bytes = FP8 ? 128 : 256;
  uint8_t* pool = static_cast<uint8_t*>(a.kv) + kv * a.stride_kv + layer * a.stride_layer +
                  (int64_t)h * a.block_size * row_bytes + lane * 16;
  if constexpr (!FP8) {
    for (int j0 = first; j0 < len; j0 += BATCH) {
      uint4 x[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u)
        if (j0 + u < len && s_off[j0 + u] >= 0) x[u] = *reinterpret_cast<const uint4*>(pool + s_src[j0 + u] * row_bytes);
#pragma unroll
      for (int u = 0; u < BATCH; ++u)
        if (j0 + u < len && s_off[j0 + u] >= 0) *reinterpret_cast<uint4*>(pool + s_dst[j0 + u] * row_bytes) = x[u];
    }
  } else {
    float* scales = a.scale + kv * a.scale_stride_kv + layer * a.scale_stride_layer + h;
    const int64_t per_block = (int64_t)a.nkv * a.block_size;
    const unsigned group = 0xffu << (threadIdx.x & 24);
    // the scales of the tree's blocks as they were: a moved first row replaces its block's
    const int blk0 = (base + first) / a.block_size;
    const int blocks = (base + min(n, a.max_nodes) - 1) / a.block_size - blk0 + 1;
    const int ld = (a.max_nodes - 1) / a.block_size + 2;
    float* old = s_scale + threadIdx.x / LANES * ld;
    for (int i = lane; i < blocks; i += LANES) {
      const int64_t r = page_row(a, b, (blk0 + i) * a.block_size);
      old[i] = r >= 0 ? scales[r / per_block * a.nkv] : 1.f;
    }
    __syncwarp(group);
    float now = old[0];  // of the destination's block
    int now_blk = 0;
    for (int j0 = first; j0 < len; j0 += BATCH) {
      uint4 x[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u)
        if (j0 + u < len && s_off[j0 + u] >= 0) x[u] = *reinterpret_cast<const uint4*>(pool + s_src[j0 + u] * row_bytes);
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int j = j0 + u;
        if (j >= len || s_off[j] < 0) continue;
        const float from = old[(base + path[j]) / a.block_size - blk0];
        const int blk = (base + j) / a.block_size - blk0;
        if (blk != now_blk) now = old[blk];
        now_blk = blk;
        float f[16];
        const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) e4m3x4_to_f32(w[k], f + 4 * k);
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          f[k] = __fmul_rn(f[k], from);
          amax = fmaxf(amax, fabsf(f[k]));
        }
        if (s_off[j] == 0) {
          // the block begins with this row: its scale, as the store of a first token sets it
#pragma unroll
          for (int o = 4; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(group, amax, o, 8));
          now = fmaxf(__fmul_rn(amax, 4.0f / 448.0f), 1e-8f);
          if (lane == 0) scales[s_dst[j] / per_block * a.nkv] = now;
        }
        if (now != from) {  // rounded to 8 bits again, to within half a step of e4m3
          uint32_t y[4];
          if (fminf(now, from) > 1e-20f && fmaxf(now, from) < 1e20f) {
            // f / now, correctly rounded, from the correctly rounded reciprocal: the remainder of f * r is exact and
            // corrects it (P. Markstein, 1990); the bounds keep the remainder above fp32's smallest
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
        *reinterpret_cast<uint4*>(pool + s_dst[j] * row_bytes) = x[u];
      }
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
  const int units = CT / (a.kv_fp8 ? 8 : 16);
  const dim3 grid((2 * a.layers * a.nkv + units - 1) / units, a.num_seqs);
  if (a.kv_fp8)
    launch_pdl(tree_commit_kernel<true>, grid, dim3(CT), units * ((a.max_nodes - 1) / a.block_size + 2) * sizeof(float),
               stream, a);
  else
    launch_pdl(tree_commit_kernel<false>, grid, dim3(CT), 0, stream, a);
  NVB_LAUNCH_CHECK();
  return cudaSuccess;
}

}  // namespace nvb
