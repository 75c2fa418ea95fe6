// Attention of a tree of drafted tokens over the paged cache.
//
// Row r = (node, query head) of a KV head sees the positions before the tree and the nodes of its mask:
//   o_r = sum_j a_rj v_j,  a = softmax_j(scale q_r . k_j)   over j < base or (j - base) in mask(node).
// All rows of a KV head (nodes x nq / nkv) share its keys, so a tree of 8 nodes and 4 heads per KV head does 32
// rows' work on each key that decode attention would read for 4: HBM still bounds it up to some 64 rows.
//
// One warp streams tiles of 64 keys with TMA into a ring; eight warps work on them: RG groups of 16 rows, the 8 / RG
// warps of a group on different keys, each with running maxima, sums and outputs of its own (fp32) that are joined
// through shared memory once per (sequence, KV head).  bf16 mma.sync tiles; an e4m3 cache is converted once per
// value, by four further warps, into f16 tiles (exact; K's scale multiplies the scores, V's is carried by the
// accumulator's unit), so all that follows is the same kernel on f16.
//
// Balance: the tiles of all (sequence, KV head) pairs are laid end to end and cut into equal stretches, one per CTA,
// whatever the sequences' lengths.  A pair that is cut leaves partial sums (at most two per CTA), which the second
// kernel joins in the order of the keys: no atomics, the same bits on every run.
//
// Masks: only tiles that reach into the tree look at them.  What a row does not see takes no part in it: scores are
// replaced by -inf, and where a value that some row must not see is infinite or NaN (0 x inf), the tile's V is
// cleaned in registers and such values are added row by row.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "tcgen05.cuh"
#include "tree.h"

namespace nvb {
namespace {

constexpr int AD = 128;      // head dim
constexpr int KT = 64;       // keys per tile
constexpr int NWARP = 8;     // warps that work on tiles
constexpr float LOG2E = 1.4426950408889634f;
constexpr uint64_t WAIT_NS = 2000000000ull;

__device__ int g_tree_error = 0;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// c += a b: 16 x 16 times 16 x 8, f16 or bf16 in, fp32 sums
template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool F16>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t d;
  if constexpr (F16)
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(d) : "f"(lo), "f"(hi));
  else
    asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(d) : "f"(lo), "f"(hi));
  return d;
}
template <bool F16>
__device__ __forceinline__ float2 unpack(uint32_t x) {
  if constexpr (F16)
    return __half22float2(*reinterpret_cast<__half2*>(&x));
  else
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&x));
}
// Set in bits 15 and 31 where a half of x is infinite or NaN (its exponent is all ones).
template <bool F16>
__device__ __forceinline__ uint32_t odd_halves(uint32_t x) {
  return ((x & 0x7fff7fffu) + (F16 ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}

struct Args {
  TreeAttn t;
  int G, row_tiles, chunks, bs_shift;
  int box_rows;     // rows per TMA box: min(64, block size)
  int oob_row;      // a row behind the pool: reads as zeros
  float scale_log2;
};

// ------------------------------------------------------------------- the list of tiles
// Sequence b with nodes has max(1, ceil(k_len / 64)) tiles for each of its KV heads (an empty context still writes
// its zeros); tile i of the list belongs to the sequence, head and key tile that come from dividing through.
__device__ __forceinline__ int seq_begin(const TreeAttn& t, int b) { return min(max(t.cu_q[b], 0), t.T); }
__device__ __forceinline__ int seq_nodes(const TreeAttn& t, int b) { return min(t.cu_q[b + 1], t.T) - seq_begin(t, b); }
__device__ __forceinline__ int seq_tiles(const TreeAttn& t, int b) {
  return seq_nodes(t, b) > 0 ? max(1, (t.ctx_lens[b] + KT - 1) / KT) : 0;
}

struct Where {
  int b;        // sequence
  int64_t rem;  // tiles between its first one and the place
};

// total number of tiles, and the sequences in which places `lo` and `hi` of chunk `c` lie.  All threads of the CTA.
struct Spot {
  int64_t total, lo, hi;
  Where at_lo, at_hi;
};

__device__ void find_chunk(const Args& a, int c, Spot* out) {
  __shared__ int64_t part[33];
  const int nt = blockDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = nt >> 5;
  const int per = (a.t.num_seqs + nt - 1) / nt;
  const int b0 = min(a.t.num_seqs, (int)threadIdx.x * per), b1 = min(a.t.num_seqs, b0 + per);
  int64_t sum = 0;
  for (int b = b0; b < b1; ++b) sum += (int64_t)seq_tiles(a.t, b) * a.t.nkv;
  int64_t incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(FULL_MASK, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) part[warp] = incl;
  __syncthreads();
  if (threadIdx.x == 0) {
    int64_t s = 0;
    for (int w = 0; w < nw; ++w) {
      const int64_t x = part[w];
      part[w] = s;
      s += x;
    }
    part[32] = s;
    out->total = s;
    out->lo = s * c / a.chunks;
    out->hi = s * (c + 1) / a.chunks;
    out->at_lo.b = out->at_hi.b = a.t.num_seqs;
    out->at_lo.rem = out->at_hi.rem = 0;
  }
  __syncthreads();
  int64_t at = part[warp] + incl - sum;
  const int64_t lo = out->lo, hi = out->hi;
  for (int b = b0; b < b1; ++b) {
    const int64_t n = (int64_t)seq_tiles(a.t, b) * a.t.nkv;
    if (lo >= at && lo < at + n) out->at_lo = {b, lo - at};
    if (hi >= at && hi < at + n) out->at_hi = {b, hi - at};
    at += n;
  }
  __syncthreads();
}

// Walks the (sequence, KV head) pairs of a stretch: tiles [t0, t1) of each.
struct Walk {
  int b, h, t0, t1, tiles;
  int64_t left;
  __device__ __forceinline__ Walk(const Args& a, const Spot& s) {
    b = s.at_lo.b;
    left = s.hi - s.lo;
    tiles = 0;
    h = t0 = t1 = 0;
    if (left > 0) {
      tiles = seq_tiles(a.t, b);
      h = (int)(s.at_lo.rem / tiles);
      t0 = (int)(s.at_lo.rem % tiles);
      t1 = (int)min((int64_t)tiles, t0 + left);
    }
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ void next(const Args& a) {
    left -= t1 - t0;
    if (left <= 0) return;
    if (t1 == tiles && ++h == a.t.nkv) {
      h = 0;
      do ++b;
      while ((tiles = seq_tiles(a.t, b)) == 0);
    }
    t0 = 0;
    t1 = (int)min((int64_t)tiles, left);
  }
  // rows of this pair in row tile rt
  __device__ __forceinline__ int rows(const Args& a, int rt, int per_tile) const {
    return min(per_tile, min(seq_nodes(a.t, b), a.t.max_nodes) * a.G - rt * per_tile);
  }
};

// Partial sums of slot s (2 per CTA): rows x 128 outputs (not divided by the sum), then rows x (maximum, sum).
__device__ __forceinline__ float* slot_o(const Args& a, int rows, int cta, int slot) {
  return a.t.ws + (int64_t)(cta * 2 + slot) * rows * (AD + 2);
}

// ------------------------------------------------------------------------ main kernel
template <bool FP8>
struct Cfg {
  static constexpr int KV_BYTES = KT * AD * 2;        // one K or V tile in 16 bits
  static constexpr int STAGE = 2 * KV_BYTES;
  static constexpr int RING = FP8 ? 2 : 4;            // 16-bit stages
  static constexpr int RAW = FP8 ? 5 : 0;             // e4m3 stages
  static constexpr int RAW_STAGE = 2 * KT * AD;
  static constexpr int CONV = FP8 ? 4 : 0;            // converting warps
  static constexpr int THREADS = (NWARP + 1 + CONV) * 32;
  static constexpr int MERGE = NWARP * 16 * AD * 4;   // the warps' outputs
  static constexpr int SMEM = 1024 + RING * STAGE + RAW * RAW_STAGE + MERGE + NWARP * 16 * 8 + 512;
};

// Byte offset of (row, 16-byte chunk) in a 16-bit tile: [2 halves of 64 dims][64 rows][128 B], 128-byte swizzle.
__device__ __forceinline__ uint32_t tile_at(int r, int c16) {
  return (uint32_t)((c16 >> 3) * (KT * 128) + r * 128 + (((c16 & 7) ^ (r & 7)) << 4));
}

template <bool FP8, int RG>
__global__ void __launch_bounds__(Cfg<FP8>::THREADS, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, Args a) {
  using C = Cfg<FP8>;
  constexpr int SH = NWARP / RG;             // warps that share a row group
  constexpr int KG = SH < 4 ? SH : 4;        // of them, on different keys of one tile
  constexpr int TG = SH / KG;                // tiles worked on at a time
  constexpr int KW = KT / KG;                // keys of a warp
  constexpr int NT = KW / 8;                 // 8-key tiles of its scores
  constexpr int ROWS = RG * 16;
  pdl_wait();     // inputs come from the previous kernel in the stream
  pdl_trigger();  // the next kernel may start its prologue
  extern __shared__ __align__(1024) uint8_t raw_sm[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw_sm) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = sm;
  uint8_t* rawr = ring + C::RING * C::STAGE;
  float* merge_o = reinterpret_cast<float*>(rawr + C::RAW * C::RAW_STAGE);
  float2* merge_ml = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(merge_o) + C::MERGE);
  uint64_t* bars = reinterpret_cast<uint64_t*>(merge_ml + NWARP * 16);
  volatile int* gave_up = reinterpret_cast<volatile int*>(bars + 2 * (C::RING + C::RAW));
  __shared__ Spot spot;
  __shared__ float2 unit_scale[C::RING][KT / 16];  // e4m3: (K, V) scales of 16 keys
  const uint32_t bar0 = smem_u32(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (C::RING + s); };
  auto raw_full = [&](int s) { return bar0 + 8u * (2 * C::RING + s); };
  auto raw_empty = [&](int s) { return bar0 + 8u * (2 * C::RING + C::RAW + s); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rt = blockIdx.x % a.row_tiles, chunk = blockIdx.x / a.row_tiles;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::RING; ++s) {
      tc::mbar_init(full(s), FP8 ? C::CONV * 32 : 1);
      tc::mbar_init(empty(s), RG * KG);
    }
    for (int s = 0; s < C::RAW; ++s) {
      tc::mbar_init(raw_full(s), 1);
      tc::mbar_init(raw_empty(s), C::CONV);
    }
    *gave_up = 0;
    tc::fence_barrier_init();
  }
  find_chunk(a, chunk, &spot);  // ends with a barrier

  // Bounded wait; on expiry every role goes on without waiting, and the outputs are not valid.
  auto wait = [&](uint32_t bar, uint32_t parity, int code) -> bool {
    if (tc::mbar_try(bar, parity)) return true;
    SpinBudget sb;
    while (!tc::mbar_try(bar, parity)) {
      if (*gave_up) return false;
      if (sb.expired(WAIT_NS)) {
        atomicCAS(&g_tree_error, 0, code);
        *gave_up = 1;
        return false;
      }
    }
    return true;
  };

  if (warp == NWARP) {
    // ------------------------------------------------------------------ TMA producer
    if (lane != 0) return;
    tc::prefetch_map(&kmap);
    tc::prefetch_map(&vmap);
    constexpr int DEPTH = FP8 ? C::RAW : C::RING;
    int i = 0;
    bool ok = true;
    for (Walk w(a, spot); w.more() && ok; w.next(a)) {
      if (w.rows(a, rt, ROWS) <= 0) continue;
      const int* bt = a.t.block_tables + w.b * a.t.bt_stride;
      for (int t = w.t0; t < w.t1; ++t, ++i) {
        const int s = i % DEPTH;
        if (!wait(FP8 ? raw_empty(s) : empty(s), ((i / DEPTH) & 1) ^ 1, 1)) {
          ok = false;
          break;
        }
        const uint32_t bar = FP8 ? raw_full(s) : full(s);
        uint8_t* kd = FP8 ? rawr + s * C::RAW_STAGE : ring + s * C::STAGE;
        uint8_t* vd = kd + (FP8 ? C::RAW_STAGE : C::STAGE) / 2;
        tc::mbar_arrive_expect_tx(bar, FP8 ? C::RAW_STAGE : C::STAGE);
        for (int r = 0; r < KT; r += a.box_rows) {
          const int tok = t * KT + r, bi = tok >> a.bs_shift;
          int row = a.oob_row;
          if (bi < a.t.W) {
            const int blk = bt[bi];
            if (blk >= 0 && blk < a.t.num_blocks)
              row = ((blk * a.t.nkv + w.h) << a.bs_shift) + (tok & (a.t.block_size - 1));
          }
          if constexpr (FP8) {
            tc::tma_load_2d(smem_u32(kd + r * AD), &kmap, bar, 0, row);
            tc::tma_load_2d(smem_u32(vd + r * AD), &vmap, bar, 0, row);
          } else {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t off = half * (KT * 128) + r * 128;
              tc::tma_load_2d(smem_u32(kd + off), &kmap, bar, half * 64, row);
              tc::tma_load_2d(smem_u32(vd + off), &vmap, bar, half * 64, row);
            }
          }
        }
      }
    }
    // Do not leave while copies of this thread may still be landing.
    for (int j = max(0, i - DEPTH); j < i; ++j)
      tc::mbar_drain(FP8 ? raw_full(j % DEPTH) : full(j % DEPTH), (j / DEPTH) & 1);
    return;
  }

  if constexpr (FP8) {
    if (warp > NWARP) {
      // ------------------------------------------------------------ e4m3 -> f16 tiles
      const int tid = threadIdx.x - (NWARP + 1) * 32;
      int i = 0;
      for (Walk w(a, spot); w.more(); w.next(a)) {
        if (w.rows(a, rt, ROWS) <= 0) continue;
        const int* bt = a.t.block_tables + w.b * a.t.bt_stride;
        const int k_len = a.t.ctx_lens[w.b];
        for (int t = w.t0; t < w.t1; ++t, ++i) {
          const int s = i % C::RAW, d = i % C::RING;
          float2 sc = make_float2(0.f, 0.f);
          if (tid < KT / 16) {
            const int bi = (t * KT + tid * 16) >> a.bs_shift;
            const int blk = bi < a.t.W ? bt[bi] : -1;
            if (blk >= 0 && blk < a.t.num_blocks) {
              const int64_t at = (int64_t)blk * a.t.nkv + w.h;
              sc = make_float2(a.t.k_scale[at], a.t.v_scale[at]);
            }
          }
          wait(raw_full(s), (i / C::RAW) & 1, 2);
          wait(empty(d), ((i / C::RING) & 1) ^ 1, 3);
          if (tid < KT / 16) unit_scale[d][tid] = sc;
          const uint8_t* src = rawr + s * C::RAW_STAGE;
          uint8_t* dst = ring + d * C::STAGE;
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const int idx = tid + (u & 3) * 128, r = idx >> 3, c = idx & 7;  // 16 values of row r
            uint4 x = *reinterpret_cast<const uint4*>(src + (u >> 2) * KT * AD + idx * 16);
            // positions behind the context may hold any bytes, a NaN included
            if (t * KT + r >= k_len) x = make_uint4(0, 0, 0, 0);
            const uint32_t in[4] = {x.x, x.y, x.z, x.w};
            uint32_t h[8];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
                  : "=r"(h[2 * e]), "=r"(h[2 * e + 1])
                  : "r"(in[e]));
            uint8_t* to = dst + (u >> 2) * C::KV_BYTES;
            *reinterpret_cast<uint4*>(to + tile_at(r, 2 * c)) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(to + tile_at(r, 2 * c + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
          }
          tc::mbar_arrive_release(full(d));
          __syncwarp();
          if (lane == 0) tc::mbar_arrive_release(raw_empty(s));
        }
      }
      return;
    }
  }

  // -------------------------------------------------------------------- working warps
  const int rg = warp % RG, kg = warp / RG % KG, tg = warp / (RG * KG);
  const int key0 = kg * KW;  // this warp's keys in a tile
  const int c2 = (lane & 3) * 2;
  int i = 0;  // tiles so far
  for (Walk w(a, spot); w.more(); w.next(a)) {
    const int rows = w.rows(a, rt, ROWS);
    if (rows <= 0) continue;
    const int qrow = seq_begin(a.t, w.b), n_nodes = seq_nodes(a.t, w.b), k_len = a.t.ctx_lens[w.b];
    const int base = k_len - n_nodes;
    const int rr[2] = {rg * 16 + (lane >> 2), rg * 16 + (lane >> 2) + 8};  // this thread's rows in the tile
    int node[2];
    uint32_t qf[8][4];
    float qmul[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bool live = rr[e] < rows;
      const int r = rt * ROWS + (live ? rr[e] : 0);
      node[e] = r / a.G;
      const uint32_t* qp = reinterpret_cast<const uint32_t*>(
          static_cast<const __nv_bfloat16*>(a.t.q) + (int64_t)(qrow + node[e]) * a.t.q_stride + (w.h * a.G + r % a.G) * AD);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        qf[kk][e] = live ? qp[kk * 8 + (lane & 3)] : 0u;
        qf[kk][2 + e] = live ? qp[kk * 8 + (lane & 3) + 4] : 0u;
      }
      qmul[e] = a.scale_log2;
      if constexpr (FP8) {
        // f16 holds 11 bits, but not bf16's range: the row by a power of two that brings it below 256
        float m = 0.f;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const float2 x = unpack<false>(qf[kk][e]), y = unpack<false>(qf[kk][2 + e]);
          m = fmaxf(m, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))));
        }
        m = fmaxf(m, __shfl_xor_sync(FULL_MASK, m, 1));
        m = fmaxf(m, __shfl_xor_sync(FULL_MASK, m, 2));
        const int ex = (int)(__float_as_uint(m) >> 23) - 127;  // m < 2^(ex + 1)
        const int by = m > 0.f && ex < 128 ? max(-126, min(126, 7 - ex)) : 0;
        const float f = __int_as_float((127 + by) << 23);
        qmul[e] *= __int_as_float((127 - by) << 23);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const float2 x = unpack<false>(qf[kk][e]), y = unpack<false>(qf[kk][2 + e]);
          qf[kk][e] = pack<true>(x.x * f, x.y * f);
          qf[kk][2 + e] = pack<true>(y.x * f, y.y * f);
        }
      }
    }
    float acc[16][4];
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float unit = 1.f;  // e4m3: V's scale that the sums are in units of

    for (int t = w.t0; t < w.t1; ++t, ++i) {
      if (TG > 1 && i % TG != tg) continue;
      const int s = i % C::RING;
      wait(full(s), (i / C::RING) & 1, 4);
      const uint32_t kb = smem_u32(ring + s * C::STAGE), vb = kb + C::KV_BYTES;
      if (rg * 16 < rows) {
        float sc[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
#pragma unroll
          for (int np = 0; np < NT / 2; ++np) {
            uint32_t kf[4];
            const int r = key0 + np * 16 + (lane & 7) + ((lane >> 4) << 3), c = kk * 2 + ((lane >> 3) & 1);
            ldsm4(kb + tile_at(r, c), kf);
            mma<FP8>(sc[2 * np], qf[kk], kf[0], kf[1]);
            mma<FP8>(sc[2 * np + 1], qf[kk], kf[2], kf[3]);
          }
        // scores in units of log2; keys that a row does not see: -inf
        const bool masked = t * KT + KT > base;
        uint64_t see[2] = {~0ull, ~0ull};
        if (masked) {
          const int d = base - t * KT;  // keys of this tile before the tree (below 0: nodes in earlier tiles)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int64_t* mw = a.t.mask + (int64_t)(qrow + node[e]) * a.t.mask_stride;
            if (d > 0) {
              see[e] = (1ull << d) - 1 | (uint64_t)mw[0] << d;
            } else {
              const int word = -d >> 6, sh = -d & 63;
              const uint64_t lo = word < a.t.words ? (uint64_t)mw[word] : 0, hi = word + 1 < a.t.words ? (uint64_t)mw[word + 1] : 0;
              see[e] = sh ? lo >> sh | hi << (64 - sh) : lo;
            }
            const int valid = k_len - t * KT;
            if (valid < KT) see[e] &= valid > 0 ? (1ull << valid) - 1 : 0ull;
            see[e] >>= key0;
          }
        }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float f = qmul[e >> 1];
            if constexpr (FP8) f *= unit_scale[s][(key0 + j * 8) >> 4].x;
            sc[j][e] *= f;
            if (masked && !(see[e >> 1] >> (j * 8 + c2 + (e & 1)) & 1)) sc[j][e] = -INFINITY;
            mx[e >> 1] = fmaxf(mx[e >> 1], sc[j][e]);
          }
        float al[2], bs[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(FULL_MASK, mx[e], 1));
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(FULL_MASK, mx[e], 2));
          mx[e] = fmaxf(mx[e], m[e]);
          bs[e] = mx[e] == -INFINITY ? 0.f : mx[e];
          al[e] = ex2(m[e] - bs[e]);
          // f16: weights up to 2^15, so that those down to 2^-29 of the largest keep 11 bits; the sums share the factor
          if constexpr (FP8) bs[e] -= 15.f;
          m[e] = mx[e];
          l[e] *= al[e];
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sc[j][e] = ex2(sc[j][e] - bs[e >> 1]);
            l[e >> 1] += sc[j][e];
          }
#pragma unroll
        for (int ks = 0; ks < KW / 16; ++ks) {  // 16 keys at a time
          float f[2] = {1.f, 1.f};
          if (ks == 0) {
            f[0] = al[0];
            f[1] = al[1];
          }
          bool gone = false;
          if constexpr (FP8) {
            const float vs = unit_scale[s][(key0 >> 4) + ks].y;
            gone = vs == 0.f;  // no block, or one of zeros
            if (!gone) {
              f[0] *= unit / vs;
              f[1] *= unit / vs;
              unit = vs;
            }
          }
          if (__any_sync(FULL_MASK, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              acc[j][0] *= f[0];
              acc[j][1] *= f[0];
              acc[j][2] *= f[1];
              acc[j][3] *= f[1];
            }
          }
          if (gone) continue;
          // P is rounded to the type of V: 2^-9 (bf16) or 2^-12 (f16) of each weight at most; the sum l is not
          const uint32_t pf[4] = {pack<FP8>(sc[2 * ks][0], sc[2 * ks][1]), pack<FP8>(sc[2 * ks][2], sc[2 * ks][3]),
                                  pack<FP8>(sc[2 * ks + 1][0], sc[2 * ks + 1][1]),
                                  pack<FP8>(sc[2 * ks + 1][2], sc[2 * ks + 1][3])};
          uint32_t keep0 = ~0u, keep1 = ~0u, odd = 0;
          if (masked) {
            // positions behind the context hold any bits
            const int k = t * KT + key0 + ks * 16 + c2;
            keep0 = (k < k_len ? 0xffffu : 0u) | (k + 1 < k_len ? 0xffff0000u : 0u);
            keep1 = (k + 8 < k_len ? 0xffffu : 0u) | (k + 9 < k_len ? 0xffff0000u : 0u);
          }
#pragma unroll
          for (int np = 0; np < 8; ++np) {
            uint32_t vf[4];
            const int r = key0 + ks * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, c = np * 2 + (lane >> 4);
            ldsm4t(vb + tile_at(r, c), vf);
            if (masked) {
              vf[0] &= keep0;
              vf[2] &= keep0;
              vf[1] &= keep1;
              vf[3] &= keep1;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t o = odd_halves<FP8>(vf[e]);
                odd |= o;
                vf[e] &= ~((o >> 15) * 0xffffu);  // to 0: added below where it is seen
              }
            }
            mma<FP8>(acc[2 * np], pf, vf[0], vf[1]);
            mma<FP8>(acc[2 * np + 1], pf, vf[2], vf[3]);
          }
          if (masked && __any_sync(FULL_MASK, odd != 0)) {
            // infinities and NaN, for the rows that see them
            for (int kx = 0; kx < 16; ++kx) {
              const int key = key0 + ks * 16 + kx;
              if (t * KT + key >= k_len) break;
              const int from = (lane & 28) | ((kx & 7) >> 1);
              float p[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float x0 = __shfl_sync(FULL_MASK, sc[2 * ks][2 * e], from), x1 = __shfl_sync(FULL_MASK, sc[2 * ks][2 * e + 1], from);
                const float y0 = __shfl_sync(FULL_MASK, sc[2 * ks + 1][2 * e], from), y1 = __shfl_sync(FULL_MASK, sc[2 * ks + 1][2 * e + 1], from);
                p[e] = kx < 8 ? (kx & 1 ? x1 : x0) : (kx & 1 ? y1 : y0);
              }
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                uint32_t x;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(vb + tile_at(key, j) + (lane & 3) * 4) : "memory");
                const uint32_t o = odd_halves<FP8>(x);
                const float2 v = unpack<FP8>(x);
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (see[e] >> (ks * 16 + kx) & 1) {
                    if (o & 0x8000u) acc[j][2 * e] += p[e] * v.x;
                    if (o & 0x80000000u) acc[j][2 * e + 1] += p[e] * v.y;
                  }
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive_release(empty(s));
    }

    // ---- join the warps of each row group
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(FULL_MASK, l[e], 1);
      l[e] += __shfl_xor_sync(FULL_MASK, l[e], 2);
    }
    // this warp's 16 x 128 outputs; columns are moved by the row so that a store's rows meet no bank twice
    float* mo = merge_o + warp * 16 * AD;
    const int r0 = lane >> 2;
    if ((lane & 3) == 0) {
      merge_ml[warp * 16 + r0] = make_float2(m[0], l[0]);
      merge_ml[warp * 16 + r0 + 8] = make_float2(m[1], l[1]);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int c = (j * 8 + c2) ^ ((r0 & 3) << 3);
      *reinterpret_cast<float2*>(mo + r0 * AD + c) = make_float2(acc[j][0] * unit, acc[j][1] * unit);
      *reinterpret_cast<float2*>(mo + (r0 + 8) * AD + c) = make_float2(acc[j][2] * unit, acc[j][3] * unit);
    }
    asm volatile("bar.sync 1, %0;" ::"n"(NWARP * 32) : "memory");
    const bool whole = w.t0 == 0 && w.t1 == w.tiles;
    float* po = slot_o(a, ROWS, blockIdx.x, w.t0 == 0);
    // a thread takes 4 columns of a row
    for (int x = threadIdx.x; x < rows * (AD / 4); x += NWARP * 32) {
      const int r = x / (AD / 4), c = x % (AD / 4) * 4, g = r >> 4, q = r & 15;
      float M = -INFINITY;
#pragma unroll
      for (int k = 0; k < SH; ++k) M = fmaxf(M, merge_ml[(k * RG + g) * 16 + q].x);
      const float mb = M == -INFINITY ? 0.f : M;
      float L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < SH; ++k) {
        const float2 ml = merge_ml[(k * RG + g) * 16 + q];
        if (ml.x == -INFINITY && ml.y == 0.f) continue;  // saw nothing
        const float f = ex2(ml.x - mb);
        const float4 v = *reinterpret_cast<const float4*>(merge_o + ((k * RG + g) * 16 + q) * AD + (c ^ ((q & 3) << 3)));
        L += f * ml.y;
        o[0] += f * v.x;
        o[1] += f * v.y;
        o[2] += f * v.z;
        o[3] += f * v.w;
      }
      if (whole) {
        const float inv = L != 0.f ? 1.f / L : 0.f;
        const int R = rt * ROWS + r;
        __nv_bfloat16* op = static_cast<__nv_bfloat16*>(a.t.out) +
                            ((int64_t)(qrow + R / a.G) * a.t.nq + w.h * a.G + R % a.G) * AD + c;
        float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
        if (L == 0.f) v[0] = v[1] = v[2] = v[3] = 0.f;
        *reinterpret_cast<uint2*>(op) = f32_to_bf16x4(v);
      } else {
        *reinterpret_cast<float4*>(po + r * AD + c) = make_float4(o[0], o[1], o[2], o[3]);
        if (c == 0) *reinterpret_cast<float2*>(po + ROWS * AD + r * 2) = make_float2(M, L);
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(NWARP * 32) : "memory");  // the outputs are read
  }
}

// ---------------------------------------------------------------------------- joining
// CTA (chunk, row tile, 16 rows) joins the pair that begins in its chunk and ends in a later one.
__global__ void __launch_bounds__(128) tree_join_kernel(Args a, int ROWS) {
  pdl_wait();     // the partial sums come from the previous kernel in the stream
  pdl_trigger();  // the next kernel may start its prologue
  __shared__ Spot spot;
  const int rt = blockIdx.x % a.row_tiles, chunk = blockIdx.x / a.row_tiles;
  find_chunk(a, chunk, &spot);
  const int64_t lo = spot.lo, hi = spot.hi;
  if (hi <= lo || hi >= spot.total) return;
  const int b = spot.at_hi.b, tiles = seq_tiles(a.t, b);
  const int h = (int)(spot.at_hi.rem / tiles), t = (int)(spot.at_hi.rem % tiles);
  const int64_t begin = hi - t, end = begin + tiles;
  if (t == 0 || begin < lo) return;  // nothing is cut here, or the pair begins in an earlier chunk
  const int rows = min(ROWS, min(seq_nodes(a.t, b), a.t.max_nodes) * a.G - rt * ROWS);
  const int qrow = seq_begin(a.t, b);
  const int r = blockIdx.y * 4 + (threadIdx.x >> 5), c = (threadIdx.x & 31) * 4;
  if (r >= rows) return;
  float M = -INFINITY, L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  int64_t from = lo, upto = hi;
  for (int k = chunk;; ++k) {
    if (upto > from) {  // with fewer tiles than chunks, some have none
      const float* po = slot_o(a, ROWS, k * a.row_tiles + rt, k == chunk);
      const float2 ml = *reinterpret_cast<const float2*>(po + ROWS * AD + r * 2);
      const float4 v = *reinterpret_cast<const float4*>(po + r * AD + c);
      if (!(ml.x == -INFINITY && ml.y == 0.f)) {
        const float nm = fmaxf(M, ml.x), nb = nm == -INFINITY ? 0.f : nm;
        const float f = L == 0.f && M == -INFINITY ? 0.f : ex2(M - nb), g = ex2(ml.x - nb);
        M = nm;
        L = L * f + g * ml.y;
        o[0] = (f == 0.f ? 0.f : o[0] * f) + g * v.x;
        o[1] = (f == 0.f ? 0.f : o[1] * f) + g * v.y;
        o[2] = (f == 0.f ? 0.f : o[2] * f) + g * v.z;
        o[3] = (f == 0.f ? 0.f : o[3] * f) + g * v.w;
      }
    }
    if (upto >= end) break;
    from = upto;
    upto = spot.total * (k + 2) / a.chunks;
  }
  const float inv = L != 0.f ? 1.f / L : 0.f;
  float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  if (L == 0.f) v[0] = v[1] = v[2] = v[3] = 0.f;
  const int R = rt * ROWS + r;
  *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.t.out) +
                            ((int64_t)(qrow + R / a.G) * a.t.nq + h * a.G + R % a.G) * AD + c) = f32_to_bf16x4(v);
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> fn{nullptr};
  auto f = fn.load();
  if (!f) {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn.store(f = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p));
  }
  return f;
}

// The pool as rows of 128 values; boxes of 64 bf16 values (the swizzle's width) or 128 e4m3 ones.
bool pool_map(CUtensorMap* m, const void* base, int64_t rows, bool fp8, int box_rows) {
  auto enc = encoder();
  if (!enc) return false;
  cuuint64_t dims[2] = {(cuuint64_t)AD, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(fp8 ? AD : AD * 2)};
  cuuint32_t box[2] = {(cuuint32_t)(fp8 ? AD : 64), (cuuint32_t)box_rows};
  cuuint32_t one[2] = {1, 1};
  return enc(m, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base),
             dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             fp8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool FP8, int RG>
cudaError_t launch_main(const CUtensorMap& km, const CUtensorMap& vm, const Args& a, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  cudaError_t e = smem_opt_in(done, tree_attn_kernel<FP8, RG>, Cfg<FP8>::SMEM);
  if (e != cudaSuccess) return e;
  return launch_pdl(tree_attn_kernel<FP8, RG>, dim3(a.chunks * a.row_tiles), dim3(Cfg<FP8>::THREADS), Cfg<FP8>::SMEM,
                    stream, km, vm, a);
}

}  // namespace

// Row groups by the rows of the largest tree; one CTA per SM (shared memory allows one).
TreeAttnPlan tree_attn_plan(int num_seqs, int max_nodes, int nq, int nkv, int num_sms) {
  TreeAttnPlan p;
  const int rows = max_nodes * (nq / nkv);
  p.rg = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  p.row_tiles = (rows + p.rg * 16 - 1) / (p.rg * 16);
  p.chunks = num_sms / p.row_tiles > 1 ? num_sms / p.row_tiles : 1;
  p.ws_floats = 2LL * p.chunks * p.row_tiles * p.rg * 16 * (AD + 2);
  (void)num_seqs;
  return p;
}

cudaError_t launch_tree_attention(const TreeAttn& t, const TreeAttnPlan& p, cudaStream_t stream) {
  const int64_t rows = (int64_t)t.num_blocks * t.nkv * t.block_size;
  if (t.num_seqs <= 0 || t.nkv <= 0 || t.nq % t.nkv || t.block_size < 16 || (t.block_size & (t.block_size - 1)) ||
      t.max_nodes < 1 || t.max_nodes > TREE_MAX_NODES || rows >= (int64_t)INT32_MAX - 256)
    return cudaErrorInvalidValue;
  Args a;
  a.t = t;
  a.G = t.nq / t.nkv;
  a.row_tiles = p.row_tiles;
  a.chunks = p.chunks;
  a.bs_shift = __builtin_ctz((unsigned)t.block_size);
  a.box_rows = t.block_size < KT ? t.block_size : KT;
  a.oob_row = (int)rows;
  a.scale_log2 = t.softmax_scale * LOG2E;
  CUtensorMap km, vm;
  if (!pool_map(&km, t.k_cache, rows, t.kv_fp8, a.box_rows) || !pool_map(&vm, t.v_cache, rows, t.kv_fp8, a.box_rows))
    return cudaErrorInvalidValue;
  cudaError_t e;
  if (t.kv_fp8)
    e = p.rg == 1 ? launch_main<true, 1>(km, vm, a, stream)
                  : p.rg == 2 ? launch_main<true, 2>(km, vm, a, stream) : launch_main<true, 4>(km, vm, a, stream);
  else
    e = p.rg == 1 ? launch_main<false, 1>(km, vm, a, stream)
                  : p.rg == 2 ? launch_main<false, 2>(km, vm, a, stream) : launch_main<false, 4>(km, vm, a, stream);
  if (e != cudaSuccess) return e;
  return launch_pdl(tree_join_kernel, dim3(a.chunks * a.row_tiles, p.rg * 4), dim3(128), 0, stream, a, p.rg * 16);
}

int tree_attn_error_code(int reset) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_tree_error, sizeof(int));
  if (reset) {
    const int z = 0;
    cudaMemcpyToSymbol(g_tree_error, &z, sizeof(int));
  }
  return v;
}

}  // namespace nvb
