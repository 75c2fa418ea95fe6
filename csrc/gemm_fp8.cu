// fp8 (e4m3) matrix product with block scales on the 5th-generation tensor cores, sm_100a.
//
//   Y[t, n] = sum_b xs[t, b] ws[n / 128, b] sum_{k in block b} xq[t, k] wq[n, k]
//
// b runs over blocks of 128 channels: activations carry a scale per token and block, weights one
// per 128 x 128 block.  The scales are arbitrary fp32 numbers, so the tensor core cannot apply
// them: every block's product is a separate MMA accumulation in TMEM, and the epilogue warps add it,
// scaled, to fp32 accumulators in registers while the tensor core works on the next block (two TMEM
// buffers).
//
// No counterpart in the reference, whose linear layers are 16-bit (nanovllm/models/qwen3.py:96-134).
//
// The bf16 output is rounded once, from the fp32 sums: RoPE, attention and the residual addition behind
// these products take bf16.  The 8-bit output of SiLU-and-mul is rounded once too, from fp32.
//
// gemm_fp8_tokens_kernel<CTAS, BN>: tiles of 128 tokens (MMA M, one TMEM lane each) x BN = 256 or 128
// features (MMA N) per CTA; CTAS = 2: a pair of CTAs (tcgen05.mma.cta_group::2) shares the weight rows of
// a tile of 256 tokens, each staging half of them.  A thread of the epilogue owns one token and 64
// features of each 128-row weight block of the tile: each scale is then one number per thread and
// k-block (no scale vector to load), and with gate and up rows in alternating blocks of 128 the thread
// holds matching gate / up pairs, so SiLU-and-mul needs no exchange and a tile of 256 is one whole group
// of 128 of the 8-bit output.
//
// What bounds it: not one thing alone, as far as is known.  Per k-block and 256 features the tensor core needs 512
// clocks.  Whole calls take 910 with 96 k-blocks per tile and 1010 with 32, the tile's end included: 8192 x
// 4096 x 12288 434 us (1.90 PFLOP/s) and gate / up of 16384 x 24576 x 4096 1.77 ms (1.87), in a row at the 1000 W
// limit, which holds the clock at 1.42 and 1.55 GHz.  In the loop the chain MMA -> commit -> poll -> TMEM loads and
// additions -> arrival -> poll -> MMA took 1540 clocks, two of them in flight, when it was last timed by itself;
// the loads and additions alone, without a tensor core at work, take 320.  16 epilogue warps of 32 features per
// block, with half the registers each, were 10% slower (386 against 350 us beside each other); asking for the
// next product's barrier ahead of the additions changed nothing.
//
// gemm_fp8_weights_kernel<NP, MW>: few tokens.  Tiles of 128 weight rows (MMA M) x NP tokens (MMA N), so a
// step of one token moves 16 activation rows beside the weights instead of 128, and K split over the
// CTAs of a cluster so that the weights of a small layer are streamed by the whole GPU.  A thread
// owns one feature and all NP tokens; the K slices' fp32 sums meet in shared memory: every CTA stores
// the sums of token c straight into CTA c mod splits (distributed shared memory), which adds them in
// the order of the slices (the result does not depend on timing), finishes and stores the token.  For
// SiLU-and-mul a CTA holds both tiles of a group: its gate rows and the matching up rows.
//
// What bounds it: the weights.  One token, 6144 x 4096: 6.8 us; 4096 x 12288: 10.9 us (4.6 TB/s); gate / up
// of 2 x 12288 x 4096: 21.2 us in a graph (4.75 TB/s), of which 14.1 us are spent streaming at 7.1 TB/s, 1.7
// pass until the first stage has landed, 2.3 until the slowest CTA is done, and 2 in the reduction and the
// next launch.  Weights are prefetched into L2 for the first ring only, while the previous kernel ends:
// two rings deep cost 2%, four 8%.
//
// Neither kernel uses a global workspace.  Every wait on an mbarrier is bounded; on expiry the kernel records
// an error code in a word of host memory, drains its copies, frees TMEM and returns, with an output that is
// not valid: whoever reads the output back checks the word (fp8_error).  Cluster barriers, TMEM allocation and
// the wait for the previous kernel have no bound of their own; every thread reaches them, on the error path too.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "fp8_quant.cuh"
#include "tcgen05.cuh"

namespace nvb {

namespace {

using namespace tc;

constexpr int BM = 128;                 // tokens per CTA
constexpr int BK = 128;                 // one scale block = one 128-byte swizzle row
constexpr int EPI_THREADS = 256;
constexpr int THREADS = 128 + EPI_THREADS;  // TMA warp, MMA warp, two scale warps; 8 epilogue warps
// Registers: the 12 warps are launched with 168 each (65536 / 384); the control warps give theirs up
// for the epilogue's, which hold 128 sums and two TMEM loads of 32 values.
constexpr int LAUNCH_REGS = 168, CONTROL_REGS = 56, EPI_REGS = 224;
static_assert(4 * CONTROL_REGS + 8 * EPI_REGS <= 12 * LAUNCH_REGS, "the launch's registers");

// CTAS CTAs share a tile of CTAS x 128 tokens x BN features.
template <int CTAS, int BN>
struct TokensCfg {
  static constexpr int BUFS = 512 / BN;     // accumulator buffers: all of TMEM
  static constexpr int BLOCKS = BN / 128;   // 128-row blocks of W in a tile, each with a scale of its own
  static constexpr int B_ROWS = BN / CTAS;  // weight rows staged by one CTA
  static constexpr int A_BYTES = BM * BK, STAGE = A_BYTES + B_ROWS * BK;  // 48 or 32 KB
  static constexpr int STAGES = STAGE == 48 * 1024 ? 4 : 6;
  static constexpr int STAGING = EPI_THREADS / 32 * 2048;
  // K-blocks whose scale products are kept, in two halves, which the epilogue gives back whole: an arrival for
  // each k-block cost 2-3%.  As many barriers announce a product and its scales, so that the scale warps run
  // ahead without looking at the products.
  static constexpr int PRODS = 8, HALF = PRODS / 2;
  static constexpr int BARS = 3 * STAGES + PRODS + 2 + 2;
  static constexpr int XLD = BN + 4;        // exchange row: 16-byte stores of 8 rows hit distinct banks
  static constexpr int SMEM = 1024 + STAGES * STAGE + STAGING + STAGES * BM * 4 + PRODS * BLOCKS * BM * 4 +
                              2 * 2 * BM * 4 + 8 * BARS + 16;
  static_assert(SMEM <= 227 * 1024, "shared memory of a CTA");
  static_assert(BM * XLD * 4 <= STAGES * STAGE, "the exchange fits over the ring");
  static_assert(BUFS <= STAGES, "a stage's barrier takes the arrivals of one k-block at a time");
  static_assert(BUFS <= PRODS, "a product's barrier takes the arrivals of one k-block at a time");
};

// Shape of gemm_fp8_weights_kernel<NP, MW>: NP tokens (rounded up), MW = 1 or (SiLU-and-mul: a block of 128
// gate rows and the matching up rows) 2 tiles of 128 weight rows per CTA.  Two CTAs fit on an SM, so
// that one streams while the other fills its pipeline or finishes, and so that the next kernel's CTAs
// start early.
template <int NP, int MW>
struct WeightsCfg {
  static constexpr int COL_SPLIT = NP >= 64 ? 2 : 1;           // warps that share a quarter of the lanes
  static constexpr int NC = NP / COL_SPLIT;                    // tokens per epilogue thread
  static constexpr int CHUNK = NC == 32 ? 32 : 16;             // TMEM columns per load
  static constexpr int EPI_WARPS = 4 * COL_SPLIT * MW;
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int ACC_BUFS = MW == 2 ? 2 : 4;             // TMEM buffers (at most as many as stages)
  static constexpr int TMEM_COLS = ACC_BUFS * MW * NP;         // 64 .. 256
  static constexpr int ROWS = 128 * MW;
  static constexpr int W_BYTES = ROWS * BK, X_BYTES = NP * BK, STAGE = W_BYTES + X_BYTES;
  // fp32 sums of the tokens this CTA finishes: slices x ceil(NP / slices) <= NP + 7 rows; beside the
  // ring where that leaves it deep enough, over it otherwise
  static constexpr int EXCHANGE = (NP + 8) * ROWS * 4;
  static constexpr bool OVER_RING = NP * MW >= 32 && !(NP == 32 && MW == 1);
  static constexpr int SLOT = NP * 4 < 128 ? 128 : NP * 4;     // activation scales of one k-block
  static constexpr int BUDGET = 113 * 1024;
  static constexpr int bars(int s) { return 4 * s + 3 * ACC_BUFS + 3; }
  static constexpr int ring_bytes(int s) {
    return OVER_RING ? (s * STAGE > EXCHANGE ? s * STAGE : EXCHANGE) : s * STAGE + EXCHANGE;
  }
  static constexpr int smem(int s) { return 1024 + ring_bytes(s) + (s + ACC_BUFS + 1) * SLOT + 8 * bars(s) + 16; }
  static constexpr int stages() {
    int s = 8;
    while (s > 2 && smem(s) > BUDGET) --s;
    return s;
  }
  static constexpr int STAGES = stages();
  static constexpr int SLOTS = STAGES + ACC_BUFS + 1;
  static constexpr int BARS = bars(STAGES);
  static constexpr int SMEM = smem(STAGES);
  static_assert(SMEM <= BUDGET, "two CTAs per SM");
  static_assert(ACC_BUFS <= STAGES, "a stage's barrier takes the arrivals of one k-block at a time");
};

// A wait of a whole warp that stays together afterwards.  All lanes poll: electing one to do it costs
// more (the divergent branch and the broadcast) than the 31 other polls of the same word.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* word, int code) {
  return __all_sync(FULL_MASK, mbar_wait(bar, parity, abort_flag, word, code));
}

struct Params {
  int splits, kb_per_split;  // K slices and their length in k-blocks
  const float* ws;
  int64_t ldws;
  int T, N, num_kb, nb;      // nb: 128-row blocks of W
  int tiles_m, tiles_n, group;
  int act, features;
  int vec, tma_out;          // bf16 rows allow 16-byte stores; the output is stored by TMA
  void* out;
  int64_t ldo;
  float* os;
  int64_t ldos;
  int* error;                // the process's error word
};

// Tile order: groups of `group` token tiles walk the features together, so that CTAs which run at
// the same time share operand tiles in L2.
__device__ __forceinline__ void tile_coords(const Params& p, int t, int& tm, int& tn) {
  const int per_group = p.group * p.tiles_n;
  const int g = t / per_group;
  const int first = g * p.group;
  const int size = min(p.group, p.tiles_m - first);
  const int r = t - g * per_group;
  tm = first + r % size;
  tn = r / size;
}

// g / (1 + e^-g) with e^-g = 2^(-g log2 e), by the approximate base-2 exponential and reciprocal (relative
// errors of 2^-22 and 2^-23; the product -g log2 e adds |g| 2^-24): far inside the 8-bit rounding that
// follows.  A reciprocal below 2^-126 counts as zero: gates below -87.3, where silu is under 1.1e-36 in magnitude.
__device__ __forceinline__ float silu_f(float g) {
  float e, q;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.44269504f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.f + e));
  return g * q;
}

// acc += s * 32 values, two per instruction: half the issue slots of scalar additions (3% of the kernel).
__device__ __forceinline__ void add32(float* acc, const uint32_t (&v)[32], float s) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) fma2(acc[i], acc[i + 1], v[i], v[i + 1], s);
}

// The scales of one 128-row block of W for k-blocks 0, 1, .. n - 1, asked for in this order by a whole
// warp.  Lane l holds those of l, l + 32, ..: 32 per load, which is under way 32 k-blocks early (a load
// per k-block, with one k-block to arrive in, held the epilogue up by 500 clocks each).
struct WeightScales {
  const float* w;
  int n, lane;
  float now, next;
  __device__ __forceinline__ WeightScales(const float* w_, int n_, int lane_) : w(w_), n(n_), lane(lane_) {
    now = lane < n ? w[lane] : 0.f;
    next = lane + 32 < n ? w[lane + 32] : 0.f;
  }
  __device__ __forceinline__ float at(int kb) {
    if ((kb & 31) == 0 && kb > 0) {
      now = next;
      next = kb + 32 + lane < n ? w[kb + 32 + lane] : 0.f;
    }
    return __shfl_sync(FULL_MASK, now, kb & 31);
  }
};

// silu(gate) * up of 4 + 4 sums of the features [f, f + 4) of token t, one warp per token and group of
// 128: the fp32 sums are rounded once, to 8 bits.
__device__ __forceinline__ void finish_silu4(const Params& p, int t, int group, int lane, const float* g, const float* u) {
  const int f = group * 128 + lane * 4;
  uint32_t m = 0;
  float h[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = f < p.features ? silu_f(g[e]) * u[e] : 0.f;
    m = max(m, __float_as_uint(h[e]) & 0x7fffffffu);
  }
  const Fp8Scale sc = fp8_scale(__reduce_max_sync(FULL_MASK, m));
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] *= sc.inv;
  if (f < p.features)
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.out) + (int64_t)t * p.ldo + f) = f32x4_to_e4m3(h);
  if (lane == 0) p.os[(int64_t)group * p.ldos + t] = sc.scale;
}

// bf16 values [n, n + 4) of token t.
__device__ __forceinline__ void finish_bf16x4(const Params& p, int t, int n, const float* o) {
  __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + (int64_t)t * p.ldo + n;
  if (p.vec && n + 4 <= p.N) {
    *reinterpret_cast<uint2*>(dst) = f32_to_bf16x4(o);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) dst[e] = __float2bfloat16_rn(o[e]);
  }
}

// Tokens [128 slice / S, 128 (slice + 1) / S) of a tile whose sums lie in the S CTAs of the cluster: added
// in the order of the slices, finished and stored.  A warp takes a token's sums of one slice and 128
// features as one 512-byte row (remote stores of each thread's own 16 bytes were slower by half) and has
// 16 of them in flight.
template <int BN, int S>
__device__ __forceinline__ void finish_rows(const Params& p, float* exchange, int slice, int row0, int tn, int w,
                                            int lane) {
  constexpr int XLD = TokensCfg<1, BN>::XLD, NB = BN / 128;
  constexpr int PER = BM / S, G = 16 / NB / S;
  for (int tl = w * G; tl < PER; tl += EPI_THREADS / 32 * G) {
    const int r0 = slice * PER + tl;
    if (row0 + r0 >= p.T) break;
    const uint32_t src = smem_u32(exchange + r0 * XLD + lane * 4);
    float4 a[G][S][NB];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const uint32_t at = cluster_map(src, s);
#pragma unroll
      for (int i = 0; i < G; ++i)
#pragma unroll
        for (int h = 0; h < NB; ++h) a[i][s][h] = ld_cluster_f32x4(at + (i * XLD + h * 128) * 4);
    }
#pragma unroll
    for (int i = 0; i < G; ++i) {
      float o[NB][4] = {};
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int h = 0; h < NB; ++h) {
          o[h][0] += a[i][s][h].x; o[h][1] += a[i][s][h].y; o[h][2] += a[i][s][h].z; o[h][3] += a[i][s][h].w;
        }
      const int row = row0 + r0 + i;
      if (row < p.T) {  // the same for the whole warp
        if (BN == 256 && p.act) {
          finish_silu4(p, row, tn, lane, o[0], o[NB - 1]);
        } else {
#pragma unroll
          for (int h = 0; h < NB; ++h) finish_bf16x4(p, row, tn * BN + h * 128 + lane * 4, o[h]);
        }
      }
    }
  }
}

// With one CTA per tile: one tile per cluster of splits CTAs, each a slice of K, or, with splits = 1,
// persistent CTAs that walk the tiles.  With pairs: persistent pairs.
template <int CTAS, int BN>
__global__ void __launch_bounds__(THREADS, 1)
    gemm_fp8_tokens_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                           const __grid_constant__ CUtensorMap map_s, const __grid_constant__ CUtensorMap map_o, Params p) {
  using C = TokensCfg<CTAS, BN>;
  constexpr int S = C::STAGES, BUFS = C::BUFS, XLD = C::XLD, PRODS = C::PRODS, HALF = C::HALF;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // the same offset in every CTA of the cluster
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* exchange = reinterpret_cast<float*>(smem);  // over the idle ring (splits > 1)
  uint8_t* staging = smem + S * C::STAGE;  // 2 KB per epilogue warp: 64 bytes of 32 rows on their way out
  float* slots = reinterpret_cast<float*>(staging + C::STAGING);  // a stage's activation scales
  float* prods = slots + S * BM;  // [k-block % PRODS][weight block][token]: activation scale x weight scale
  uint32_t* amax = reinterpret_cast<uint32_t*>(prods + PRODS * C::BLOCKS * BM);  // [tile parity][half][token]
  uint64_t* bars = reinterpret_cast<uint64_t*>(amax + 2 * 2 * BM);
  const uint32_t bar0 = smem_u32(bars);
  // go (the even CTA's): the operands of the k-block in this stage have landed and the epilogue warps have
  // emptied its accumulator buffer.  One barrier for both: a poll costs the MMA warp 200 clocks or more
  // beside the epilogue's additions, even when its answer is yes.
  auto go = [&](int s) { return bar0 + 8u * s; };
  // empty: the stage's product has read its operands, the scale warps its scales.  sfull: these have landed.
  auto empty = [&](int s) { return bar0 + 8u * (S + s); };
  auto sfull = [&](int s) { return bar0 + 8u * (2 * S + s); };
  // tfull: the product of k-block % PRODS has landed, and the products of its scales are laid out.  pempty: the
  // epilogue warps have read a half of these.
  auto tfull = [&](int k) { return bar0 + 8u * (3 * S + k); };
  auto pempty = [&](int h) { return bar0 + 8u * (3 * S + PRODS + h); };
  const uint32_t final_bar = bar0 + 8u * (3 * S + PRODS + 2);
  const uint32_t amax_bar = final_bar + 8u;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + C::BARS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::BARS) + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CTAS == 2 || p.splits > 1 ? (int)cluster_rank() : 0;
  const int r = CTAS == 2 ? rank : 0, slice = CTAS == 2 ? 0 : rank;  // CTA of the pair; slice of K
  const int splits = CTAS == 2 ? 1 : p.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(go(s), 1 + CTAS * EPI_THREADS / 32);
      mbar_init(empty(s), 1 + C::BLOCKS);
      mbar_init(sfull(s), 1);
    }
    for (int k = 0; k < PRODS; ++k) mbar_init(tfull(k), 1 + C::BLOCKS);
    for (int h = 0; h < 2; ++h) mbar_init(pempty(h), EPI_THREADS / 32);
    mbar_init(final_bar, 1);
    mbar_init(amax_bar, EPI_THREADS / 32);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc<CTAS>(smem_u32(tmem_slot), BUFS * BN);
  fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) {  // both CTAs' barriers are initialised before any load, commit or arrival reaches them
    cluster_arrive();
    cluster_wait();
  }
  fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();

  const int tiles = p.tiles_m * p.tiles_n;
  const int t0 = blockIdx.x / (splits * CTAS), dt = gridDim.x / (splits * CTAS);
  const int kb0 = slice * p.kb_per_split;
  const int nkb = max(0, min(p.num_kb - kb0, p.kb_per_split));
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CONTROL_REGS));
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------------- producer
      prefetch_map(&map_x);
      prefetch_map(&map_w);
      prefetch_map(&map_s);
      if (t0 < tiles) {  // into L2 only, ahead of the previous kernel's end
        int tm, tn;
        tile_coords(p, t0, tm, tn);
        for (int i = 0; i < min(nkb, S); ++i) tma_prefetch_2d(&map_w, (kb0 + i) * BK, tn * BN + r * C::B_ROWS);
      }
      pdl_wait();
      uint32_t it = 0;
      bool ok = true;
      for (int t = t0; t < tiles && ok; t += dt) {
        int tm, tn;
        tile_coords(p, t, tm, tn);
        const int row0 = (tm * CTAS + r) * BM;
        for (int i = 0; i < nkb; ++i, ++it) {
          const int s = it % S, k = (kb0 + i) * BK;
          if (!mbar_wait(empty(s), ((it / S) & 1) ^ 1, abort_flag, p.error, 501)) {
            ok = false;
            break;
          }
          const uint32_t st = smem_u32(smem + s * C::STAGE);
          if constexpr (CTAS == 1) {
            mbar_arrive_expect_tx(go(s), C::STAGE);
            tma_load_2d(st, &map_x, go(s), k, row0);
            tma_load_2d(st + C::A_BYTES, &map_w, go(s), k, tn * BN);
          } else {
            if (r == 0) mbar_arrive_expect_tx(go(s), 2 * C::STAGE);
            const uint32_t gb = cluster_map(go(s), 0);
            tma_load_2d_pair(st, &map_x, gb, k, row0);
            tma_load_2d_pair(st + C::A_BYTES, &map_w, gb, k, tn * BN + r * C::B_ROWS);
          }
          mbar_arrive_expect_tx(sfull(s), BM * 4);
          tma_load_2d(smem_u32(slots + s * BM), &map_s, sfull(s), row0, kb0 + i);
        }
      }
      if (!ok) {
        const uint32_t n = it < (uint32_t)S ? it : (uint32_t)S;
        for (uint32_t j = it - n; j < it; ++j) {
          if (r == 0) mbar_drain(go(j % S), (j / S) & 1);
          mbar_drain(sfull(j % S), (j / S) & 1);
        }
      }
    } else if (warp == 1 && r == 0) {
      // ---------------------------------------------------------------- MMA issuer (a pair's even CTA)
      const uint32_t tbase = __shfl_sync(FULL_MASK, tmem, 0);
      const uint32_t total = (uint32_t)nkb * (t0 < tiles ? (tiles - t0 + dt - 1) / dt : 0);
      const uint64_t ad0 = sdesc(smem_u32(smem)), bd0 = sdesc(smem_u32(smem) + C::A_BYTES);
      int s = 0, phase = 0;
      pdl_wait();  // as in every role: the bounds of its waits do not count the previous kernel's time
      for (uint32_t it = 0; it < total; ++it) {
        if (!warp_wait(go(s), phase, abort_flag, p.error, 503)) break;
        fence_after();
        const uint32_t off = s * (C::STAGE >> 4);  // the descriptors count in 16 bytes
        const uint64_t ad = ad0 + off, bd = bd0 + off;
        const uint32_t d = tbase + (it % BUFS) * BN;
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            mma_f8<CTAS>(d, ad + 2 * k, bd + 2 * k, idesc_f8(CTAS * BM, BN), k > 0 ? 1u : 0u);
          commit<CTAS>(empty(s));
          commit<CTAS>(tfull(it % PRODS));
        }
        __syncwarp();
        if (++s == S) {
          s = 0;
          phase ^= 1;
        }
      }
      if (elect_one()) commit<CTAS>(final_bar);
      if (lane == 0) mbar_drain(final_bar, 0);
    } else if (warp >= 2 && warp - 2 < C::BLOCKS) {
      // ---------------------------------------------------------------- scales of weight block warp - 2
      // Each k-block's products of activation and weight scale, so that the epilogue has one barrier to
      // wait for and one number per column half to load.
      pdl_wait();
      uint32_t it = 0;
      int s = 0, phase = 0;
      bool ok = true;
      for (int t = t0; t < tiles && ok; t += dt) {
        int tm, tn;
        tile_coords(p, t, tm, tn);
        WeightScales ws(p.ws + (int64_t)min(C::BLOCKS * tn + warp - 2, p.nb - 1) * p.ldws + kb0, nkb, lane);
        for (int kb = 0; kb < nkb; ++kb, ++it) {
          const float w = ws.at(kb);
          // The half that holds k-block it - PRODS has been read: its products may be overwritten, and the
          // barrier that announced it takes the arrival below.
          ok = (it % HALF || warp_wait(pempty(it / HALF & 1), ((it / PRODS) & 1) ^ 1, abort_flag, p.error, 502)) &&
               warp_wait(sfull(s), phase, abort_flag, p.error, 506);
          if (!ok) break;
          float4 x = reinterpret_cast<const float4*>(slots + s * BM)[lane];
          x.x *= w; x.y *= w; x.z *= w; x.w *= w;
          reinterpret_cast<float4*>(prods + ((it % PRODS) * C::BLOCKS + warp - 2) * BM)[lane] = x;
          __syncwarp();
          if (lane == 0) {
            mbar_arrive_release(tfull(it % PRODS));
            mbar_arrive_release(empty(s));
          }
          if (++s == S) {
            s = 0;
            phase ^= 1;
          }
        }
      }
    }
    __syncwarp();
    if (splits > 1) {
      cluster_arrive();  // (the epilogue's phases, see there)
      cluster_wait();
      cluster_arrive();
      cluster_wait();
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(EPI_REGS));
    const int q4 = warp & 3, wg = (warp - 4) >> 2;
    const int lt = q4 * 32 + lane;  // this thread's token of the CTA's 128
    const uint32_t ta0 = tmem + ((uint32_t)(q4 * 32) << 16) + wg * 64;
    // (in the cluster's window for one CTA too: an arrival that returns no state is not waited for)
    const uint32_t go0 = cluster_map(go(0), CTAS == 2 ? 0 : rank);
    int gs = BUFS % S;  // stage of the k-block that takes over the buffer of k-block `it`, it + BUFS
    if (lane == 0)
      for (int b = 0; b < BUFS; ++b) mbar_arrive_cluster(go0 + 8u * b);  // every buffer is empty
    float acc[C::BLOCKS][64];
    uint32_t it = 0, tile_parity = 0;
    bool ok = true;
    pdl_wait();
    for (int t = t0; t < tiles; t += dt, tile_parity ^= 1) {
      int tm, tn;
      tile_coords(p, t, tm, tn);
      const int row = (tm * CTAS + r) * BM + lt;
#pragma unroll
      for (int h = 0; h < C::BLOCKS; ++h)
#pragma unroll
        for (int i = 0; i < 64; ++i) acc[h][i] = 0.f;
      if (nkb > 0) {
        // A k-block is 2 loads of 32 columns per block of W, through two register buffers.  The loads of
        // the next half are issued between the additions of this one, across k-blocks too; the buffer goes
        // back to the tensor core before its last half is added.
        uint32_t v[2][32];
        float s[C::BLOCKS];
        auto landed = [&](uint32_t it) {  // the product of k-block `it`; its scales
          if (!warp_wait(tfull(it % PRODS), (it / PRODS) & 1, abort_flag, p.error, 504)) return false;
          fence_after();
          return true;
        };
        auto scales = [&](uint32_t it) {
#pragma unroll
          for (int h = 0; h < C::BLOCKS; ++h) s[h] = prods[((it % PRODS) * C::BLOCKS + h) * BM + lt];
        };
        ok = landed(it);
        if (!ok) break;
        scales(it);
        tmem_ld(ta0 + (it % BUFS) * BN, v[0]);
        tmem_ld(ta0 + (it % BUFS) * BN + 32, v[1]);
        for (int kb = 0; kb < nkb; ++kb, ++it) {
          const bool more = kb + 1 < nkb;
          const uint32_t ta = ta0 + (it % BUFS) * BN, nx = ta0 + ((it + 1) % BUFS) * BN;
          const float last = s[C::BLOCKS - 1];
          ld_wait(v[0]);
          ld_wait(v[1]);
          if constexpr (C::BLOCKS == 2) {
            add32(acc[0], v[0], s[0]);
            tmem_ld(ta + 128, v[0]);
            add32(acc[0] + 32, v[1], s[0]);
            tmem_ld(ta + 160, v[1]);
            ld_wait(v[0]);
            ld_wait(v[1]);
          }
          fence_before();
          __syncwarp();
          // this buffer has been read: the tensor core may overwrite it, and the scale warps its products
          if (lane == 0) {
            mbar_arrive_cluster(go0 + 8u * gs);
            if (it % HALF == HALF - 1) mbar_arrive_release(pempty(it / HALF & 1));
          }
          if (++gs == S) gs = 0;
          float* a = acc[C::BLOCKS - 1];
          add32(a, v[0], last);
          if (more) {
            ok = landed(it + 1);
            if (!ok) break;
            tmem_ld(nx, v[0]);
            scales(it + 1);
          }
          add32(a + 32, v[1], last);
          if (more) tmem_ld(nx + 32, v[1]);
        }
        if (!ok) break;
      }
      if (splits > 1) break;  // one tile per cluster; finished below
      // Each warp stores pieces of 32 rows x 64 bytes through shared memory by TMA, which writes whole
      // sectors and drops what lies outside (stores of each thread's own row took 9000 clocks per tile,
      // a quarter of it, as long as nothing overlaps them).
      const int row0 = (tm * CTAS + r) * BM + q4 * 32;
      uint8_t* mine = staging + (warp - 4) * 2048;
      auto piece = [&](const uint4* w4, int col) {
        if (lane == 0 && p.tma_out) bulk_wait_read();  // the piece before has left
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 4; ++c)  // 64-byte swizzle: no bank conflicts
          *reinterpret_cast<uint4*>(mine + lane * 64 + (c ^ ((lane >> 1) & 3)) * 16) = w4[c];
        if (p.tma_out) {
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&map_o, smem_u32(mine), col, row0);
            bulk_commit();
          }
        } else {  // bf16 rows that TMA cannot address: a lane per column, one row at a time
          __syncwarp();
          if (col + lane < p.N) {
            __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + (int64_t)row0 * p.ldo + col + lane;
            const int n = min(32, p.T - row0);
            for (int i = 0; i < n; ++i, dst += p.ldo)
              *dst = *reinterpret_cast<const __nv_bfloat16*>(mine + i * 64 + ((lane >> 3) ^ ((i >> 1) & 3)) * 16 +
                                                             (lane & 7) * 2);
          }
        }
      };
      if (BN == 128 || !p.act) {
#pragma unroll
        for (int h = 0; h < C::BLOCKS; ++h)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int col = tn * BN + h * 128 + wg * 64 + c * 32;
            const float* a = acc[h] + c * 32;
            const uint4 w4[4] = {f32_to_bf16x8(a), f32_to_bf16x8(a + 8), f32_to_bf16x8(a + 16), f32_to_bf16x8(a + 24)};
            if (row0 < p.T && col < p.N) piece(w4, col);
          }
      } else {
        // SiLU-and-mul; the values stay fp32 up to the 8-bit rounding
        const int f = tn * 128 + wg * 64;
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 64; ++i) acc[0][i] = silu_f(acc[0][i]) * acc[C::BLOCKS - 1][i];
        if (f + 64 > p.features) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (f + i >= p.features) acc[0][i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 64; ++i) m = max(m, __float_as_uint(acc[0][i]) & 0x7fffffffu);
        // the other half of the group of 128 belongs to the other warpgroup's thread of this token;
        // two buffers: a warp may be one tile ahead of the reader of the one before
        uint32_t* am = amax + tile_parity * 2 * BM + lt;
        am[wg * BM] = m;
        __syncwarp();
        if (lane == 0) mbar_arrive_release(amax_bar);
        ok = warp_wait(amax_bar, tile_parity, abort_flag, p.error, 505);
        if (!ok) break;
        const Fp8Scale sc = fp8_scale(max(m, am[(wg ^ 1) * BM]));
        uint4 w4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint2 a = f32x8_to_e4m3(acc[0] + 16 * i, sc.inv), b = f32x8_to_e4m3(acc[0] + 16 * i + 8, sc.inv);
          w4[i] = make_uint4(a.x, a.y, b.x, b.y);
        }
        if (row0 < p.T && f < p.features) piece(w4, f);
        if (wg == 0 && row < p.T) p.os[(int64_t)tn * p.ldos + row] = sc.scale;
      }
    }
    if (lane == 0) bulk_wait();  // every piece has been written
    __syncwarp();
    if (splits > 1) {
      // Every CTA lays its sums out in its own shared memory, over its idle ring (the last MMA has
      // completed), [token][feature]; after the cluster's barrier each slice finishes its share.
      int tm, tn;
      tile_coords(p, t0, tm, tn);
      float* dst = exchange + lt * XLD + wg * 64;
#pragma unroll
      for (int h = 0; h < C::BLOCKS; ++h)
#pragma unroll
        for (int i = 0; i < 64; i += 4)
          *reinterpret_cast<float4*>(dst + h * 128 + i) =
              make_float4(acc[h][i], acc[h][i + 1], acc[h][i + 2], acc[h][i + 3]);
      cluster_arrive();
      cluster_wait();  // every slice's sums are laid out
      if (!*abort_flag) {
        if (splits == 2) finish_rows<BN, 2>(p, exchange, slice, tm * BM, tn, warp - 4, lane);
        else finish_rows<BN, 4>(p, exchange, slice, tm * BM, tn, warp - 4, lane);
      }
      cluster_arrive();
      cluster_wait();  // nobody reads this CTA's shared memory any more
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) {  // the pair's MMAs, loads, commits and arrivals are done before TMEM is freed
    if (r == 1 && threadIdx.x == 32) mbar_drain(final_bar, 0);  // the last commit has reached this CTA too
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    fence_after();
    tmem_dealloc<CTAS>(tmem, BUFS * BN);
  }
}

template <int NP, int MW>
__global__ void __launch_bounds__(WeightsCfg<NP, MW>::THREADS, 2)
    gemm_fp8_weights_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                            const __grid_constant__ CUtensorMap map_s, Params p) {
  using C = WeightsCfg<NP, MW>;
  constexpr int S = C::STAGES, NB = C::ACC_BUFS, SL = C::SLOTS;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // the same offset in every CTA of the cluster
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* exchange = reinterpret_cast<float*>(smem + (C::OVER_RING ? 0 : S * C::STAGE));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::SMEM - 1024 - 8 * C::BARS - 16);
  uint8_t* slots = reinterpret_cast<uint8_t*>(bars) - SL * C::SLOT;
  const uint32_t bar0 = smem_u32(bars);
  // go: the operands of the k-block in this stage have landed and the epilogue warps have emptied its
  // accumulator buffer (one poll for both, see gemm_fp8_tokens_kernel)
  auto go = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (S + s); };
  auto tfull = [&](int b) { return bar0 + 8u * (2 * S + b); };
  auto sfull = [&](int l) { return bar0 + 8u * (2 * S + NB + l); };
  auto sempty = [&](int l) { return bar0 + 8u * (2 * S + NB + SL + l); };  // a slot's scales have been read
  const uint32_t final_bar = bar0 + 8u * (2 * S + NB + 2 * SL);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + C::BARS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::BARS) + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = p.splits > 1 ? (int)cluster_rank() : 0;
  const int tile = blockIdx.x / p.splits;
  const int kb0 = slice * p.kb_per_split;
  const int nkb = max(0, min(p.num_kb - kb0, p.kb_per_split));

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(go(s), 1 + C::EPI_WARPS);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < NB; ++b) mbar_init(tfull(b), 1);
    for (int l = 0; l < SL; ++l) {
      mbar_init(sfull(l), 1);
      mbar_init(sempty(l), C::EPI_WARPS);
    }
    mbar_init(final_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc<1>(smem_u32(tmem_slot), C::TMEM_COLS);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  // this CTA's exchange area may be written: now, or once its ring is idle (waited on below)
  if (!C::OVER_RING && p.splits > 1) cluster_arrive();
  pdl_trigger();

  if (warp == 0 && lane == 0) {
    // ------------------------------------------------------------------ producer
    prefetch_map(&map_w);
    prefetch_map(&map_x);
    prefetch_map(&map_s);
    // Into L2 only, ahead of the previous kernel's end: whoever writes the weights writes there too
    for (int i = 0; i < min(nkb, S); ++i) tma_prefetch_2d(&map_w, (kb0 + i) * BK, tile * C::ROWS);
    pdl_wait();
    bool ok = true;
    int i = 0;
    for (; i < nkb; ++i) {
      const int s = i % S, l = i % SL;
      if (!mbar_wait(empty(s), ((i / S) & 1) ^ 1, abort_flag, p.error, 511) ||
          !mbar_wait(sempty(l), ((i / SL) & 1) ^ 1, abort_flag, p.error, 512)) {
        ok = false;
        break;
      }
      const uint32_t st = smem_u32(smem + s * C::STAGE);
      mbar_arrive_expect_tx(go(s), C::STAGE);
      tma_load_2d(st, &map_w, go(s), (kb0 + i) * BK, tile * C::ROWS);
      tma_load_2d(st + C::W_BYTES, &map_x, go(s), (kb0 + i) * BK, 0);
      mbar_arrive_expect_tx(sfull(l), NP * 4);
      tma_load_2d(smem_u32(slots + l * C::SLOT), &map_s, sfull(l), 0, kb0 + i);
    }
    if (!ok) {
      for (int j = max(0, i - S); j < i; ++j) {
        mbar_drain(go(j % S), (j / S) & 1);
        mbar_drain(sfull(j % SL), (j / SL) & 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    const uint32_t tbase = __shfl_sync(FULL_MASK, tmem, 0);
    pdl_wait();  // as in every role: the bounds of its waits do not count the previous kernel's time
    for (int i = 0; i < nkb; ++i) {
      const int s = i % S, b = i % NB;
      if (!warp_wait(go(s), (i / S) & 1, abort_flag, p.error, 513)) break;
      fence_after();
      const uint32_t st = smem_u32(smem + s * C::STAGE);
      const uint64_t wd = sdesc(st), xd = sdesc(st + C::W_BYTES);
      if (elect_one()) {
#pragma unroll
        for (int m = 0; m < MW; ++m)
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            mma_f8<1>(tbase + (b * MW + m) * NP, wd + m * (128 * BK >> 4) + 2 * k, xd + 2 * k, idesc_f8(128, NP),
                      k > 0 ? 1u : 0u);
        commit<1>(empty(s));
        commit<1>(tfull(b));
      }
      __syncwarp();
    }
    if (elect_one()) commit<1>(final_bar);
    if (lane == 0) mbar_drain(final_bar, 0);
    __syncwarp();
  } else if (warp >= 2) {
    // ------------------------------------------------------------------ epilogue
    // lane quarter, 128-row block of the tile, share of the tokens
    const int q4 = warp & 3, m = ((warp - 2) >> 2) % MW, cs = ((warp - 2) >> 2) / MW;
    const uint32_t go0 = cluster_map(go(0), slice);
    if (lane == 0)
      for (int b = 0; b < NB; ++b) mbar_arrive_cluster(go0 + 8u * b);  // every buffer is empty
    float acc[C::NC];
#pragma unroll
    for (int i = 0; i < C::NC; ++i) acc[i] = 0.f;
    pdl_wait();
    WeightScales ws(p.ws + (int64_t)min(tile * MW + m, p.nb - 1) * p.ldws + kb0, nkb, lane);
    bool ok = true;
    for (int i = 0; i < nkb; ++i) {
      const float wsc = ws.at(i);
      const int b = i % NB, l = i % SL;
      ok = warp_wait(sfull(l), (i / SL) & 1, abort_flag, p.error, 514) && warp_wait(tfull(b), (i / NB) & 1, abort_flag, p.error, 515);
      if (!ok) break;
      fence_after();
      const uint32_t ta = tmem + ((uint32_t)(q4 * 32) << 16) + (b * MW + m) * NP + cs * C::NC;
      const float4* xs = reinterpret_cast<const float4*>(slots + l * C::SLOT) + cs * (C::NC / 4);
#pragma unroll
      for (int c = 0; c < C::NC / C::CHUNK; ++c) {
        uint32_t v[C::CHUNK];
        tmem_ld(ta + c * C::CHUNK, v);
        ld_wait(v);
        if (c + 1 == C::NC / C::CHUNK) {  // this buffer has been read: the tensor core may overwrite it
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(go0 + 8u * ((i + NB) % S));
        }
#pragma unroll
        for (int j = 0; j < C::CHUNK / 4; ++j) {
          const float4 sx = xs[c * (C::CHUNK / 4) + j];  // 4 tokens' scales, the same for every lane
          float* a = acc + c * C::CHUNK + 4 * j;
          a[0] = fmaf(__uint_as_float(v[4 * j]), sx.x * wsc, a[0]);
          a[1] = fmaf(__uint_as_float(v[4 * j + 1]), sx.y * wsc, a[1]);
          a[2] = fmaf(__uint_as_float(v[4 * j + 2]), sx.z * wsc, a[2]);
          a[3] = fmaf(__uint_as_float(v[4 * j + 3]), sx.w * wsc, a[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_release(sempty(l));
    }
    // sums of token c to CTA c mod splits: [slice][c / splits][feature]
    if (p.splits > 1) {
      if (C::OVER_RING) cluster_arrive();  // the last MMA has completed: nothing reads the ring any more
      cluster_wait();
    }
    const int f = m * 128 + q4 * 32 + lane;
    const int per = (NP + p.splits - 1) / p.splits;
    int owner = (cs * C::NC) % p.splits, tl = (cs * C::NC) / p.splits;
#pragma unroll
    for (int c = 0; c < C::NC; ++c)
      if (cs * C::NC + c < p.T) {
        float* dst = exchange + (slice * per + tl) * C::ROWS + f;
        if (p.splits > 1)
          st_cluster_f32(cluster_map(smem_u32(dst), owner), acc[c]);
        else
          *dst = acc[c];
        if (++owner == p.splits) {
          owner = 0;
          ++tl;
        }
      }
  }
  __syncwarp();
  fence_before();
  if (p.splits > 1) {
    if (warp < 2) {
      if (C::OVER_RING) cluster_arrive();
      cluster_wait();
    }
    cluster_arrive();
    cluster_wait();  // every slice's sums have arrived
  } else {
    __syncthreads();
  }
  if (warp >= 2 && !*abort_flag) {
    const int per = (NP + p.splits - 1) / p.splits;
    const int mine = (p.T - slice + p.splits - 1) / p.splits;  // tokens slice, slice + splits, ...
    for (int tl = warp - 2; tl < mine; tl += C::EPI_WARPS) {
      const int t = slice + tl * p.splits;
      float o[MW][4] = {};
      for (int r = 0; r < p.splits; ++r) {
        const float4* row = reinterpret_cast<const float4*>(exchange + (r * per + tl) * C::ROWS);
#pragma unroll
        for (int m = 0; m < MW; ++m) {
          const float4 v = row[m * 32 + lane];
          o[m][0] += v.x; o[m][1] += v.y; o[m][2] += v.z; o[m][3] += v.w;
        }
      }
      if constexpr (MW == 1) finish_bf16x4(p, t, tile * 128 + lane * 4, o[0]);
      else finish_silu4(p, t, tile, lane, o[0], o[1]);
    }
  }
  if (warp == 1) {
    fence_after();
    tmem_dealloc<1>(tmem, C::TMEM_COLS);
  }
}

// The error word: pinned host memory that every GPU of the process can write, so that reading it after a
// synchronisation costs no copy and covers all of them.  Null where it cannot be had.
std::atomic<int*> g_error_word{nullptr};
int* error_word() {
  int* w = g_error_word.load(std::memory_order_acquire);
  if (w) return w;
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  if ((w = g_error_word.load(std::memory_order_acquire))) return w;
  // the first call may lie inside a stream capture, which this allocation does not concern
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
  void* m = nullptr;
  const cudaError_t e = cudaHostAlloc(&m, sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  w = static_cast<int*>(m);
  *w = 0;
  g_error_word.store(w, std::memory_order_release);
  return w;
}

// A wait that nothing ends, given up after budget_ns.
__global__ void wait_check_kernel(int* word, uint64_t budget_ns) {
  __shared__ uint64_t bar;
  __shared__ int abort_flag;
  mbar_init(smem_u32(&bar), 1);
  abort_flag = 0;
  mbar_wait(smem_u32(&bar), 0, &abort_flag, word, 599, budget_ns);
}

PFN_cuTensorMapEncodeTiled_v12000 get_encode() {
  static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> cached{nullptr};
  auto fn = cached.load(std::memory_order_acquire);
  if (!fn) {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess) {
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
      cached.store(fn, std::memory_order_release);
    }
  }
  return fn;
}

// e4m3 [rows, k] with row stride ld; boxes of 128 channels x box_rows, 128-byte swizzle; elements
// outside are read as zero.
bool make_map(CUtensorMap* m, const void* base, int rows, int k, int64_t ld, int box_rows) {
  auto enc = get_encode();
  if (!enc) return false;
  cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// fp32 scales [blocks][tokens] with row stride ld; boxes of one block's scales of `box` tokens.
bool make_scale_map(CUtensorMap* m, const float* base, int blocks, int tokens, int64_t ld, int box) {
  auto enc = get_encode();
  if (!enc) return false;
  cuuint64_t dims[2] = {(cuuint64_t)tokens, (cuuint64_t)blocks};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 4};
  cuuint32_t boxd[2] = {(cuuint32_t)box, 1};
  cuuint32_t estr[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<float*>(base), dims, strides, boxd, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaLaunchConfig_t cluster_config(int grid, int threads, int smem, int cluster, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cfg;
}

// Shared-memory opt-in, and the check that the kernel is launched with the registers that its
// warps redistribute (fewer would leave the epilogue waiting for them).
template <int CTAS, int BN>
cudaError_t tokens_opt_in() {
  static std::atomic<uint64_t> done{0};
  return once_per_device(done, []() -> cudaError_t {
    cudaFuncAttributes a;
    cudaError_t e = cudaFuncGetAttributes(&a, gemm_fp8_tokens_kernel<CTAS, BN>);
    if (e != cudaSuccess) return e;
    if (a.numRegs < LAUNCH_REGS) return cudaErrorInvalidDeviceFunction;
    return cudaFuncSetAttribute(gemm_fp8_tokens_kernel<CTAS, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                TokensCfg<CTAS, BN>::SMEM);
  });
}

template <int NP, int MW>
cudaError_t weights_opt_in() {
  static std::atomic<uint64_t> done{0};
  return smem_opt_in(done, gemm_fp8_weights_kernel<NP, MW>, WeightsCfg<NP, MW>::SMEM);
}

// Clusters of 1 .. 8 CTAs that a GPU of num_sms SMs holds at once, with one CTA per SM and with two: a cluster
// lies within one of the GPU's processing clusters, so fewer fit than num_sms / cluster.  These are what
// cudaOccupancyMaxActiveClusters answers on a B200 of 148 SMs, scaled to other sizes, but for 3 and 5 CTAs of two
// per SM: 93 and 56 are its answers, and of launches behind one another 92 and 53 ran at once (1 x 4096 x 11904,
// 93 tiles, in 3 slices 14.9 us, in 2 13.0; 7040, 55 tiles, in 5 slices 10.2, in 4 8.6; past the others' figures as
// well: 9216, 72 tiles, in 4 slices 14.2, in 3 9.7).  They are not asked of
// the GPU at hand, on which parts of one model can differ: a plan fixes the order of the fp32 sums, and that
// is the same wherever a size runs.  A GPU that holds fewer runs the rest in a second round: slower, with the
// same result.
constexpr int CLUSTERS_OF_SMS[9] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
constexpr int CLUSTERS_OF_HALF_SMS[9] = {0, 296, 148, 92, 71, 53, 45, 37, 33};
int clusters_of_sms(int cluster, int num_sms) { return std::max(1, CLUSTERS_OF_SMS[cluster] * num_sms / 148); }
int clusters_of_half_sms(int cluster, int num_sms) { return std::max(1, CLUSTERS_OF_HALF_SMS[cluster] * num_sms / 148); }

// The output of the token-major kernel: bf16 [T, N] or e4m3 [T, features], pieces of 64 bytes x 32 rows.
bool make_out_map(CUtensorMap* m, const Fp8Gemm& g) {
  auto enc = get_encode();
  if (!enc) return false;
  const int bytes = g.act ? 1 : 2;
  cuuint64_t dims[2] = {(cuuint64_t)(g.act ? g.features : g.N), (cuuint64_t)g.T};
  cuuint64_t strides[1] = {(cuuint64_t)g.ldo * bytes};
  cuuint32_t box[2] = {(cuuint32_t)(64 / bytes), 32};
  cuuint32_t estr[2] = {1, 1};
  return enc(m, g.act ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, g.out, dims, strides, box,
             estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NP, int MW>
cudaError_t run_weights(const Fp8Gemm& g, Params p, int splits, cudaStream_t stream) {
  using C = WeightsCfg<NP, MW>;
  if (splits < 1 || splits > 8 || g.T > NP) return cudaErrorInvalidValue;
  CUtensorMap mx, mw, ms;
  if (!make_map(&mx, g.xq, g.T, g.K, g.ldx, NP) || !make_map(&mw, g.wq, g.N, g.K, g.ldw, C::ROWS) ||
      !make_scale_map(&ms, g.xs, p.num_kb, g.T, g.ldxs, NP))
    return cudaErrorInvalidValue;
  p.splits = splits;
  p.kb_per_split = (p.num_kb + splits - 1) / splits;
  cudaError_t e = weights_opt_in<NP, MW>();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = cluster_config((g.N + C::ROWS - 1) / C::ROWS * splits, C::THREADS, C::SMEM, splits, attr);
  cfg.stream = stream;
  return cudaLaunchKernelEx(&cfg, gemm_fp8_weights_kernel<NP, MW>, mx, mw, ms, p);
}

template <int CTAS, int BN>
cudaError_t run_tokens(const Fp8Gemm& g, Params p, int splits, int num_sms, cudaStream_t stream) {
  using C = TokensCfg<CTAS, BN>;
  if ((splits != 1 && (CTAS == 2 || (splits != 2 && splits != 4))) || (g.act && BN != 256)) return cudaErrorInvalidValue;
  CUtensorMap mx, mw, ms;
  if (!make_map(&mx, g.xq, g.T, g.K, g.ldx, BM) || !make_map(&mw, g.wq, g.N, g.K, g.ldw, C::B_ROWS) ||
      !make_scale_map(&ms, g.xs, p.num_kb, g.T, g.ldxs, BM))
    return cudaErrorInvalidValue;
  p.tiles_m = (g.T + CTAS * BM - 1) / (CTAS * BM);
  p.tiles_n = (g.N + BN - 1) / BN;
  p.group = 16;
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  if (tiles > 0x7fffffff / 16) return cudaErrorInvalidValue;
  p.splits = splits;
  p.kb_per_split = (p.num_kb + splits - 1) / splits;
  cudaError_t e = tokens_opt_in<CTAS, BN>();
  if (e != cudaSuccess) return e;
  CUtensorMap mo = mx;  // not used without p.tma_out
  p.tma_out = g.act || p.vec;
  if (p.tma_out && !make_out_map(&mo, g)) return cudaErrorInvalidValue;
  const int64_t most = splits > 1 ? tiles : std::min<int64_t>(tiles, clusters_of_sms(CTAS, num_sms));
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = cluster_config((int)most * splits * CTAS, THREADS, C::SMEM, splits * CTAS, attr);
  cfg.stream = stream;
  return cudaLaunchKernelEx(&cfg, gemm_fp8_tokens_kernel<CTAS, BN>, mx, mw, ms, mo, p);
}

}  // namespace

Fp8Plan fp8_plan(int T, int N, int K, int act, int num_sms) {
  Fp8Plan pl;
  const int num_kb = (K + BK - 1) / BK;
  if (T <= (act ? 32 : 64)) {
    // Few tokens: the weights are streamed once, by as many CTAs as the GPU holds.
    pl.np = T <= 16 ? 16 : T <= 32 ? 32 : 64;
    const int rows = act ? 256 : 128, tiles = (N + rows - 1) / rows;
    for (int s = 2; s <= 8; ++s)
      if (num_kb >= s && tiles <= clusters_of_half_sms(s, num_sms)) pl.splits = s;
    // .. unless there is little to stream per tile: 61 x 7216 x 624 takes 8.3 us so, 5.3 us below
    if (pl.np < 64 || pl.splits >= 4 || num_kb > 8) {
      // as many slices as the length of the longest one leaves any work: 9 blocks in 8 slices are 5 of 2
      const int per = (num_kb + pl.splits - 1) / pl.splits;
      pl.splits = (num_kb + per - 1) / per;
      return pl;
    }
    pl = Fp8Plan{};
  }
  // Fewest nanoseconds by a model of one CTA's time: its k-blocks at 460 ns for a tile of 256 features and 310
  // ns for one of 128, and the exchange of the slices' sums, 5.0 and 6.2 us for 2 and 4 slices of 256
  // features, 2.4 and 3.2 us of 128.  (The slope over K is 440 and 296 ns with 32 CTAs at work, 430 in pairs, which
  // load 32 KB per k-block and CTA instead of 48: it is the CTA's own chain, not the delivery of operands.  With all
  // SMs at work it is 440-620 and 290-380, the more the longer K: power and memory.  What a call takes besides, 3.5 to
  // 4.6 us, is the same for all.)  Examples of both sides, T x N x K: 256 x 4096 x 4096, 128 features in 2
  // slices 11.3 us, 256 features in 4 slices 13.2 us, neither split 13.1 and 18.7 us; 512 x 6144 x
  // 4096, 128 features 24.2 us, 256 features 19.3 us.  Where 256 features in one slice win, pairs of
  // CTAs run them if that takes no more rounds of the GPU, and K fills 8 blocks or there are three rounds
  // of it: 4699 x 6416 x 9456, pairs 288 us, single CTAs 338 us; 8192 x 8192 x 640 61.7 and 62.5 us; equal for
  // one round of 512 x 6144 x 4096.  The other side: 300 x 12288 x 1024, pairs (two rounds) 13.7 us, single
  // CTAs (one) 8.8 us; two rounds of 1024 x 8192 x 384 9.9 and 9.3 us.
  int64_t best = -1;
  for (int bn = 256; bn >= (act ? 256 : 128); bn /= 2) {
    const int64_t tiles = (int64_t)((T + BM - 1) / BM) * ((N + bn - 1) / bn);
    for (int s = 1; s <= 4; s *= 2) {
      if (s > 1 && (num_kb / s < 4 || tiles > clusters_of_sms(s, num_sms))) continue;
      const int64_t rounds = s > 1 ? 1 : (tiles + num_sms - 1) / num_sms, kbs = (num_kb + s - 1) / s * rounds;
      const int64_t exchange = s == 1 ? 0 : bn == 256 ? 3800 + 600 * s : 1600 + 400 * s;
      const int64_t ns = kbs * (bn == 256 ? 460 : 310) + exchange;
      if (best >= 0 && ns >= best) continue;
      best = ns;
      const int64_t pair_tiles = (int64_t)((T + 2 * BM - 1) / (2 * BM)) * ((N + bn - 1) / bn);
      const int pairs = clusters_of_sms(2, num_sms);
      const bool paired = s == 1 && T > BM && (pair_tiles + pairs - 1) / pairs <= rounds && (num_kb >= 8 || rounds >= 3);
      pl.np = bn == 128 ? -3 : paired ? -2 : -1;
      pl.splits = s;
    }
  }
  return pl;
}

cudaError_t gemm_fp8(const Fp8Gemm& g, const Fp8Plan& pl, int num_sms, cudaStream_t stream) {
  if (g.T == 0 || g.N == 0) return cudaSuccess;
  Params p{};
  p.error = error_word();
  if (!p.error) return cudaErrorMemoryAllocation;
  p.ws = g.ws;
  p.ldws = g.ldws;
  p.T = g.T;
  p.N = g.N;
  p.num_kb = (g.K + BK - 1) / BK;
  p.nb = (g.N + FP8_GROUP - 1) / FP8_GROUP;
  p.act = g.act;
  p.features = g.features;
  p.out = g.out;
  p.ldo = g.ldo;
  p.os = g.os;
  p.ldos = g.ldos;
  p.vec = g.ldo % 8 == 0 && (reinterpret_cast<uintptr_t>(g.out) & 15) == 0;
  switch (pl.np) {
    case -1: return run_tokens<1, 256>(g, p, pl.splits, num_sms, stream);
    case -2: return run_tokens<2, 256>(g, p, pl.splits, num_sms, stream);
    case -3: return run_tokens<1, 128>(g, p, pl.splits, num_sms, stream);
    case 16: return g.act ? run_weights<16, 2>(g, p, pl.splits, stream) : run_weights<16, 1>(g, p, pl.splits, stream);
    case 32: return g.act ? run_weights<32, 2>(g, p, pl.splits, stream) : run_weights<32, 1>(g, p, pl.splits, stream);
    case 64: return g.act ? cudaErrorInvalidValue : run_weights<64, 1>(g, p, pl.splits, stream);
    default: return cudaErrorInvalidValue;
  }
}

int gemm_fp8_error_code(int reset) {
  int* w = g_error_word.load(std::memory_order_acquire);
  if (!w) return 0;  // no product was ever launched
  return reset ? __atomic_exchange_n(w, 0, __ATOMIC_ACQ_REL) : __atomic_load_n(w, __ATOMIC_ACQUIRE);
}

cudaError_t gemm_fp8_wait_check(uint64_t budget_ns, cudaStream_t stream) {
  int* w = error_word();
  if (!w) return cudaErrorMemoryAllocation;
  wait_check_kernel<<<1, 1, 0, stream>>>(w, std::min<uint64_t>(budget_ns, WAIT_BUDGET_NS));
  return cudaGetLastError();
}

}  // namespace nvb
