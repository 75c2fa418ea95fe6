// Attention of a tree of drafted tokens over the paged cache.
//
// Row r = (node, query head) of a KV head sees the positions before the tree and the nodes of its mask:
//   o_r = sum_j a_rj v_j,  a = softmax_j(scale q_r . k_j)   over j < base or (j - base) in mask(node).
// All rows of a KV head (nodes x nq / nkv) share its keys.  One CTA takes up to 256 rows of a (sequence, KV head) and
// tiles of 128 keys:
//   S = Q K^T    tcgen05, Q and K in shared memory, S [128 rows x 128 keys] fp32 in TMEM
//   P = exp2(S - m), rounded to bf16, written over S: one row per thread, no shuffles
//   O += P V     tcgen05, P in TMEM, V in shared memory, O [128 x 128] fp32 in TMEM
// Two groups of four warps, each with an S, an O, a running maximum and a running sum of its own, work on alternate
// steps, so that one's products run beside the other's exponentials: with up to 128 rows they take every other key
// tile and are joined at the end, with more they take 128 rows each of every tile.
// An e4m3 cache is converted once per value by four more warps, to bf16 (exact); K's scale multiplies the scores, V's
// the weights before they are rounded.
//
// Up to 64 rows (nodes x query heads of a KV head) the roles of the product's sides are exchanged: tree_attn_few_kernel.
//
// Balance: the tiles of all (sequence, 256 rows, KV head) are laid end to end and cut into stretches of equal work, one
// per CTA, whatever the sequences' lengths.  One that is cut leaves partial sums (at most two per CTA), which a second
// kernel joins in the order of the keys: no atomics, the same bits on every run.
//
// Masks: only tiles that reach into the tree look at them.  What a row does not see takes no part in it: its score is
// -inf, and a value that is infinite or NaN (0 x inf), of itself or by its scale, is taken out of such a tile in shared
// memory and added at the end to the rows that see it.
//
// What bounds it.  Up to 64 rows the bytes of K and V should: 64 trees of 16 nodes, 32 query and 8 KV heads, 2048
// tokens, bf16: 127 us, 4.35 TB/s (a tile's round of product, maximum, weights and store is longer than its bytes take);
// 128 trees of 8 on e4m3: 295 us, 1.9 TB/s (a round takes twice as long beside the eight warps that convert).  Beyond, the
// exponentials: 24 trees of up to 64 nodes, 64 and 8 heads, up to 8191 tokens: 252-261 us, 530-550 TFLOP/s; two groups'
// weights of a tile take 3800 clocks in turn, the products 2048.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "common.cuh"
#include "device_error.h"
#include "tcgen05.cuh"
#include "tree.h"

#include <algorithm>
#include <type_traits>

namespace nvb {
namespace {

constexpr int AD = 128;                 // head dim
constexpr int KT = 128;                 // keys per tile
constexpr int HALF = KT * 128;          // bytes of 64 dims of a 128-row tile
constexpr int TILE = 2 * HALF;          // a 128 x 128 tile of 16-bit values
constexpr int RAW_TILE = KT * AD;       // of 8-bit values
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RAISE = 8.f;            // the running maximum follows once a row's grows by 2^8
// First warp of each role; 0-7: softmax (the polling MMA warps share the schedulers of warps 2, 3, 6 and 7, whose rows are
// the last); 9 has none: registers are moved between whole warpgroups.
constexpr int W_TMA = 8, W_MMA = 10, W_CONV = 12;
constexpr int BAD_WORDS = TREE_MAX_NODES / 32 + 1;  // the nodes, and keys ahead of them (bad_from)
constexpr float NOTHING = -3e38f;       // below any score

constexpr int ERROR_BASE = 600;         // of the codes in the process's error word

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(d) : "f"(lo), "f"(hi));
  return d;
}
// Set in bits 15 and 31 where a bf16 half of x is infinite or NaN (its exponent is all ones).
__device__ __forceinline__ uint32_t odd_halves(uint32_t x) { return ((x & 0x7fff7fffu) + 0x00800080u) & 0x80008000u; }

struct Args {
  TreeAttn t;
  int G, chunks, bs_shift;
  int rows_cap;     // rows of a CTA: 16 to 256
  int slots;        // tiles of the 16-bit ring (K and V in turn)
  int raw_slots;    // and of the e4m3 ring
  int box_rows;     // rows per TMA box: min(128, block size)
  int oob_row;      // a row behind the pool: reads as zeros
  int q16;          // q's rows are 16-byte aligned
  float scale_log2;
  int* error;       // the process's error word
};

// ------------------------------------------------------------------- the list of tiles
// Sequence b with nodes has max(1, ceil(k_len / 128)) tiles for each KV head and stretch of rows (an empty context
// still writes its zeros).  The list runs over sequences, stretches of rows, KV heads and tiles.
__device__ __forceinline__ int seq_begin(const TreeAttn& t, int b) { return min(max(t.cu_q[b], 0), t.T); }
__device__ __forceinline__ int seq_nodes(const TreeAttn& t, int b) { return min(t.cu_q[b + 1], t.T) - seq_begin(t, b); }
__device__ __forceinline__ int seq_rows(const Args& a, int b) { return min(seq_nodes(a.t, b), a.t.max_nodes) * a.G; }
__device__ __forceinline__ int seq_tiles(const TreeAttn& t, int b) { return max(1, (t.ctx_lens[b] + KT - 1) / KT); }
// Its work, in units of some 1000 clocks: a tile that meets more than 128 rows takes ALL_ROWS (the exponentials), one
// that meets fewer takes FEW_ROWS (its bytes, or up to 64 rows a tile's round), and an item (a sequence, a stretch of
// rows, a KV head) ITEM_WORK whatever its tiles (queries, first maximum, outputs).  With stretches of equal products the
// slowest CTA took 470000 clocks where most took 335000, with ITEM_WORK 0 more (24 x up to 64 nodes, 64 heads, 600 to
// 8000 tokens).
constexpr int ALL_ROWS = 4, FEW_ROWS = 3, ITEM_WORK = 12;
struct Work {
  int tiles;
  int64_t twice;  // items of more than 128 rows, which come first
  int64_t per2, per1;  // work of an item
  __device__ __forceinline__ Work(const Args& a, int b) {
    const int rows = seq_rows(a, b);
    tiles = seq_tiles(a.t, b);
    twice = a.rows_cap > 128 ? (int64_t)a.t.nkv * (rows / 256 + (rows % 256 > 128 ? 1 : 0)) : 0;
    per2 = ITEM_WORK + (int64_t)ALL_ROWS * tiles;
    per1 = ITEM_WORK + (int64_t)FEW_ROWS * tiles;
  }
  // the tile (of sequence b's part of the list) in which its work unit `w` lies; the first one takes the item's own
  __device__ __forceinline__ int64_t tile(int64_t w) const {
    const bool two = w < twice * per2;
    if (!two) w -= twice * per2;
    const int64_t item = w / (two ? per2 : per1), at = w % (two ? per2 : per1) - ITEM_WORK;
    return (item + (two ? 0 : twice)) * tiles + (at <= 0 ? 0 : at / (two ? ALL_ROWS : FEW_ROWS));
  }
  // the units ahead of the item that begins with tile i
  __device__ __forceinline__ int64_t ahead(int64_t i) const {
    const int64_t item = i / tiles;
    return item <= twice ? item * per2 : twice * per2 + (item - twice) * per1;
  }
};
__device__ __forceinline__ int64_t seq_work(const Args& a, int b) {
  const int rows = seq_rows(a, b);
  if (rows <= 0) return 0;
  const Work w(a, b);
  return w.ahead((int64_t)a.t.nkv * ((rows + a.rows_cap - 1) / a.rows_cap) * w.tiles);
}

// Stretch c of the list: from tile lo_tile of sequence lo_seq to ahead of tile hi_tile of hi_seq.  In units of work:
// the whole list's, and those ahead of hi_seq.
struct Spot {
  int64_t total, hi_ahead, lo_tile, hi_tile;
  int lo_seq, hi_seq;
};

// All threads of the CTA.
__device__ void find_chunk(const Args& a, int c, Spot* out, int64_t* part) {
  const int nt = blockDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = nt >> 5;
  const int per = (a.t.num_seqs + nt - 1) / nt;
  const int b0 = min(a.t.num_seqs, (int)threadIdx.x * per), b1 = min(a.t.num_seqs, b0 + per);
  int64_t sum = 0;
  for (int b = b0; b < b1; ++b) sum += seq_work(a, b);
  int64_t incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(FULL_MASK, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) part[warp] = incl;
  if (threadIdx.x == 0) {
    out->lo_seq = out->hi_seq = a.t.num_seqs;
    out->lo_tile = out->hi_tile = 0;
  }
  __syncthreads();
  int64_t before = 0, total = 0;
  for (int w = 0; w < nw; ++w) {
    if (w < warp) before += part[w];
    total += part[w];
  }
  const int64_t lo = total * c / a.chunks, hi = total * (c + 1) / a.chunks;
  if (threadIdx.x == 0) out->total = total;
  int64_t at = before + incl - sum;
  for (int b = b0; b < b1; ++b) {
    const int64_t n = seq_work(a, b);
    if (lo >= at && lo < at + n) {
      out->lo_seq = b;
      out->lo_tile = Work(a, b).tile(lo - at);
    }
    if (hi >= at && hi < at + n) {
      out->hi_seq = b;
      out->hi_tile = Work(a, b).tile(hi - at);
      out->hi_ahead = at;
    }
    at += n;
  }
  __syncthreads();
}

// Walks the items of a stretch: tiles [t0, t1) of KV head h and rows [rt * rows_cap, ...) of sequence b.
struct Walk {
  int b, rt, h, t0, t1, tiles, rts, hi_seq;
  int64_t at, hi_tile;  // the item's first tile in the sequence's part of the list; the stretch's end in hi_seq's
  __device__ __forceinline__ void enter(const Args& a) {
    tiles = seq_tiles(a.t, b);
    rts = (seq_rows(a, b) + a.rows_cap - 1) / a.rows_cap;
  }
  __device__ __forceinline__ void to_end() {
    t1 = b == hi_seq ? (int)min((int64_t)tiles, hi_tile - at) : tiles;
  }
  __device__ __forceinline__ Walk(const Args& a, const Spot& s) {
    b = s.lo_seq;
    hi_seq = s.hi_seq;
    hi_tile = s.hi_tile;
    rt = h = t0 = t1 = tiles = rts = 0;
    at = 0;
    if (b < a.t.num_seqs) {
      enter(a);
      const int per = tiles * a.t.nkv;  // below 2^31: k_len / 128 x nkv
      rt = (int)(s.lo_tile / per);
      const int r = (int)(s.lo_tile % per);
      h = r / tiles;
      t0 = r % tiles;
      at = s.lo_tile - t0;
      to_end();
    }
  }
  __device__ __forceinline__ bool more() const { return t1 > t0; }
  __device__ __forceinline__ void next(const Args& a) {
    if (t1 < tiles) {
      t0 = t1;  // the stretch's end
      return;
    }
    at += tiles;
    if (++h == a.t.nkv) {
      h = 0;
      if (++rt == rts) {
        rt = 0;
        at = 0;
        do ++b;
        while (b < a.t.num_seqs && seq_rows(a, b) <= 0);
        if (b >= a.t.num_seqs) {
          t0 = t1 = 0;
          return;
        }
        enter(a);
      }
    }
    t0 = 0;
    to_end();
  }
  __device__ __forceinline__ int rows(const Args& a) const { return min(a.rows_cap, seq_rows(a, b) - rt * a.rows_cap); }
};

// Partial sums of slot s (2 per CTA): rows x 128 outputs (not divided by the sum), then rows x (maximum, sum).
__device__ __forceinline__ float* slot_o(const Args& a, int cta, int slot) {
  return a.t.ws + (int64_t)(cta * 2 + slot) * a.rows_cap * (AD + 2);
}
// Behind them each CTA's end in the list, for the join.
__device__ __forceinline__ Spot* spot_of(const Args& a, int cta) {
  return reinterpret_cast<Spot*>(a.t.ws + 2LL * a.chunks * a.rows_cap * (AD + 2)) + cta;
}

// ------------------------------------------------------------------------ main kernel
// Byte offset of (row, 16-byte chunk) in a tile: [2 halves of 64 dims][128 rows][128 B], 128-byte swizzle.
__device__ __forceinline__ uint32_t tile_at(int r, int c16) {
  return (uint32_t)((c16 >> 3) * HALF + r * 128 + (((c16 & 7) ^ (r & 7)) << 4));
}

struct Small {  // shared memory besides the tiles
  uint64_t full[8], empty[8], raw_full[8], raw_empty[8];
  // q_full: one per group, and only items in which the group has steps arrive at it.  With one barrier for both, an item
  // of a single step, which group 1 takes no part in, could be over before group 1's MMA warp had looked: two such
  // items on, the barrier's parity is what it was and the warp waits for an item that it is already behind.
  uint64_t q_full[2], s_full[2], p_ready[2], o_done[2], o_empty, drain[2];
  uint64_t scale_full[4];
  float2 ml[2][128];        // (maximum, sum) of the groups' rows
  float2 scale[4][KT / 16];  // e4m3: (K, V) scales of 16 keys, of the last four tiles
  uint32_t bad[2][BAD_WORDS];  // keys from bad_from() on whose values are not finite
  int64_t part[16];
  Spot spot;
  uint32_t tmem;
  int gave_up;
};

__host__ __device__ constexpr int smem_bytes(int q_tiles, int slots, int raw_slots) {
  return q_tiles * TILE + slots * TILE + raw_slots * RAW_TILE + (int)sizeof(Small);
}

// e4m3 x 4 -> bf16 x 4, exactly (4 significant bits; a NaN stays one), by f16 and fp32.
__device__ __forceinline__ void e4m3x4_to_bf16(uint32_t x, uint32_t& lo, uint32_t& hi) {
  float f[4];
  e4m3x4_to_f32(x, f);
  lo = pack_bf16(f[0], f[1]);
  hi = pack_bf16(f[2], f[3]);
}

// A tile of e4m3 values (rows of 128 bytes) -> bf16 in a swizzled tile.  128 threads.
__device__ __forceinline__ void convert_tile(const uint8_t* src, uint8_t* dst, int tid) {
  uint4 x[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) x[u] = *reinterpret_cast<const uint4*>(src + (tid + u * 128) * 16);
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int idx = tid + u * 128, r = idx >> 3, i = idx & 7;  // 16 values of row r
    const uint32_t in[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
    uint32_t h[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) e4m3x4_to_bf16(in[e], h[2 * e], h[2 * e + 1]);
    // half of a row's eight lanes store their second 16 bytes first: the two halves of 64 dims lie in the same banks
    // (a tile: 645 -> 400 clocks of stores and loads)
    const int late = i >> 2;
    uint4 v0 = make_uint4(h[0], h[1], h[2], h[3]), v1 = make_uint4(h[4], h[5], h[6], h[7]);
    *reinterpret_cast<uint4*>(dst + tile_at(r, 2 * i + late)) = late ? v1 : v0;
    *reinterpret_cast<uint4*>(dst + tile_at(r, 2 * i + 1 - late)) = late ? v0 : v1;
  }
}

// One warp: queries of rows R .. R + rows - 1 (at most 128) of KV head h as a tile of the products (dims 64.. `half` bytes
// on).  Two rows a step, four steps at a time, whose places in the tile repeat every 1024 bytes.
__device__ __forceinline__ void load_q(const Args& a, int b, int h, int R, int rows, uint32_t dst, int half, int lane) {
  const int c = lane & 15, r0 = lane >> 4, two_gh = 2 % a.G;
  const int64_t stride = a.t.q_stride, two = 2 / a.G * stride;
  int gh = (R + r0) % a.G;
  const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.t.q) + (seq_begin(a.t, b) + (R + r0) / a.G) * stride +
                           (int64_t)h * a.G * AD + c * 8;
  dst += (c >> 3) * half + r0 * 128;
  for (int r = r0; r < rows; r += 8, dst += 1024) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat16* src = q + gh * AD;
      const uint32_t to = dst + j * 256 + (((c & 7) ^ (r0 + 2 * j)) << 4);
      if (r + 2 * j < rows) {
        if (a.q16) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(src) : "memory");
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + 4 * e), "l"(src + 2 * e) : "memory");
        }
      }
      gh += two_gh;
      q += two;
      if (gh >= a.G) {
        gh -= a.G;
        q += stride;
      }
    }
  }
}

// The first key that is looked at for values that are not finite: the tree's, or of an 8-bit cache the first of the 16
// (of one scale) in which the tree begins.
template <bool FP8>
__device__ __forceinline__ int bad_from(int base) {
  return FP8 ? base & ~15 : base;
}

// V's scale of a key is not finite, and not every row sees the 16 keys that share it (or they lie behind the context,
// where the block may be anybody's): their weights are 0, and their values count as not finite.
template <bool FP8>
__device__ __forceinline__ bool odd_scale(int key, int base, float vs) {
  return key >= bad_from<FP8>(base) && !(fabsf(vs) < INFINITY);
}

// Row r of a V tile without its infinities and NaN, all zeros `behind` the context; whether there were any.
__device__ __forceinline__ bool clean_row(uint8_t* v, int r, bool behind) {
  uint32_t any = 0;
#pragma unroll
  for (int h = 0; h < 16 && !behind; h += 8) {  // eight loads on their way: nearly all rows are left as they are
    uint4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const uint4*>(v + tile_at(r, h + i));
#pragma unroll
    for (int i = 0; i < 8; ++i) any |= odd_halves(x[i].x) | odd_halves(x[i].y) | odd_halves(x[i].z) | odd_halves(x[i].w);
  }
  if (behind) {
#pragma unroll
    for (int i = 0; i < 16; ++i) *reinterpret_cast<uint4*>(v + tile_at(r, i)) = make_uint4(0, 0, 0, 0);
  }
  if (any) {
#pragma unroll 1
    for (int i = 0; i < 16; ++i) {
      uint4& at = *reinterpret_cast<uint4*>(v + tile_at(r, i));
      uint4 x = at;
      x.x &= ~((odd_halves(x.x) >> 15) * 0xffffu);
      x.y &= ~((odd_halves(x.y) >> 15) * 0xffffu);
      x.z &= ~((odd_halves(x.z) >> 15) * 0xffffu);
      x.w &= ~((odd_halves(x.w) >> 15) * 0xffffu);
      at = x;
    }
  }
  return any != 0;
}

// Keys [key0, key0 + 64) that a row sees, as bits: those before the tree and its mask's, within the context.
__device__ __forceinline__ uint64_t visible(const uint64_t (&mask)[TREE_WORDS], int key0, int base, int k_len) {
  const int d = base - key0;
  uint64_t see;
  if (d >= 64) {
    see = ~0ull;
  } else if (d > 0) {
    see = ((1ull << d) - 1) | (mask[0] << d);
  } else {
    const int word = -d >> 6, sh = -d & 63;
    uint64_t lo = 0, hi = 0;
#pragma unroll
    for (int i = 0; i < TREE_WORDS; ++i) {
      if (i == word) lo = mask[i];
      if (i == word + 1) hi = mask[i];
    }
    see = sh ? lo >> sh | hi << (64 - sh) : lo;
  }
  const int valid = k_len - key0;
  if (valid < 64) see &= valid > 0 ? (1ull << valid) - 1 : 0ull;
  return see;
}

// 32 bytes of a row in one store: whole sectors.
__device__ __forceinline__ void st32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// The block starts with 128 (e4m3: 512 threads) or 168 registers per thread; the softmax warps take more from the
// other warpgroups: 2 x 176 + 56 + 104 = 4 x 128, 2 x 208 + 88 = 3 x 168.
template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// (a, b) * f + c and (a, b) + (c, d) in one instruction each
__device__ __forceinline__ float2 fma2(uint32_t a, uint32_t b, float f, float c) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %4};\n mov.b64 z, {%5, %5};\n"
      " fma.rn.f32x2 z, x, y, z;\n mov.b64 {%0, %1}, z;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "r"(a), "r"(b), "f"(f), "f"(c));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

// An error, in the process's error word: the outputs are not valid.
__device__ __forceinline__ void give_up(int* word, int code) {
  *reinterpret_cast<volatile int*>(word) = ERROR_BASE + code;
  __threadfence_system();
}

// Bounded wait of a whole warp; on expiry every role goes on without waiting, and the kernel's end reports the code that
// it finds in *gave_up.  The same answer in every lane.  One lane polls.
__device__ __forceinline__ bool warp_poll(uint32_t bar, uint32_t parity, volatile int* gave_up, int code,
                                          uint64_t budget_ns = tc::WAIT_BUDGET_NS) {
  int ok = 1;
  if ((threadIdx.x & 31) == 0) {
    SpinBudget sb;
    while (!tc::mbar_try(bar, parity)) {
      if (*gave_up) {
        ok = 0;
        break;
      }
      if (sb.expired(budget_ns)) {
        *gave_up = code;
        ok = 0;
        break;
      }
    }
  }
  ok = __shfl_sync(FULL_MASK, ok, 0);
  if (ok) tc::mbar_try(bar, parity);  // the phase is complete: this orders the other lanes' accesses
  return ok != 0;
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* gave_up, int code) {
  if (__all_sync(FULL_MASK, tc::mbar_try(bar, parity))) return true;
  return warp_poll(bar, parity, gave_up, code);
}

// A wait that nothing ends, given up after budget_ns.
__global__ void tree_wait_check_kernel(int* word, uint64_t budget_ns) {
  __shared__ uint64_t bar;
  __shared__ int gave_up;
  if (threadIdx.x == 0) {
    tc::mbar_init(smem_u32(&bar), 1);
    gave_up = 0;
    tc::fence_barrier_init();
  }
  __syncthreads();
  warp_poll(smem_u32(&bar), 0, &gave_up, 99, budget_ns);
  __syncthreads();
  if (threadIdx.x == 0 && gave_up) give_up(word, gave_up);
}

// The part of keys whose values were taken out of the products in a row that sees them, from the cache: the values
// themselves (infinite or NaN), added to the row's outputs [d0, d0 + n) at `out`.
template <bool FP8, typename T>
__device__ __forceinline__ void add_bad(const Args& a, const Walk& w, const uint32_t* bad, int node, int d0, int n, T* out) {
  const int qrow = seq_begin(a.t, w.b), nodes = seq_nodes(a.t, w.b), base = a.t.ctx_lens[w.b] - nodes;
  const int from = bad_from<FP8>(base), last = base + min(nodes, min(TREE_WORDS, a.t.words) * 64);
  for (int pos = from; pos < last; ++pos) {
    const int nd = pos - base;
    if (!(bad[(pos - from) >> 5] >> ((pos - from) & 31) & 1) ||
        (nd >= 0 && !(a.t.mask[(int64_t)(qrow + node) * a.t.mask_stride + (nd >> 6)] >> (nd & 63) & 1)))
      continue;
    if (pos < w.t0 * KT || pos >= w.t1 * KT || (pos >> a.bs_shift) >= a.t.W) continue;
    const int blk = a.t.block_tables[w.b * a.t.bt_stride + (pos >> a.bs_shift)];
    if (blk < 0 || blk >= a.t.num_blocks) continue;
    const int64_t row = (int64_t)blk * a.t.nkv + w.h, at = ((row << a.bs_shift) + (pos & (a.t.block_size - 1))) * AD + d0;
    for (int i = 0; i < n; ++i) {
      float z;
      if constexpr (FP8) {
        __half_raw x = __nv_cvt_fp8_to_halfraw(static_cast<const uint8_t*>(a.t.v_cache)[at + i], __NV_E4M3);
        z = __half2float(*reinterpret_cast<__half*>(&x)) * a.t.v_scale[row];
      } else {
        z = __bfloat162float(static_cast<const __nv_bfloat16*>(a.t.v_cache)[at + i]);
      }
      if (!(fabsf(z) < INFINITY)) {
        if constexpr (sizeof(T) == 2)
          out[i] = __float2bfloat16_rn(__bfloat162float(out[i]) + z);
        else
          out[i] += z;
      }
    }
  }
}

// A place in a ring of S slots.
struct Place {
  int s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void step(int by, int S) {  // by <= S
    s += by;
    if (s >= S) {
      s -= S;
      ph ^= 1;
    }
  }
};

template <bool FP8>
__global__ void __launch_bounds__(FP8 ? 512 : 384, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, Args a) {
  pdl_wait();     // inputs come from the previous kernel in the stream
  pdl_trigger();  // the next kernel may start its prologue
  extern __shared__ __align__(1024) uint8_t sm[];
  const int q_tiles = a.rows_cap / 128, S = a.slots, RS = a.raw_slots;
  uint8_t* sq = sm;
  uint8_t* ring = sq + q_tiles * TILE;
  uint8_t* rawr = ring + S * TILE;
  Small& sh = *reinterpret_cast<Small*>(rawr + RS * RAW_TILE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto bar = [](uint64_t& b) { return smem_u32(&b); };
  if (smem_u32(sm) & 1023) {  // the swizzle goes by the address
    if (threadIdx.x == 0) {
      give_up(a.error, 9);
      spot_of(a, blockIdx.x)->hi_seq = a.t.num_seqs;  // nothing to join
    }
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < 8; ++s) {
      tc::mbar_init(bar(sh.full[s]), FP8 ? 4 : 1);
      tc::mbar_init(bar(sh.empty[s]), 2);
      tc::mbar_init(bar(sh.raw_full[s]), 1);
      tc::mbar_init(bar(sh.raw_empty[s]), 4);
    }
    for (int g = 0; g < 2; ++g) {
      tc::mbar_init(bar(sh.q_full[g]), 8);
      tc::mbar_init(bar(sh.s_full[g]), 1);
      tc::mbar_init(bar(sh.p_ready[g]), 4);
      tc::mbar_init(bar(sh.o_done[g]), 1);
      tc::mbar_init(bar(sh.drain[g]), 1);
    }
    tc::mbar_init(bar(sh.o_empty), 8);
    for (int s = 0; s < 4; ++s) tc::mbar_init(bar(sh.scale_full[s]), 1);
    sh.gave_up = 0;
    tc::fence_barrier_init();
  }
  if (threadIdx.x < 2 * BAD_WORDS) sh.bad[threadIdx.x / BAD_WORDS][threadIdx.x % BAD_WORDS] = 0;
  if (warp == W_MMA) tc::tmem_alloc<1>(smem_u32(&sh.tmem), 512);
  tc::fence_before();
  find_chunk(a, blockIdx.x, &sh.spot, sh.part);  // ends with a barrier
  if (threadIdx.x == 0) *spot_of(a, blockIdx.x) = sh.spot;
  tc::fence_after();
  const uint32_t tmem = sh.tmem;
  volatile int* gave_up = &sh.gave_up;

  auto wait = [&](uint64_t& b, uint32_t parity, int code) { return warp_wait(bar(b), parity, &sh.gave_up, code); };

  if (warp < W_TMA) {
    // ------------------------------------------------------------------ softmax, outputs
    regs_inc<FP8 ? 176 : 208>();
    const int g = warp >> 2, q4 = warp & 3, lr = q4 * 32 + lane;  // TMEM lane = row of the group
    const uint32_t lanes = (uint32_t)(q4 * 32) << 16;
    const uint32_t s_tm = tmem + g * 128u + lanes, o_tm = tmem + 256u + lanes;  // O of group k: + 128 k
    uint32_t n_done = 0;  // steps of this group so far
    // The groups make their weights in turn: left alone they fall into step, and then both wait for products at a
    // time and share the exponentials' units at another.
    auto turn_take = [&]() { asm volatile("bar.sync %0, 256;" ::"r"(2 + g) : "memory"); };
    auto turn_pass = [&]() { asm volatile("bar.arrive %0, 256;" ::"r"(3 - g) : "memory"); };
    if (g == 1) turn_pass();
    int tile0 = 0, items = 0;  // tiles before this item
    // An item's queries, by the eight warps: one alone took 20000 clocks for 256 rows.  The next item's are on their way
    // while this one's outputs are written.
    auto fetch_q = [&](const Walk& w) {
      const int rows = w.rows(a), per = rows > 128 ? 32 : 16, r = warp * per;
      load_q(a, w.b, w.h, w.rt * a.rows_cap + r, min(per, rows - r), smem_u32(sq) + (r >> 7) * TILE + (r & 127) * 128, HALF, lane);
    };
    struct Row {  // what a thread has to know of its row
      int row, qrow, nodes, k_len, node, gh;
      uint64_t bits[TREE_WORDS];  // the mask
    };
    auto row_of = [&](const Walk& w) {
      Row r;
      const int rows = w.rows(a);
      r.row = rows > 128 ? g * 128 + lr : lr;
      const int R = w.rt * a.rows_cap + r.row;
      const bool live = r.row < rows;
      r.qrow = seq_begin(a.t, w.b);
      r.nodes = seq_nodes(a.t, w.b);
      r.k_len = a.t.ctx_lens[w.b];
      r.node = live ? R / a.G : 0;
      r.gh = live ? R % a.G : 0;
#pragma unroll
      for (int i = 0; i < TREE_WORDS; ++i)
        r.bits[i] = i < a.t.words ? (uint64_t)a.t.mask[(int64_t)(r.qrow + r.node) * a.t.mask_stride + i] : 0ull;
      return r;
    };
    Walk next(a, sh.spot);
    Row next_row;
    if (next.more()) {
      fetch_q(next);
      next_row = row_of(next);
    }
    for (; next.more(); ++items) {
      const Walk w = next;
      next.next(a);
      asm volatile("cp.async.wait_all;" ::: "memory");
      tc::fence_proxy_async();
      __syncwarp();
      const int n = w.t1 - w.t0, rows = w.rows(a), two = rows > 128, steps = two ? 2 * n : n;
      if (lane == 0) {
        tc::mbar_arrive_release(bar(sh.q_full[0]));
        if (steps > 1) tc::mbar_arrive_release(bar(sh.q_full[1]));
      }
      const Row me = next_row;
      const int row = me.row, qrow = me.qrow, k_len = me.k_len, base = k_len - me.nodes, node = me.node, head = w.h * a.G + me.gh;
      const bool live = row < rows, work = __any_sync(FULL_MASK, live);
      float m = -INFINITY, l = 0.f;
      int mine = 0;
      for (int st = g; st < steps; st += 2, ++mine, ++n_done) {
        const int j = two ? st >> 1 : st, t = w.t0 + j;
        wait(sh.s_full[g], n_done & 1, 8);
        tc::fence_after();
        const bool masked = t * KT + KT > base;
        const float2* scl = sh.scale[(tile0 + j) & 3];
        // (not K's own barrier: its slot may have been filled again by now.  This one is filled for the fourth tile
        // from here, once this one's weights are used.)
        if constexpr (FP8) wait(sh.scale_full[(tile0 + j) & 3], ((tile0 + j) >> 2) & 1, 10);
        auto softmax = [&](auto with_mask) {
          constexpr bool MASK = decltype(with_mask)::value;
          uint32_t see[4] = {~0u, ~0u, ~0u, ~0u}, x[2][16], p[64];
          if constexpr (MASK) {
            const uint64_t s0 = visible(me.bits, t * KT, base, k_len), s1 = visible(me.bits, t * KT + 64, base, k_len);
            see[0] = (uint32_t)s0;
            see[1] = (uint32_t)(s0 >> 32);
            see[2] = (uint32_t)s1;
            see[3] = (uint32_t)(s1 >> 32);
          }
          // 16 columns (keys) at a time, the next ones on their way: f(column group, their scores in units of log2
          // of weights, times K's scale)
          auto columns = [&](auto&& f) {
            tc::tmem_ld(s_tm, x[0]);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              tc::ld_wait(x[c & 1]);
              if (c < 7) tc::tmem_ld(s_tm + 16 * (c + 1), x[(c + 1) & 1]);
              f(c, x[c & 1]);
            }
          };
          auto seen = [&](int c, int i) { return !MASK || (see[c >> 1] >> (16 * (c & 1) + i) & 1); };
          auto factor = [&](int c) { return FP8 ? a.scale_log2 * scl[c].x : a.scale_log2; };
          float2 ls[2];
          float top;
          // weights relative to `sub`, their sum, and the largest exponent
          auto weights = [&](float sub) {
            ls[0] = ls[1] = make_float2(0.f, 0.f);
            float mx[2] = {-INFINITY, -INFINITY};
            columns([&](int c, uint32_t(&v)[16]) {
              const float f = factor(c);
              [[maybe_unused]] float vs = 1.f;
              if constexpr (FP8) {
                vs = scl[c].y;
                if (MASK && odd_scale<FP8>(t * KT + 16 * c, base, vs)) vs = 0.f;
              }
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                float2 y = fma2(v[i], v[i + 1], f, -sub);
                if (!seen(c, i)) y.x = -INFINITY;
                if (!seen(c, i + 1)) y.y = -INFINITY;
                mx[0] = fmaxf(mx[0], y.x);
                mx[1] = fmaxf(mx[1], y.y);
                y = make_float2(ex2(y.x), ex2(y.y));
                ls[i >> 1 & 1] = add2(ls[i >> 1 & 1], y);
                if constexpr (FP8) {
                  y.x *= vs;
                  y.y *= vs;
                }
                // rounded by 2^-8 of a weight at most; the sum takes the weights as they were
                p[8 * c + (i >> 1)] = pack_bf16(y.x, y.y);
              }
            });
            top = fmaxf(mx[0], mx[1]);
          };
          if (mine == 0) {  // the first tile's maximum; later ones mostly stay within 2^RAISE of it
            top = -INFINITY;
            columns([&](int c, uint32_t(&v)[16]) {
              const float f = factor(c);  // of either sign
              float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (seen(c, i)) mx[i & 1] = fmaxf(mx[i & 1], __uint_as_float(v[i]) * f);
              top = fmaxf(top, fmaxf(mx[0], mx[1]));
            });
            m = top;
          }
          weights(m == -INFINITY ? 0.f : m);
          const bool raise = top > RAISE || (m == -INFINITY && top > -INFINITY);
          if (mine > 0 && __any_sync(FULL_MASK, raise)) {
            // the outputs so far move to the new maximum, and the weights are made again
            const float nm = raise ? (m == -INFINITY ? top : m + top) : m, f = raise ? ex2(m - nm) : 1.f;
            wait(sh.o_done[g], (n_done - 1) & 1, 11);
            tc::fence_after();
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t o[16];
              tc::tmem_ld(o_tm + 128 * g + 16 * c, o);
              tc::ld_wait(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tc::tmem_st(o_tm + 128 * g + 16 * c, o);
            }
            l *= f;
            m = nm;
            weights(m == -INFINITY ? 0.f : m);
          }
          turn_pass();
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t(&pc)[16] = *reinterpret_cast<uint32_t(*)[16]>(p + 16 * c);
            tc::tmem_st(s_tm + 16 * c, pc);  // over the scores
          }
          ls[0] = add2(ls[0], ls[1]);
          l += ls[0].x + ls[0].y;
          tc::st_wait();
        };
        turn_take();
        if (work) {
          if (masked)
            softmax(std::true_type());
          else
            softmax(std::false_type());
        } else {
          turn_pass();
        }
        if (masked) {
          // this group's threads look through V, a key each: positions behind the context hold any bits, and
          // a node's infinities and NaN go to the rows that see it at the end.  (Where both groups use the tile, both
          // do, since neither's product waits for the other's threads; they write the same.)
          const int c = 2 * (tile0 + j) + 1, pos = t * KT + lr;
          wait(sh.full[c % S], (c / S) & 1, 12);
          uint8_t* v = ring + (c % S) * TILE;
          if (pos >= bad_from<FP8>(base)) {
            bool odd = clean_row(v, lr, pos >= k_len);
            if constexpr (FP8) odd |= pos < k_len && odd_scale<FP8>(pos, base, scl[lr >> 4].y);
            const int i = pos - bad_from<FP8>(base);
            if (odd && i < BAD_WORDS * 32) atomicOr(&sh.bad[items & 1][i >> 5], 1u << (i & 31));
          }
          tc::fence_proxy_async();
        }
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_release(bar(sh.p_ready[g]));
      }
      if (g == 1 && !two && (n & 1)) {  // the other group had a step more
        turn_take();
        turn_pass();
      }
      // ---- outputs
      sh.ml[g][lr] = make_float2(m, l);
      if (mine) wait(sh.o_done[g], (n_done - 1) & 1, 13);
      tc::fence_before();
      asm volatile("bar.sync 1, 256;" ::: "memory");
      tc::fence_after();
      if (next.more()) {  // every product with this item's queries has been waited for
        fetch_q(next);
        next_row = row_of(next);
      }
      const float2 ml0 = sh.ml[0][lr], ml1 = sh.ml[1][lr];
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < BAD_WORDS; ++i) any |= sh.bad[items & 1][i];
      if (g == 0 && lr < BAD_WORDS) sh.bad[(items + 1) & 1][lr] = 0;
      // the groups' sums by their weights: with more than 128 rows a group has rows of its own
      float w0 = 0.f, w1 = 0.f, M = m, L = l;
      bool has0, has1;
      if (two) {
        has0 = g == 0 && !(m == -INFINITY && l == 0.f);
        has1 = g == 1 && !(m == -INFINITY && l == 0.f);
        w0 = w1 = 1.f;
      } else {
        M = fmaxf(ml0.x, ml1.x);
        const float mb = M == -INFINITY ? 0.f : M;
        has0 = !(ml0.x == -INFINITY && ml0.y == 0.f);
        has1 = steps > 1 && !(ml1.x == -INFINITY && ml1.y == 0.f);
        L = 0.f;
        if (has0) L += (w0 = ex2(ml0.x - mb)) * ml0.y;
        if (has1) L += (w1 = ex2(ml1.x - mb)) * ml1.y;
      }
      const bool whole = w.t0 == 0 && w.t1 == w.tiles;
      const float inv = whole ? (L != 0.f ? 1.f / L : 0.f) : 1.f;
      float* slot = slot_o(a, blockIdx.x, w.t0 == 0);
      if (work) {
        const int c0 = two ? 0 : 4 * g, c1 = two ? 8 : 4 * g + 4;  // chunks of 16 dims
        const bool r0 = !two || g == 0, r1 = two ? g == 1 : steps > 1;  // uniform
        if (!has0) w0 = 0.f;
        if (!has1) w1 = 0.f;
        __nv_bfloat16* op = static_cast<__nv_bfloat16*>(a.t.out) + ((int64_t)(qrow + node) * a.t.nq + head) * AD;
        float* po = slot + (int64_t)row * AD;
#pragma unroll 1
        for (int c = c0; c < c1; ++c) {
          uint32_t x0[16], x1[16], v[8];
          if (r0) tc::tmem_ld(o_tm + 16 * c, x0);
          if (r1) tc::tmem_ld(o_tm + 128 + 16 * c, x1);
          float o[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = 0.f;
          if (r0) {
            tc::ld_wait(x0);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = has0 ? w0 * __uint_as_float(x0[i]) : 0.f;
          }
          if (r1) {
            tc::ld_wait(x1);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] += has1 ? w1 * __uint_as_float(x1[i]) : 0.f;
          }
          if (!live) continue;
          if (whole) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = L == 0.f ? 0u : pack_bf16(o[2 * i] * inv, o[2 * i + 1] * inv);
            st32(op + 16 * c, v);
          } else {
#pragma unroll
            for (int k = 0; k < 16; k += 8) {
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = __float_as_uint(o[k + i]);
              st32(po + 16 * c + k, v);
            }
          }
        }
        if (any && live && k_len > 0) {
          if (whole)
            add_bad<FP8>(a, w, sh.bad[items & 1], node, 16 * c0, 16 * (c1 - c0), op + 16 * c0);
          else
            add_bad<FP8>(a, w, sh.bad[items & 1], node, 16 * c0, 16 * (c1 - c0), po + 16 * c0);
        }
        if (!whole && live && (two || g == 0))
          *reinterpret_cast<float2*>(slot + (int64_t)a.rows_cap * AD + row * 2) = make_float2(M, L);
      }
      tc::fence_before();
      asm volatile("bar.sync 1, 256;" ::: "memory");  // ml and bad have been read
      if (lane == 0) tc::mbar_arrive_release(bar(sh.o_empty));
      tile0 += n;
    }
    tc::fence_before();
  } else if (warp < W_CONV) {
    regs_dec<FP8 ? 56 : 88>();
    if (warp == W_TMA) {
      // ---------------------------------------------------------------- TMA producer
      if (lane == 0) {
        tc::prefetch_map(&kmap);
        tc::prefetch_map(&vmap);
      }
      const int depth = FP8 ? RS : S;
      Place at;
      int c = 0;  // tiles so far (K and V in turn)
      bool ok = true;
      for (Walk w(a, sh.spot); w.more() && ok; w.next(a)) {
        const int* bt = a.t.block_tables + w.b * a.t.bt_stride;
        for (int t = w.t0; t < w.t1 && ok; ++t) {
          // one lane per box
          int row = a.oob_row;
          const int r = lane << (a.bs_shift < 7 ? a.bs_shift : 7);
          if (r < KT) {
            const int tok = t * KT + r, bi = tok >> a.bs_shift;
            if (bi < a.t.W) {
              const int blk = bt[bi];
              if (blk >= 0 && blk < a.t.num_blocks) row = ((blk * a.t.nkv + w.h) << a.bs_shift) + (tok & (a.t.block_size - 1));
            }
          }
          for (int kv = 0; kv < 2 && ok; ++kv, ++c) {
            if (!wait(FP8 ? sh.raw_empty[at.s] : sh.empty[at.s], at.ph ^ 1, 1)) {
              ok = false;
              break;
            }
            const uint32_t full = bar(FP8 ? sh.raw_full[at.s] : sh.full[at.s]);
            const uint32_t dst = FP8 ? smem_u32(rawr + at.s * RAW_TILE) : smem_u32(ring + at.s * TILE);
            const CUtensorMap* map = kv ? &vmap : &kmap;
            if (lane == 0) tc::mbar_arrive_expect_tx(full, FP8 ? RAW_TILE : TILE);
            __syncwarp();
            if (r < KT) {
              tc::tma_load_2d(dst + r * 128, map, full, 0, row);
              if (!FP8) tc::tma_load_2d(dst + HALF + r * 128, map, full, 64, row);
            }
            at.step(1, depth);
          }
        }
      }
      if (*gave_up)  // copies that nobody waited for may still be landing
        for (int k = max(0, c - depth); k < c; ++k)
          tc::mbar_drain(bar(FP8 ? sh.raw_full[k % depth] : sh.full[k % depth]), (k / depth) & 1);
    } else if (warp >= W_MMA) {
      // ---------------------------------------------------------------- MMA issuers, one per group
      const int g = warp - W_MMA;
      constexpr uint32_t id_qk = tc::idesc_bf16(128, 128, false), id_pv = tc::idesc_bf16(128, 128, true);
      const uint32_t s_tm = tmem + g * 128u, o_tm = tmem + 256u + g * 128u;
      const uint64_t ring_k = tc::sdesc(smem_u32(ring)), ring_v = tc::sdesc_mn(smem_u32(ring), HALF), q0 = tc::sdesc(smem_u32(sq));
      bool ok = true;
      uint32_t done = 0;  // steps so far
      int items = 0;
      uint32_t q_items = 0;  // of them with steps of this group
      Place begin;  // of the item's first K
      for (Walk w(a, sh.spot); w.more() && ok; w.next(a), ++items) {
        const int n = w.t1 - w.t0, two = w.rows(a) > 128;
        const int mine = two ? n : (n + 1 - g) >> 1, by = two ? 2 : 4;  // this group's steps; their distance in the ring
        const uint64_t qd = q0 + (two ? g * (TILE >> 4) : 0);
        Place k_at = begin, v_at;
        if (!two && g) k_at.step(2, S);
        v_at = k_at;
        v_at.step(1, S);
        if (mine > 0) ok = wait(sh.q_full[g], q_items++ & 1, 2);
        for (int i = 0; i <= mine && ok; ++i) {
          if (i > 0) {  // P V of the step before
            ok = wait(sh.p_ready[g], (done - 1) & 1, 3) && wait(sh.full[v_at.s], v_at.ph, 4) &&
                 // the outputs of the item before have been read
                 (i > 1 || items == 0 || wait(sh.o_empty, (items - 1) & 1, 5));
            if (!ok) break;
            tc::fence_after();
            if (elect_one()) {
              const uint64_t vd = ring_v + (uint64_t)v_at.s * (TILE >> 4);
#pragma unroll
              for (int k = 0; k < 8; ++k)  // 16 keys: packed columns 8 k of P, rows 16 k of V
                tc::mma_bf16_ts(o_tm, s_tm + 8 * k, vd + k * (16 * 128 >> 4), id_pv, i > 1 || k > 0);
              tc::commit<1>(bar(sh.o_done[g]));
              tc::commit<1>(bar(sh.empty[v_at.s]));
              if (!two) tc::commit<1>(bar(sh.empty[v_at.s]));
            }
            __syncwarp();
            v_at.step(by, S);
          }
          if (i < mine) {
            ok = wait(sh.full[k_at.s], k_at.ph, 6) &&
                 (done == 0 || wait(sh.o_done[g], (done - 1) & 1, 7));  // S overwrites the P of this group's last step
            if (!ok) break;
            if (elect_one()) {
              const uint64_t kd = ring_k + (uint64_t)k_at.s * (TILE >> 4);
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const uint32_t at = ((k >> 2) * HALF + (k & 3) * 32) >> 4;
                tc::mma_bf16_ss(s_tm, qd + at, kd + at, id_qk, k > 0);
              }
              tc::commit<1>(bar(sh.s_full[g]));
              tc::commit<1>(bar(sh.empty[k_at.s]));
              if (!two) tc::commit<1>(bar(sh.empty[k_at.s]));
            }
            __syncwarp();
            k_at.step(by, S);
            ++done;
          }
        }
        const int on = begin.s + 2 * n;
        begin.ph ^= (uint32_t)(on / S) & 1;
        begin.s = on % S;
      }
      if (elect_one()) tc::commit<1>(bar(sh.drain[g]));  // every MMA of this thread
      __syncwarp();
      if (lane == 0) tc::mbar_drain(bar(sh.drain[g]), 0);
      __syncwarp();
    }
  } else if constexpr (FP8) {
    // ------------------------------------------------------------------ e4m3 -> bf16 tiles
    regs_dec<104>();
    const int tid = threadIdx.x - W_CONV * 32;
    Place from, to;
    int tile = 0;
    for (Walk w(a, sh.spot); w.more(); w.next(a)) {
      const int* bt = a.t.block_tables + w.b * a.t.bt_stride;
      for (int t = w.t0; t < w.t1; ++t, ++tile)
        for (int kv = 0; kv < 2; ++kv) {
          float2 sc = make_float2(0.f, 0.f);
          if (kv == 0 && tid < KT / 16) {
            const int bi = (t * KT + tid * 16) >> a.bs_shift;
            const int blk = bi < a.t.W ? bt[bi] : -1;
            if (blk >= 0 && blk < a.t.num_blocks) {
              const int64_t at = (int64_t)blk * a.t.nkv + w.h;
              sc = make_float2(a.t.k_scale[at], a.t.v_scale[at]);
            }
          }
          wait(sh.raw_full[from.s], from.ph, 15);
          wait(sh.empty[to.s], to.ph ^ 1, 16);
          if (kv == 0 && tid < 32) {
            if (tid < KT / 16) sh.scale[tile & 3][tid] = sc;
            __syncwarp();
            if (tid == 0) tc::mbar_arrive_release(bar(sh.scale_full[tile & 3]));
          }
          convert_tile(rawr + from.s * RAW_TILE, ring + to.s * TILE, tid);
          tc::fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            tc::mbar_arrive_release(bar(sh.full[to.s]));
            tc::mbar_arrive_release(bar(sh.raw_empty[from.s]));
          }
          from.step(1, RS);
          to.step(1, S);
        }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && sh.gave_up) give_up(a.error, sh.gave_up);
  if (warp == W_MMA) {
    tc::fence_after();
    tc::tmem_dealloc<1>(tmem, 512);
  }
}

// ------------------------------------------------------------------ kernel for few rows
// Up to 64 rows: keys on the products' M side, so that nothing is computed for rows that are not there.
//   S^T = K Q^T     [128 keys x N rows], two buffers in TMEM
//   P^T             one key per thread, N weights, as bf16 into shared memory (two buffers)
//   O^T += V^T P^T  [128 dims x N rows] in TMEM, two buffers, one per item in turn
// A row's maximum and sum run over threads: the maximum is taken from the first tile and raised only when a score
// passes it by 2^8 (one vote per tile), the sums are kept per thread and added up at the item's end.
struct Few {  // shared memory besides the tiles
  uint64_t full[8], empty[8], raw_full[8], raw_empty[8];
  uint64_t q_full[2], q_empty[2], s_full[2], p_ready[2], o_done[2], o_empty[2], scale_full[4], drain;
  alignas(16) float mrow[64];  // maxima (units of log2); read four at a time
  alignas(16) float inv[64];   // 1 / sums
  alignas(16) float red[4][64];
  float2 scale[4][KT / 16];
  uint32_t bad[2][BAD_WORDS];
  int64_t part[16];
  Spot spot;
  uint32_t tmem;
  int gave_up;
};

// Buffers of Q and P: two each; e4m3, which needs the room for its 8-bit tiles: one of P, and with 64 rows one of Q.
template <bool FP8, int N>
struct Bufs {
  static constexpr int Q = FP8 && N == 64 ? 1 : 2, P = FP8 ? 1 : 2;
  __host__ __device__ static constexpr int bytes(int slots, int raw_slots) {
    return Q * N * 256 + P * HALF + slots * TILE + raw_slots * RAW_TILE + (int)sizeof(Few);
  }
};

__device__ __forceinline__ bool vote_any(bool p) {  // over the 128 softmax threads
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 128, p;\n selp.b32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"((int)p)
      : "memory");
  return r != 0;
}
// (a, b) * f - (c, d)
__device__ __forceinline__ float2 fms2(uint32_t a, uint32_t b, float f, float c, float d) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %4};\n mov.b64 z, {%5, %6};\n"
      " fma.rn.f32x2 z, x, y, z;\n mov.b64 {%0, %1}, z;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "r"(a), "r"(b), "f"(f), "f"(-c), "f"(-d));
  return r;
}

template <bool FP8, int N>
__global__ void __launch_bounds__(FP8 ? 512 : 256, 1)
    tree_attn_few_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, Args a) {
  pdl_wait();     // inputs come from the previous kernel in the stream
  pdl_trigger();  // the next kernel may start its prologue
  extern __shared__ __align__(1024) uint8_t sm[];
  constexpr int QT = N * 256, QHALF = N * 128;
  constexpr int F_TMA = 4, F_Q = 5, F_MMA = 6, F_CONV = 8;  // first warp of each role; 0-3: softmax
  const int S = a.slots, RS = a.raw_slots;
  uint8_t* ring = sm;
  uint8_t* pbuf = ring + S * TILE;
  constexpr int QB = Bufs<FP8, N>::Q, PB = Bufs<FP8, N>::P;
  uint8_t* rawr = pbuf + PB * HALF;
  uint8_t* sq = rawr + RS * RAW_TILE;
  Few& sh = *reinterpret_cast<Few*>(sq + QB * QT);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto bar = [](uint64_t& b) { return smem_u32(&b); };
  if (smem_u32(sm) & 1023) {  // the swizzle goes by the address
    if (threadIdx.x == 0) {
      give_up(a.error, 9);
      spot_of(a, blockIdx.x)->hi_seq = a.t.num_seqs;  // nothing to join
    }
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < 8; ++s) {
      tc::mbar_init(bar(sh.full[s]), FP8 ? 4 : 1);
      tc::mbar_init(bar(sh.empty[s]), 1);
      tc::mbar_init(bar(sh.raw_full[s]), 1);
      tc::mbar_init(bar(sh.raw_empty[s]), 4);
    }
    for (int k = 0; k < 2; ++k) {
      tc::mbar_init(bar(sh.q_full[k]), 1);
      tc::mbar_init(bar(sh.q_empty[k]), 1);
      tc::mbar_init(bar(sh.s_full[k]), 1);
      tc::mbar_init(bar(sh.p_ready[k]), 4);
      tc::mbar_init(bar(sh.o_done[k]), 1);
      tc::mbar_init(bar(sh.o_empty[k]), 4);
    }
    for (int k = 0; k < 4; ++k) tc::mbar_init(bar(sh.scale_full[k]), 1);
    tc::mbar_init(bar(sh.drain), 1);
    sh.gave_up = 0;
    tc::fence_barrier_init();
  }
  if (threadIdx.x < 2 * BAD_WORDS) sh.bad[threadIdx.x / BAD_WORDS][threadIdx.x % BAD_WORDS] = 0;
  if (warp == F_MMA) tc::tmem_alloc<1>(smem_u32(&sh.tmem), 256);
  tc::fence_before();
  find_chunk(a, blockIdx.x, &sh.spot, sh.part);  // ends with a barrier
  if (threadIdx.x == 0) *spot_of(a, blockIdx.x) = sh.spot;
  tc::fence_after();
  const uint32_t tmem = sh.tmem;  // S^T at 0 and 64, O^T at 128 and 192
  volatile int* gave_up = &sh.gave_up;
  auto wait = [&](uint64_t& b, uint32_t parity, int code) { return warp_wait(bar(b), parity, &sh.gave_up, code); };

  // e4m3: 512 threads begin with 128 registers each, of which the softmax warps take more: 216 + 72 + 2 x 104 < 4 x 128
  if constexpr (FP8) {
    if (warp < F_TMA)
      regs_inc<216>();
    else if (warp < F_CONV)
      regs_dec<72>();
    else
      regs_dec<104>();
  }
  if (warp < F_TMA) {
    // ------------------------------------------------------------------ softmax, outputs
    const int kq = threadIdx.x;  // TMEM lane: a key of the tile, a dim of the outputs
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    uint32_t cnt = 0;  // tiles so far
    int items = 0;
    for (Walk w(a, sh.spot); w.more(); w.next(a), ++items) {
      const int rows = w.rows(a);  // all of the tree's
      const int qrow = seq_begin(a.t, w.b), nodes = seq_nodes(a.t, w.b), k_len = a.t.ctx_lens[w.b], base = k_len - nodes;
      float l[N];
#pragma unroll
      for (int i = 0; i < N; ++i) l[i] = 0.f;
      for (int t = w.t0; t < w.t1; ++t, ++cnt) {
        const int buf = cnt & 1, pos = t * KT + kq;
        const bool masked = t * KT + KT > base;
        uint64_t see = ~0ull;  // rows that see this thread's key
        if (masked) {
          see = pos < base ? ~0ull : 0ull;
          const int nd = pos - base;
          if (pos >= base && pos < k_len && nd >= 0 && (nd >> 6) < a.t.words) {
            const int64_t* mw = a.t.mask + (int64_t)qrow * a.t.mask_stride + (nd >> 6);
            const uint64_t ones = a.G >= 64 ? ~0ull : (1ull << a.G) - 1;
#pragma unroll 4
            for (int r = 0; r < rows; r += a.G, mw += a.t.mask_stride) see |= (*mw >> (nd & 63) & 1) ? ones << r : 0ull;
          }
        }
        wait(sh.s_full[buf], (cnt >> 1) & 1, 8);
        tc::fence_after();
        float f = a.scale_log2, vs = 1.f;
        if constexpr (FP8) {
          wait(sh.scale_full[cnt & 3], (cnt >> 2) & 1, 10);
          const float2 sc = sh.scale[cnt & 3][kq >> 4];
          f *= sc.x;
          vs = sc.y;
        }
        const uint32_t s_tm = tmem + 64u * buf + lanes;
        auto seen = [&](int r) { return (uint32_t)(see >> (r & 32)) >> (r & 31) & 1; };
        // this key's scores, kept in registers where there are enough (e4m3 with 64 rows: read again each time)
        constexpr bool KEEP = !(FP8 && N == 64);
        uint32_t x[KEEP ? N / 16 : 2][16];
        if constexpr (KEEP) {
#pragma unroll
          for (int c = 0; c < N / 16; ++c) tc::tmem_ld(s_tm + 16 * c, x[c]);
#pragma unroll
          for (int c = 0; c < N / 16; ++c) tc::ld_wait(x[c]);
        }
        auto columns = [&](auto&& fn) {
          if constexpr (KEEP) {
#pragma unroll
            for (int c = 0; c < N / 16; ++c) fn(c, x[c]);
          } else {
            tc::tmem_ld(s_tm, x[0]);
#pragma unroll
            for (int c = 0; c < N / 16; ++c) {
              tc::ld_wait(x[c & 1]);
              if (c + 1 < N / 16) tc::tmem_ld(s_tm + 16 * (c + 1), x[(c + 1) & 1]);
              fn(c, x[c & 1]);
            }
          }
        };
        const float4* mr = reinterpret_cast<const float4*>(sh.mrow);
        bool raise = true;
        if (t > w.t0) {
          float mx[2] = {-INFINITY, -INFINITY};
          columns([&](int c, uint32_t(&v)[16]) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const float4 m = mr[4 * c + (i >> 2)];
              float2 y0 = fms2(v[i], v[i + 1], f, m.x, m.y), y1 = fms2(v[i + 2], v[i + 3], f, m.z, m.w);
              if (masked) {
                if (!seen(16 * c + i)) y0.x = -INFINITY;
                if (!seen(16 * c + i + 1)) y0.y = -INFINITY;
                if (!seen(16 * c + i + 2)) y1.x = -INFINITY;
                if (!seen(16 * c + i + 3)) y1.y = -INFINITY;
              }
              mx[0] = fmaxf(mx[0], fmaxf(y0.x, y0.y));
              mx[1] = fmaxf(mx[1], fmaxf(y1.x, y1.y));
            }
          });
          raise = vote_any(fmaxf(mx[0], mx[1]) > RAISE);
        }
        if (raise) {
          // every row's maximum over the tile: within the warp as ordered integers, then over the warps
          columns([&](int c, uint32_t(&v)[16]) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float y = fmaxf(__uint_as_float(v[i]) * f, -INFINITY);  // a NaN sets no maximum
              if (!seen(16 * c + i)) y = -INFINITY;
              const int o = __float_as_int(y) ^ ((__float_as_int(y) >> 31) & 0x7fffffff);
              const int mo = __reduce_max_sync(FULL_MASK, o);
              if (lane == i) sh.red[warp][16 * c + i] = __int_as_float(mo ^ ((mo >> 31) & 0x7fffffff));
            }
          });
          asm volatile("bar.sync 1, 128;" ::: "memory");
          if (kq < N) {
            const float top = fmaxf(fmaxf(sh.red[0][kq], sh.red[1][kq]), fmaxf(sh.red[2][kq], sh.red[3][kq]));
            // a row that has seen nothing yet has a maximum that any score passes
            const float old = t > w.t0 ? sh.mrow[kq] : NOTHING, nm = fmaxf(old, top);
            sh.mrow[kq] = nm;
            sh.red[0][kq] = ex2(old - nm);  // what the sums so far are multiplied by
          }
          asm volatile("bar.sync 1, 128;" ::: "memory");
          if (t > w.t0) {
            wait(sh.o_done[(cnt - 1) & 1], ((cnt - 1) >> 1) & 1, 11);
            tc::fence_after();
            const uint32_t o_tm = tmem + 128u + 64u * (items & 1) + lanes;
#pragma unroll
            for (int c = 0; c < N / 16; ++c) {
              uint32_t o[16];
              tc::tmem_ld(o_tm + 16 * c, o);
              tc::ld_wait(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float g = sh.red[0][16 * c + i];
                o[i] = g == 0.f ? 0u : __float_as_uint(__uint_as_float(o[i]) * g);
                l[16 * c + i] = g == 0.f ? 0.f : l[16 * c + i] * g;
              }
              tc::tmem_st(o_tm + 16 * c, o);
            }
            tc::st_wait();
          }
          asm volatile("bar.sync 1, 128;" ::: "memory");  // red has been read
        }
        // weights: rounded to bf16 (2^-8 of each at most; e4m3: times V's scale), their sums taken as they were
        uint32_t p[N / 2];
        columns([&](int c, uint32_t(&v)[16]) {
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float2 m = reinterpret_cast<const float2*>(sh.mrow)[8 * c + (i >> 1)];
            float2 y = fms2(v[i], v[i + 1], f, m.x, m.y);
            if (masked) {
              if (!seen(16 * c + i)) y.x = -INFINITY;
              if (!seen(16 * c + i + 1)) y.y = -INFINITY;
            }
            y = make_float2(ex2(y.x), ex2(y.y));
            const float2 ls = add2(make_float2(l[16 * c + i], l[16 * c + i + 1]), y);
            l[16 * c + i] = ls.x;
            l[16 * c + i + 1] = ls.y;
            p[8 * c + (i >> 1)] = FP8 ? pack_bf16(y.x * vs, y.y * vs) : pack_bf16(y.x, y.y);
          }
        });
        // the product that read this buffer
        if (cnt >= (uint32_t)PB) wait(sh.o_done[(cnt - PB) & 1], ((cnt - PB) >> 1) & 1, 17);
        uint8_t* pb = pbuf + (PB == 2 ? buf : 0) * HALF;
#pragma unroll
        for (int c = 0; c < N / 8; ++c)
          *reinterpret_cast<uint4*>(pb + tile_at(kq, c)) = make_uint4(p[4 * c], p[4 * c + 1], p[4 * c + 2], p[4 * c + 3]);
        if (masked) {
          // positions behind the context hold any bits, and a node's infinities and NaN go to the rows that
          // see it at the end
          const int c = 2 * cnt + 1;
          wait(sh.full[c % S], (c / S) & 1, 12);
          uint8_t* v = ring + (c % S) * TILE;
          if (pos >= bad_from<FP8>(base)) {
            bool odd = clean_row(v, kq, pos >= k_len);
            if constexpr (FP8)
              if (odd_scale<FP8>(pos, base, sh.scale[cnt & 3][kq >> 4].y)) {
                odd = pos < k_len;
#pragma unroll 1
                for (int c = 0; c < N / 8; ++c) *reinterpret_cast<uint4*>(pb + tile_at(kq, c)) = make_uint4(0, 0, 0, 0);
              }
            const int i = pos - bad_from<FP8>(base);
            if (odd && i < BAD_WORDS * 32) atomicOr(&sh.bad[items & 1][i >> 5], 1u << (i & 31));
          }
        }
        tc::fence_proxy_async();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_release(bar(sh.p_ready[buf]));
      }
      // ---- sums over the threads: each exchange halves what a lane holds
      int at = 0, held = N;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        if (held > 1) {
          const bool up = lane & o;
          held >>= 1;
          at += up ? held : 0;
#pragma unroll
          for (int i = 0; i < N / 2; ++i)
            if (i < held) {
              const float keep = up ? l[i + held] : l[i], give = up ? l[i] : l[i + held];
              l[i] = keep + __shfl_xor_sync(FULL_MASK, give, o);
            }
        } else {
          l[0] += __shfl_xor_sync(FULL_MASK, l[0], o);
        }
      }
#pragma unroll
      for (int i = 0; i < (N > 32 ? N / 32 : 1); ++i) sh.red[warp][at + i] = l[i];
      asm volatile("bar.sync 1, 128;" ::: "memory");
      const bool whole = w.t0 == 0 && w.t1 == w.tiles;
      float* slot = slot_o(a, blockIdx.x, w.t0 == 0);
      if (kq < N) {
        const float L = (sh.red[0][kq] + sh.red[1][kq]) + (sh.red[2][kq] + sh.red[3][kq]);
        sh.inv[kq] = !whole ? 1.f : L == 0.f ? 0.f : 1.f / L;
        if (!whole && kq < rows)
          *reinterpret_cast<float2*>(slot + (int64_t)a.rows_cap * AD + kq * 2) = make_float2(L == 0.f ? -INFINITY : sh.mrow[kq], L);
      }
      wait(sh.o_done[(cnt - 1) & 1], ((cnt - 1) >> 1) & 1, 13);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      tc::fence_after();
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < BAD_WORDS; ++i) any |= sh.bad[items & 1][i];
      if (kq < BAD_WORDS) sh.bad[(items + 1) & 1][kq] = 0;
      const uint32_t o_tm = tmem + 128u + 64u * (items & 1) + lanes;
      {
        // eight rows at a time: a warp writes 32 dims of each
        __nv_bfloat16* op = static_cast<__nv_bfloat16*>(a.t.out) + ((int64_t)qrow * a.t.nq + w.h * a.G) * AD + kq;
        float* po = slot + kq;
        const int64_t jump = (int64_t)(a.t.nq - a.G) * AD;
        int gh = 0;
#pragma unroll 1
        for (int r = 0; r < rows; r += 8) {
          uint32_t o[8];
          tc::tmem_ld(o_tm + r, o);
          const float4 i0 = *reinterpret_cast<const float4*>(sh.inv + r), i1 = *reinterpret_cast<const float4*>(sh.inv + r + 4);
          const float inv[8] = {i0.x, i0.y, i0.z, i0.w, i1.x, i1.y, i1.z, i1.w};
          tc::ld_wait(o);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (r + i < rows) {
              const float v = inv[i] == 0.f ? 0.f : __uint_as_float(o[i]) * inv[i];
              if (whole)
                *op = __float2bfloat16_rn(v);
              else
                *po = v;
            }
            po += AD;
            op += AD;
            if (++gh == a.G) {
              gh = 0;
              op += jump;
            }
          }
        }
        if (any && k_len > 0)
          for (int r = 0; r < rows; ++r) {
            if (whole)
              add_bad<FP8>(a, w, sh.bad[items & 1], r / a.G, kq, 1,
                           static_cast<__nv_bfloat16*>(a.t.out) + ((int64_t)(qrow + r / a.G) * a.t.nq + w.h * a.G + r % a.G) * AD + kq);
            else
              add_bad<FP8>(a, w, sh.bad[items & 1], r / a.G, kq, 1, slot + (int64_t)r * AD + kq);
          }
      }
      tc::fence_before();
      asm volatile("bar.sync 1, 128;" ::: "memory");  // mrow, inv, red and bad have been read
      if (lane == 0) tc::mbar_arrive_release(bar(sh.o_empty[items & 1]));
    }
    tc::fence_before();
  } else if (warp == F_TMA) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      tc::prefetch_map(&kmap);
      tc::prefetch_map(&vmap);
    }
    const int depth = FP8 ? RS : S;
    Place at;
    int c = 0;  // tiles so far (K and V in turn)
    bool ok = true;
    for (Walk w(a, sh.spot); w.more() && ok; w.next(a)) {
      const int* bt = a.t.block_tables + w.b * a.t.bt_stride;
      for (int t = w.t0; t < w.t1 && ok; ++t) {
        // one lane per box
        int row = a.oob_row;
        const int r = lane << (a.bs_shift < 7 ? a.bs_shift : 7);
        if (r < KT) {
          const int tok = t * KT + r, bi = tok >> a.bs_shift;
          if (bi < a.t.W) {
            const int blk = bt[bi];
            if (blk >= 0 && blk < a.t.num_blocks) row = ((blk * a.t.nkv + w.h) << a.bs_shift) + (tok & (a.t.block_size - 1));
          }
        }
        for (int kv = 0; kv < 2 && ok; ++kv, ++c) {
          if (!wait(FP8 ? sh.raw_empty[at.s] : sh.empty[at.s], at.ph ^ 1, 1)) {
            ok = false;
            break;
          }
          const uint32_t full = bar(FP8 ? sh.raw_full[at.s] : sh.full[at.s]);
          const uint32_t dst = FP8 ? smem_u32(rawr + at.s * RAW_TILE) : smem_u32(ring + at.s * TILE);
          const CUtensorMap* map = kv ? &vmap : &kmap;
          if (lane == 0) tc::mbar_arrive_expect_tx(full, FP8 ? RAW_TILE : TILE);
          __syncwarp();
          if (r < KT) {
            tc::tma_load_2d(dst + r * 128, map, full, 0, row);
            if (!FP8) tc::tma_load_2d(dst + HALF + r * 128, map, full, 64, row);
          }
          at.step(1, depth);
        }
      }
    }
    if (*gave_up)  // copies that nobody waited for may still be landing
      for (int k = max(0, c - depth); k < c; ++k)
        tc::mbar_drain(bar(FP8 ? sh.raw_full[k % depth] : sh.full[k % depth]), (k / depth) & 1);
  } else if (warp == F_Q) {
    // ------------------------------------------------------------------ Q, two buffers
    int items = 0;
    for (Walk w(a, sh.spot); w.more(); w.next(a), ++items) {
      const int qb = items % QB;
      if (items >= QB) wait(sh.q_empty[qb], (items / QB - 1) & 1, 14);
      const int rows = w.rows(a), c = lane & 15;
      load_q(a, w.b, w.h, 0, rows, smem_u32(sq + qb * QT), QHALF, lane);
      for (int r = rows + (lane >> 4); r < N; r += 2)  // no row: scores of 0
        *reinterpret_cast<uint4*>(sq + qb * QT + (c >> 3) * QHALF + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
      asm volatile("cp.async.wait_all;" ::: "memory");
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive_release(bar(sh.q_full[qb]));
    }
  } else if (warp == F_MMA) {
    // ------------------------------------------------------------------ MMA issuer
    constexpr uint32_t id_s = tc::idesc_bf16(128, N, false), id_o = tc::idesc_bf16(128, N, true) | (1u << 15);
    const uint64_t ring_k = tc::sdesc(smem_u32(ring)), ring_v = tc::sdesc_mn(smem_u32(ring), HALF);
    const uint64_t p0 = tc::sdesc_mn(smem_u32(pbuf), HALF), q0 = tc::sdesc(smem_u32(sq));
    bool ok = true;
    uint32_t cnt = 0;
    int items = 0;
    Place at;  // of the next K
    // the product with V that is still to come: its tile's number, V's place, the item
    bool pending = false, p_first = false;
    uint32_t p_cnt = 0;
    int p_item = 0;
    Place p_at;
    auto product = [&]() {
      const int buf = p_cnt & 1, ob = p_item & 1;
      pending = false;
      ok = wait(sh.p_ready[buf], (p_cnt >> 1) & 1, 3) && wait(sh.full[p_at.s], p_at.ph, 4) &&
           // the outputs of the item before last have been read
           (!p_first || p_item < 2 || wait(sh.o_empty[ob], ((p_item >> 1) - 1) & 1, 5));
      if (!ok) return;
      tc::fence_after();
      if (elect_one()) {
        const uint64_t vd = ring_v + (uint64_t)p_at.s * (TILE >> 4), pd = p0 + (uint64_t)(PB == 2 ? buf : 0) * (HALF >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k)  // 16 keys
          tc::mma_bf16_ss(tmem + 128u + 64u * ob, vd + k * (16 * 128 >> 4), pd + k * (16 * 128 >> 4), id_o, !p_first || k > 0);
        tc::commit<1>(bar(sh.o_done[buf]));
        tc::commit<1>(bar(sh.empty[p_at.s]));
      }
      __syncwarp();
    };
    for (Walk w(a, sh.spot); w.more() && ok; w.next(a), ++items) {
      const int qb = items % QB;
      for (int t = w.t0; t < w.t1 && ok; ++t, ++cnt) {
        const int buf = cnt & 1;
        // the last tile's product goes first unless this tile's keys are there already
        int ready = 0;
        if (lane == 0) ready = tc::mbar_try(bar(sh.full[at.s]), at.ph);
        if (pending && !__shfl_sync(FULL_MASK, ready, 0)) product();
        if (!ok) break;
        if (t == w.t0) ok = wait(sh.q_full[qb], (items / QB) & 1, 2);
        ok = ok && wait(sh.full[at.s], at.ph, 6);
        if (!ok) break;
        if (cnt >= 2) tc::fence_after();  // the buffer's last reader has announced its weights
        if constexpr (FP8) tc::fence_after();
        if (elect_one()) {
          const uint64_t kd = ring_k + (uint64_t)at.s * (TILE >> 4), qd = q0 + (uint64_t)qb * (QT >> 4);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            tc::mma_bf16_ss(tmem + 64u * buf, kd + (((k >> 2) * HALF + (k & 3) * 32) >> 4), qd + (((k >> 2) * QHALF + (k & 3) * 32) >> 4), id_s, k > 0);
          tc::commit<1>(bar(sh.s_full[buf]));
          tc::commit<1>(bar(sh.empty[at.s]));
          if (t == w.t1 - 1) tc::commit<1>(bar(sh.q_empty[qb]));
        }
        __syncwarp();
        if (pending) product();
        pending = true;
        p_first = t == w.t0;
        p_cnt = cnt;
        p_item = items;
        at.step(1, S);
        p_at = at;
        at.step(1, S);
      }
    }
    if (ok && pending) product();
    if (elect_one()) tc::commit<1>(bar(sh.drain));  // every MMA of this thread
    __syncwarp();
    if (lane == 0) tc::mbar_drain(bar(sh.drain), 0);
    __syncwarp();
  } else if (FP8 && warp >= F_CONV) {
    // ------------------------------------------------------------------ e4m3 -> bf16 tiles: four warps for K, four for V
    const int tid = (threadIdx.x - F_CONV * 32) & 127, kv = (warp - F_CONV) >> 2;
    Place from, to;
    from.step(kv, RS);
    to.step(kv, S);
    int tile = 0;
    // the scales of a tile, asked for while the one before is converted
    auto scales = [&](const Walk& w, int t) {
      float2 sc = make_float2(0.f, 0.f);
      if (kv == 0 && tid < KT / 16) {
        const int bi = (t * KT + tid * 16) >> a.bs_shift;
        const int blk = bi < a.t.W ? a.t.block_tables[w.b * a.t.bt_stride + bi] : -1;
        if (blk >= 0 && blk < a.t.num_blocks) {
          const int64_t k = (int64_t)blk * a.t.nkv + w.h;
          sc = make_float2(a.t.k_scale[k], a.t.v_scale[k]);
        }
      }
      return sc;
    };
    for (Walk w(a, sh.spot); w.more(); w.next(a)) {
      float2 next = scales(w, w.t0);
      for (int t = w.t0; t < w.t1; ++t, ++tile) {
        const float2 sc = next;
        wait(sh.raw_full[from.s], from.ph, 15);
        if (t + 1 < w.t1) next = scales(w, t + 1);
        wait(sh.empty[to.s], to.ph ^ 1, 16);
        if (kv == 0 && tid < 32) {
          // (K's slot is free: the weights of the fourth tile before this one are done, and with them its scales)
          if (tid < KT / 16) sh.scale[tile & 3][tid] = sc;
          __syncwarp();
          if (tid == 0) tc::mbar_arrive_release(bar(sh.scale_full[tile & 3]));
        }
        convert_tile(rawr + from.s * RAW_TILE, ring + to.s * TILE, tid);
        tc::fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          tc::mbar_arrive_release(bar(sh.full[to.s]));
          tc::mbar_arrive_release(bar(sh.raw_empty[from.s]));
        }
        from.step(2, RS);
        to.step(2, S);
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && sh.gave_up) give_up(a.error, sh.gave_up);
  if (warp == F_MMA) {
    tc::fence_after();
    tc::tmem_dealloc<1>(tmem, 256);
  }
}

// ---------------------------------------------------------------------------- joining
// CTA (chunk, JOIN_ROWS rows) joins the item that begins in its chunk and ends in a later one, a warp four rows at a
// time: their loads are independent.
constexpr int JOIN_ROWS = 16;
__global__ void __launch_bounds__(128) tree_join_kernel(Args a) {
  pdl_wait();     // the partial sums come from the previous kernel in the stream
  pdl_trigger();  // the next kernel may start its prologue
  const int chunk = blockIdx.x;
  const Spot spot = *spot_of(a, chunk);
  const int b = spot.hi_seq;
  if (b >= a.t.num_seqs) return;  // the list's end
  const int tiles = seq_tiles(a.t, b), per = tiles * a.t.nkv;
  const int rt = (int)(spot.hi_tile / per), r0 = (int)(spot.hi_tile % per), h = r0 / tiles, t = r0 % tiles;
  // the item that this chunk's end cuts: its first tile and its work
  const Work work(a, b);
  const int64_t first = spot.hi_tile - t, begin = spot.hi_ahead + work.ahead(first);
  const int unit = first < work.twice * tiles ? ALL_ROWS : FEW_ROWS;
  // tiles of it ahead of a place in the list
  auto ahead = [&](int64_t w) {
    w -= begin + ITEM_WORK;
    return w <= 0 ? (int64_t)0 : min((int64_t)tiles, w / unit);
  };
  auto edge = [&](int k) { return spot.total * k / a.chunks; };
  // (a chunk whose place lies inside the item's first tile begins with it)
  if (t == 0 || edge(chunk) >= begin + ITEM_WORK + unit) return;  // nothing is cut here, or it begins in an earlier chunk
  const int rows = min(a.rows_cap, seq_rows(a, b) - rt * a.rows_cap);
  constexpr int N = JOIN_ROWS / 4;
  const int row0 = blockIdx.y * JOIN_ROWS + (threadIdx.x >> 5) * N, c = (threadIdx.x & 31) * 4;
  if (row0 >= rows) return;
  float M[N], L[N], o[N][4];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    M[i] = -INFINITY;
    L[i] = o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  }
  int64_t from = 0;
  for (int k = chunk; from < tiles; ++k) {
    const int64_t upto = ahead(edge(k + 1));
    if (upto > from) {  // with less work than chunks, some have none
      const float* po = slot_o(a, k, from == 0);
      float2 ml[N];
      float4 v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = min(row0 + i, rows - 1);
        ml[i] = *reinterpret_cast<const float2*>(po + (int64_t)a.rows_cap * AD + r * 2);
        v[i] = *reinterpret_cast<const float4*>(po + (int64_t)r * AD + c);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (ml[i].x == -INFINITY && ml[i].y == 0.f) continue;
        const float nm = fmaxf(M[i], ml[i].x), nb = nm == -INFINITY ? 0.f : nm;
        const float f = L[i] == 0.f && M[i] == -INFINITY ? 0.f : ex2(M[i] - nb), g = ex2(ml[i].x - nb);
        M[i] = nm;
        L[i] = L[i] * f + g * ml[i].y;
        o[i][0] = (f == 0.f ? 0.f : o[i][0] * f) + g * v[i].x;
        o[i][1] = (f == 0.f ? 0.f : o[i][1] * f) + g * v[i].y;
        o[i][2] = (f == 0.f ? 0.f : o[i][2] * f) + g * v[i].z;
        o[i][3] = (f == 0.f ? 0.f : o[i][3] * f) + g * v[i].w;
      }
      from = upto;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (row0 + i >= rows) return;
    const float inv = L[i] != 0.f ? 1.f / L[i] : 0.f;
    float v[4] = {o[i][0] * inv, o[i][1] * inv, o[i][2] * inv, o[i][3] * inv};
    if (L[i] == 0.f) v[0] = v[1] = v[2] = v[3] = 0.f;
    const int R = rt * a.rows_cap + row0 + i;
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.t.out) +
                              ((int64_t)(seq_begin(a.t, b) + R / a.G) * a.t.nq + h * a.G + R % a.G) * AD + c) =
        f32_to_bf16x4(v);
  }
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

}  // namespace

// Rows per CTA by the largest tree: the kernel for few rows up to 64.  One CTA per SM (shared memory allows one).
TreeAttnPlan tree_attn_plan(int max_nodes, int nq, int nkv, int num_sms) {
  TreeAttnPlan p;
  const int rows = max_nodes * (nq / nkv);
  p.rows_cap = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
  p.chunks = num_sms;
  p.ws_floats = 2LL * p.chunks * p.rows_cap * (AD + 2) + p.chunks * (int64_t)(sizeof(Spot) / sizeof(float));
  return p;
}

namespace {
constexpr int SMEM_MOST = 232448;  // 227 KB

template <typename K>
cudaError_t launch_main(K kern, int threads, int smem, std::atomic<uint64_t>& done, const CUtensorMap& km,
                        const CUtensorMap& vm, const Args& a, cudaStream_t stream) {
  cudaError_t e = smem_opt_in(done, kern, SMEM_MOST);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, dim3(a.chunks), dim3(threads), smem, stream, km, vm, a);
}

template <bool FP8, int N>
cudaError_t launch_few(const CUtensorMap& km, const CUtensorMap& vm, Args& a, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  // The rest of shared memory: K and V tiles.  e4m3: four of them, and four 8-bit ones - even numbers, so that K and V,
  // which are converted by warps of their own, have slots of their own.
  const int left = SMEM_MOST - Bufs<FP8, N>::bytes(0, 0);
  a.slots = FP8 ? 4 : std::min(left / TILE, 8);
  a.raw_slots = FP8 ? 4 : 0;
  static_assert(Bufs<true, N>::bytes(4, 4) <= SMEM_MOST, "");
  return launch_main(tree_attn_few_kernel<FP8, N>, FP8 ? 512 : 256, Bufs<FP8, N>::bytes(a.slots, a.raw_slots), done, km, vm, a, stream);
}

template <bool FP8>
cudaError_t launch_wide(const CUtensorMap& km, const CUtensorMap& vm, Args& a, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  const int qt = a.rows_cap / 128;
  static_assert(smem_bytes(2, FP8 ? 4 : 5, FP8 ? 2 : 0) <= SMEM_MOST && smem_bytes(1, FP8 ? 4 : 6, FP8 ? 4 : 0) <= SMEM_MOST, "");
  a.slots = FP8 ? 4 : 7 - qt;
  a.raw_slots = FP8 ? (qt == 1 ? 4 : 2) : 0;
  return launch_main(tree_attn_kernel<FP8>, FP8 ? 512 : 384, smem_bytes(qt, a.slots, a.raw_slots), done, km, vm, a, stream);
}

template <bool FP8>
cudaError_t launch_rows(const CUtensorMap& km, const CUtensorMap& vm, Args& a, cudaStream_t stream) {
  switch (a.rows_cap) {
    case 16: return launch_few<FP8, 16>(km, vm, a, stream);
    case 32: return launch_few<FP8, 32>(km, vm, a, stream);
    case 64: return launch_few<FP8, 64>(km, vm, a, stream);
    default: return launch_wide<FP8>(km, vm, a, stream);
  }
}
}  // namespace

cudaError_t launch_tree_attention(const TreeAttn& t, const TreeAttnPlan& p, cudaStream_t stream) {
  const int64_t rows = (int64_t)t.num_blocks * t.nkv * t.block_size;
  if (t.num_seqs <= 0 || t.nkv <= 0 || t.nq % t.nkv || t.block_size < 16 || (t.block_size & (t.block_size - 1)) ||
      t.max_nodes < 1 || t.max_nodes > TREE_MAX_NODES || rows >= (int64_t)INT32_MAX - 256)
    return cudaErrorInvalidValue;
  Args a;
  a.t = t;
  a.G = t.nq / t.nkv;
  a.chunks = p.chunks;
  a.rows_cap = p.rows_cap;
  a.slots = a.raw_slots = 0;
  a.bs_shift = __builtin_ctz((unsigned)t.block_size);
  a.box_rows = t.block_size < KT ? t.block_size : KT;
  a.oob_row = (int)rows;
  a.q16 = t.q_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(t.q) & 15) == 0;
  a.scale_log2 = t.softmax_scale * LOG2E;
  a.error = device_error_word();
  if (!a.error) return cudaErrorMemoryAllocation;
  CUtensorMap km, vm;
  if (!pool_map(&km, t.k_cache, rows, t.kv_fp8, a.box_rows) || !pool_map(&vm, t.v_cache, rows, t.kv_fp8, a.box_rows))
    return cudaErrorInvalidValue;
  cudaError_t e = t.kv_fp8 ? launch_rows<true>(km, vm, a, stream) : launch_rows<false>(km, vm, a, stream);
  if (e != cudaSuccess) return e;
  return launch_pdl(tree_join_kernel, dim3(a.chunks, a.rows_cap / JOIN_ROWS), dim3(128), 0, stream, a);
}

cudaError_t launch_tree_wait_check(uint64_t budget_ns, cudaStream_t stream) {
  int* word = device_error_word();
  if (!word) return cudaErrorMemoryAllocation;
  tree_wait_check_kernel<<<1, 32, 0, stream>>>(word, std::min<uint64_t>(budget_ns, tc::WAIT_BUDGET_NS));
  return cudaGetLastError();
}

}  // namespace nvb
