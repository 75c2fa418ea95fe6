// bf16 -> e4m3 with one scale per token and 128 channels, alone and behind residual add + RMSNorm.
//
// No counterpart in the reference (its products are all 16-bit); the norm is its RMSNorm
// (nanovllm/layers/RMSNorm.py:11-17) with the 8-bit rounding of the next product's input fused in.
// Both are bound by memory traffic: 3 bytes per value for the quantisation (2 read, 1 written), 7
// for the norm (x and the residual read, the residual and the 8-bit value written).
#include "fp8_quant.cuh"

namespace nvb {
namespace {

constexpr int QROWS = 8;    // rows per CTA: one half-warp each
constexpr int QGROUPS = 4;  // groups per half-warp, all of whose loads are in flight together

// A half-warp holds a group of 128 as 16 lanes x 8 values.  The half-warps of a CTA take consecutive
// tokens of the same groups, so that a group's scales leave as one 32-byte sector (scales are stored
// token-contiguous, the order in which the products read them).  With a reduction and two divisions
// per group in every lane the kernel was bound by its instructions (79% of the issue slots, 33.8 us at
// 16384 x 4096); with the four groups' maxima and divisions spread over the lanes it is bound by
// memory: 31.0 us, 6.5 TB/s.  2 groups per half-warp 35.7 us; 16 rows per CTA, 8 or 16 groups were
// slower as well.
__global__ void __launch_bounds__(QROWS * 16) quant_fp8_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx,
                                                               uint8_t* __restrict__ q, float* __restrict__ s,
                                                               int64_t lds, int T, int K) {
  pdl_wait();     // inputs come from the previous kernel in the stream
  pdl_trigger();  // the next kernel may start its prologue
  const int hw = threadIdx.x >> 4, l = threadIdx.x & 15;
  const int kb = (K + FP8_GROUP - 1) / FP8_GROUP;
  const int64_t t = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * QROWS + hw;
  const int g0 = (int)blockIdx.x * QGROUPS;
  uint4 v[QGROUPS];
#pragma unroll
  for (int i = 0; i < QGROUPS; ++i) {
    const int c = (g0 + i) * FP8_GROUP + l * 8;
    v[i] = make_uint4(0, 0, 0, 0);
    if (t < T && c < K) v[i] = *reinterpret_cast<const uint4*>(x + t * ldx + c);
  }
  uint32_t m[QGROUPS];
#pragma unroll
  for (int i = 0; i < QGROUPS; ++i) {
    // |bf16| as 16-bit integers, two per word
    m[i] = __vmaxu2(__vmaxu2(v[i].x & 0x7fff7fffu, v[i].y & 0x7fff7fffu),
                    __vmaxu2(v[i].z & 0x7fff7fffu, v[i].w & 0x7fff7fffu));
    m[i] = max(m[i] & 0xffff0000u, m[i] << 16);  // as an fp32 magnitude
  }
  constexpr int LPG = 16 / QGROUPS;  // lanes that hold a group's maximum
  const Fp8Scale sc = fp8_scale(half_warp_umax(m));
  if (l % LPG == 0 && t < T && g0 + l / LPG < kb) s[(g0 + l / LPG) * lds + t] = sc.scale;
#pragma unroll
  for (int i = 0; i < QGROUPS; ++i) {
    const float inv = __shfl_sync(FULL_MASK, sc.inv, i * LPG, 16);
    const int c = (g0 + i) * FP8_GROUP + l * 8;
    if (t < T && c < K) {
      float f[8];
      bf16x8_to_f32(v[i], f);
      *reinterpret_cast<uint2*>(q + t * K + c) = f32x8_to_e4m3(f, inv);
    }
  }
}

constexpr int TPR = 128;    // threads per row of the norm

// One CTA of 128 threads per row, 8 values per thread and step; a group of 128 is the 16 lanes of a
// half-warp.  The row is kept as bf16 between the two passes over it (the residual's rounding is exact
// in it): half the registers of fp32, so that enough rows are in flight to cover the latency.
// The 8-bit values are taken from r * f * w, where f is the root's factor without its mantissa: scaling by a
// power of two and the product of two bf16 values are exact in fp32.  The mantissa is the same for the whole
// row and enters the scales alone.  The power of two keeps the products in range whatever the row's
// magnitude: between half of the normalised values and these, so that 448 over a group's largest one is
// finite wherever that lies above the floor.  The squares are summed in fp32, as in the 16-bit norm: rows of a
// root mean square below 1e-19 rest on eps, and rows above 1e19 come out as zeros.
// Measured, inputs out of the cache and launches back to back: 8191 x 5120 48.4 us (6.1 TB/s), 8192 x 8192
// 77.6 us; without the power of two 48.1 and 77.4 us.  Scales of one group at a time 83.8 us (8192 x 8192); 256
// threads per row 54 us, two rows per CTA 51 us, fp32 in between 63 us (8191 x 5120).
template <int NI>
__global__ void __launch_bounds__(TPR) add_rmsnorm_fp8_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx,
                                                              __nv_bfloat16* __restrict__ residual,
                                                                  const __nv_bfloat16* __restrict__ w,
                                                                  uint8_t* __restrict__ q, float* __restrict__ s,
                                                                  int64_t lds, int K, float eps) {
  pdl_wait();     // inputs come from the previous kernel in the stream
  pdl_trigger();  // the next kernel may start its prologue
  const int tid = threadIdx.x, row = blockIdx.x;
  const int nvec = K >> 3;
  const uint4* xr = reinterpret_cast<const uint4*>(x + (int64_t)row * ldx);
  uint4* rr = reinterpret_cast<uint4*>(residual + (int64_t)row * K);
  uint4 v[NI];
  float ss = 0.f;
  if (residual) {
    uint4 b[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = tid + i * TPR;
      v[i] = b[i] = make_uint4(0, 0, 0, 0);
      if (c < nvec) {
        v[i] = xr[c];
        b[i] = rr[c];
      }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = tid + i * TPR;
      // the residual stream stays bf16, as an eager bf16 add keeps it
      float f[8], r[8];
      bf16x8_to_f32(v[i], f);
      bf16x8_to_f32(b[i], r);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] += r[j];
      v[i] = f32_to_bf16x8(f);
      if (c < nvec) rr[c] = v[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = tid + i * TPR;
      v[i] = make_uint4(0, 0, 0, 0);
      if (c < nvec) v[i] = xr[c];
    }
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    float f[8];
    bf16x8_to_f32(v[i], f);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
  }
  ss = warp_sum(ss);
  __shared__ float red[TPR / 32];
  if ((tid & 31) == 0) red[tid >> 5] = ss;
  __syncthreads();
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < TPR / 32; ++i) ss += red[i];
  const uint32_t inv_rms = __float_as_uint(rsqrtf(ss / (float)K + eps));
  const float pow2 = __uint_as_float(inv_rms & 0x7f800000u);  // (infinite for a factor that is not finite)
  const float mant = __uint_as_float((inv_rms & 0x007fffffu) | 0x3f800000u);
  const uint4* wr = reinterpret_cast<const uint4*>(w);
  constexpr int G = NI < 3 ? NI : 4;  // groups per half-warp whose scales are made at once
  constexpr int LPG = 16 / G;
#pragma unroll
  for (int i0 = 0; i0 < NI; i0 += G) {
    uint32_t m[G];
    float o[G][8];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int c = tid + (i0 + g) * TPR;
      m[g] = 0;
      if (i0 + g < NI && c < nvec) {
        float wf[8];
        bf16x8_to_f32(v[i0 + g], o[g]);
        bf16x8_to_f32(wr[c], wf);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          o[g][j] = o[g][j] * pow2 * wf[j];
          m[g] = max(m[g], __float_as_uint(o[g][j]) & 0x7fffffffu);
        }
      }
    }
    const float mr = __uint_as_float(half_warp_umax(m));
    float a = mr * mant, mine = __fdiv_rn(FP8_E4M3_MAX, mr);
    if (a < FP8_AMAX_MIN) {  // false for NaN, which stays
      a = FP8_AMAX_MIN;
      mine = mant * (FP8_E4M3_MAX / FP8_AMAX_MIN);
    }
    const int cs = (tid & ~15) + (i0 + (tid & 15) / LPG) * TPR;  // first vector of this lane's group
    if ((tid & 15) % LPG == 0 && i0 + (tid & 15) / LPG < NI && cs < nvec) 
      s[(int64_t)(cs >> 4) * lds + row] = __fdiv_rn(a, FP8_E4M3_MAX);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int c = tid + (i0 + g) * TPR;
      const float inv = __shfl_sync(FULL_MASK, mine, g * LPG, 16);
      if (i0 + g < NI && c < nvec) *reinterpret_cast<uint2*>(q + (int64_t)row * K + c * 8) = f32x8_to_e4m3(o[g], inv);
    }
  }
}

}  // namespace

cudaError_t launch_quant_fp8(const void* x, int64_t ldx, void* q, float* s, int64_t lds, int T, int K,
                             cudaStream_t stream) {
  if (T == 0) return cudaSuccess;
  const int kb = (K + FP8_GROUP - 1) / FP8_GROUP;
  const int64_t rows = ((int64_t)T + QROWS - 1) / QROWS;  // in CTAs; a grid's y goes to 65535 only
  const int64_t ny = rows < 32768 ? rows : 32768, nz = (rows + ny - 1) / ny;
  const int chunks = (kb + QGROUPS - 1) / QGROUPS;
  if (K % 16 || ldx % 8 || nz > 65535) return cudaErrorInvalidValue;
  return launch_pdl(quant_fp8_kernel, dim3(chunks, (unsigned)ny, (unsigned)nz), dim3(QROWS * 16), 0, stream,
                    static_cast<const __nv_bfloat16*>(x), ldx, static_cast<uint8_t*>(q), s, lds, T, K);
}

cudaError_t launch_add_rmsnorm_fp8(const void* x, int64_t ldx, void* residual, const void* w, void* q, float* s,
                                   int64_t lds, int T, int K, float eps, cudaStream_t stream) {
  if (T == 0) return cudaSuccess;
  const int ni = (K / 8 + TPR - 1) / TPR;
  if (K % 16 || ldx % 8 || ni > 16) return cudaErrorInvalidValue;
  auto go = [&](auto kern) {
    return launch_pdl(kern, dim3(T), dim3(TPR), 0, stream, static_cast<const __nv_bfloat16*>(x), ldx,
                      static_cast<__nv_bfloat16*>(residual), static_cast<const __nv_bfloat16*>(w),
                      static_cast<uint8_t*>(q), s, lds, K, eps);
  };
  if (ni == 1) return go(add_rmsnorm_fp8_kernel<1>);
  if (ni == 2) return go(add_rmsnorm_fp8_kernel<2>);
  if (ni == 3) return go(add_rmsnorm_fp8_kernel<3>);
  if (ni == 4) return go(add_rmsnorm_fp8_kernel<4>);
  if (ni == 5) return go(add_rmsnorm_fp8_kernel<5>);
  if (ni == 6) return go(add_rmsnorm_fp8_kernel<6>);
  if (ni <= 8) return go(add_rmsnorm_fp8_kernel<8>);
  if (ni <= 12) return go(add_rmsnorm_fp8_kernel<12>);
  return go(add_rmsnorm_fp8_kernel<16>);
}

}  // namespace nvb
