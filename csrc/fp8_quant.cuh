// Quantisation of groups of 128 channels to fp8 e4m3, shared by the norm, quantisation and GEMM
// epilogue kernels:
//   a = max(max |x|, 1e-30),  scale = a / 448,  q = e4m3(x * (448 / a))   (saturating, nearest even)
// so that scale * q is the value q stands for and the group's largest magnitude maps to e4m3's
// largest, 448.  The floor keeps 448 / a finite for a group of zeros.  Maxima are taken over the
// magnitude's bits as integers, which orders NaN above infinity above every finite value: a group
// that holds a NaN or an infinity gets that scale and dequantises to NaN instead of hiding it.
#pragma once
#include "common.cuh"
#include "fp8.h"

namespace nvb {

constexpr float FP8_E4M3_MAX = 448.f;
constexpr float FP8_AMAX_MIN = 1e-30f;

struct Fp8Scale {
  float scale, inv;
};

__device__ __forceinline__ Fp8Scale fp8_scale(uint32_t amax_bits) {
  float a = __uint_as_float(amax_bits);
  if (a < FP8_AMAX_MIN) a = FP8_AMAX_MIN;  // false for NaN, which stays
  return {__fdiv_rn(a, FP8_E4M3_MAX), __fdiv_rn(FP8_E4M3_MAX, a)};
}

// Maxima over the 16 lanes of a half-warp, of G values per lane at once (all 32 lanes call it).  Each
// step halves the values that a lane still holds, until lane l has that of value l / (16 / G); the
// division that follows is then made once per lane instead of once per value.
template <int G>
__device__ __forceinline__ uint32_t half_warp_umax(const uint32_t (&v)[G]) {
  static_assert(G == 1 || G == 2 || G == 4, "values per lane");
  const int l = threadIdx.x & 15;
  uint32_t m[G];
#pragma unroll
  for (int i = 0; i < G; ++i) m[i] = v[i];
  int o = 8;
#pragma unroll
  for (int n = G / 2; n > 0; n >>= 1, o >>= 1) {
    const bool hi = l & o;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const uint32_t send = hi ? m[i] : m[i + n], keep = hi ? m[i + n] : m[i];
      m[i] = max(keep, __shfl_xor_sync(FULL_MASK, send, o));
    }
  }
#pragma unroll
  for (; o > 0; o >>= 1) m[0] = max(m[0], __shfl_xor_sync(FULL_MASK, m[0], o));
  return m[0];
}

// 8 values as 8 bytes.
__device__ __forceinline__ uint2 f32x8_to_e4m3(const float* v, float inv) {
  float t[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = v[j] * inv;
  return make_uint2(f32x4_to_e4m3(t), f32x4_to_e4m3(t + 4));
}

}  // namespace nvb
