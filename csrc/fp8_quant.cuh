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

// Maximum over the 16 lanes of a half-warp (all 32 lanes call it).
__device__ __forceinline__ uint32_t half_warp_umax(uint32_t v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(FULL_MASK, v, o));
  return v;
}

// 8 values as 8 bytes.
__device__ __forceinline__ uint2 f32x8_to_e4m3(const float* v, float inv) {
  float t[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = v[j] * inv;
  return make_uint2(f32x4_to_e4m3(t), f32x4_to_e4m3(t + 4));
}

}  // namespace nvb
