// Host interface of the fp8 (e4m3) layer kernels: quantisation, norm and matrix products with
// block scales (raw pointers, no torch types).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace nvb {

constexpr int FP8_GROUP = 128;  // channels of one activation scale; side of one weight scale's block

// q[T, K] (e4m3) and s (one fp32 scale per token and 128 channels, s[g * lds + t]) of x[T, K] (bf16,
// row stride ldx).  K % 16 == 0, ldx % 8 == 0, 16-byte aligned x, 8-byte aligned q.
cudaError_t launch_quant_fp8(const void* x, int64_t ldx, void* q, float* s, int64_t lds, int T, int K,
                             cudaStream_t stream);

// r = bf16(x + residual) (written back to `residual`), or x where residual is null;
// (q, s) = quantised rmsnorm(r) * w.  K % 16 == 0, K <= 16384.
cudaError_t launch_add_rmsnorm_fp8(const void* x, int64_t ldx, void* residual, const void* w, void* q, float* s,
                                   int64_t lds, int T, int K, float eps, cudaStream_t stream);

// Y[T, N] = sum over 128-blocks b of k of xs[b * ldxs + t] ws[(n / 128) * ldws + b] sum_k xq wq.
struct Fp8Gemm {
  const void* xq;    // e4m3 [T, K], row stride ldx (bytes, a multiple of 16), 16-byte aligned
  const float* xs;   // [K / 128][T], row stride ldxs (a multiple of 4), 16-byte aligned
  const void* wq;    // e4m3 [N, K], row stride ldw
  const float* ws;   // [N / 128][K / 128], row stride ldws
  int64_t ldx, ldxs, ldw, ldws;
  int T, N, K;
  // act = 0: out is bf16 [T, N], row stride ldo.  act = 1 (SiLU-and-mul): W's rows are alternating
  // blocks of 128 gate rows and the 128 matching up rows; out is e4m3 [T, features], row stride
  // ldo (a multiple of 16), and os (os[g * ldos + t]) its scales.
  int act;
  int features;
  void* out;
  int64_t ldo;
  float* os;
  int64_t ldos;
};

// Which kernel computes a product, and over how many CTAs of a cluster K is split.  np = -1, -2, -3: the
// kernel with the tokens on the MMA's M side (any T), 1 CTA per tile of 256 features (splits 1, 2, 4), 2
// CTAs per tile of 256 (splits 1), 1 CTA per tile of 128 (splits 1, 2, 4; not with act).
// np = 16, 32, 64 (with act 16, 32): the weights on the M side, np >= T tokens, 1 .. 8 splits.
struct Fp8Plan {
  int np = -1, splits = 1;
};
// The plan of a product, from its sizes and the GPU's number of SMs alone (the same in every process and every
// call, whatever the GPU): equal operands give equal bits on every GPU of one model.
Fp8Plan fp8_plan(int T, int N, int K, int act, int num_sms);
cudaError_t gemm_fp8(const Fp8Gemm& g, const Fp8Plan& plan, int num_sms, cudaStream_t stream);

// Error word written by a product that gave up on a bounded wait (0 = none; the last code wins): its output is
// not valid.  One word for all GPUs of the process, in host memory: what a launch wrote is seen once its stream
// has been synchronised.
int gemm_fp8_error_code(int reset);
// Runs a wait that nothing ends, for at most budget_ns (up to 2 s), through the same path: error code 599.
cudaError_t gemm_fp8_wait_check(uint64_t budget_ns, cudaStream_t stream);

}  // namespace nvb
