// Python bindings of the fp8 layer kernels.  Each call checks its arguments, allocates its outputs and
// launches on the current stream of the inputs' device; none keeps a workspace.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "device_error.h"
#include "fp8.h"

namespace {

using Pair = std::tuple<at::Tensor, at::Tensor>;

void ok(cudaError_t e, const char* what) { TORCH_CHECK(e == cudaSuccess, what, " failed: ", cudaGetErrorString(e)); }

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

int64_t groups(int64_t k) { return (k + nvb::FP8_GROUP - 1) / nvb::FP8_GROUP; }

bool aligned(const at::Tensor& t, uintptr_t a) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & (a - 1)) == 0; }

// Outputs come straight from the caching allocator: the smallest calls are bound by the host, and the
// dispatcher's way there costs as much as the launch.
at::Tensor new_cuda(at::IntArrayRef size, at::ScalarType dtype, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(size, dtype, like.device(), c10::nullopt));
}

// e4m3 [t, k] and its scales [t, k / 128], token-contiguous (strides (1, t rounded up to 4)).
Pair new_pair(const at::Tensor& like, int64_t t, int64_t k) {
  const int64_t ld = std::max<int64_t>((t + 3) / 4 * 4, 4);
  return {new_cuda({t, k}, at::kFloat8_e4m3fn, like),
          at::Tensor(at::detail::empty_strided_cuda({t, groups(k)}, {1, ld}, at::kFloat, like.device()))};
}

// The device is checked last: every other refusal then also holds for CPU tensors.
void check_cuda(const at::Tensor& x, const char* what) {
  TORCH_CHECK(x.is_cuda(), what, ": the operands must be CUDA tensors");
}

void check_rows(const at::Tensor& x, const char* what) {
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, what, ": x must be bfloat16");
  TORCH_CHECK(x.dim() == 2 && (x.stride(1) == 1 || x.size(1) == 1), what, ": x must be [rows, K] with unit inner stride");
  TORCH_CHECK(x.size(1) > 0 && x.size(1) % 16 == 0, what, ": K must be a positive multiple of 16, got ", x.size(1));
  TORCH_CHECK(x.size(0) < (1LL << 31) - 65536 && x.size(1) < (1LL << 31) - 65536, what, ": too large");
  TORCH_CHECK(x.size(0) <= 1 || (x.stride(0) % 8 == 0 && x.stride(0) >= x.size(1)), what,
              ": x's row stride must be a multiple of 8 and at least K");
  TORCH_CHECK(aligned(x, 16), what, ": x must be 16-byte aligned");
}

int64_t row_stride(const at::Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

// Whether a row of x, [T, K] bf16 with any row stride, shares an element with the `n` bf16 values at `other`.
bool rows_meet(const at::Tensor& x, const at::Tensor& other) {
  const int64_t T = x.size(0), K = x.size(1), n = other.numel(), ld = row_stride(x);
  if (T == 0 || n == 0) return false;
  const int64_t d = (static_cast<const char*>(other.data_ptr()) - static_cast<const char*>(x.data_ptr())) / 2;
  const int64_t i = d < K ? 0 : (d - K) / ld + 1;  // the first row that ends behind other's beginning
  return i < T && i * ld < d + n;
}

Pair quant_fp8(const at::Tensor& x) {
  check_rows(x, "quant_fp8");
  check_cuda(x, "quant_fp8");
  const int64_t T = x.size(0), K = x.size(1);
  at::cuda::CUDAGuard g(x.device());
  auto [q, s] = new_pair(x, T, K);
  ok(nvb::launch_quant_fp8(x.data_ptr(), row_stride(x), q.data_ptr(), s.data_ptr<float>(), s.stride(1), (int)T, (int)K,
                           stream()),
     "quant_fp8");
  return {q, s};
}

Pair add_rmsnorm_fp8(const at::Tensor& x, const c10::optional<at::Tensor>& residual, const at::Tensor& w, double eps) {
  check_rows(x, "add_rmsnorm_fp8");
  const int64_t T = x.size(0), K = x.size(1);
  TORCH_CHECK(K <= 16384, "add_rmsnorm_fp8: K must be at most 16384, got ", K);
  TORCH_CHECK(w.device() == x.device() && w.scalar_type() == at::kBFloat16 && w.is_contiguous() && w.numel() == K &&
                  aligned(w, 16),
              "add_rmsnorm_fp8: w must be ", K, " contiguous bfloat16 values on x's device");
  void* r = nullptr;
  if (residual.has_value()) {
    TORCH_CHECK(residual->device() == x.device() && residual->scalar_type() == at::kBFloat16 &&
                    residual->sizes() == x.sizes() && residual->is_contiguous() && aligned(*residual, 16),
                "add_rmsnorm_fp8: the residual must be contiguous bfloat16 of x's shape on x's device");
    // rows are read and written by CTAs of their own, in any order
    TORCH_CHECK(!rows_meet(*residual, w) && (!rows_meet(x, *residual) ||
                                           (x.data_ptr() == residual->data_ptr() && row_stride(x) == K)),
                "add_rmsnorm_fp8: x and the residual must be the same memory or have none in common, and w none of the "
                "residual's");
    r = residual->data_ptr();
  }
  check_cuda(x, "add_rmsnorm_fp8");
  at::cuda::CUDAGuard g(x.device());
  auto [q, s] = new_pair(x, T, K);
  ok(nvb::launch_add_rmsnorm_fp8(x.data_ptr(), row_stride(x), r, w.data_ptr(), q.data_ptr(), s.data_ptr<float>(),
                                 s.stride(1), (int)T, (int)K, (float)eps, stream()),
     "add_rmsnorm_fp8");
  return {q, s};
}

nvb::Fp8Gemm gemm_args(const at::Tensor& xq, const at::Tensor& xs, const at::Tensor& wq, const at::Tensor& ws,
                       const char* what) {
  TORCH_CHECK(xs.device() == xq.device() && wq.device() == xq.device() && ws.device() == xq.device(),
              what, ": all operands must be on one device");
  TORCH_CHECK(xq.scalar_type() == at::kFloat8_e4m3fn && wq.scalar_type() == at::kFloat8_e4m3fn, what,
              ": x and w must be float8_e4m3fn");
  TORCH_CHECK(xs.scalar_type() == at::kFloat && ws.scalar_type() == at::kFloat, what, ": scales must be float32");
  TORCH_CHECK(xq.dim() == 2 && wq.dim() == 2 && xs.dim() == 2 && ws.dim() == 2, what, ": 2-D tensors required");
  const int64_t T = xq.size(0), K = xq.size(1), N = wq.size(0);
  TORCH_CHECK(K > 0 && K % 16 == 0 && wq.size(1) == K, what, ": x [T, K] and w [N, K] with K a multiple of 16, got ",
              xq.sizes(), " and ", wq.sizes());
  TORCH_CHECK(T < (1LL << 31) - 65536 && N < (1LL << 31) - 65536 && K < (1LL << 31) - 65536, what, ": too large");
  TORCH_CHECK(xq.stride(1) == 1 && wq.stride(1) == 1 && (T <= 1 || (xq.stride(0) % 16 == 0 && xq.stride(0) >= K)) &&
                  (N <= 1 || (wq.stride(0) % 16 == 0 && wq.stride(0) >= K)) && aligned(xq, 16) && aligned(wq, 16),
              what, ": x and w need unit inner strides, row strides that are multiples of 16 and 16-byte alignment");
  TORCH_CHECK(xs.size(0) == T && xs.size(1) == groups(K), what, ": x's scales must be [T, ceil(K / 128)], got ",
              xs.sizes());
  TORCH_CHECK((T <= 1 || xs.stride(0) == 1) &&
                  (xs.size(1) <= 1 || (xs.stride(1) % 4 == 0 && xs.stride(1) >= T)) && aligned(xs, 16),
              what, ": x's scales must be token-contiguous (strides (1, a multiple of 4)) and 16-byte aligned, as "
              "quant_fp8 returns them");
  TORCH_CHECK(ws.size(0) == groups(N) && ws.size(1) == groups(K) && (ws.size(1) <= 1 || ws.stride(1) == 1), what,
              ": w's scales must be [ceil(N / 128), ceil(K / 128)] with unit inner stride, got ", ws.sizes());
  nvb::Fp8Gemm a{};
  a.xq = xq.data_ptr();
  a.xs = xs.data_ptr<float>();
  a.wq = wq.data_ptr();
  a.ws = ws.data_ptr<float>();
  a.ldx = row_stride(xq);
  a.ldxs = xs.size(1) > 1 ? xs.stride(1) : (T + 3) / 4 * 4;
  a.ldw = row_stride(wq);
  a.ldws = ws.size(0) > 1 ? ws.stride(0) : ws.size(1);
  a.T = (int)T;
  a.N = (int)N;
  a.K = (int)K;
  return a;
}

// plan: empty (chosen from the sizes) or (np, splits), see Fp8Plan.
nvb::Fp8Plan plan_of(const nvb::Fp8Gemm& a, const std::vector<int64_t>& plan, int num_sms) {
  if (plan.empty()) return nvb::fp8_plan(a.T, a.N, a.K, a.act, num_sms);
  TORCH_CHECK(plan.size() == 2 && plan[0] >= -3 && plan[0] <= 64 && plan[1] >= 1 && plan[1] <= 8,
              "plan: (np, splits) with np from -3 to 64 and splits from 1 to 8");
  nvb::Fp8Plan p;
  p.np = (int)plan[0];
  p.splits = (int)plan[1];
  return p;
}

std::vector<int64_t> fp8_plan(int64_t T, int64_t N, int64_t K, int64_t act, int64_t num_sms) {
  const int64_t most = (1LL << 31) - 65536;
  TORCH_CHECK(T >= 0 && T < most && N >= 0 && N < most && K > 0 && K < most && (act == 0 || act == 1) && num_sms > 0 &&
                  num_sms < 4096,
              "fp8_plan: sizes from 0 (K: 1) to below 2^31 - 65536, act 0 or 1, and a GPU's number of SMs");
  const auto p = nvb::fp8_plan((int)T, (int)N, (int)K, (int)act, (int)num_sms);
  return {p.np, p.splits};
}

int sms() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

at::Tensor linear_fp8(const at::Tensor& xq, const at::Tensor& xs, const at::Tensor& wq, const at::Tensor& ws,
                      const c10::optional<at::Tensor>& out, const std::vector<int64_t>& plan) {
  nvb::Fp8Gemm a = gemm_args(xq, xs, wq, ws, "linear_fp8");
  if (out.has_value()) {
    const at::Tensor& y = *out;
    TORCH_CHECK(y.device() == xq.device() && y.scalar_type() == at::kBFloat16 && y.dim() == 2 && y.size(0) == a.T &&
                    y.size(1) == a.N && (a.N <= 1 || y.stride(1) == 1) && (a.T <= 1 || y.stride(0) >= a.N),
                "linear_fp8: out must be bfloat16 [", a.T, ", ", a.N, "] with unit inner stride on x's device");
  }
  check_cuda(xq, "linear_fp8");
  at::cuda::CUDAGuard g(xq.device());
  at::Tensor y = out.has_value() ? *out : new_cuda({a.T, a.N}, at::kBFloat16, xq);
  a.out = y.data_ptr();
  a.ldo = row_stride(y);
  ok(nvb::gemm_fp8(a, plan_of(a, plan, sms()), sms(), stream()), "linear_fp8");
  return y;
}

Pair linear_silu_fp8(const at::Tensor& xq, const at::Tensor& xs, const at::Tensor& wq, const at::Tensor& ws,
                     int64_t features, const std::vector<int64_t>& plan) {
  nvb::Fp8Gemm a = gemm_args(xq, xs, wq, ws, "linear_silu_fp8");
  TORCH_CHECK(features > 0 && features % 16 == 0 && wq.size(0) == 2 * nvb::FP8_GROUP * groups(features),
              "linear_silu_fp8: features must be a positive multiple of 16 and w must hold 2 x ceil(features / 128) "
              "blocks of 128 rows, got ", features, " features and ", wq.size(0), " rows");
  check_cuda(xq, "linear_silu_fp8");
  at::cuda::CUDAGuard g(xq.device());
  auto [q, s] = new_pair(xq, a.T, features);
  a.act = 1;
  a.features = (int)features;
  a.out = q.data_ptr();
  a.ldo = features;
  a.os = s.data_ptr<float>();
  a.ldos = s.stride(1);
  ok(nvb::gemm_fp8(a, plan_of(a, plan, sms()), sms(), stream()), "linear_silu_fp8");
  return {q, s};
}

int64_t fp8_error(bool reset) { return nvb::device_error_code(reset ? 1 : 0); }

void fp8_wait_check(int64_t budget_ns) {
  TORCH_CHECK(budget_ns >= 0, "fp8_wait_check: the budget must not be negative");
  ok(nvb::gemm_fp8_wait_check((uint64_t)budget_ns, stream()), "fp8_wait_check");
}

}  // namespace

void register_fp8(pybind11::module& m) {
  m.def("quant_fp8", &quant_fp8);
  m.def("add_rmsnorm_fp8", &add_rmsnorm_fp8);
  m.def("linear_fp8", &linear_fp8, pybind11::arg("xq"), pybind11::arg("xs"), pybind11::arg("wq"), pybind11::arg("ws"),
        pybind11::arg("out") = c10::nullopt, pybind11::arg("plan") = std::vector<int64_t>{});
  m.def("linear_silu_fp8", &linear_silu_fp8, pybind11::arg("xq"), pybind11::arg("xs"), pybind11::arg("wq"),
        pybind11::arg("ws"), pybind11::arg("features"), pybind11::arg("plan") = std::vector<int64_t>{});
  m.def("fp8_plan", &fp8_plan);
  m.def("fp8_error", &fp8_error, pybind11::arg("reset") = false);
  m.def("fp8_wait_check", &fp8_wait_check, pybind11::arg("budget_ns") = 1000000);
}
