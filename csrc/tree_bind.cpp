// Python bindings of the kernels for trees of drafted tokens.  Each call checks its arguments, allocates its outputs
// and, where it has one, its workspace (from the caching allocator, so that calls on other streams and replays of
// other graphs have their own), and launches on the current stream of the inputs' device.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "device_error.h"
#include "tree.h"

namespace {

using Opt = c10::optional<at::Tensor>;

void ok(cudaError_t e, const char* what) { TORCH_CHECK(e == cudaSuccess, what, " failed: ", cudaGetErrorString(e)); }

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// Straight from the caching allocator: the smallest calls are bound by the host.
at::Tensor new_cuda(at::IntArrayRef size, at::ScalarType dtype, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(size, dtype, like.device(), c10::nullopt));
}

bool aligned(const at::Tensor& t, uintptr_t a) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & (a - 1)) == 0; }

// n contiguous values of a type on the device of `like`
void check_vec(const at::Tensor& t, int64_t n, at::ScalarType dtype, const at::Tensor& like, const char* op,
               const char* name) {
  TORCH_CHECK(t.device() == like.device(), op, ": ", name, " must be on the device of the other operands");
  TORCH_CHECK(t.scalar_type() == dtype && t.dim() == 1 && t.size(0) == n && (n <= 1 || t.stride(0) == 1), op, ": ", name,
              " must be ", n, " contiguous values of ", at::toString(dtype), ", got ", t.sizes(), " of ",
              t.scalar_type());
}

// The device is checked last: every other refusal then also holds for CPU tensors.
void check_cuda(const at::Tensor& x, const char* op) {
  TORCH_CHECK(x.is_cuda(), op, ": the operands must be CUDA tensors");
}

int64_t check_batch(const at::Tensor& cu_q, int64_t num_seqs, int64_t max_nodes, const at::Tensor& like, const char* op) {
  TORCH_CHECK(num_seqs >= 0 && num_seqs <= 65535, op, ": up to 65535 sequences, got ", num_seqs);
  TORCH_CHECK(max_nodes >= 1 && max_nodes <= nvb::TREE_MAX_NODES, op, ": trees have 1 to ", nvb::TREE_MAX_NODES,
              " nodes, got max_seqlen_q = ", max_nodes);
  TORCH_CHECK(cu_q.dim() == 1 && cu_q.size(0) >= num_seqs + 1, op, ": cu_seqlens_q must hold ", num_seqs + 1, " values");
  check_vec(cu_q, cu_q.size(0), at::kInt, like, op, "cu_seqlens_q");
  return (max_nodes + 63) / 64;
}

void check_tables(const at::Tensor& bt, const at::Tensor& ctx_lens, int64_t num_seqs, const at::Tensor& like,
                  const char* op) {
  TORCH_CHECK(ctx_lens.dim() == 1 && ctx_lens.size(0) >= num_seqs, op, ": context_lens must hold ", num_seqs, " values");
  check_vec(ctx_lens, ctx_lens.size(0), at::kInt, like, op, "context_lens");
  TORCH_CHECK(bt.device() == like.device() && bt.scalar_type() == at::kInt && bt.dim() == 2 && bt.size(0) >= num_seqs &&
                  (bt.size(1) <= 1 || bt.stride(1) == 1),
              op, ": block_tables must be int32 [", num_seqs, ", blocks] with unit inner stride");
}

std::tuple<at::Tensor, at::Tensor> tree_mask(const at::Tensor& parents, const at::Tensor& cu_q, int64_t num_seqs,
                                             int64_t max_nodes) {
  const char* op = "tree_mask";
  const int64_t words = check_batch(cu_q, num_seqs, max_nodes, parents, op);
  check_vec(parents, parents.numel(), at::kInt, parents, op, "parents");
  const int64_t T = parents.size(0);
  TORCH_CHECK(T < (1LL << 31) - 65536, op, ": too large");
  check_cuda(parents, op);
  at::cuda::CUDAGuard g(parents.device());
  at::Tensor mask = new_cuda({T, words}, at::kLong, parents), depth = new_cuda({T}, at::kInt, parents);
  if (T == 0) return {mask, depth};
  if (num_seqs == 0) return {mask.zero_(), depth.zero_()};
  ok(nvb::launch_tree_mask(parents.data_ptr<int>(), cu_q.data_ptr<int>(), (int)num_seqs, (int)T, (int)max_nodes,
                           mask.data_ptr<int64_t>(), (int)words, depth.data_ptr<int>(), stream()),
     op);
  return {mask, depth};
}

at::Tensor tree_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                          const Opt& k_scale, const Opt& v_scale, const at::Tensor& mask, const at::Tensor& block_tables,
                          const at::Tensor& cu_q, const at::Tensor& ctx_lens, int64_t num_seqs, int64_t max_nodes,
                          double scale) {
  const char* op = "attention_tree";
  TORCH_CHECK(q.scalar_type() == at::kBFloat16, op, ": q must be bfloat16");
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes() && k_cache.is_contiguous() &&
                  v_cache.is_contiguous() && k_cache.scalar_type() == v_cache.scalar_type(),
              op, ": the caches must be contiguous [blocks, KV heads, block size, head dim] of one type");
  const bool fp8 = k_cache.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(fp8 || k_cache.scalar_type() == at::kBFloat16, op, ": the cache must be bfloat16 or float8_e4m3fn");
  const int64_t NB = k_cache.size(0), nkv = k_cache.size(1), bs = k_cache.size(2), D = k_cache.size(3);
  TORCH_CHECK(D == 128, op, ": the head dim must be 128, got ", D);
  TORCH_CHECK(bs >= 16 && (bs & (bs - 1)) == 0, op, ": the block size must be a power of two from 16 on, got ", bs);
  TORCH_CHECK(NB > 0 && nkv > 0 && NB * nkv * bs < (1LL << 31) - 1024, op, ": too many rows in the cache");
  TORCH_CHECK((q.dim() == 2 && q.size(1) % D == 0 && (q.stride(1) == 1 || q.size(1) <= 1)) ||
                  (q.dim() == 3 && q.size(2) == D && q.stride(2) == 1 && (q.size(1) <= 1 || q.stride(1) == D)),
              op, ": q must be [tokens, heads * 128] or [tokens, heads, 128], its heads contiguous");
  const int64_t T = q.size(0), nq = q.dim() == 2 ? q.size(1) / D : q.size(1);
  TORCH_CHECK(nq > 0 && nq % nkv == 0, op, ": ", nkv, " KV heads do not divide ", nq, " query heads");
  TORCH_CHECK(nq <= 65536 && T < (1LL << 31) - 65536, op, ": too large");
  const int64_t ldq = T > 1 ? q.stride(0) : nq * D;
  TORCH_CHECK(ldq % 2 == 0 && aligned(q, 4), op, ": q's rows must be 4-byte aligned");
  const int64_t words = check_batch(cu_q, num_seqs, max_nodes, q, op);
  check_tables(block_tables, ctx_lens, num_seqs, q, op);
  TORCH_CHECK(mask.device() == q.device() && mask.scalar_type() == at::kLong && mask.dim() == 2 && mask.size(0) == T &&
                  mask.size(1) >= words && (mask.size(1) <= 1 || mask.stride(1) == 1),
              op, ": mask must be int64 [", T, ", ", words, " words or more] with unit inner stride, got ", mask.sizes());
  TORCH_CHECK(k_cache.device() == q.device() && v_cache.device() == q.device(), op, ": all operands must be on one device");
  TORCH_CHECK(aligned(k_cache, 16) && aligned(v_cache, 16), op, ": the caches must be 16-byte aligned");
  if (fp8) {
    TORCH_CHECK(k_scale.has_value() && v_scale.has_value(), op, ": an fp8 cache needs its scales");
    for (const at::Tensor* s : {&*k_scale, &*v_scale})
      TORCH_CHECK(s->device() == q.device() && s->scalar_type() == at::kFloat && s->is_contiguous() && s->dim() == 2 &&
                      s->size(0) == NB && s->size(1) == nkv,
                  op, ": scales must be contiguous float32 [", NB, ", ", nkv, "], got ", s->sizes());
  }
  check_cuda(q, op);
  at::cuda::CUDAGuard g(q.device());
  at::Tensor out = new_cuda({T, nq * D}, at::kBFloat16, q);
  if (T == 0 || num_seqs == 0) return out;
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const nvb::TreeAttnPlan p = nvb::tree_attn_plan((int)max_nodes, (int)nq, (int)nkv, sms);
  at::Tensor ws = new_cuda({p.ws_floats}, at::kFloat, q);
  nvb::TreeAttn a{};
  a.q = q.data_ptr();
  a.q_stride = ldq;
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.k_scale = fp8 ? k_scale->data_ptr<float>() : nullptr;
  a.v_scale = fp8 ? v_scale->data_ptr<float>() : nullptr;
  a.mask = mask.data_ptr<int64_t>();
  a.mask_stride = T > 1 ? mask.stride(0) : mask.size(1);
  a.words = (int)mask.size(1);
  a.block_tables = block_tables.data_ptr<int>();
  a.bt_stride = num_seqs > 1 ? block_tables.stride(0) : block_tables.size(1);
  a.W = (int)block_tables.size(1);
  a.cu_q = cu_q.data_ptr<int>();
  a.ctx_lens = ctx_lens.data_ptr<int>();
  a.out = out.data_ptr();
  a.ws = ws.data_ptr<float>();
  a.T = (int)T;
  a.nq = (int)nq;
  a.nkv = (int)nkv;
  a.block_size = (int)bs;
  a.num_blocks = (int)NB;
  a.num_seqs = (int)num_seqs;
  a.max_nodes = (int)max_nodes;
  a.kv_fp8 = fp8;
  a.softmax_scale = (float)scale;
  ok(nvb::launch_tree_attention(a, p, stream()), op);
  return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> tree_verify(const at::Tensor& logits, const at::Tensor& tokens,
                                                           const at::Tensor& parents, const at::Tensor& cu_q,
                                                           const at::Tensor& temps, const at::Tensor& u,
                                                           const at::Tensor& u_draw, const Opt& draft, int64_t num_seqs,
                                                           int64_t max_nodes) {
  const char* op = "verify_tree";
  const bool bf16 = logits.scalar_type() == at::kBFloat16;
  TORCH_CHECK(bf16 || logits.scalar_type() == at::kFloat, op, ": logits must be bfloat16 or float32");
  TORCH_CHECK(logits.dim() == 2 && logits.size(1) > 0 && (logits.stride(1) == 1 || logits.size(1) == 1), op,
              ": logits must be [tokens, vocabulary] with unit inner stride");
  const int64_t T = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V < (1 << 22) && T < (1LL << 31) - 65536, op, ": vocabularies of up to 4194303 tokens, got ", V);
  check_batch(cu_q, num_seqs, max_nodes, logits, op);
  check_vec(tokens, T, at::kInt, logits, op, "tokens");
  check_vec(parents, T, at::kInt, logits, op, "parents");
  check_vec(u, T, at::kFloat, logits, op, "uniforms");
  check_vec(temps, num_seqs, at::kFloat, logits, op, "temperatures");
  check_vec(u_draw, num_seqs, at::kFloat, logits, op, "draw_uniforms");
  if (draft.has_value())
    TORCH_CHECK(draft->device() == logits.device() && draft->scalar_type() == at::kFloat && draft->sizes() == logits.sizes() &&
                    (draft->stride(1) == 1 || V == 1),
                op, ": draft_probs must be float32 of the logits' shape with unit inner stride");
  check_cuda(logits, op);
  at::cuda::CUDAGuard g(logits.device());
  at::Tensor path = new_cuda({num_seqs, max_nodes}, at::kInt, logits), length = new_cuda({num_seqs}, at::kInt, logits),
             next = new_cuda({num_seqs}, at::kInt, logits);
  if (num_seqs == 0) return {path, length, next};
  nvb::TreeVerify a{};
  a.logits = logits.data_ptr();
  a.logits_bf16 = bf16;
  a.ld = T > 1 ? logits.stride(0) : V;
  if (draft.has_value()) {
    a.draft = draft->data_ptr<float>();
    a.ld_draft = T > 1 ? draft->stride(0) : V;
  }
  a.tokens = tokens.data_ptr<int>();
  a.parents = parents.data_ptr<int>();
  a.cu_q = cu_q.data_ptr<int>();
  a.temps = temps.data_ptr<float>();
  a.u = u.data_ptr<float>();
  a.u_draw = u_draw.data_ptr<float>();
  a.path = path.data_ptr<int>();
  a.length = length.data_ptr<int>();
  a.next_token = next.data_ptr<int>();
  a.num_seqs = (int)num_seqs;
  a.max_nodes = (int)max_nodes;
  a.V = (int)V;
  a.T = (int)T;
  ok(nvb::launch_tree_verify(a, stream()), op);
  return {path, length, next};
}

void tree_commit(const at::Tensor& kv, const at::Tensor& path, const at::Tensor& length, const at::Tensor& block_tables,
                 const at::Tensor& cu_q, const at::Tensor& ctx_lens, const Opt& scale, int64_t num_seqs,
                 int64_t max_nodes) {
  const char* op = "commit_tree";
  const bool fp8 = kv.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(fp8 || kv.scalar_type() == at::kBFloat16, op, ": the cache must be bfloat16 or float8_e4m3fn");
  TORCH_CHECK(kv.dim() == 6 && kv.size(0) == 2, op,
              ": the cache must be [2, layers, blocks, KV heads, block size, head dim], got ", kv.sizes());
  const int64_t L = kv.size(1), NB = kv.size(2), nkv = kv.size(3), bs = kv.size(4), D = kv.size(5);
  TORCH_CHECK(D == 128, op, ": the head dim must be 128, got ", D);
  TORCH_CHECK(bs > 0 && bs < (1 << 24) && nkv > 0 && NB > 0 && NB < (1LL << 31) && L * nkv < (1LL << 24), op, ": too large");
  TORCH_CHECK(kv.stride(5) == 1 && kv.stride(4) == D && (nkv == 1 || kv.stride(3) == bs * D) &&
                  (NB == 1 || kv.stride(2) == nkv * bs * D),
              op, ": a layer's blocks must be contiguous");
  const int64_t elt = fp8 ? 1 : 2;
  TORCH_CHECK(aligned(kv, 16) && kv.stride(0) * elt % 16 == 0 && kv.stride(1) * elt % 16 == 0, op,
              ": the cache must be 16-byte aligned");
  check_batch(cu_q, num_seqs, max_nodes, kv, op);
  check_tables(block_tables, ctx_lens, num_seqs, kv, op);
  check_vec(length, num_seqs, at::kInt, kv, op, "lengths");
  TORCH_CHECK(path.device() == kv.device() && path.scalar_type() == at::kInt && path.dim() == 2 &&
                  path.size(0) == num_seqs && (path.size(1) <= 1 || path.stride(1) == 1),
              op, ": path must be int32 [", num_seqs, ", nodes] with unit inner stride");
  TORCH_CHECK(!fp8 || scale.has_value(), op, ": an fp8 cache needs its scales");
  if (fp8)
    TORCH_CHECK(scale->device() == kv.device() && scale->scalar_type() == at::kFloat && scale->dim() == 4 &&
                    scale->size(0) == 2 && scale->size(1) == L && scale->size(2) == NB && scale->size(3) == nkv &&
                    (nkv == 1 || scale->stride(3) == 1) && (NB == 1 || scale->stride(2) == nkv),
                op, ": scales must be float32 [2, ", L, ", ", NB, ", ", nkv, "], a layer's contiguous");
  check_cuda(kv, op);
  if (num_seqs == 0 || L == 0 || path.size(1) == 0) return;
  at::cuda::CUDAGuard g(kv.device());
  nvb::TreeCommit a{};
  a.kv = kv.data_ptr();
  a.stride_kv = kv.stride(0) * elt;
  a.stride_layer = kv.stride(1) * elt;
  if (fp8) {
    a.scale = scale->data_ptr<float>();
    a.scale_stride_kv = scale->stride(0);
    a.scale_stride_layer = scale->stride(1);
  }
  a.path = path.data_ptr<int>();
  a.path_stride = num_seqs > 1 ? path.stride(0) : path.size(1);
  a.length = length.data_ptr<int>();
  a.block_tables = block_tables.data_ptr<int>();
  a.bt_stride = num_seqs > 1 ? block_tables.stride(0) : block_tables.size(1);
  a.W = (int)block_tables.size(1);
  a.cu_q = cu_q.data_ptr<int>();
  a.ctx_lens = ctx_lens.data_ptr<int>();
  a.layers = (int)L;
  a.num_blocks = (int)NB;
  a.nkv = (int)nkv;
  a.block_size = (int)bs;
  a.num_seqs = (int)num_seqs;
  a.max_nodes = (int)max_nodes;
  a.max_path = (int)path.size(1);
  a.kv_fp8 = fp8;
  ok(nvb::launch_tree_commit(a, stream()), op);
}

int64_t tree_error(bool reset) { return nvb::device_error_code(reset ? 1 : 0); }

void tree_wait_check(int64_t budget_ns) {
  TORCH_CHECK(budget_ns >= 0, "tree_wait_check: the budget must not be negative");
  ok(nvb::launch_tree_wait_check((uint64_t)budget_ns, stream()), "tree_wait_check");
}

}  // namespace

void register_tree(pybind11::module& m) {
  m.def("tree_mask", &tree_mask);
  m.def("tree_attention", &tree_attention);
  m.def("tree_verify", &tree_verify);
  m.def("tree_commit", &tree_commit);
  m.def("tree_error", &tree_error, pybind11::arg("reset") = false);
  m.def("tree_wait_check", &tree_wait_check, pybind11::arg("budget_ns") = 1000000);
}
