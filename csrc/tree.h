// Host-side launch entry points of the kernels for trees of drafted tokens (raw pointers, no torch types).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace nvb {

constexpr int TREE_MAX_NODES = 256;
constexpr int TREE_WORDS = TREE_MAX_NODES / 64;

// mask [T, words], depth [T]; rows behind the last sequence, and nodes from max_nodes on, are zero.
cudaError_t launch_tree_mask(const int* parents, const int* cu_q, int num_seqs, int T, int max_nodes, int64_t* mask,
                             int words, int* depth, cudaStream_t stream);

struct TreeAttn {
  const void* q;  // bf16, row t at q + t * q_stride
  int64_t q_stride;
  const void* k_cache;  // [num_blocks, nkv, block_size, 128] bf16 or e4m3
  const void* v_cache;
  const float* k_scale;  // [num_blocks, nkv] (e4m3)
  const float* v_scale;
  const int64_t* mask;  // [T, words]
  int64_t mask_stride;
  int words;
  const int* block_tables;
  int64_t bt_stride;
  int W;
  const int* cu_q;
  const int* ctx_lens;
  void* out;  // bf16 [T, nq, 128]
  float* ws;  // tree_attn_plan().ws_floats
  int T;  // rows of q, mask and out: cu_q is clamped to them
  int nq, nkv, block_size, num_blocks, num_seqs, max_nodes, kv_fp8;
  float softmax_scale;
};
struct TreeAttnPlan {
  int rows_cap;  // (node, query head) rows per CTA
  int chunks;    // CTAs
  int64_t ws_floats;
};
TreeAttnPlan tree_attn_plan(int max_nodes, int nq, int nkv, int num_sms);
cudaError_t launch_tree_attention(const TreeAttn& a, const TreeAttnPlan& p, cudaStream_t stream);
// Runs a wait that nothing ends, for at most budget_ns (up to 2 s), as attention waits: error code 699.
cudaError_t launch_tree_wait_check(uint64_t budget_ns, cudaStream_t stream);

struct TreeVerify {
  const void* logits;  // [T, V]
  int logits_bf16;
  int64_t ld;
  const float* draft;  // [T, V] or null
  int64_t ld_draft;
  const int* tokens;
  const int* parents;
  const int* cu_q;
  const float* temps;
  const float* u;
  const float* u_draw;
  int* path;  // [B, max_nodes]
  int* length;
  int* next_token;
  int num_seqs, max_nodes, V;
  int T;  // rows of logits: cu_q is clamped to them
};
cudaError_t launch_tree_verify(const TreeVerify& a, cudaStream_t stream);

struct TreeCommit {
  void* kv;  // row (kv, layer, block, head, offset) of 128 values
  int64_t stride_kv, stride_layer;  // in bytes
  float* scale;  // e4m3: (kv, layer, block, head)
  int64_t scale_stride_kv, scale_stride_layer;
  const int* path;
  int64_t path_stride;
  const int* length;
  const int* block_tables;
  int64_t bt_stride;
  int W;
  const int* cu_q;
  const int* ctx_lens;
  int layers, num_blocks, nkv, block_size, num_seqs, max_nodes, max_path, kv_fp8;
};
cudaError_t launch_tree_commit(const TreeCommit& a, cudaStream_t stream);

}  // namespace nvb
