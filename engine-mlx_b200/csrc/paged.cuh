// paged.cuh — batched operators over a paged K/V cache.
#pragma once
#include "common.cuh"
#include "paged_plan.h"

namespace emx {

// The cache of one layer and a batch over it, as the kernels take them
// (emx_paged_kv / emx_paged_batch with everything checked by the host).
struct PagedArgs {
  bf16* k;  // [n_pages, n_kv, page_size, head_dim]
  bf16* v;
  int n_pages, page_size, n_kv, head_dim;
  int n_seqs, n_rows, max_pages;
  const int* indptr;   // [n_seqs + 1]
  const int* lengths;  // [n_seqs]
  const int* table;    // [n_seqs, max_pages]
  int n_q;
  int* status;
};

struct PagedAppendArgs {
  PagedArgs p;
  const bf16* qkv;     // [n_rows, (n_q + 2 n_kv) * head_dim]
  const bf16* q_norm;  // [head_dim] or null
  const bf16* k_norm;
  float eps;
  double log2_theta;   // 0: no rotation
  int rotate;
  bf16* q_out;         // [n_rows, n_q, head_dim]
};
cudaError_t paged_append_launch(const PagedAppendArgs& a, int num_sms, cudaStream_t st);

struct PagedAttnArgs {
  PagedArgs p;
  const bf16* q;  // [n_rows, n_q, head_dim]
  bf16* out;
  int shared_len;
  const int* shared_pages;
  float scale;
  void* workspace;
};
// Bytes of workspace for a batch of this size (the same whatever its lengths).
size_t paged_attn_workspace(int n_rows, int n_q, int n_kv, int head_dim, int shared_len, int num_sms);
cudaError_t paged_attn_launch(const PagedAttnArgs& a, int num_sms, cudaStream_t st);

struct VerifyArgs {
  const void* target;  // [n_seqs, n_draft + 1, vocab] f32 or bf16
  const void* draft;   // [n_seqs, n_draft, vocab] or null
  int is_bf16;
  const int* tokens;   // [n_seqs, n_draft]
  const int* counts;   // [n_seqs] or null
  const float* uniforms;  // [n_seqs, n_draft + 1]
  int n_seqs, n_draft, vocab;
  int* out;       // [n_seqs, n_draft + 1]
  int* accepted;  // [n_seqs]
  int* status;
};
cudaError_t verify_launch(const VerifyArgs& a, int num_sms, cudaStream_t st);

}  // namespace emx
