// paged_api.cu — C ABI of the batched operators: a paged K/V cache filled and
// attended by a batch of sequences, and drafted tokens verified for it.  Each
// call checks its arguments on the host (the context last, so that a shape is
// refused without a device), enqueues on the context's stream and allocates
// nothing, so it may be captured into a graph.
#include <cfloat>
#include <cmath>

#include "ctx.cuh"
#include "paged.cuh"

using namespace emx;

#define PG_REQUIRE(cond, ...) \
  do {                        \
    if (!(cond)) return fail(EMX_ERR_INVALID, __VA_ARGS__); \
  } while (0)

namespace {

constexpr int kMaxSeqs = 1024;

// The context's device is current within the scope.
struct DeviceScope {
  int prev = -1;
  cudaError_t err;
  explicit DeviceScope(int device) {
    err = cudaGetDevice(&prev);
    if (err == cudaSuccess && prev != device) err = cudaSetDevice(device);
    else prev = -1;
  }
  ~DeviceScope() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_shape(const char* op, const emx_paged_kv* kv, const emx_paged_batch* b, int n_q) {
  PG_REQUIRE(kv && b, "%s: null argument", op);
  PG_REQUIRE(kv->head_dim == 64 || kv->head_dim == 128, "%s: head_dim must be 64 or 128 (got %d)", op, kv->head_dim);
  PG_REQUIRE(kv->n_kv >= 1 && n_q >= 1 && n_q % kv->n_kv == 0, "%s: n_q %d must be a positive multiple of n_kv %d", op, n_q,
             kv->n_kv);
  PG_REQUIRE(n_q <= 1024, "%s: n_q %d exceeds 1024", op, n_q);
  PG_REQUIRE(kv->n_pages >= 0 && kv->page_size >= 1, "%s: bad cache: %d pages of %d", op, kv->n_pages, kv->page_size);
  // row numbers are int32 coordinates of a tensor map; with 64-element rows that cache would be 256 GB
  PG_REQUIRE((double)kv->n_pages * kv->n_kv * kv->page_size < 2147483647.0, "%s: cache of %d x %d x %d rows is too large", op,
             kv->n_pages, kv->n_kv, kv->page_size);
  PG_REQUIRE(b->n_seqs >= 0 && b->n_seqs <= kMaxSeqs, "%s: n_seqs %d outside [0, %d]", op, b->n_seqs, kMaxSeqs);
  PG_REQUIRE(b->n_rows >= 0 && (int64_t)b->n_rows * n_q <= 0x7fffffff, "%s: n_rows %d is negative or too large for %d heads",
             op, b->n_rows, n_q);
  // the last key tile ends up to 127 positions behind a sequence, still in int32
  PG_REQUIRE(b->max_pages >= 1 && (int64_t)b->max_pages * kv->page_size <= 0x7fffffff - 255,
             "%s: max_pages %d of %d positions outside [1, 2^31 - 256]", op, b->max_pages, kv->page_size);
  return EMX_OK;
}

int check_paged(const char* op, const emx_paged_kv* kv, const emx_paged_batch* b, int n_q) {
  int rc = check_shape(op, kv, b, n_q);
  if (rc) return rc;
  PG_REQUIRE(kv->k && kv->v && b->indptr && b->lengths && b->table, "%s: null argument", op);
  PG_REQUIRE(aligned(kv->k, 16) && aligned(kv->v, 16), "%s: the cache must be 16-byte aligned", op);
  PG_REQUIRE(aligned(b->indptr, 4) && aligned(b->lengths, 4) && aligned(b->table, 4), "%s: misaligned batch", op);
  return EMX_OK;
}

PagedArgs paged_args(const emx_ctx* c, const emx_paged_kv* kv, const emx_paged_batch* b, int n_q) {
  PagedArgs p = {};
  p.k = static_cast<bf16*>(kv->k);
  p.v = static_cast<bf16*>(kv->v);
  p.n_pages = kv->n_pages;
  p.page_size = kv->page_size;
  p.n_kv = kv->n_kv;
  p.head_dim = kv->head_dim;
  p.n_seqs = b->n_seqs;
  p.n_rows = b->n_rows;
  p.max_pages = b->max_pages;
  p.indptr = b->indptr;
  p.lengths = b->lengths;
  p.table = b->table;
  p.n_q = n_q;
  p.status = c->status;
  return p;
}

}  // namespace

extern "C" {

int emx_paged_append(emx_ctx* c, const void* qkv, const void* q_norm, const void* k_norm, float eps, float rope_theta,
                     int n_q, const emx_paged_kv* kv, const emx_paged_batch* b, void* q_out) {
  PG_REQUIRE(qkv && q_out, "emx_paged_append: null argument");
  int rc = check_paged("emx_paged_append", kv, b, n_q);
  if (rc) return rc;
  PG_REQUIRE(rope_theta >= 0.f && rope_theta < INFINITY, "emx_paged_append: rope_theta %g must be positive, or 0 for no rotation",
             rope_theta);
  PG_REQUIRE((int64_t)b->n_rows * (n_q + 2 * (int64_t)kv->n_kv) <= 0x7fffffff, "emx_paged_append: n_rows %d is too large",
             b->n_rows);
  PG_REQUIRE(aligned(qkv, 8) && aligned(q_out, 8) && aligned(q_norm, 8) && aligned(k_norm, 8),
             "emx_paged_append: qkv, the norm weights and q_out must be 8-byte aligned");
  PG_REQUIRE(c, "emx_paged_append: null context");
  if (b->n_rows == 0 || b->n_seqs == 0) return EMX_OK;
  DeviceScope dev(c->device);
  EMX_CHECK_CUDA(dev.err, "emx_paged_append");
  PagedAppendArgs a = {};
  a.p = paged_args(c, kv, b, n_q);
  a.qkv = static_cast<const bf16*>(qkv);
  a.q_norm = static_cast<const bf16*>(q_norm);
  a.k_norm = static_cast<const bf16*>(k_norm);
  a.eps = eps;
  a.rotate = rope_theta > 0.f;
  a.log2_theta = a.rotate ? std::log2((double)rope_theta) : 0.0;
  a.q_out = static_cast<bf16*>(q_out);
  EMX_CHECK_CUDA(paged_append_launch(a, c->num_sms, c->stream), "emx_paged_append");
  return EMX_OK;
}

int emx_sdpa_paged_workspace(emx_ctx* c, const emx_paged_kv* kv, const emx_paged_batch* b, int n_q, int shared_len,
                             size_t* bytes) {
  PG_REQUIRE(bytes, "emx_sdpa_paged_workspace: null argument");
  int rc = check_shape("emx_sdpa_paged_workspace", kv, b, n_q);
  if (rc) return rc;
  PG_REQUIRE(shared_len >= 0, "emx_sdpa_paged_workspace: shared_len %d", shared_len);
  PG_REQUIRE(c, "emx_sdpa_paged_workspace: null context");
  *bytes = paged_attn_workspace(b->n_rows, n_q, kv->n_kv, kv->head_dim, shared_len, c->num_sms);
  return EMX_OK;
}

int emx_sdpa_paged(emx_ctx* c, const void* q, const emx_paged_kv* kv, const emx_paged_batch* b, int n_q, float scale,
                   int shared_len, const int32_t* shared_pages, void* out, void* workspace, size_t workspace_bytes) {
  PG_REQUIRE(q && out && workspace, "emx_sdpa_paged: null argument");
  int rc = check_paged("emx_sdpa_paged", kv, b, n_q);
  if (rc) return rc;
  PG_REQUIRE(shared_len >= 0 && shared_len % kv->page_size == 0,
             "emx_sdpa_paged: shared_len %d must be whole pages of %d positions", shared_len, kv->page_size);
  PG_REQUIRE(shared_len == 0 || shared_pages, "emx_sdpa_paged: shared_len %d without shared_pages", shared_len);
  PG_REQUIRE((int64_t)shared_len <= (int64_t)b->max_pages * kv->page_size,
             "emx_sdpa_paged: shared_len %d exceeds the page table's %d x %d positions", shared_len, b->max_pages, kv->page_size);
  PG_REQUIRE(aligned(q, 16) && aligned(out, 16), "emx_sdpa_paged: q and out must be 16-byte aligned");
  PG_REQUIRE(aligned(workspace, 256), "emx_sdpa_paged: the workspace must be 256-byte aligned");
  PG_REQUIRE(aligned(shared_pages, 4), "emx_sdpa_paged: misaligned shared_pages");
  PG_REQUIRE(c, "emx_sdpa_paged: null context");
  const size_t need = paged_attn_workspace(b->n_rows, n_q, kv->n_kv, kv->head_dim, shared_len, c->num_sms);
  PG_REQUIRE(workspace_bytes >= need, "emx_sdpa_paged: workspace of %zu bytes, %zu needed (emx_sdpa_paged_workspace)",
             workspace_bytes, need);
  if (b->n_rows == 0 || b->n_seqs == 0) return EMX_OK;
  DeviceScope dev(c->device);
  EMX_CHECK_CUDA(dev.err, "emx_sdpa_paged");
  PagedAttnArgs a = {};
  a.p = paged_args(c, kv, b, n_q);
  a.q = static_cast<const bf16*>(q);
  a.out = static_cast<bf16*>(out);
  a.shared_len = shared_len;
  a.shared_pages = shared_pages;
  // equal weights for a scale of 0: the kernels mask by infinite scores, which 0 would turn to NaN
  a.scale = scale == 0.f ? FLT_MIN : scale;
  a.workspace = workspace;
  EMX_CHECK_CUDA(paged_attn_launch(a, c->num_sms, c->stream), "emx_sdpa_paged");
  return EMX_OK;
}

int emx_verify_draft(emx_ctx* c, const void* target, const void* draft, emx_dtype dtype, const int32_t* tokens,
                     const int32_t* counts, const float* uniforms, int n_seqs, int n_draft, int vocab, int32_t* out,
                     int32_t* accepted) {
  PG_REQUIRE(n_seqs >= 0 && n_seqs <= 65535 && n_draft >= 0 && n_draft <= 4096 && vocab >= 1 && vocab <= (1 << 30),
             "emx_verify_draft: bad shape: %d sequences, %d drafts, vocabulary %d", n_seqs, n_draft, vocab);
  PG_REQUIRE(target && uniforms && out && accepted && (tokens || n_draft == 0), "emx_verify_draft: null argument");
  PG_REQUIRE(dtype == EMX_F32 || dtype == EMX_BF16, "emx_verify_draft: probabilities must be f32 or bf16");
  const uintptr_t size = dtype == EMX_F32 ? 4 : 2;
  PG_REQUIRE(aligned(target, size) && aligned(draft, size) && aligned(tokens, 4) && aligned(counts, 4) && aligned(uniforms, 4) &&
                 aligned(out, 4) && aligned(accepted, 4),
             "emx_verify_draft: misaligned argument");
  PG_REQUIRE(c, "emx_verify_draft: null context");
  if (n_seqs == 0) return EMX_OK;
  DeviceScope dev(c->device);
  EMX_CHECK_CUDA(dev.err, "emx_verify_draft");
  VerifyArgs a = {};
  a.target = target;
  a.draft = n_draft > 0 ? draft : nullptr;
  a.is_bf16 = dtype == EMX_BF16;
  a.tokens = tokens;
  a.counts = counts;
  a.uniforms = uniforms;
  a.n_seqs = n_seqs;
  a.n_draft = n_draft;
  a.vocab = vocab;
  a.out = out;
  a.accepted = accepted;
  a.status = c->status;
  EMX_CHECK_CUDA(verify_launch(a, c->num_sms, c->stream), "emx_verify_draft");
  return EMX_OK;
}

}  // extern "C"
