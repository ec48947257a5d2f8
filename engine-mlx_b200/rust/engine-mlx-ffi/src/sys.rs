// @generated by engine-mlx_b200/rust/gen_sys.py from include/emx.h -- do not edit.
#![allow(non_camel_case_types, non_snake_case, dead_code)]

use std::os::raw::{c_char, c_int, c_void};

pub const EMX_OK: c_int = 0;
pub const EMX_ERR_INVALID: c_int = 1;
pub const EMX_ERR_CUDA: c_int = 2;
pub const EMX_ERR_OOM: c_int = 3;
pub const EMX_ERR_DEVICE: c_int = 4;
pub const EMX_ERR_NCCL: c_int = 5;
pub const EMX_ERR_STATE: c_int = 6;
pub const EMX_DEV_OK: c_int = 0;
pub const EMX_DEV_TIMEOUT_MBAR: c_int = 1;
pub const EMX_DEV_TIMEOUT_PEER: c_int = 2;
pub const EMX_DEV_BAD_TOKEN: c_int = 3;
pub const EMX_DEV_KV_OVERFLOW: c_int = 4;
pub const EMX_DEV_BAD_PAGE: c_int = 5;
pub const EMX_DEV_BAD_BATCH: c_int = 6;
pub const EMX_UNIQUE_ID_BYTES: c_int = 128;

pub const EMX_BF16: c_int = 0;
pub const EMX_F32: c_int = 1;
pub const EMX_U32: c_int = 2;
pub const EMX_I32: c_int = 3;

#[repr(C)]
pub struct emx_ctx {
    _private: [u8; 0],
}
#[repr(C)]
pub struct emx_comm {
    _private: [u8; 0],
}
#[repr(C)]
pub struct emx_qwen3 {
    _private: [u8; 0],
}

pub type emx_error_handler = Option<unsafe extern "C" fn(msg: *const c_char, data: *mut c_void)>;
pub type emx_token_cb = Option<unsafe extern "C" fn(token: i32, index: c_int, user: *mut c_void) -> c_int>;

#[repr(C)]
#[derive(Clone, Copy)]
pub struct emx_qwen3_config {
    pub hidden: c_int,
    pub layers: c_int,
    pub n_q: c_int,
    pub n_kv: c_int,
    pub head_dim: c_int,
    pub inter: c_int,
    pub vocab: c_int,
    pub eps: f32,
    pub rope_theta: f32,
    pub tied: c_int,
    pub norm_groups: c_int,
    pub attn_bits: c_int,
    pub attn_group: c_int,
    pub mlp_bits: c_int,
    pub mlp_group: c_int,
    pub embed_bits: c_int,
    pub embed_group: c_int,
    pub lm_bits: c_int,
    pub lm_group: c_int,
    pub n_experts: c_int,
    pub top_k: c_int,
    pub moe_inter: c_int,
    pub norm_topk: c_int,
    pub router_bits: c_int,
    pub router_group: c_int,
    pub expert_bits: c_int,
    pub expert_group: c_int,
    pub kv_cap: c_int,
    pub max_prefill: c_int,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct emx_st_tensor {
    pub name: [c_char; 256],
    pub dtype: [c_char; 12],
    pub ndim: c_int,
    pub shape: [i64; 8],
    pub offset: u64,
    pub bytes: u64,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct emx_paged_kv {
    pub k: *mut c_void,
    pub v: *mut c_void,
    pub n_pages: c_int,
    pub page_size: c_int,
    pub n_kv: c_int,
    pub head_dim: c_int,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct emx_paged_batch {
    pub n_seqs: c_int,
    pub n_rows: c_int,
    pub max_pages: c_int,
    pub indptr: *const i32,
    pub lengths: *const i32,
    pub table: *const i32,
}

extern "C" {
    pub fn emx_set_error_handler(handler: emx_error_handler, data: *mut c_void);
    pub fn emx_last_error() -> *const c_char;
    pub fn emx_version() -> *const c_char;
    pub fn emx_ctx_create(device: c_int, out: *mut *mut emx_ctx) -> c_int;
    pub fn emx_ctx_create_on_stream(device: c_int, cuda_stream: *mut c_void, out: *mut *mut emx_ctx) -> c_int;
    pub fn emx_ctx_destroy(ctx: *mut emx_ctx) -> c_int;
    pub fn emx_ctx_stream(ctx: *mut emx_ctx, cuda_stream: *mut *mut c_void) -> c_int;
    pub fn emx_ctx_num_sms(ctx: *mut emx_ctx, n: *mut c_int) -> c_int;
    pub fn emx_synchronize(ctx: *mut emx_ctx) -> c_int;
    pub fn emx_device_status(ctx: *mut emx_ctx, status: *mut c_int, clear: c_int) -> c_int;
    pub fn emx_malloc(ctx: *mut emx_ctx, bytes: usize, ptr: *mut *mut c_void) -> c_int;
    pub fn emx_free(ctx: *mut emx_ctx, ptr: *mut c_void) -> c_int;
    pub fn emx_memcpy_h2d(ctx: *mut emx_ctx, dst: *mut c_void, src: *const c_void, bytes: usize) -> c_int;
    pub fn emx_memcpy_d2h(ctx: *mut emx_ctx, dst: *mut c_void, src: *const c_void, bytes: usize) -> c_int;
    pub fn emx_memset(ctx: *mut emx_ctx, dst: *mut c_void, value: c_int, bytes: usize) -> c_int;
    pub fn emx_get_active_memory(ctx: *mut emx_ctx, bytes: *mut usize) -> c_int;
    pub fn emx_get_peak_memory(ctx: *mut emx_ctx, bytes: *mut usize) -> c_int;
    pub fn emx_set_memory_limit(ctx: *mut emx_ctx, limit: usize, previous: *mut usize) -> c_int;
    pub fn emx_quantized_matmul(ctx: *mut emx_ctx, x: *const c_void, w: *const c_void, scales: *const c_void, biases: *const c_void, y: *mut c_void, M: c_int, N: c_int, K: c_int, transpose: c_int, group_size: c_int, bits: c_int) -> c_int;
    pub fn emx_qpack_bytes(N: c_int, K: c_int, group_size: c_int, bits: c_int, bytes: *mut usize) -> c_int;
    pub fn emx_qpack(ctx: *mut emx_ctx, w: *const c_void, scales: *const c_void, biases: *const c_void, out: *mut c_void, N: c_int, K: c_int, group_size: c_int, bits: c_int) -> c_int;
    pub fn emx_quantized_matvec_packed(ctx: *mut emx_ctx, x: *const c_void, packed: *const c_void, y: *mut c_void, N: c_int, K: c_int, group_size: c_int, bits: c_int) -> c_int;
    pub fn emx_quantized_matmul_packed(ctx: *mut emx_ctx, x: *const c_void, packed: *const c_void, y: *mut c_void, M: c_int, N: c_int, K: c_int, group_size: c_int, bits: c_int) -> c_int;
    pub fn emx_dequantize(ctx: *mut emx_ctx, w: *const c_void, scales: *const c_void, biases: *const c_void, out: *mut c_void, N: c_int, K: c_int, group_size: c_int, bits: c_int) -> c_int;
    pub fn emx_quantize(ctx: *mut emx_ctx, src: *const c_void, src_dtype: c_int, w: *mut c_void, scales: *mut c_void, biases: *mut c_void, N: c_int, K: c_int, group_size: c_int, bits: c_int) -> c_int;
    pub fn emx_rms_norm(ctx: *mut emx_ctx, x: *const c_void, weight: *const c_void, out: *mut c_void, rows: c_int, dims: c_int, eps: f32) -> c_int;
    pub fn emx_grouped_rms_norm(ctx: *mut emx_ctx, x: *const c_void, weight: *const c_void, out: *mut c_void, rows: c_int, dims: c_int, eps: f32, groups: c_int) -> c_int;
    pub fn emx_rope(ctx: *mut emx_ctx, x: *const c_void, out: *mut c_void, heads: c_int, T: c_int, dims: c_int, theta: f32, offset: c_int, offset_dev: *const i32) -> c_int;
    pub fn emx_sdpa_causal(ctx: *mut emx_ctx, q: *const c_void, k: *const c_void, v: *const c_void, out: *mut c_void, nq: c_int, nkv: c_int, T: c_int, head_dim: c_int, scale: f32, out_tnd: c_int) -> c_int;
    pub fn emx_sdpa_decode(ctx: *mut emx_ctx, q: *const c_void, k_cache: *const c_void, v_cache: *const c_void, out: *mut c_void, nq: c_int, nkv: c_int, cap: c_int, head_dim: c_int, length: c_int, scale: f32) -> c_int;
    pub fn emx_sdpa_decode_noalloc(ctx: *mut emx_ctx, q: *const c_void, k_cache: *const c_void, v_cache: *const c_void, out: *mut c_void, nq: c_int, nkv: c_int, cap: c_int, head_dim: c_int, length: c_int, scale: f32) -> c_int;
    pub fn emx_silu(ctx: *mut emx_ctx, x: *const c_void, out: *mut c_void, n: usize) -> c_int;
    pub fn emx_multiply(ctx: *mut emx_ctx, a: *const c_void, b: *const c_void, out: *mut c_void, n: usize) -> c_int;
    pub fn emx_add(ctx: *mut emx_ctx, a: *const c_void, b: *const c_void, out: *mut c_void, n: usize) -> c_int;
    pub fn emx_argmax(ctx: *mut emx_ctx, x: *const c_void, rows: c_int, n: c_int, out: *mut i32) -> c_int;
    pub fn emx_sample_token(ctx: *mut emx_ctx, logits: *const c_void, n: c_int, temperature: f32, top_p: f32, top_k: c_int, rng_state: *mut u64, token: *mut i32) -> c_int;
    pub fn emx_softmax(ctx: *mut emx_ctx, x: *const c_void, out: *mut c_void, rows: c_int, n: c_int) -> c_int;
    pub fn emx_embed_quantized(ctx: *mut emx_ctx, w: *const c_void, scales: *const c_void, biases: *const c_void, ids: *const i32, T: c_int, hidden: c_int, vocab: c_int, group_size: c_int, bits: c_int, out: *mut c_void) -> c_int;
    pub fn emx_slice_update(ctx: *mut emx_ctx, cache: *mut c_void, upd: *const c_void, nkv: c_int, cap: c_int, head_dim: c_int, offset: c_int, T: c_int) -> c_int;
    pub fn emx_scatter_single(ctx: *mut emx_ctx, cache: *mut c_void, offset: *const i32, upd: *const c_void, nkv: c_int, cap: c_int, head_dim: c_int) -> c_int;
    pub fn emx_moe_route(ctx: *mut emx_ctx, router_logits: *const c_void, n_experts: c_int, top_k: c_int, normalize: c_int, idx: *mut i32, weights: *mut f32) -> c_int;
    pub fn emx_gather_qmm(ctx: *mut emx_ctx, x: *const c_void, x_per_slot: c_int, w: *const c_void, scales: *const c_void, biases: *const c_void, idx: *const i32, n_slots: c_int, y: *mut c_void, n_experts: c_int, N: c_int, K: c_int, group_size: c_int, bits: c_int) -> c_int;
    pub fn emx_paged_append(ctx: *mut emx_ctx, qkv: *const c_void, q_norm: *const c_void, k_norm: *const c_void, eps: f32, rope_theta: f32, n_q: c_int, kv: *const emx_paged_kv, batch: *const emx_paged_batch, q_out: *mut c_void) -> c_int;
    pub fn emx_sdpa_paged_workspace(ctx: *mut emx_ctx, kv: *const emx_paged_kv, batch: *const emx_paged_batch, n_q: c_int, shared_len: c_int, bytes: *mut usize) -> c_int;
    pub fn emx_sdpa_paged(ctx: *mut emx_ctx, q: *const c_void, kv: *const emx_paged_kv, batch: *const emx_paged_batch, n_q: c_int, scale: f32, shared_len: c_int, shared_pages: *const i32, out: *mut c_void, workspace: *mut c_void, workspace_bytes: usize) -> c_int;
    pub fn emx_verify_draft(ctx: *mut emx_ctx, target: *const c_void, draft: *const c_void, dtype: c_int, tokens: *const i32, counts: *const i32, uniforms: *const f32, n_seqs: c_int, n_draft: c_int, vocab: c_int, out: *mut i32, accepted: *mut i32) -> c_int;
    pub fn emx_comm_unique_id(id_out: *mut c_void) -> c_int;
    pub fn emx_comm_init(ctx: *mut emx_ctx, unique_id: *const c_void, nranks: c_int, rank: c_int, out: *mut *mut emx_comm) -> c_int;
    pub fn emx_comm_destroy(comm: *mut emx_comm) -> c_int;
    pub fn emx_all_reduce_sum(comm: *mut emx_comm, buf: *mut c_void, count: usize, dtype: c_int) -> c_int;
    pub fn emx_qwen3_config_from_dir(model_dir: *const c_char, kv_cap: c_int, max_prefill: c_int, out: *mut emx_qwen3_config) -> c_int;
    pub fn emx_qwen3_create(ctx: *mut emx_ctx, cfg: *const emx_qwen3_config, comm: *mut emx_comm, out: *mut *mut emx_qwen3) -> c_int;
    pub fn emx_qwen3_destroy(m: *mut emx_qwen3) -> c_int;
    pub fn emx_qwen3_load_tensor(m: *mut emx_qwen3, name: *const c_char, host: *const c_void, bytes: usize) -> c_int;
    pub fn emx_qwen3_read_tensor(m: *mut emx_qwen3, name: *const c_char, host: *mut c_void, bytes: usize) -> c_int;
    pub fn emx_qwen3_load_safetensors(m: *mut emx_qwen3, path: *const c_char, n_loaded: *mut c_int) -> c_int;
    pub fn emx_qwen3_tensor_names(m: *mut emx_qwen3, buf: *mut c_char, cap: usize, need: *mut usize) -> c_int;
    pub fn emx_qwen3_tensor_shape(m: *mut emx_qwen3, name: *const c_char, shape3: *mut i64, ndim: *mut c_int, dtype: *mut c_int) -> c_int;
    pub fn emx_qwen3_set_sampling(m: *mut emx_qwen3, temperature: f32, top_p: f32, top_k: c_int, seed: u64) -> c_int;
    pub fn emx_safetensors_index(file: *const c_char, out: *mut emx_st_tensor, cap: c_int, n: *mut c_int) -> c_int;
    pub fn emx_qwen3_read_kv(m: *mut emx_qwen3, layer: c_int, which: c_int, host: *mut c_void, bytes: usize) -> c_int;
    pub fn emx_qwen3_init_random(m: *mut emx_qwen3, seed: u64) -> c_int;
    pub fn emx_qwen3_reset(m: *mut emx_qwen3) -> c_int;
    pub fn emx_qwen3_offset(m: *mut emx_qwen3, offset: *mut c_int) -> c_int;
    pub fn emx_qwen3_prefill(m: *mut emx_qwen3, tokens: *const i32, T: c_int, next_token: *mut i32, logits: *mut c_void) -> c_int;
    pub fn emx_qwen3_prefill_chunked(m: *mut emx_qwen3, tokens: *const i32, T: c_int, chunk: c_int, next_token: *mut i32, logits: *mut c_void) -> c_int;
    pub fn emx_qwen3_decode_step(m: *mut emx_qwen3, token: i32, next_token: *mut i32, logits: *mut c_void) -> c_int;
    pub fn emx_qwen3_decode(m: *mut emx_qwen3, token: i32, n: c_int, tokens_out: *mut i32) -> c_int;
    pub fn emx_qwen3_decode_stream(m: *mut emx_qwen3, token: i32, n: c_int, cb: emx_token_cb, user: *mut c_void, n_done: *mut c_int) -> c_int;
    pub fn emx_qwen3_prefill_device(m: *mut emx_qwen3, tokens_dev: *const i32, T: c_int) -> c_int;
    pub fn emx_qwen3_decode_device(m: *mut emx_qwen3, n: c_int) -> c_int;
    pub fn emx_qwen3_shard(cfg: *const emx_qwen3_config, world: c_int, rank: c_int, name: *const c_char, out6: *mut i32) -> c_int;
    pub fn emx_qwen3_set_compiled(m: *mut emx_qwen3, compiled: c_int) -> c_int;
    pub fn emx_qwen3_is_compiled(m: *mut emx_qwen3, compiled: *mut c_int) -> c_int;
    pub fn emx_qwen3_set_fused(m: *mut emx_qwen3, fused: c_int) -> c_int;
    pub fn emx_qwen3_is_fused(m: *mut emx_qwen3, fused: *mut c_int) -> c_int;
    pub fn emx_qwen3_step_launches(m: *mut emx_qwen3, n: *mut c_int) -> c_int;
}
