//! engine-mlx-ffi on libemx: the crate crates/serve links for the quantized
//! Qwen3 forward pass, with the MLX / mlx-c backend
//! (crates/mlx-ffi/src/ops/real/mod.rs:4-41, src/lib.rs:24-25) replaced by the
//! B200 kernels of libemx.
//!
//! * `sys` — every declaration of include/emx.h (generated by
//!   engine-mlx_b200/rust/gen_sys.py; a test keeps it equal to the header).
//! * `MlxCtx` — the context (one CUDA stream) and the op-level methods the
//!   engine's ops crates call, named as MlxCtx names them, on device buffers
//!   instead of lazy `mlx_array` handles: work is enqueued in call order and
//!   `synchronize` / the device-to-host copies are the sync points.
//! * `Qwen3Engine` — the whole-model engine: load, prefill, decode, per-token
//!   streaming, sampling; what crates/serve's Qwen3Engine
//!   (crates/serve/src/engine.rs:62-227, forward_qwen3.rs, decode_compiled.rs)
//!   does through MlxCtx.
//!
//! Errors: every call returns a code; non-zero becomes an `anyhow::Error`
//! carrying `emx_last_error()`, as `MlxCtx::check` maps MLX's status
//! (crates/mlx-ffi/src/ops/real/mod.rs:35-40).
pub mod sys;

use anyhow::{anyhow, Result};
use std::ffi::{c_void, CStr, CString};
use std::os::raw::c_int;

/// The message of the last failed call on this thread.
pub fn last_error() -> String {
    unsafe {
        let p = sys::emx_last_error();
        if p.is_null() {
            String::new()
        } else {
            CStr::from_ptr(p).to_string_lossy().into_owned()
        }
    }
}

fn check(rc: c_int, op: &str) -> Result<()> {
    if rc == sys::EMX_OK {
        Ok(())
    } else {
        Err(anyhow!("{op} failed (code {rc}): {}", last_error()))
    }
}

/// libemx's version string.
pub fn version() -> String {
    unsafe { CStr::from_ptr(sys::emx_version()).to_string_lossy().into_owned() }
}

/// A CUDA context and stream on one device (MlxCtx::new / gpu with
/// mlx_default_gpu_stream_new, crates/serve/src/engine.rs:69-80).
pub struct MlxCtx {
    raw: *mut sys::emx_ctx,
}

// One owner thread drives the context, as the reference's single "MLX
// thread" does (crates/mlx-ffi/src/lib.rs:188-208); moving it between threads
// is allowed, sharing it is not.
unsafe impl Send for MlxCtx {}

/// Device memory allocated through a context; freed on drop.
pub struct DeviceBuffer<'c> {
    ctx: &'c MlxCtx,
    ptr: *mut c_void,
    bytes: usize,
}

impl DeviceBuffer<'_> {
    pub fn as_ptr(&self) -> *const c_void {
        self.ptr
    }
    pub fn as_mut_ptr(&mut self) -> *mut c_void {
        self.ptr
    }
    pub fn len(&self) -> usize {
        self.bytes
    }
    pub fn is_empty(&self) -> bool {
        self.bytes == 0
    }
    /// Host -> device copy of `src` (bytes <= len), stream-ordered.
    pub fn upload<T: Copy>(&mut self, src: &[T]) -> Result<()> {
        let n = std::mem::size_of_val(src);
        if n > self.bytes {
            return Err(anyhow!("upload of {n} bytes into a {}-byte buffer", self.bytes));
        }
        check(unsafe { sys::emx_memcpy_h2d(self.ctx.raw, self.ptr, src.as_ptr() as *const c_void, n) }, "upload")
    }
    /// Device -> host copy into `dst`; returns after all prior work is done.
    pub fn download<T: Copy>(&self, dst: &mut [T]) -> Result<()> {
        let n = std::mem::size_of_val(dst);
        if n > self.bytes {
            return Err(anyhow!("download of {n} bytes from a {}-byte buffer", self.bytes));
        }
        check(unsafe { sys::emx_memcpy_d2h(self.ctx.raw, dst.as_mut_ptr() as *mut c_void, self.ptr, n) },
              "download")
    }
}

impl Drop for DeviceBuffer<'_> {
    fn drop(&mut self) {
        unsafe {
            sys::emx_free(self.ctx.raw, self.ptr);
        }
    }
}

impl MlxCtx {
    /// MlxCtx::gpu: a context on CUDA device `device`.
    pub fn gpu(device: i32) -> Result<Self> {
        let mut raw = std::ptr::null_mut();
        check(unsafe { sys::emx_ctx_create(device, &mut raw) }, "emx_ctx_create")?;
        Ok(Self { raw })
    }
    /// A context that runs on a CUDA stream of the caller's (null: the default stream).
    ///
    /// # Safety
    /// `stream` must be a stream of `device` and outlive the context.
    pub unsafe fn on_stream(device: i32, stream: *mut std::os::raw::c_void) -> Result<Self> {
        let mut raw = std::ptr::null_mut();
        check(sys::emx_ctx_create_on_stream(device, stream, &mut raw), "emx_ctx_create_on_stream")?;
        Ok(Self { raw })
    }
    pub fn raw(&self) -> *mut sys::emx_ctx {
        self.raw
    }
    /// mlx_synchronize.
    pub fn synchronize(&self) -> Result<()> {
        check(unsafe { sys::emx_synchronize(self.raw) }, "emx_synchronize")
    }
    pub fn alloc(&self, bytes: usize) -> Result<DeviceBuffer<'_>> {
        let mut ptr = std::ptr::null_mut();
        check(unsafe { sys::emx_malloc(self.raw, bytes, &mut ptr) }, "emx_malloc")?;
        Ok(DeviceBuffer { ctx: self, ptr, bytes })
    }
    /// mlx_get_active_memory / mlx_get_peak_memory / mlx_set_memory_limit
    /// (crates/serve/src/engine.rs:84-110).
    pub fn active_memory(&self) -> Result<usize> {
        let mut b = 0usize;
        check(unsafe { sys::emx_get_active_memory(self.raw, &mut b) }, "emx_get_active_memory")?;
        Ok(b)
    }
    pub fn peak_memory(&self) -> Result<usize> {
        let mut b = 0usize;
        check(unsafe { sys::emx_get_peak_memory(self.raw, &mut b) }, "emx_get_peak_memory")?;
        Ok(b)
    }
    pub fn set_memory_limit(&self, limit: usize) -> Result<usize> {
        let mut prev = 0usize;
        check(unsafe { sys::emx_set_memory_limit(self.raw, limit, &mut prev) }, "emx_set_memory_limit")?;
        Ok(prev)
    }

    // ---- op-level methods (crates/mlx-ffi/src/ops/real/*.rs), device buffers
    /// MlxCtx::quantized_matmul (transform.rs:77-89): y[m,n] = x[m,k] . dequant(w)^T.
    #[allow(clippy::too_many_arguments)]
    pub fn quantized_matmul(&self, x: &DeviceBuffer, w: &DeviceBuffer, scales: &DeviceBuffer,
                            biases: &DeviceBuffer, y: &mut DeviceBuffer, m: i32, n: i32, k: i32, group_size: i32,
                            bits: i32) -> Result<()> {
        check(unsafe {
            sys::emx_quantized_matmul(self.raw, x.as_ptr(), w.as_ptr(), scales.as_ptr(), biases.as_ptr(),
                                      y.as_mut_ptr(), m, n, k, 1, group_size, bits)
        }, "quantized_matmul")
    }
    /// MlxCtx::dequantize_weight (transform.rs:45-60): bf16 [n, k].
    #[allow(clippy::too_many_arguments)]
    pub fn dequantize_weight(&self, w: &DeviceBuffer, scales: &DeviceBuffer, biases: &DeviceBuffer,
                             out: &mut DeviceBuffer, n: i32, k: i32, group_size: i32, bits: i32) -> Result<()> {
        check(unsafe {
            sys::emx_dequantize(self.raw, w.as_ptr(), scales.as_ptr(), biases.as_ptr(), out.as_mut_ptr(), n, k,
                                group_size, bits)
        }, "dequantize_weight")
    }
    /// MlxCtx::rms_norm (blas.rs:5-9) over `rows` rows of `dims`.
    pub fn rms_norm(&self, x: &DeviceBuffer, weight: &DeviceBuffer, out: &mut DeviceBuffer, rows: i32, dims: i32,
                    eps: f32) -> Result<()> {
        check(unsafe {
            sys::emx_rms_norm(self.raw, x.as_ptr(), weight.as_ptr(), out.as_mut_ptr(), rows, dims, eps)
        }, "rms_norm")
    }
    /// MlxCtx::grouped_rms_norm (grouped_norm.rs:50-135).
    #[allow(clippy::too_many_arguments)]
    pub fn grouped_rms_norm(&self, x: &DeviceBuffer, weight: &DeviceBuffer, out: &mut DeviceBuffer, rows: i32,
                            dims: i32, eps: f32, groups: i32) -> Result<()> {
        check(unsafe {
            sys::emx_grouped_rms_norm(self.raw, x.as_ptr(), weight.as_ptr(), out.as_mut_ptr(), rows, dims, eps,
                                      groups)
        }, "grouped_rms_norm")
    }
    /// MlxCtx::silu / multiply / add (blas.rs:17-37) on n bf16 elements.
    pub fn silu(&self, x: &DeviceBuffer, out: &mut DeviceBuffer, n: usize) -> Result<()> {
        check(unsafe { sys::emx_silu(self.raw, x.as_ptr(), out.as_mut_ptr(), n) }, "silu")
    }
    pub fn multiply(&self, a: &DeviceBuffer, b: &DeviceBuffer, out: &mut DeviceBuffer, n: usize) -> Result<()> {
        check(unsafe { sys::emx_multiply(self.raw, a.as_ptr(), b.as_ptr(), out.as_mut_ptr(), n) }, "multiply")
    }
    pub fn add(&self, a: &DeviceBuffer, b: &DeviceBuffer, out: &mut DeviceBuffer, n: usize) -> Result<()> {
        check(unsafe { sys::emx_add(self.raw, a.as_ptr(), b.as_ptr(), out.as_mut_ptr(), n) }, "add")
    }
    /// MlxCtx::argmax + to_vec_u32 (array.rs:6-11, 103-118): the first index of
    /// the maximum of each of `rows` rows of n bf16 values.
    pub fn argmax(&self, x: &DeviceBuffer, rows: i32, n: i32, out: &mut DeviceBuffer) -> Result<()> {
        check(unsafe { sys::emx_argmax(self.raw, x.as_ptr(), rows, n, out.as_mut_ptr() as *mut i32) }, "argmax")
    }

    // ---- a batch of sequences over a paged cache (emx.h describes the two
    // structs; their device arrays must outlive the enqueued work, and what
    // they hold is read on the device)
    /// Per-head norm and rotation of q and k, k and v to their pages of the cache.
    ///
    /// # Safety
    /// The pointers in `kv` and `batch` must be device arrays of the sizes they state.
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn paged_append(&self, qkv: &DeviceBuffer, q_norm: Option<&DeviceBuffer>,
                               k_norm: Option<&DeviceBuffer>, eps: f32, rope_theta: f32, n_q: i32,
                               kv: &sys::emx_paged_kv, batch: &sys::emx_paged_batch, q_out: &mut DeviceBuffer)
                               -> Result<()> {
        let opt = |b: Option<&DeviceBuffer>| b.map_or(std::ptr::null(), |b| b.as_ptr());
        check(sys::emx_paged_append(self.raw, qkv.as_ptr(), opt(q_norm), opt(k_norm), eps, rope_theta, n_q, kv, batch,
                                    q_out.as_mut_ptr()), "paged_append")
    }
    /// Bytes of workspace that `sdpa_paged` needs.
    pub fn sdpa_paged_workspace(&self, kv: &sys::emx_paged_kv, batch: &sys::emx_paged_batch, n_q: i32,
                                shared_len: i32) -> Result<usize> {
        let mut n = 0usize;
        check(unsafe { sys::emx_sdpa_paged_workspace(self.raw, kv, batch, n_q, shared_len, &mut n) },
              "sdpa_paged_workspace")?;
        Ok(n)
    }
    /// Attention of a batch's rows over the cache, the pages `shared_pages` of
    /// the first `shared_len` positions read once for all sequences.
    ///
    /// # Safety
    /// As `paged_append`.
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn sdpa_paged(&self, q: &DeviceBuffer, kv: &sys::emx_paged_kv, batch: &sys::emx_paged_batch, n_q: i32,
                             scale: f32, shared_len: i32, shared_pages: Option<&DeviceBuffer>,
                             out: &mut DeviceBuffer, workspace: &mut DeviceBuffer) -> Result<()> {
        let pages = shared_pages.map_or(std::ptr::null(), |b| b.as_ptr() as *const i32);
        let bytes = workspace.len();
        check(sys::emx_sdpa_paged(self.raw, q.as_ptr(), kv, batch, n_q, scale, shared_len, pages, out.as_mut_ptr(),
                                  workspace.as_mut_ptr(), bytes), "sdpa_paged")
    }
    /// Speculative sampling's acceptance of drafted tokens (`dtype`: sys::EMX_F32 or sys::EMX_BF16).
    #[allow(clippy::too_many_arguments)]
    pub fn verify_draft(&self, target: &DeviceBuffer, draft: Option<&DeviceBuffer>, dtype: i32, tokens: &DeviceBuffer,
                        counts: Option<&DeviceBuffer>, uniforms: &DeviceBuffer, n_seqs: i32, n_draft: i32, vocab: i32,
                        out: &mut DeviceBuffer, accepted: &mut DeviceBuffer) -> Result<()> {
        let opt = |b: Option<&DeviceBuffer>| b.map_or(std::ptr::null(), |b| b.as_ptr());
        check(unsafe {
            sys::emx_verify_draft(self.raw, target.as_ptr(), opt(draft), dtype, tokens.as_ptr() as *const i32,
                                  opt(counts) as *const i32, uniforms.as_ptr() as *const f32, n_seqs, n_draft, vocab,
                                  out.as_mut_ptr() as *mut i32, accepted.as_mut_ptr() as *mut i32)
        }, "verify_draft")
    }
}

impl Drop for MlxCtx {
    fn drop(&mut self) {
        unsafe {
            sys::emx_ctx_destroy(self.raw);
        }
    }
}

/// Sampling parameters (crates/serve/src/sampler.rs SamplingParams): greedy
/// when temperature < 1e-6.
#[derive(Clone, Copy, Debug)]
pub struct SamplingParams {
    pub temperature: f32,
    pub top_p: f32,
    pub top_k: usize,
    pub seed: u64,
}

/// The Qwen3 engine on libemx: weights, the static KV cache and the decode
/// state live on the device; the calls mirror crates/serve's Qwen3Engine.
pub struct Qwen3Engine<'c> {
    raw: *mut sys::emx_qwen3,
    cfg: sys::emx_qwen3_config,
    _ctx: &'c MlxCtx,
}

unsafe impl Send for Qwen3Engine<'_> {}

impl<'c> Qwen3Engine<'c> {
    /// Qwen3Config::from_dir (crates/serve/src/config.rs:77-90) plus the
    /// engine's own KV capacity and largest prefill.
    pub fn config_from_dir(model_dir: &str, kv_cap: i32, max_prefill: i32) -> Result<sys::emx_qwen3_config> {
        let dir = CString::new(model_dir)?;
        let mut cfg = std::mem::MaybeUninit::<sys::emx_qwen3_config>::zeroed();
        check(unsafe { sys::emx_qwen3_config_from_dir(dir.as_ptr(), kv_cap, max_prefill, cfg.as_mut_ptr()) },
              "config_from_dir")?;
        Ok(unsafe { cfg.assume_init() })
    }

    /// Qwen3Engine::from_init (crates/serve/src/engine.rs:62-227): allocates
    /// the model of shape `cfg` on `ctx` (one GPU; tensor / expert parallel
    /// ranks go through emx_comm_init and the raw `sys` calls).
    pub fn new(ctx: &'c MlxCtx, cfg: &sys::emx_qwen3_config) -> Result<Self> {
        let mut raw = std::ptr::null_mut();
        check(unsafe { sys::emx_qwen3_create(ctx.raw, cfg, std::ptr::null_mut(), &mut raw) }, "emx_qwen3_create")?;
        Ok(Self { raw, cfg: *cfg, _ctx: ctx })
    }

    /// load_weights_from_manifest (crates/serve/src/loader/weights.rs:17-284):
    /// an MLX model directory or .safetensors file; returns the tensors loaded.
    pub fn load_safetensors(&mut self, path: &str) -> Result<i32> {
        let p = CString::new(path)?;
        let mut n: c_int = 0;
        check(unsafe { sys::emx_qwen3_load_safetensors(self.raw, p.as_ptr(), &mut n) }, "load_safetensors")?;
        Ok(n)
    }

    /// Seeded synthetic weights (benchmarks and tests).
    pub fn init_random(&mut self, seed: u64) -> Result<()> {
        check(unsafe { sys::emx_qwen3_init_random(self.raw, seed) }, "init_random")
    }

    /// Qwen3Engine::reset (crates/serve/src/engine_ext.rs:10-36).
    pub fn reset(&mut self) -> Result<()> {
        check(unsafe { sys::emx_qwen3_reset(self.raw) }, "reset")
    }

    pub fn offset(&self) -> Result<usize> {
        let mut o: c_int = 0;
        check(unsafe { sys::emx_qwen3_offset(self.raw, &mut o) }, "offset")?;
        Ok(o as usize)
    }

    /// Qwen3Engine::set_sampling (crates/serve/src/engine.rs:230-233).
    pub fn set_sampling(&mut self, p: SamplingParams) -> Result<()> {
        check(unsafe { sys::emx_qwen3_set_sampling(self.raw, p.temperature, p.top_p, p.top_k as i32, p.seed) },
              "set_sampling")
    }

    fn ids(tokens: &[u32]) -> Vec<i32> {
        tokens.iter().map(|&t| t as i32).collect()
    }

    /// Qwen3Engine::prefill (crates/serve/src/forward_qwen3.rs:12-200): the
    /// prompt at the current offset; returns the next token.
    pub fn prefill(&mut self, tokens: &[u32]) -> Result<u32> {
        let ids = Self::ids(tokens);
        let mut next: i32 = 0;
        check(unsafe {
            sys::emx_qwen3_prefill(self.raw, ids.as_ptr(), ids.len() as i32, &mut next, std::ptr::null_mut())
        }, "prefill")?;
        Ok(next as u32)
    }

    /// The prefill pipeline (crates/prefill/src/pipeline.rs:60-117): chunks
    /// of at most `chunk` tokens, each attending the cache before it.
    pub fn prefill_chunked(&mut self, tokens: &[u32], chunk: usize) -> Result<u32> {
        let ids = Self::ids(tokens);
        let mut next: i32 = 0;
        check(unsafe {
            sys::emx_qwen3_prefill_chunked(self.raw, ids.as_ptr(), ids.len() as i32, chunk as i32, &mut next,
                                           std::ptr::null_mut())
        }, "prefill_chunked")?;
        Ok(next as u32)
    }

    /// One decode step (decode_compiled.rs:113-120): the token after `token`.
    pub fn decode_step(&mut self, token: u32) -> Result<u32> {
        let mut next: i32 = 0;
        check(unsafe { sys::emx_qwen3_decode_step(self.raw, token as i32, &mut next, std::ptr::null_mut()) },
              "decode_step")?;
        Ok(next as u32)
    }

    /// `n` steps from `token` with one host synchronisation.
    pub fn decode(&mut self, token: u32, n: usize) -> Result<Vec<u32>> {
        let mut out = vec![0i32; n];
        check(unsafe { sys::emx_qwen3_decode(self.raw, token as i32, n as i32, out.as_mut_ptr()) }, "decode")?;
        Ok(out.into_iter().map(|t| t as u32).collect())
    }

    /// Per-token streaming for the server's SSE path
    /// (crates/serve/src/server.rs:131-181): `on_token(token, index)` runs as
    /// each token is produced; returning `false` stops after that token (an
    /// end-of-sequence id, a closed client), leaving the engine just after
    /// it.  Returns the tokens delivered.
    pub fn decode_stream<F: FnMut(u32, usize) -> bool>(&mut self, token: u32, n: usize, mut on_token: F)
                                                       -> Result<usize> {
        unsafe extern "C" fn tramp<F: FnMut(u32, usize) -> bool>(tok: i32, idx: c_int, user: *mut c_void) -> c_int {
            let f = &mut *(user as *mut F);
            // a panic must not unwind into C: it stops the stream
            match std::panic::catch_unwind(std::panic::AssertUnwindSafe(|| f(tok as u32, idx as usize))) {
                Ok(true) => 0,
                _ => 1,
            }
        }
        let mut done: c_int = 0;
        check(unsafe {
            sys::emx_qwen3_decode_stream(self.raw, token as i32, n as i32, Some(tramp::<F>),
                                         &mut on_token as *mut F as *mut c_void, &mut done)
        }, "decode_stream")?;
        Ok(done as usize)
    }

    pub fn config(&self) -> &sys::emx_qwen3_config {
        &self.cfg
    }
}

impl Drop for Qwen3Engine<'_> {
    fn drop(&mut self) {
        unsafe {
            sys::emx_qwen3_destroy(self.raw);
        }
    }
}
