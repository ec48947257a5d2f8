// paged_dev.cuh — device helpers of the paged-cache kernels.
#pragma once
#include "paged.cuh"

namespace emx {

// Two fp32 values of one register pair, and the instructions on both.
__device__ __forceinline__ uint64_t pair32(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split32(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Two weights, each as the sum of two bf16: hi below the weight, lo what is left, rounded (off by at most 2^-14 of the
// weight).  Both are positive where the weight is, so that an infinite V stays what it is.
__device__ __forceinline__ void split_weights(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  constexpr float kBelow = 1.f - 0x1p-20f;
  const uint64_t p = pair32(p0, p1);
  float h0, h1, l0, l1;
  split32(mul2(p, pair32(kBelow, kBelow)), h0, h1);
  hi = __byte_perm(__float_as_uint(h0), __float_as_uint(h1), 0x7632);  // truncated
  split32(fma2(pair32(__uint_as_float(hi << 16), __uint_as_float(hi & 0xffff0000u)), pair32(-1.f, -1.f), p), l0, l1);
  const __nv_bfloat162 l = __floats2bfloat162_rn(l0, l1);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ SeqInfo load_seq(const PagedArgs& p, int i, int shared) {
  return seq_info(p.indptr[i], p.indptr[i + 1], p.lengths[i], p.n_rows, shared, (int64_t)p.max_pages * p.page_size);
}

__device__ __forceinline__ Line make_line(const PagedArgs& p, int shared_len, bool own, int mt, int keys, int setup,
                                          const int64_t* starts) {
  return Line{own, p.n_seqs, p.n_rows, p.n_kv, p.n_q / p.n_kv, shared_len, mt, keys, setup, (int64_t)p.max_pages * p.page_size,
              p.indptr, p.lengths, starts};
}

// The status a sequence that is not in order reports.
__device__ __forceinline__ int seq_status(const PagedArgs& p, int i) {
  return (int64_t)p.lengths[i] > (int64_t)p.max_pages * p.page_size ? kDevKvOverflow : kDevBadBatch;
}

// The sequence that batch row `row` belongs to: the first i with
// indptr[i + 1] > row, by all 32 lanes of a warp, or n_seqs.  Every read is
// inside indptr whatever it holds; the caller checks indptr[i] <= row, which
// an indptr that does not ascend may break.
__device__ __forceinline__ int warp_find_seq(const int* indptr, int n_seqs, int row) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = n_seqs;  // the answer is in [lo, lo + n]
  while (n > 0) {
    const int stride = (n + 31) / 32;
    const int at = min(lo + (lane + 1) * stride, lo + n);  // lane's block of sequences ends before `at`
    const unsigned hit = __ballot_sync(0xffffffffu, indptr[at] > row);
    if (!hit) return lo + n;
    const int first = __ffs(hit) - 1;
    const int b = lo + first * stride, e = min(b + stride, lo + n);
    lo = b;
    n = e - b - 1;  // the answer is one of [b, e): e - 1 if no earlier one has it
  }
  return lo;
}

// An attribute of a kernel, before its launch on the current device.
template <typename K>
inline cudaError_t attribute(std::atomic<uint64_t>& done, K kernel, cudaFuncAttribute which, int value) {
  int device = -1;
  const cudaError_t e = cudaGetDevice(&device);
  return e != cudaSuccess ? e : once_a_device(done, device, [&] { return cudaFuncSetAttribute(kernel, which, value); });
}

// A launch that may begin while the kernel before it in the stream still runs:
// the kernel waits (pdl_wait) before it reads or writes anything but its own
// shared and tensor memory.
inline void overlapped(cudaLaunchConfig_t& cfg, cudaLaunchAttribute& at, unsigned grid, int threads, int smem, cudaStream_t st) {
  cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
}

}  // namespace emx
