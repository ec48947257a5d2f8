// paged_append.cu — the rows of a batch on their way from the q|k|v
// projection: per-head RMSNorm of q and k, the rotation of both to their
// positions, k and v to their pages of the cache, q to the attention.
//
// For a head x of row r at position p, D = head_dim:
//   n_d = x_d / sqrt(mean_d x_d^2 + eps) * w_d            (w given)
//   y_d         = n_d cos a_d - n_{d+D/2} sin a_d
//   y_{d+D/2}   = n_d sin a_d + n_{d+D/2} cos a_d,  a_d = p theta^(-2d/D), d < D/2
// all in fp32 and rounded to bf16 once.  Every byte of qkv is read once and
// every byte of q, k, v written once: memory bounds it, at few rows the
// latency of the row's own chain (indptr -> length -> page -> store).
//
// A far position's angle does not fit fp32 (p = 1e5 would leave errors of
// 1e-2 rad), so turns p * theta^(-2d/D) / 2pi are taken in fp64, their whole
// part is dropped there, and only the rest, in [-1/2, 1/2], goes to fp32.
//
// One warp per item, an item being some heads of one row.  A lane holds
// elements 4d..4d+3 of both halves of a head (two 8-byte loads, 128 contiguous
// bytes a half at D = 128): the pair that a rotation mixes sits in one lane,
// and its four angles serve every head of the row.
#include "paged_dev.cuh"

namespace emx {

namespace {

constexpr int kThreads = 256;

template <int HD>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const PagedAppendArgs a, int parts, int iters) {
  constexpr int LPH = HD / 8;    // lanes a head
  constexpr int HPI = 32 / LPH;  // heads a step of the warp
  constexpr int U = 4;           // steps whose loads are in flight together
  const PagedArgs& p = a.p;
  const int lane = threadIdx.x & 31;
  const int d0 = 4 * (lane % LPH), sub = lane / LPH;
  const int n_heads = p.n_q + 2 * p.n_kv;
  const int64_t items = (int64_t)p.n_rows * parts;
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  const int64_t first = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (first >= items) return;

  double turn[4];  // theta^(-2d/D) / 2pi of this lane's four pairs
#pragma unroll
  for (int e = 0; e < 4; ++e)
    turn[e] = exp2(a.log2_theta * (-2.0 * (d0 + e) / HD)) * 0.15915494309189533577;

  uint2 wq[2], wk[2];
  const bool norm_q = a.q_norm != nullptr, norm_k = a.k_norm != nullptr;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    wq[b] = norm_q ? *reinterpret_cast<const uint2*>(a.q_norm + d0 + b * (HD / 2)) : make_uint2(0u, 0u);
    wk[b] = norm_k ? *reinterpret_cast<const uint2*>(a.k_norm + d0 + b * (HD / 2)) : make_uint2(0u, 0u);
  }

  for (int64_t item = first; item < items; item += warps) {
    const int row = (int)(item / parts);
    const int it0 = (int)(item - (int64_t)row * parts) * iters;
    const bf16* src = a.qkv + (size_t)row * n_heads * HD;
    uint2 x[U][2];
    auto load = [&](int it) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = (it + u) * HPI + sub;
        const bool on = it + u < it0 + iters && h < n_heads;
#pragma unroll
        for (int b = 0; b < 2; ++b)
          x[u][b] = on ? __ldcs(reinterpret_cast<const uint2*>(src + (size_t)h * HD + d0 + b * (HD / 2)))
                       : make_uint2(0u, 0u);
      }
    };
    load(it0);
    const int i = warp_find_seq(p.indptr, p.n_seqs, row);
    if (i >= p.n_seqs || row < p.indptr[i]) continue;  // behind the last sequence: left as it was
    const SeqInfo s = load_seq(p, i, 0);
    if (!s.ok) {
      if (lane == 0) report_status(p.status, seq_status(p, i));
      continue;
    }
    const int pos = s.len - s.rows + (row - s.row0);
    const int page = p.table[(size_t)i * p.max_pages + pos / p.page_size];
    const bool store = page >= 0 && page < p.n_pages;
    if (!store && lane == 0) report_status(p.status, kDevBadPage);
    float sn[4], cs[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (a.rotate) {
        double t = (double)pos * turn[e];
        t -= rint(t);
        sincospif((float)(2.0 * t), &sn[e], &cs[e]);
      } else {
        sn[e] = 0.f;
        cs[e] = 1.f;
      }
    }
    for (int it = it0; it < it0 + iters; it += U) {
      if (it != it0) load(it);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = (it + u) * HPI + sub;
        const bool on = it + u < it0 + iters && h < n_heads;
        uint2 y[2] = {x[u][0], x[u][1]};
        float f[2][4];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          f[b][0] = __uint_as_float(x[u][b].x << 16);
          f[b][1] = __uint_as_float(x[u][b].x & 0xffff0000u);
          f[b][2] = __uint_as_float(x[u][b].y << 16);
          f[b][3] = __uint_as_float(x[u][b].y & 0xffff0000u);
        }
        float ss = 0.f;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) ss = fmaf(f[b][e], f[b][e], ss);
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const bool is_q = h < p.n_q, is_v = h >= p.n_q + p.n_kv;
        if (!is_v) {
          if (is_q ? norm_q : norm_k) {
            const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)HD), a.eps)));
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const uint2 w = is_q ? wq[b] : wk[b];
              f[b][0] *= inv * __uint_as_float(w.x << 16);
              f[b][1] *= inv * __uint_as_float(w.x & 0xffff0000u);
              f[b][2] *= inv * __uint_as_float(w.y << 16);
              f[b][3] *= inv * __uint_as_float(w.y & 0xffff0000u);
            }
          }
          float g[2][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            g[0][e] = a.rotate ? f[0][e] * cs[e] - f[1][e] * sn[e] : f[0][e];
            g[1][e] = a.rotate ? f[0][e] * sn[e] + f[1][e] * cs[e] : f[1][e];
          }
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            y[b].x = (uint32_t)f2bits(g[b][0]) | ((uint32_t)f2bits(g[b][1]) << 16);
            y[b].y = (uint32_t)f2bits(g[b][2]) | ((uint32_t)f2bits(g[b][3]) << 16);
          }
        }
        if (!on || (!is_q && !store)) continue;
        bf16* dst;
        if (is_q) {
          dst = a.q_out + ((size_t)row * p.n_q + h) * HD;
        } else {
          const int hk = is_v ? h - p.n_q - p.n_kv : h - p.n_q;
          dst = (is_v ? p.v : p.k) + (size_t)cache_row(page, p.n_kv, hk, p.page_size, pos % p.page_size) * HD;
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) *reinterpret_cast<uint2*>(dst + d0 + b * (HD / 2)) = y[b];
      }
    }
  }
}

}  // namespace

cudaError_t paged_append_launch(const PagedAppendArgs& a, int num_sms, cudaStream_t st) {
  const PagedArgs& p = a.p;
  const int hpi = 32 / (p.head_dim / 8);
  const int steps = (p.n_q + 2 * p.n_kv + hpi - 1) / hpi;
  // a row to a warp when the rows alone fill the SMs' warps; below that its
  // heads are spread over more warps, four steps (one batch of loads) at
  // least each, so that a few rows are not one warp's serial work
  const int64_t want = (int64_t)num_sms * 32;
  int parts = (int)((want + p.n_rows - 1) / p.n_rows);
  const int most = (steps + 3) / 4;
  if (parts > most) parts = most;
  const int iters = (steps + parts - 1) / parts;
  parts = (steps + iters - 1) / iters;
  const int64_t items = (int64_t)p.n_rows * parts;
  int64_t grid = (items + kThreads / 32 - 1) / (kThreads / 32);
  const int64_t cap = (int64_t)num_sms * 8;  // eight CTAs of eight warps fill an SM: more would only repeat the set-up
  if (grid > cap) grid = cap;
  if (p.head_dim == 128) paged_append_kernel<128><<<(int)grid, kThreads, 0, st>>>(a, parts, iters);
  else paged_append_kernel<64><<<(int)grid, kThreads, 0, st>>>(a, parts, iters);
  return cudaGetLastError();
}

}  // namespace emx
