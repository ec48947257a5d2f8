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
// One warp per item, an item being some heads of one row, in steps of two heads
// (four at D = 64) of one kind.  A lane holds elements 4d..4d+3 of both halves of
// a head (two 8-byte loads, 128 contiguous bytes a half at D = 128): the pair
// that a rotation mixes sits in one lane, and its four angles, multiplied into
// the norm's weights once a row, serve every head of the row.  Four steps' loads
// are in flight together, and 32 warps an SM.
#include "paged_dev.cuh"

namespace emx {

namespace {

constexpr int kThreads = 256;
constexpr int kSteps = 4;  // whose loads are in flight together

__device__ __forceinline__ void unpack(const uint2& u, float (&f)[4]) {
  f[0] = __uint_as_float(u.x << 16);
  f[1] = __uint_as_float(u.x & 0xffff0000u);
  f[2] = __uint_as_float(u.y << 16);
  f[3] = __uint_as_float(u.y & 0xffff0000u);
}

__device__ __forceinline__ uint2 pack(const float (&f)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 4) paged_append_kernel(const PagedAppendArgs a, int parts, int iters) {
  constexpr int LPH = HD / 8;    // lanes a head
  constexpr int HPI = 32 / LPH;  // heads a step
  __shared__ double turns[HD / 2];  // theta^(-2d/D) / 2pi
  const PagedArgs& p = a.p;
  const int lane = threadIdx.x & 31;
  const int d0 = 4 * (lane % LPH), sub = lane / LPH;
  const int n_heads = p.n_q + 2 * p.n_kv;
  const int q_steps = (p.n_q + HPI - 1) / HPI, k_steps = (p.n_kv + HPI - 1) / HPI, steps = q_steps + 2 * k_steps;
  if (threadIdx.x < HD / 2) turns[threadIdx.x] = exp2(a.log2_theta * (-2.0 * threadIdx.x / HD)) * 0.15915494309189533577;
  __syncthreads();
  pdl_wait();
  pdl_trigger();

  const int64_t items = (int64_t)p.n_rows * parts;
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t item = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); item < items; item += warps) {
    const int row = (int)(item / parts);
    const int it0 = (int)(item - (int64_t)row * parts) * iters, it1 = min(it0 + iters, steps);
    const bf16* src = a.qkv + (size_t)row * n_heads * HD + d0;
    // the head of this lane in step `it` (in q | k | v), and whether there is one
    auto head_of = [&](int it, bool& on) {
      const int kind = it < q_steps ? 0 : it < q_steps + k_steps ? 1 : 2;
      const int h = (it - (kind == 0 ? 0 : q_steps + (kind - 1) * k_steps)) * HPI + sub;
      on = it < it1 && h < (kind == 0 ? p.n_q : p.n_kv);
      return h + (kind == 0 ? 0 : p.n_q + (kind - 1) * p.n_kv);
    };
    uint2 x[kSteps][2];
    auto load = [&](int it) {
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        bool on;
        const int h = head_of(it + u, on);
#pragma unroll
        for (int b = 0; b < 2; ++b)
          x[u][b] = on ? __ldcs(reinterpret_cast<const uint2*>(src + (size_t)h * HD + b * (HD / 2))) : make_uint2(0u, 0u);
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
    const size_t at = store ? (size_t)cache_row(page, p.n_kv, 0, p.page_size, pos % p.page_size) * HD + d0 : 0;
    // a lane's four angles are those of the lanes with the same columns of the step's other heads: each works out its part
    constexpr int kMine = 4 / HPI;
    float sn[4], cs[4], my_sn[kMine], my_cs[kMine];
#pragma unroll
    for (int x = 0; x < kMine; ++x) {
      my_sn[x] = 0.f;
      my_cs[x] = 1.f;
      if (a.rotate) {
        double t = (double)pos * turns[d0 + sub * kMine + x];
        t -= rint(t);
        sincospif((float)(2.0 * t), &my_sn[x], &my_cs[x]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sn[e] = __shfl_sync(0xffffffffu, my_sn[e % kMine], e / kMine * LPH + lane % LPH);
      cs[e] = __shfl_sync(0xffffffffu, my_cs[e % kMine], e / kMine * LPH + lane % LPH);
    }
    // y_d = inv (x_d c0 - x_{d+D/2} s1), y_{d+D/2} = inv (x_d s0 + x_{d+D/2} c1), the weights in c and s
    float c0[4], s0[4], c1[4], s1[4];
    auto weigh = [&](const bf16* w) {
      float w0[4] = {1.f, 1.f, 1.f, 1.f}, w1[4] = {1.f, 1.f, 1.f, 1.f};
      if (w) {
        unpack(*reinterpret_cast<const uint2*>(w + d0), w0);
        unpack(*reinterpret_cast<const uint2*>(w + d0 + HD / 2), w1);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c0[e] = cs[e] * w0[e];
        s0[e] = sn[e] * w0[e];
        c1[e] = cs[e] * w1[e];
        s1[e] = sn[e] * w1[e];
      }
    };
    int weighed = -1;
    for (int it = it0; it < it1; it += kSteps) {
      if (it != it0) load(it);
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        if (it + u >= it1) break;
        bool on;
        const int h = head_of(it + u, on), kind = it + u < q_steps ? 0 : it + u < q_steps + k_steps ? 1 : 2;
        if (kind < 2) {
          const bf16* w = kind == 0 ? a.q_norm : a.k_norm;
          if (weighed != kind) weigh(w);
          weighed = kind;
          float f[2][4], y[2][4];
          unpack(x[u][0], f[0]);
          unpack(x[u][1], f[1]);
          float inv = 1.f;
          if (w) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) ss = fmaf(f[0][e], f[0][e], fmaf(f[1][e], f[1][e], ss));
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            inv = rsqrtf(fmaf(ss, 1.0f / HD, a.eps));  // 2 ulp of fp32
          }
          const bool norm = w != nullptr, turn = a.rotate != 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // without a rotation x passes untouched: 0 * inf would not be 0
            const float r0 = turn ? fmaf(f[0][e], c0[e], -(f[1][e] * s1[e])) : f[0][e] * c0[e];
            const float r1 = turn ? fmaf(f[0][e], s0[e], f[1][e] * c1[e]) : f[1][e] * c1[e];
            y[0][e] = norm ? r0 * inv : r0;
            y[1][e] = norm ? r1 * inv : r1;
          }
          x[u][0] = pack(y[0]);
          x[u][1] = pack(y[1]);
        }
        if (!on || (kind > 0 && !store)) continue;
        bf16* dst;
        if (kind == 0) {
          dst = a.q_out + ((size_t)row * p.n_q + h) * HD + d0;
        } else {
          const int hk = h - p.n_q - (kind - 1) * p.n_kv;
          dst = (kind == 1 ? p.k : p.v) + at + (size_t)hk * p.page_size * HD;
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) *reinterpret_cast<uint2*>(dst + b * (HD / 2)) = x[u][b];
      }
    }
  }
}

}  // namespace

cudaError_t paged_append_launch(const PagedAppendArgs& a, int num_sms, cudaStream_t st) {
  const PagedArgs& p = a.p;
  const int hpi = 32 / (p.head_dim / 8);
  const int steps = (p.n_q + hpi - 1) / hpi + 2 * ((p.n_kv + hpi - 1) / hpi);
  // a row to a warp when the rows alone fill the SMs' warps; below that its
  // heads are spread over more warps, four steps (one batch of loads) at
  // least each, so that a few rows are not one warp's serial work
  const int64_t want = (int64_t)num_sms * 32;
  int parts = (int)((want + p.n_rows - 1) / p.n_rows);
  const int most = (steps + kSteps - 1) / kSteps;
  if (parts > most) parts = most;
  const int iters = (steps + parts - 1) / parts;
  parts = (steps + iters - 1) / iters;
  const int64_t items = (int64_t)p.n_rows * parts;
  int64_t grid = (items + kThreads / 32 - 1) / (kThreads / 32);
  const int64_t cap = (int64_t)num_sms * 8;  // two rounds of four CTAs an SM: beyond that a warp takes further items
  if (grid > cap) grid = cap;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute at;
  overlapped(cfg, at, (unsigned)grid, kThreads, 0, st);
  return p.head_dim == 128 ? cudaLaunchKernelEx(&cfg, paged_append_kernel<128>, a, parts, iters)
                           : cudaLaunchKernelEx(&cfg, paged_append_kernel<64>, a, parts, iters);
}

}  // namespace emx
