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
// 8190 rows of 16 + 8 + 8 heads (134 MB): 27.4 us, 4.9 TB/s; the rest is
// instructions (issue slots 70% busy where a step took 170, now about 90).  Up to 500
// rows 4.2 to 5.7 us, a row's chain of latencies.
//
// One warp per item, an item being some heads of one row, in batches of four
// steps: of q, or two of k and the same two of v; a step is two heads (four at
// D = 64).  A lane holds elements 4d..4d+3 of both halves of a head (two 8-byte
// loads, 128 contiguous bytes a half at D = 128): the pair that a rotation mixes
// sits in one lane, and its four angles, multiplied into the norm's weights once a
// row, serve every head of the row.  A batch's loads are in flight together, and 32
// warps an SM.  The fp32 steps go two to an instruction (f32x2).
#include "paged_dev.cuh"

namespace emx {

namespace {

constexpr int kThreads = 256;
constexpr int kSteps = 4;  // of a batch

__device__ __forceinline__ uint64_t unpack(uint32_t u) { return pair32(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
__device__ __forceinline__ uint32_t pack(uint64_t v) {
  float a, b;
  split32(v, a, b);
  const __nv_bfloat162 two = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&two);
}

// The norm's weights (w, or 1) times the row's cosines and sines.
struct Turn {
  uint64_t c_lo[2], s_lo[2], c_hi[2], s_hi[2];  // s_hi negated
};

template <int HD, bool TURN>
__global__ void __launch_bounds__(kThreads, 4) paged_append_kernel(const PagedAppendArgs a, int parts, int each) {
  constexpr int LPH = HD / 8;    // lanes a head
  constexpr int HPI = 32 / LPH;  // heads a step
  __shared__ double turns[HD / 2];  // theta^(-2d/D) / 2pi
  const PagedArgs& p = a.p;
  const int lane = threadIdx.x & 31;
  const int d0 = 4 * (lane % LPH), sub = lane / LPH;
  const int n_heads = p.n_q + 2 * p.n_kv;
  const int q_batches = ceil_div(p.n_q, HPI * kSteps), batches = q_batches + ceil_div(p.n_kv, HPI * kSteps / 2);
  if (TURN && threadIdx.x < HD / 2) turns[threadIdx.x] = exp2(a.log2_theta * (-2.0 * threadIdx.x / HD)) * 0.15915494309189533577;
  __syncthreads();
  pdl_wait();
  pdl_trigger();

  const int64_t items = (int64_t)p.n_rows * parts;
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t item = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); item < items; item += warps) {
    const int row = share_of(item, parts);
    const int b0 = (int)(item - (int64_t)row * parts) * each, b1 = min(b0 + each, batches);
    const bf16* src = a.qkv + (size_t)row * n_heads * HD + d0;
    uint2 x[kSteps][2];
    // head of slot u in batch b: of q, or of k (slots 0, 1) and v (2, 3)
    auto q_head = [&](int b, int u) { return (b * kSteps + u) * HPI + sub; };
    auto kv_head = [&](int b, int u) { return ((b - q_batches) * (kSteps / 2) + (u & 1)) * HPI + sub; };
    auto load = [&](int b) {
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        int h = q_head(b, u);
        bool on = h < p.n_q;
        if (b >= q_batches) {
          h = kv_head(b, u);
          on = h < p.n_kv;
          h += p.n_q + (u >> 1) * p.n_kv;
        }
#pragma unroll
        for (int y = 0; y < 2; ++y)
          x[u][y] = on ? __ldcs(reinterpret_cast<const uint2*>(src + h * HD + y * (HD / 2))) : make_uint2(0u, 0u);
      }
    };
    load(b0);
    const int i = warp_find_seq(p.indptr, p.n_seqs, row);
    if (i >= p.n_seqs || row < p.indptr[i]) continue;  // behind the last sequence: left as it was
    const SeqInfo s = load_seq(p, i, 0);
    if (!s.ok) continue;
    const int pos = s.len - s.rows + (row - s.row0);
    const int pg = pos / p.page_size, page = p.table[(size_t)i * p.max_pages + pg];
    const bool store = page >= 0 && page < p.n_pages;
    if (!store && lane == 0) report_status(p.status, kDevBadPage);
    const size_t at = store ? (size_t)cache_row(page, p.n_kv, 0, p.page_size, pos - pg * p.page_size) * HD + d0 : 0;
    float sn[4], cs[4];
    if (TURN) {
      // a lane's four angles are those of the lanes with the same columns of the step's other heads: each works out its part
      constexpr int kMine = 4 / HPI;
      float my_sn[kMine], my_cs[kMine];
#pragma unroll
      for (int e = 0; e < kMine; ++e) {
        double t = (double)pos * turns[d0 + sub * kMine + e];
        t -= rint(t);
        sincospif((float)(2.0 * t), &my_sn[e], &my_cs[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sn[e] = __shfl_sync(0xffffffffu, my_sn[e % kMine], e / kMine * LPH + lane % LPH);
        cs[e] = __shfl_sync(0xffffffffu, my_cs[e % kMine], e / kMine * LPH + lane % LPH);
      }
    }
    // y_d = inv (x_d c_lo + x_{d+D/2} s_hi), y_{d+D/2} = inv (x_d s_lo + x_{d+D/2} c_hi)
    Turn t;
    auto weigh = [&](const bf16* w) {
      uint2 lo = make_uint2(0x3f803f80u, 0x3f803f80u), hi = lo;  // ones
      if (w) {
        lo = *reinterpret_cast<const uint2*>(w + d0);
        hi = *reinterpret_cast<const uint2*>(w + d0 + HD / 2);
      }
      const uint64_t l[2] = {unpack(lo.x), unpack(lo.y)}, h[2] = {unpack(hi.x), unpack(hi.y)};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        t.c_lo[e] = TURN ? mul2(pair32(cs[2 * e], cs[2 * e + 1]), l[e]) : l[e];
        t.c_hi[e] = TURN ? mul2(pair32(cs[2 * e], cs[2 * e + 1]), h[e]) : h[e];
        if (TURN) {
          t.s_lo[e] = mul2(pair32(sn[2 * e], sn[2 * e + 1]), l[e]);
          t.s_hi[e] = mul2(pair32(-sn[2 * e], -sn[2 * e + 1]), h[e]);
        }
      }
    };
    // a head: its norm (w given) and rotation
    auto turn = [&](uint2 (&v)[2], bool norm) {
      const uint64_t lo[2] = {unpack(v[0].x), unpack(v[0].y)}, hi[2] = {unpack(v[1].x), unpack(v[1].y)};
      float inv = 1.f;
      if (norm) {
        float s0, s1;
        split32(fma2(lo[0], lo[0], fma2(lo[1], lo[1], fma2(hi[0], hi[0], mul2(hi[1], hi[1])))), s0, s1);
        float ss = s0 + s1;
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        inv = rsqrtf(fmaf(ss, 1.0f / HD, a.eps));  // 2 ulp of fp32
      }
      const uint64_t by = pair32(inv, inv);
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // without a rotation x passes untouched: 0 * inf would not be 0
        uint64_t y0 = mul2(lo[e], t.c_lo[e]), y1 = mul2(hi[e], t.c_hi[e]);
        if (TURN) {
          y0 = fma2(hi[e], t.s_hi[e], y0);
          y1 = fma2(lo[e], t.s_lo[e], y1);
        }
        u[e] = pack(mul2(y0, by));
        u[2 + e] = pack(mul2(y1, by));
      }
      v[0] = make_uint2(u[0], u[1]);
      v[1] = make_uint2(u[2], u[3]);
    };
    auto put = [&](bf16* dst, const uint2 (&v)[2]) {
      *reinterpret_cast<uint2*>(dst) = v[0];
      *reinterpret_cast<uint2*>(dst + HD / 2) = v[1];
    };
    int b = b0;
    if (b < q_batches) {
      bf16* dst = a.q_out + (size_t)row * p.n_q * HD + d0;
      weigh(a.q_norm);
      for (; b < min(b1, q_batches); ++b) {
        if (b != b0) load(b);
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
          turn(x[u], a.q_norm != nullptr);
          const int h = q_head(b, u);
          if (h < p.n_q) put(dst + h * HD, x[u]);
        }
      }
    }
    if (b >= b1) continue;
    weigh(a.k_norm);
    for (; b < b1; ++b) {
      if (b != b0) load(b);
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        if (u < kSteps / 2) turn(x[u], a.k_norm != nullptr);
        const int h = kv_head(b, u);
        if (store && h < p.n_kv) put((u < kSteps / 2 ? p.k : p.v) + at + (size_t)h * p.page_size * HD, x[u]);
      }
    }
  }
  // sequences out of order report, those among them too that no row was found to belong to
  if (blockIdx.x == gridDim.x - 1)
    for (int i = threadIdx.x; i < p.n_seqs; i += kThreads)
      if (!load_seq(p, i, 0).ok) report_status(p.status, seq_status(p, i));
}

template <int HD, bool TURN>
cudaError_t launch(const PagedAppendArgs& a, int num_sms, cudaStream_t st) {
  const PagedArgs& p = a.p;
  constexpr int kHeads = 256 / HD * kSteps;  // of a batch of q
  const int batches = ceil_div(p.n_q, kHeads) + ceil_div(p.n_kv, kHeads / 2);
  // a row to a warp when the rows alone fill the SMs' warps (two warps a row took
  // 38.9 us where one took 33.0: each works out the row's angles); below that its
  // batches are spread over more warps (4, 64 and 500 rows of 40 heads: 4.3, 4.3 and
  // 5.7 us, with a warp a row 7.2, 8.1 and 9.4)
  int parts = min(batches, ceil_div((int64_t)num_sms * 32, p.n_rows));
  const int each = ceil_div(batches, parts);
  parts = ceil_div(batches, each);
  // two rounds of four CTAs an SM: beyond that a warp takes further items
  const int64_t grid = min(((int64_t)p.n_rows * parts + kThreads / 32 - 1) / (kThreads / 32), (int64_t)num_sms * 8);
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute at;
  overlapped(cfg, at, (unsigned)grid, kThreads, 0, st);
  return cudaLaunchKernelEx(&cfg, paged_append_kernel<HD, TURN>, a, parts, each);
}

}  // namespace

cudaError_t paged_append_launch(const PagedAppendArgs& a, int num_sms, cudaStream_t st) {
  if (a.p.head_dim == 128) return a.rotate ? launch<128, true>(a, num_sms, st) : launch<128, false>(a, num_sms, st);
  return a.rotate ? launch<64, true>(a, num_sms, st) : launch<64, false>(a, num_sms, st);
}

}  // namespace emx
