// verify.cu — drafted tokens against the target's probabilities, from given
// random numbers (speculative sampling).
//
// Sequence i has drafts x_0 .. x_{c-1}, drawn from q_0 .. q_{c-1}; p_j is the
// target's distribution where x_j stands, p_c the one after the last draft.
//   draft j is accepted while u_j q_j(x_j) < p_j(x_j)        (probability min(1, p/q))
//   n = the accepted ones; the next token is drawn from
//     r = max(p_n - q_n, 0)   when draft n was refused (p_n if r is 0 everywhere)
//     r = p_n                 when none was
//   as the first index whose running sum of r exceeds u_last * sum r,
// which leaves every token distributed as p.  Comparisons and sums are in
// fp64: u q is exact there (24 + 24 bits), and a running sum over 10^5 fp32
// values keeps a border's place to ~1e-11 of the mass.
//
// Only the row that the next token is drawn from is read whole: V values of p
// and, after a refusal, V of q, once; that stream bounds a batch, and one
// sequence the latency of its chain (drafts -> their p and q -> the row ->
// the sums of all CTAs -> the token).  A thread-block cluster has a sequence:
// each CTA a slice of the vocabulary, each warp a run of it, the sums meet in
// distributed shared memory, and the one warp whose run the token lies in
// walks it again (out of L2) with a running sum.
#include <cooperative_groups.h>

#include "paged.cuh"

namespace emx {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

template <typename T>
__device__ __forceinline__ float val(T v);
template <>
__device__ __forceinline__ float val<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ float val<bf16>(bf16 v) {
  return bf2f(v);
}

// Mass of a value: nothing but a positive, finite one has any.
__device__ __forceinline__ double mass(float v) { return v > 0.f && v < INFINITY ? (double)v : 0.0; }

// r at one index: p there, less what the draft had.
__device__ __forceinline__ double rest(float p, float q) {
  const double d = mass(p) - mass(q);
  return d > 0.0 ? d : 0.0;
}

// Values [at, at + VEC) of a row, one vector load where VEC > 1.
template <typename T, int VEC>
__device__ __forceinline__ void load(const T* row, int at, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = val<T>(row[at]);
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(row + at);
    const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 4) {
        v[e] = __uint_as_float(x[e]);
      } else {
        v[2 * e] = __uint_as_float(x[e] << 16);
        v[2 * e + 1] = __uint_as_float(x[e] & 0xffff0000u);
      }
    }
  }
}

struct Shared {
  int accepted, count, stop;
  double warp_sum[kWarps];
  double sum;  // of this CTA's slice, read by the cluster
};

// r over [at, at + VEC) of the row, after `how`: 0 p alone, 1 p - q, 2 p less 1 at the index `one`.
template <typename T, int VEC>
__device__ __forceinline__ void rests(const T* p, const T* q, int how, int one, int at, double (&r)[VEC]) {
  float a[VEC];
  load<T, VEC>(p, at, a);
  if (how == 1) {
    float b[VEC];
    load<T, VEC>(q, at, b);
#pragma unroll
    for (int e = 0; e < VEC; ++e) r[e] = rest(a[e], b[e]);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) r[e] = how == 2 && at + e == one ? rest(a[e], 1.f) : mass(a[e]);
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) verify_kernel(const VerifyArgs a) {
  __shared__ Shared S;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int i = blockIdx.x / parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int m = a.n_draft;
  const int* tokens = a.tokens + (size_t)i * m;
  const float* u = a.uniforms + (size_t)i * (m + 1);
  const T* target = static_cast<const T*>(a.target) + (size_t)i * (m + 1) * a.vocab;
  const T* draft = a.draft ? static_cast<const T*>(a.draft) + (size_t)i * m * a.vocab : nullptr;

  // ---- the accepted drafts (every CTA of the cluster finds them for itself)
  if (warp == 0) {
    int count = a.counts ? a.counts[i] : m;
    if (count > m) count = m;
    int n = 0;
    for (int j0 = 0; j0 < count; j0 += 32) {
      const int j = j0 + lane;
      bool ok = true;
      if (j < count) {
        const int x = tokens[j];
        if (x < 0 || x >= a.vocab) {
          ok = false;
          report_status(a.status, kDevBadToken);
        } else {
          const float q = draft ? val<T>(draft[(size_t)j * a.vocab + x]) : 1.f;
          ok = (double)u[j] * (double)q < (double)val<T>(target[(size_t)j * a.vocab + x]);
        }
      }
      const unsigned bad = __ballot_sync(0xffffffffu, !ok);
      if (bad) {
        n = j0 + __ffs(bad) - 1;
        break;
      }
      n = min(count, j0 + 32);
    }
    if (lane == 0) {
      S.accepted = n;
      S.count = count;
    }
  }
  __syncthreads();
  const int n = S.accepted, count = S.count;
  int* out = a.out + (size_t)i * (m + 1);
  if (count < 0) {  // an empty slot
    if (part == 0) {
      for (int j = tid; j <= m; j += kThreads) out[j] = -1;
      if (tid == 0) a.accepted[i] = 0;
    }
    return;  // the whole cluster
  }
  if (part == 0) {
    for (int j = tid; j <= m; j += kThreads)
      if (j != n) out[j] = j < n ? tokens[j] : -1;
    if (tid == 0) a.accepted[i] = n;
  }

  // ---- this warp's run [b, e) of the row
  const T* p = target + (size_t)n * a.vocab;
  const T* q = draft && n < count ? draft + (size_t)n * a.vocab : nullptr;
  const int one = !draft && n < count ? tokens[n] : -1;
  constexpr int kTile = 32 * VEC;
  const int tiles = (a.vocab + kTile - 1) / kTile, each = (tiles + parts * kWarps - 1) / (parts * kWarps);
  const int run = part * kWarps + warp;
  const int b = min((int64_t)run * each, (int64_t)tiles) * kTile;
  const int e = min(min((int64_t)(run + 1) * each, (int64_t)tiles) * kTile, (int64_t)a.vocab);
  for (int how = n < count ? (draft ? 1 : 2) : 0;; how = 0) {
    double sum = 0.0;
    int at = b + lane * VEC;
    // four tiles' loads in flight
    for (; at + 3 * kTile + VEC <= e; at += 4 * kTile) {
      double r[4][VEC];
#pragma unroll
      for (int k = 0; k < 4; ++k) rests<T, VEC>(p, q, how, one, at + k * kTile, r[k]);
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int x = 0; x < VEC; ++x) sum += r[k][x];
    }
    for (; at + VEC <= e; at += kTile) {  // VEC divides the vocabulary
      double r[VEC];
      rests<T, VEC>(p, q, how, one, at, r);
#pragma unroll
      for (int x = 0; x < VEC; ++x) sum += r[x];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) S.warp_sum[warp] = sum;
    __syncthreads();
    if (tid == 0) {
      double t = 0.0;
      for (int k = 0; k < kWarps; ++k) t += S.warp_sum[k];
      S.sum = t;
    }
    cluster.sync();
    // every warp takes the sums of all CTAs, in order
    double before = 0.0, total = 0.0;
    int last = -1;  // the last CTA with any mass
    for (int k = 0; k < parts; ++k) {
      const double t = *cluster.map_shared_rank(&S.sum, k);
      if (k < part) before += t;
      total += t;
      if (t > 0.0) last = k;
    }
    if (total <= 0.0) {
      if (how == 0) {
        if (part == 0 && tid == 0) out[n] = -1;  // no mass at all
        break;
      }
      cluster.sync();  // all have read the sums of this turn
      continue;        // nothing left of p - q: p itself
    }
    // The token's CTA is the first whose end passes the goal (the last with
    // mass if rounding leaves none), its warp and index likewise.
    const double goal = (double)u[m] * total;
    int mine = 0;
    if (before + S.sum > goal || part == last) {
      bool earlier = false;  // does an earlier CTA's end pass it?
      double end = 0.0;
      for (int k = 0; k < part; ++k) {
        end += *cluster.map_shared_rank(&S.sum, k);
        earlier |= end > goal;
      }
      mine = !earlier && S.sum > 0.0;
    }
    if (mine) {
      double from = before;
      int at_warp = -1, last_warp = -1;
      double start = 0.0;
      for (int k = 0; k < kWarps; ++k) {
        const double t = S.warp_sum[k];
        if (t > 0.0) {
          last_warp = k;
          if (at_warp < 0 && from + t > goal) {
            at_warp = k;
            start = from;
          }
        }
        from += t;
      }
      if (at_warp < 0) {
        at_warp = last_warp;
        start = INFINITY;  // rounding: the last index with mass
      }
      if (warp == at_warp) {
        int found = -1, fallback = -1;
        double base = start;
        for (int t0 = b; t0 < e && found < 0; t0 += kTile) {
          const int at2 = t0 + lane * VEC;
          double r[VEC];
          if (at2 + VEC <= e) {
            rests<T, VEC>(p, q, how, one, at2, r);
          } else {
#pragma unroll
            for (int x = 0; x < VEC; ++x) r[x] = 0.0;
          }
          double own = 0.0;
          int lastx = -1;
#pragma unroll
          for (int x = 0; x < VEC; ++x) {
            own += r[x];
            if (r[x] > 0.0) lastx = at2 + x;
          }
          double incl = own;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
          }
          if (start < INFINITY) {
            double s = base + (incl - own);
            int hit = -1;
#pragma unroll
            for (int x = 0; x < VEC; ++x) {
              s += r[x];
              if (hit < 0 && r[x] > 0.0 && s > goal) hit = at2 + x;
            }
            const unsigned who = __ballot_sync(0xffffffffu, hit >= 0);
            if (who) found = __shfl_sync(0xffffffffu, hit, __ffs(who) - 1);
            base += __shfl_sync(0xffffffffu, incl, 31);
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) lastx = max(lastx, __shfl_xor_sync(0xffffffffu, lastx, o));
          fallback = max(fallback, lastx);
        }
        if (lane == 0) out[n] = found >= 0 ? found : fallback;
      }
    }
    break;
  }
  cluster.sync();  // no CTA leaves while another may read its sum
}

template <typename T, int VEC>
cudaError_t run(const VerifyArgs& a, int parts, cudaStream_t st) {
  static cudaError_t once =
      cudaFuncSetAttribute(verify_kernel<T, VEC>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (once != cudaSuccess) return once;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n_seqs * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, verify_kernel<T, VEC>, a);
}

}  // namespace

cudaError_t verify_launch(const VerifyArgs& a, int num_sms, cudaStream_t st) {
  const int parts = 8;
  const int vec = a.is_bf16 ? 8 : 4;
  // rows keep the first one's 16-byte alignment only if they are whole vectors long
  const bool whole = a.vocab % vec == 0 && ((reinterpret_cast<uintptr_t>(a.target) | reinterpret_cast<uintptr_t>(a.draft)) & 15) == 0;
  if (a.is_bf16) return whole ? run<bf16, 8>(a, parts, st) : run<bf16, 1>(a, parts, st);
  return whole ? run<float, 4>(a, parts, st) : run<float, 1>(a, parts, st);
}

}  // namespace emx
