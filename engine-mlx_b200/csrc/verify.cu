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
// values keeps a border's place to ~1e-11 of the mass.  (Of p - q, its rounding to
// fp32 is summed in fp64 and what that leaves, below 2^-24 of it, in fp32 beside.)
//
// Only the row that the next token is drawn from is read whole: V values of p
// and, after a refusal, V of q, once; that stream bounds a batch, and one
// sequence the latency of its chain (drafts -> their p and q -> the row ->
// the sums of all CTAs -> the token).  A thread-block cluster has a sequence:
// each CTA a slice of the vocabulary, each warp a run of it.  Every CTA stores
// its sum in all CTAs' shared memory before the one cluster barrier, so nothing
// remote is touched behind it; the CTA whose slice holds the token then walks
// the run of the warp that does, all its threads together, out of L2.
//
// 64 sequences over 151936 fp32 values, p and q (78 MB): 23.4 us, 3.3 TB/s, half of
// which are the chain's other links (7.0 us for one sequence: the drafts' two
// dependent loads, the row, two reductions, the walk).
#include <cooperative_groups.h>

#include "paged_dev.cuh"

namespace emx {

namespace {

namespace cg = cooperative_groups;

constexpr int kMost = 16;  // CTAs of a cluster
constexpr int kLoads = 4;  // steps whose loads are in flight together

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
__device__ __forceinline__ float mass(float v) { return v > 0.f && v < INFINITY ? v : 0.f; }

// Sixteen bytes of a row (VEC values), or one value.
template <typename T, int VEC>
struct Raw {
  uint4 u;
  __device__ __forceinline__ void load(const T* p) { u = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ float get(int e) const {
    const uint32_t x[4] = {u.x, u.y, u.z, u.w};
    if constexpr (sizeof(T) == 4) return __uint_as_float(x[e]);
    else return __uint_as_float(e & 1 ? x[e >> 1] & 0xffff0000u : x[e >> 1] << 16);
  }
};
template <typename T>
struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ float get(int) const { return val<T>(v); }
};

// r at one index: p there, less q (both finite and not negative or without
// mass); in fp64 exact wherever their exponents are within 29 of each other.
__device__ __forceinline__ double rest(float p, float q) {
  const float a = mass(p), b = mass(q);
  return a > b ? (double)a - (double)b : 0.0;
}

template <int WARPS>
struct Shared {
  int accepted, count;
  double warp_sum[WARPS];
  double cta_sum[2][kMost];  // of the cluster's CTAs, by turn
  double scan[WARPS];
  int found;
};

// Inclusive sum over the lanes, right in the first N.
template <int N = 32>
__device__ __forceinline__ double warp_scan(double v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < N; o <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

template <typename T, int VEC, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) verify_kernel(const VerifyArgs a) {
  constexpr int kWarps = THREADS / 32;
  constexpr int kTile = 32 * VEC;  // values of one step of a warp
  __shared__ Shared<kWarps> S;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int i = blockIdx.x / parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int m = a.n_draft;
  const int* tokens = a.tokens + (size_t)i * m;
  const float* u = a.uniforms + (size_t)i * (m + 1);
  const T* target = static_cast<const T*>(a.target) + (size_t)i * (m + 1) * a.vocab;
  const T* draft = a.draft ? static_cast<const T*>(a.draft) + (size_t)i * m * a.vocab : nullptr;
  // nobody stores into a CTA that has not begun: arrives here, waits before the stores
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  auto all_began = [] { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); };
  pdl_wait();
  pdl_trigger();

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
      S.found = -1;
    }
  }
  __syncthreads();
  const int n = S.accepted, count = S.count;
  int* out = a.out + (size_t)i * (m + 1);
  if (count < 0) {  // an empty slot
    if (part == 0) {
      for (int j = tid; j <= m; j += THREADS) out[j] = -1;
      if (tid == 0) a.accepted[i] = 0;
    }
    all_began();
    return;  // the whole cluster
  }
  if (part == 0) {
    for (int j = tid; j <= m; j += THREADS)
      if (j != n) out[j] = j < n ? tokens[j] : -1;
    if (tid == 0) a.accepted[i] = n;
  }

  // ---- the sums: this warp's run is [begin(run), begin(run + 1)) of the row
  const T* p = target + (size_t)n * a.vocab;
  const T* q = draft && n < count ? draft + (size_t)n * a.vocab : nullptr;
  const int one = !draft && n < count ? tokens[n] : -1;
  const int tiles = (a.vocab + kTile - 1) / kTile, each = (tiles + parts * kWarps - 1) / (parts * kWarps);
  auto begin = [&](int run) { return (int)min((int64_t)run * each * kTile, (int64_t)a.vocab); };
  const int b = begin(part * kWarps + warp), e = begin(part * kWarps + warp + 1);
  // r of value x of a vector at `at`; minus: p - q, else p (less 1 at the draft)
  auto r_of = [&](const Raw<T, VEC>& x, const Raw<T, VEC>& y, bool minus, bool certain, int at, int k) {
    return minus ? rest(x.get(k), y.get(k)) : certain && at + k == one ? rest(x.get(k), 1.f) : (double)mass(x.get(k));
  };
  for (int turn = 0;; ++turn) {
    const bool minus = turn == 0 && q, certain = turn == 0 && one >= 0;
    constexpr int U = kLoads;
    double sums[U] = {};  // one chain of additions would take longer than the loads
    float rests[U] = {};
    for (int at0 = b + lane * VEC; at0 < e; at0 += U * kTile) {
      Raw<T, VEC> x[U], y[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (at0 + k * kTile < e) {  // VEC divides the vocabulary, and the runs' ends
          x[k].load(p + at0 + k * kTile);
          if (minus) y[k].load(q + at0 + k * kTile);
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (at0 + k * kTile < e)
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            // An SM converts 16 values to fp64 a clock, so p - q goes there once: rounded to fp32, and what the
            // rounding left (exact: a - b = d + e for a > b) is summed beside, 2^-24 of it in 24 bits.
            if (minus) {
              const float f = mass(x[k].get(v)), g = mass(y[k].get(v)), d = f - g;
              if (d > 0.f) {
                sums[k] += (double)d;
                rests[k] += (f - d) - g;
              }
            } else {
              sums[k] += r_of(x[k], y[k], minus, certain, at0 + k * kTile, v);
            }
          }
    }
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < U; ++k) sum += sums[k] + (double)rests[k];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) S.warp_sum[warp] = sum;
    __syncthreads();
    // every warp has the CTA's warps' running sums in its lanes
    const double w_sum = lane < kWarps ? S.warp_sum[lane] : 0.0, w_incl = warp_scan<kWarps>(w_sum);
    const double cta = __shfl_sync(0xffffffffu, w_incl, kWarps - 1);
    if (turn == 0) all_began();
    if (tid < parts) *cluster.map_shared_rank(&S.cta_sum[turn & 1][part], tid) = cta;
    cluster.sync();
    // ... and, in the same way, the cluster's CTAs'
    const double c_sum = lane < parts ? S.cta_sum[turn & 1][lane] : 0.0, c_incl = warp_scan<kMost>(c_sum);
    const double total = __shfl_sync(0xffffffffu, c_incl, kMost - 1);
    if (!(total > 0.0)) {
      if (minus || certain) continue;  // nothing left of p - q: p itself
      if (part == 0 && tid == 0) out[n] = -1;  // no mass at all
      return;
    }
    // The token's CTA is the first whose running sum passes the goal (where
    // rounding leaves none, the last with mass), its warp and index likewise.
    const double goal = (double)u[m] * total;
    const unsigned c_past = __ballot_sync(0xffffffffu, lane < parts && c_sum > 0.0 && c_incl > goal);
    const unsigned c_any = __ballot_sync(0xffffffffu, c_sum > 0.0);
    const int owner = c_past ? __ffs(c_past) - 1 : 31 - __clz(c_any);
    if (owner != part) return;
    const double before = __shfl_sync(0xffffffffu, c_incl - c_sum, part);
    const unsigned w_past = __ballot_sync(0xffffffffu, lane < kWarps && before + w_incl > goal && w_sum > 0.0);
    const unsigned w_any = __ballot_sync(0xffffffffu, w_sum > 0.0);
    const int run = w_past ? __ffs(w_past) - 1 : 31 - __clz(w_any);
    double base = before + __shfl_sync(0xffffffffu, w_incl - w_sum, run);
    const int rb = begin(part * kWarps + run), re = begin(part * kWarps + run + 1);
    // ---- the index: the CTA walks the run, VEC values a thread
    int fallback = -1;
    for (int c0 = rb; c0 < re; c0 += THREADS * VEC) {
      const int at = c0 + tid * VEC;
      double r[VEC];
      double own = 0.0;
      Raw<T, VEC> x, y;
      if (at < re) {
        x.load(p + at);
        if (minus) y.load(q + at);
      }
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        r[v] = at < re ? r_of(x, y, minus, certain, at, v) : 0.0;
        own += r[v];
      }
      const double incl = warp_scan(own);
      if (lane == 31) S.scan[warp] = incl;
      __syncthreads();
      const double ws = lane < kWarps ? S.scan[lane] : 0.0, wi = warp_scan<kWarps>(ws);
      double s = base + __shfl_sync(0xffffffffu, wi - ws, warp) + (incl - own);
      int hit = -1, last = -1;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        s += r[v];
        if (r[v] > 0.0) {
          last = at + v;
          if (hit < 0 && s > goal) hit = at + v;
        }
      }
      // the first index past the goal; where there is none in the run, the last with mass
      if (hit >= 0) atomicMin(reinterpret_cast<unsigned*>(&S.found), (unsigned)hit);  // -1: the largest
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
      fallback = max(fallback, last);
      base += __shfl_sync(0xffffffffu, wi, kWarps - 1);
      __syncthreads();  // found is there; scan may be written again
      if (S.found >= 0) break;
    }
    if (S.found < 0) {
      // (all threads are here: found is the same for them)
      if (lane == 0) S.scan[warp] = (double)fallback;
      __syncthreads();
      if (tid == 0) {
        for (int k = 0; k < kWarps; ++k) fallback = max(fallback, (int)S.scan[k]);
        out[n] = fallback;
      }
    } else if (tid == 0) {
      out[n] = S.found;
    }
    return;
  }
}

template <typename T, int VEC, int THREADS>
cudaError_t run(const VerifyArgs& a, int parts, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = attribute(done, verify_kernel<T, VEC, THREADS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n_seqs * parts));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, verify_kernel<T, VEC, THREADS>, a);
}

template <typename T, int VEC>
cudaError_t run(const VerifyArgs& a, int num_sms, cudaStream_t st) {
  // As many threads as there is room for, so that a thread's share of the row is a
  // load or two: sixteen CTAs of 512 a sequence while each has an SM of its own (one
  // sequence of 151936: 7.0 us, with eight 9.3), then eight, of 512 threads where
  // 256 would take more than one round of loads (24 and 32 sequences of 151936: 14.7
  // and 16.0 us, of 256 17.8 and 18.1; of 32000 8.4 and 8.9 against 7.8).  Beyond seven
  // quarters of an SM's worth each eight of 256, four on an SM, as all then begin
  // at once (37 sequences: 22.5 us, of 512 threads 23.2; 64: 23.4 and 28.4); they go
  // through the chain's links in step, so little of one's hides another's.
  if (a.n_seqs * 16 <= num_sms) return run<T, VEC, 512>(a, 16, st);
  const bool rounds = a.vocab > 8 * 256 * VEC * kLoads;
  if (rounds && a.n_seqs * 8 <= num_sms * 7 / 4) return run<T, VEC, 512>(a, 8, st);
  return run<T, VEC, 256>(a, 8, st);
}

}  // namespace

cudaError_t verify_launch(const VerifyArgs& a, int num_sms, cudaStream_t st) {
  const int vec = a.is_bf16 ? 8 : 4;
  // rows keep the first one's 16-byte alignment only if they are whole vectors long
  const bool whole = a.vocab % vec == 0 && ((reinterpret_cast<uintptr_t>(a.target) | reinterpret_cast<uintptr_t>(a.draft)) & 15) == 0;
  if (a.is_bf16) return whole ? run<bf16, 8>(a, num_sms, st) : run<bf16, 1>(a, num_sms, st);
  return whole ? run<float, 4>(a, num_sms, st) : run<float, 1>(a, num_sms, st);
}

}  // namespace emx
