// paged_attn.cu — attention of a batch's new rows over a paged K/V cache
// whose first positions all sequences share.
//
// Row r of sequence i (q head g of KV head h) at position p:
//   o = sum_j e^{s_j} v_j / sum_j e^{s_j},  s_j = scale q . k_j,  j <= p.
// The positions fall in two parts, the common prefix [0, S) and the
// sequence's own [S, p], and each part in pieces; a piece gives
//   m = max s_j, l = sum e^{s_j - m}, O = sum e^{s_j - m} v_j   (base 2, fp32)
// and pieces join as O = sum_x 2^{m_x - m} O_x, l likewise, o = O / l.  So the
// prefix is read once for all rows of the batch, as one sequence whose rows
// are every row, and the own parts once for their few rows.
//
// Workers.  A worker — a warp with 16 rows and tiles of 16 keys, or a CTA with
// 64 and 64 — takes an even share of the key tiles of all segments (sequence,
// KV head, row tile) in one line (paged_plan.h), so lengths from one to the
// longest balance to within a tile, without the host knowing them.  A share's
// pieces: a segment's first tiles go to the piece slot of its rows, a share that
// begins inside a segment to the slot of its worker; a second kernel joins the
// pieces of each row (and a segment that one worker has whole is written by it).
//
// The own part reads every K and V once and for few rows: memory bounds it where
// there is enough of it (32 sequences of 17 to 8192 positions, 269 MB: 50 us
// alone, 5.4 TB/s; 54.3 us with the join), and a warp's own chain of latencies
// elsewhere: a 16-key tile takes it 1.3 to 1.45 us, whether or not the SM's other
// warps want memory.  Twelve warps an SM with two tiles each (against eight with
// three) took 55.3 us where these took 53.5, fewer instructions for the copies nothing off.  A short
// sequence alone (132 positions) takes 8.7 us: three dependent loads (rows,
// page, keys) and two kernels.
#include "paged_attn.cuh"

namespace emx {

namespace {

constexpr int kWarps = 4;   // of a CTA
constexpr int kStages = 3;  // tiles a worker keeps, two of them in flight
// Units of a segment's set-up (q, its pieces): a worker's share of 14 one-tile
// segments took 38 us where 14 tiles of one or two segments took 23.
constexpr int kSetup = 1;
constexpr int kMaxSeqs = 1024;
constexpr int kCtasPerSm = 2;
// ns of a tcgen05 tile of 256 rows and of 128, and of an own part's unit by a
// warp and by a CTA, of those that run beside them (with the longer shares 128 rows
// on 16384 take 75.5 us, with even ones 75.9; 24 drafted sequences on 8192 83.0 and 83.7).
constexpr int kPairNs = 2480, kHalfNs = 1610, kWarpNs = 1450, kCtaNs = 4000;

// `policy`: first out of L2.  K and V are read once or, by a sequence's next row
// tile, soon again; the pieces, which the join reads, are to stay.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on, uint64_t policy) {
  const int n = on ? 16 : 0;  // 0: the 16 bytes become zeros, nothing is read
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(n), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// starts[0..n_seqs] of all sequences into shared memory, by the whole CTA.
template <int THREADS>
__device__ __forceinline__ void plan_starts(const PagedAttnArgs& a, const Line& line, int64_t* starts, bool report) {
  __shared__ int64_t wsum[THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.p.n_seqs + THREADS - 1) / THREADS;  // consecutive sequences of a thread
  const int i0 = min(a.p.n_seqs, tid * per), i1 = min(a.p.n_seqs, i0 + per);
  int64_t sum = 0;
  for (int i = i0; i < i1; ++i) {
    const SeqInfo s = line.seq(i);
    if (!s.ok && report) report_status(a.p.status, seq_status(a.p, i));
    const int64_t t = line.units(s);
    starts[i] = t;
    sum += t;
  }
  int64_t incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  int64_t run = incl - sum;
  for (int w = 0; w < warp; ++w) run += wsum[w];
  for (int i = i0; i < i1; ++i) {
    const int64_t t = starts[i];
    starts[i] = run;
    run += t;
  }
  if (tid == THREADS - 1) {  // its run ends the line
    starts[a.p.n_seqs] = run;
  }
  __syncthreads();
}

// K and V of 16 or 64 keys in shared memory: 16-byte chunk c of row r.  Rows of
// a tile hit all banks of ldmatrix.
template <int HD>
__device__ __forceinline__ uint32_t at(int r, int c) {
  return (uint32_t)(r * HD * 2 + ((c ^ (r & 7)) << 4));
}

// The page of a key and its place there, -1 where there is none.  Loaded ahead
// of its use and not looked at before: a look would wait for it.
struct Key {
  int page, off;
};

template <bool SHARED>
__device__ __forceinline__ Key key_at(const PagedAttnArgs& a, const Cursor& c, int pos) {
  Key key{0, -1};
  if (pos < c.s.len) {
    const int pg = pos / a.p.page_size;
    key.page = SHARED ? a.shared_pages[pg] : a.p.table[(size_t)c.seq * a.p.max_pages + pg];
    key.off = pos - pg * a.p.page_size;
  }
  return key;
}

// Its cache row, ~0 where there is none.
__device__ __forceinline__ uint32_t key_row(const PagedAttnArgs& a, const Key& key, int head) {
  if (key.off < 0) return ~0u;
  if (key.page >= 0 && key.page < a.p.n_pages) return cache_row(key.page, a.p.n_kv, head, a.p.page_size, key.off);
  report_status(a.p.status, kDevBadPage);
  return ~0u;
}

// Copies 16 bytes of K and of V; row ~0 reads as zeros.
template <int HD>
__device__ __forceinline__ void copy_kv(const PagedAttnArgs& a, uint32_t to_k, uint32_t to_v, uint32_t row, int c,
                                        uint64_t policy) {
  const bool on = row != ~0u;
  const size_t off = (on ? (size_t)row * HD : 0) + c * 8;
  cp_async16(to_k, a.p.k + off, on, policy);
  cp_async16(to_v, a.p.v + off, on, policy);
}

// Sixteen rows of one segment, by a warp: q as MMA operands, the running
// maximum and sum of each row and its O.
template <int HD, bool SHARED, bool FEW_ROWS>
struct Rows {
  uint32_t qf[HD / 16][4];
  float o[HD / 8][4];
  float m[2], l[2];
  int vis[2];  // keys of this part that the row sees
  int least;   // fewest of them over the rows
  int R, base, h;

  // Rows base .. base + 15 (of R) of the cursor's segment.
  __device__ __forceinline__ void begin(const PagedWork& w, const Cursor& c, int hpg, int first_row) {
    const PagedAttnArgs& a = w.a;
    const int lane = threadIdx.x & 31, quad = lane >> 2, col = (lane & 3) * 2;
    h = c.head();
    base = first_row;
    R = c.s.rows * hpg;
    least = 0x7fffffff;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int r = base + quad + b * 8;
      const bool on = r < R;
      const int tok = r / hpg;
      vis[b] = !on ? 0 : SHARED ? a.shared_len : c.s.len - c.s.rows + tok + 1 - a.shared_len;
      if (on) least = min(least, vis[b]);
      m[b] = -INFINITY;
      l[b] = 0.f;
      const bf16* qr = a.q + ((size_t)(c.s.row0 + (on ? tok : 0)) * a.p.n_q + h * hpg + (on ? r - tok * hpg : 0)) * HD;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        qf[ks][b] = on ? *reinterpret_cast<const uint32_t*>(qr + ks * 16 + col) : 0u;
        qf[ks][b + 2] = on ? *reinterpret_cast<const uint32_t*>(qr + ks * 16 + col + 8) : 0u;
      }
    }
#pragma unroll
    for (int d = 0; d < HD / 8; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[d][e] = 0.f;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, x));
  }

  // Up to eight rows: the other eight of the operands hold the low parts of the weights.
  __device__ __forceinline__ bool few() const { return R - base <= 8; }

  // 16 G keys, key0 of the part the first, rows r0 .. r0 + 16 G - 1 of the tiles at K and V; bit j of `there`: key j is.
  template <int G, bool FEW>
  __device__ __forceinline__ void keys(float sl2, uint32_t K, uint32_t V, int r0, int key0, uint32_t there) {
    constexpr uint32_t kAll = G == 2 ? 0xffffffffu : 0xffffu;
    constexpr int B = FEW ? 1 : 2;  // rows of a thread
    const int lane = threadIdx.x & 31, col = (lane & 3) * 2;
    const float nothing = sl2 < 0.f ? INFINITY : -INFINITY;  // the score of a key that is not seen
    float s[2 * G][4];
#pragma unroll
    for (int j = 0; j < 2 * G; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint32_t kf[4];  // keys 0-7 (dims lo, hi), keys 8-15 (dims lo, hi)
        ldsm4(kf, K + at<HD>(r0 + 16 * g + (lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)));
        mma_bf16_16816(s[2 * g], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], kf[0], kf[1]);
        mma_bf16_16816(s[2 * g + 1], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], kf[2], kf[3]);
      }
    // m is the maximum of s * scale * log2 e.  Masks only where a key is missing
    // or some row does not see the whole tile.
    const bool cut = key0 + 16 * G > least, masked = there != kAll || cut;
    uint32_t ph[G][4], pl[G][4];
    bool moved = false;
    float alpha[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      if (masked) {
#pragma unroll
        for (int j = 0; j < 2 * G; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = j * 8 + col + e;
            if (!(key0 + key < vis[b] && ((there >> key) & 1u))) s[j][2 * b + e] = nothing;
          }
      }
      float mx = fmaxf(s[0][2 * b] * sl2, s[0][2 * b + 1] * sl2);
#pragma unroll
      for (int j = 1; j < 2 * G; ++j) mx = fmaxf(mx, fmaxf(s[j][2 * b] * sl2, s[j][2 * b + 1] * sl2));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float to = fmaxf(m[b], mx);
      const float from = to == -INFINITY ? 0.f : to;  // nothing seen yet: weights 2^-inf = 0
      alpha[b] = ex2f(m[b] - from);
      moved |= to > m[b];
      m[b] = to;
      // weights go to the products as two bf16 (split_weights), which takes twice the MMAs of more than eight rows
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 2 * G; ++j) {
        const float p0 = ex2f(fmaf(s[j][2 * b], sl2, -from)), p1 = ex2f(fmaf(s[j][2 * b + 1], sl2, -from));
        sum += p0 + p1;
        const int at = b + 2 * (j & 1);
        split_weights(p0, p1, ph[j >> 1][at], FEW ? ph[j >> 1][at + 1] : pl[j >> 1][at]);
      }
      l[b] = l[b] * alpha[b] + sum;
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int d = 0; d < HD / 8; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][e] *= alpha[FEW ? 0 : e >> 1];
    }
    // A row that does not see a key gives it weight 0, and 0 * inf is NaN: where
    // some rows see further than others and V holds something not finite, the
    // products are taken one visible key at a time.
    bool odd = false;
    if (!SHARED && cut) {
#pragma unroll
      for (int i = 0; i < G * HD / 16; ++i) {
        const uint4 u = *reinterpret_cast<const uint4*>(__cvta_shared_to_generic(V + r0 * HD * 2 + (i * 32 + lane) * 16));
        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= (x[e] & 0x7f80u) == 0x7f80u || (x[e] & 0x7f800000u) == 0x7f800000u;
      }
      odd = __any_sync(0xffffffffu, odd);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (!odd) {
        // high parts of four 16-column blocks, then their low parts: a product does not wait for the one before
#pragma unroll
        for (int d0 = 0; d0 < HD / 16; d0 += 4) {
          uint32_t vf[4][4];  // dims lo (keys lo, hi), dims hi (keys lo, hi)
#pragma unroll
          for (int d = 0; d < 4; ++d)
            ldsm4t(vf[d], V + at<HD>(r0 + 16 * g + (lane & 7) + (((lane >> 3) & 1) << 3), (d0 + d) * 2 + (lane >> 4)));
#pragma unroll
          for (int part = 0; part < B; ++part) {
            const uint32_t(&p)[4] = part ? pl[g] : ph[g];
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              mma_bf16_16816(o[2 * (d0 + d)], p[0], p[1], p[2], p[3], vf[d][0], vf[d][1]);
              mma_bf16_16816(o[2 * (d0 + d) + 1], p[0], p[1], p[2], p[3], vf[d][2], vf[d][3]);
            }
          }
        }
      } else {
        for (int key = 0; key < 16; ++key) {
          const int from = (lane & ~3) | ((key & 7) >> 1);
#pragma unroll
          for (int b = 0; b < B; ++b) {
            const uint32_t(&rest)[4] = FEW ? ph[g] : pl[g];
            const uint32_t hi = __shfl_sync(0xffffffffu, key < 8 ? ph[g][b] : ph[g][b + 2], from);
            const uint32_t lo = __shfl_sync(0xffffffffu, key < 8 ? rest[b + FEW] : rest[b + 2 + FEW], from);
            const float pw = (key & 1) ? __uint_as_float(hi & 0xffff0000u) + __uint_as_float(lo & 0xffff0000u)
                                       : __uint_as_float(hi << 16) + __uint_as_float(lo << 16);
            const bool on = key0 + 16 * g + key < vis[b] && ((there >> (16 * g + key)) & 1u);
#pragma unroll
            for (int d = 0; d < HD / 8; ++d) {
              const uint32_t x = *reinterpret_cast<const uint32_t*>(
                  __cvta_shared_to_generic(V + at<HD>(r0 + 16 * g + key, d) + (lane & 3) * 4));
              if (on) {
                o[d][2 * b] = fmaf(pw, __uint_as_float(x << 16), o[d][2 * b]);
                o[d][2 * b + 1] = fmaf(pw, __uint_as_float(x & 0xffff0000u), o[d][2 * b + 1]);
              }
            }
          }
        }
      }
    }
  }

  // The rows' piece of the segment: to the output (`direct`: it is all there is), to the rows' first slots (the
  // segment's first tile was this worker's) or, from slot `more` on, to the worker's.
  __device__ __forceinline__ void end(const PagedWork& w, const Cursor& c, int hpg, bool direct, bool first, size_t more) {
    const PagedAttnArgs& a = w.a;
    const Pieces& pc = SHARED ? w.shared : w.own;
    const int lane = threadIdx.x & 31, quad = lane >> 2, col = (lane & 3) * 2;
    if (FEW_ROWS && few()) {
#pragma unroll
      for (int d = 0; d < HD / 8; ++d)
#pragma unroll
        for (int e = 0; e < 2; ++e) o[d][e] += o[d][e + 2];
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      float ls = l[b];
      ls += __shfl_xor_sync(0xffffffffu, ls, 1);
      ls += __shfl_xor_sync(0xffffffffu, ls, 2);
      const int r = base + quad + b * 8;
      if (r >= R) continue;
      const int tok = r / hpg;
      const size_t head = (size_t)(c.s.row0 + tok) * a.p.n_q + h * hpg + (r - tok * hpg);
      if (direct) {
        const float inv = ls > 0.f ? 1.f / ls : ls == 0.f ? 0.f : ls;  // no key seen: zeros; NaN stays
#pragma unroll
        for (int d = 0; d < HD / 8; ++d)
          *reinterpret_cast<__nv_bfloat162*>(a.out + head * HD + d * 8 + col) =
              __floats2bfloat162_rn(o[d][2 * b] * inv, o[d][2 * b + 1] * inv);
      } else {
        const size_t slot = first ? head : more + quad + b * 8;
        float* dst = (first ? pc.first_o : pc.more_o) + slot * HD;
#pragma unroll
        for (int d = 0; d < HD / 8; ++d) *reinterpret_cast<float2*>(dst + d * 8 + col) = make_float2(o[d][2 * b], o[d][2 * b + 1]);
        if ((lane & 3) == 0) (first ? pc.first_ml : pc.more_ml)[slot] = make_float2(m[b], ls);
      }
    }
  }
};

// A worker's place in the line, for the loads and for the products, which run
// kStages - 1 tiles behind: the tiles among units [.., x1).
struct Share {
  Cursor ld, cc;
  int64_t x1;
  __device__ __forceinline__ bool begin(const Line& line, int64_t x0, int64_t end) {
    x1 = end;
    cc.seek(line, x0);
    ld = cc;
    return cc.x < x1;  // else nothing but a set-up
  }
  __device__ __forceinline__ bool loading() const { return ld.x < x1; }
  __device__ __forceinline__ void loaded(const Line& line) {
    if (ld.x + 1 < x1) ld.next(line);
    else ld.x = x1;
  }
  __device__ __forceinline__ bool last() const { return cc.k + 1 == cc.kt; }
  // the next tile is this worker's if its unit is; a segment's last is followed by a set-up
  __device__ __forceinline__ bool more(const Line& line) const { return cc.x + 1 + (last() ? line.setup : 0) < x1; }
};

// Few rows (up to 32 a sequence and KV head): a warp is a worker, with 16 rows, 16 keys
// a tile and three tiles in flight of its own, and never meets another.
template <int HD, bool SHARED>
struct WarpWorker {
  static_assert(!SHARED, "a prefix has more rows");
  static constexpr int kRows = 16, kKeys = 16, kPerCta = kWarps;
  static constexpr int kTileB = kKeys * HD * 2;  // one tile of K (or V)
  static constexpr int kSmem = kWarps * kStages * 2 * kTileB;

  static __device__ __forceinline__ void run(const PagedWork& w, const Line& line, unsigned char* smem, int worker, int64_t x0,
                                             int64_t x1) {
    __shared__ uint32_t there_[kWarps][kStages];  // bit j: key j of the tile is there
    const PagedAttnArgs& a = w.a;
    const int lane = threadIdx.x & 31;
    const uint32_t ring = smem_u32(smem) + (threadIdx.x >> 5) * (uint32_t)(kStages * 2 * kTileB);
    uint32_t* there = there_[threadIdx.x >> 5];
    Share sh;
    if (!sh.begin(line, x0, x1)) return;
    const uint64_t policy = l2_evict_first_policy();
    auto next_key = [&]() {
      return key_at<false>(a, sh.ld, a.shared_len + sh.ld.k * kKeys + (lane & 15));
    };
    Key key = next_key();
    int at_stage = 0;  // of the next load
    auto load = [&]() {
      if (sh.loading()) {
        const uint32_t row = key_row(a, key, sh.ld.head());
        const unsigned mask = __ballot_sync(0xffffffffu, row != ~0u) & 0xffffu;
        if (lane == 0) there[at_stage] = mask;
        constexpr int kChunks = HD / 8, kPer = 32 / kChunks;  // of a row; rows of one copy of the warp
        const int sub = lane / kChunks, c = lane % kChunks;
        const uint32_t dst = ring + at_stage * 2 * kTileB + at<HD>(sub, c);
#pragma unroll
        for (int i = 0; i < kKeys / kPer; ++i) {
          const uint32_t src = __shfl_sync(0xffffffffu, row, i * kPer + sub);
          // chunk c of row i * kPer + sub: the swizzle's bits of the two parts of the row number do not meet
          const uint32_t to = (dst ^ (uint32_t)(((i * kPer) & 7) << 4)) + (uint32_t)(i * kPer * HD * 2);
          copy_kv<HD>(a, to, to + kTileB, src, c, policy);
        }
        sh.loaded(line);
        if (sh.loading()) key = next_key();
      }
      at_stage = at_stage + 1 == kStages ? 0 : at_stage + 1;
      cp_commit();
    };
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) load();
    const float sl2 = a.scale * kLog2e;
    Rows<HD, false, true> rows;
    bool fresh = true, first = false;
    for (int stage = 0;; stage = stage + 1 == kStages ? 0 : stage + 1) {
      if (fresh) {
        first = sh.cc.k == 0;
        rows.begin(w, sh.cc, line.hpg, (sh.cc.seg - sh.cc.head() * sh.cc.mt) * kRows);
      }
      load();
      cp_wait<kStages - 1>();
      __syncwarp();
      const uint32_t K = ring + stage * 2 * kTileB;
      if (rows.few()) rows.template keys<1, true>(sl2, K, K + kTileB, 0, sh.cc.k * kKeys, there[stage]);
      else rows.template keys<1, false>(sl2, K, K + kTileB, 0, sh.cc.k * kKeys, there[stage]);
      __syncwarp();  // the stage may be filled again
      const bool last = sh.last(), more = sh.more(line);
      fresh = last || !more;
      if (fresh) rows.end(w, sh.cc, line.hpg, first && last && a.shared_len == 0, first, (size_t)worker * kRows);
      if (!more) break;
      sh.cc.next(line);
    }
    cp_wait<0>();
  }
};

// More rows: a CTA is a worker, 64 rows (16 a warp) against tiles of 64 keys
// that its warps load together.  One barrier a tile: behind it the tile's keys
// are there, every warp is done with the tile before, whose stage the next load
// takes, and the rows of that load's keys are known.
template <int HD, bool SHARED>
struct CtaWorker {
  static constexpr int kRows = 16 * kWarps, kKeys = 64, kPerCta = 1;
  static constexpr int kTileB = kKeys * HD * 2;
  static constexpr int kSmem = kStages * 2 * kTileB;

  static __device__ __forceinline__ void run(const PagedWork& w, const Line& line, unsigned char* smem, int worker, int64_t x0,
                                             int64_t x1) {
    __shared__ uint32_t row_[2][kKeys];        // cache rows of the next load's keys
    __shared__ uint32_t there[kStages + 1][2];  // bit j: key j of the tile is there (one more than tiles are kept)
    const PagedAttnArgs& a = w.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t ring = smem_u32(smem);
    Share sh;
    if (!sh.begin(line, x0, x1)) return;
    const uint64_t policy = l2_evict_first_policy();
    auto next_key = [&]() {  // threads 0-63
      return tid < kKeys ? key_at<SHARED>(a, sh.ld, (SHARED ? 0 : a.shared_len) + sh.ld.k * kKeys + tid) : Key{0, -1};
    };
    Key key = next_key();
    int tile = 0;  // of the next load
    // the rows of the next load's keys, for all warps after the next barrier
    auto name = [&]() {
      if (sh.loading() && tid < kKeys) {
        const uint32_t row = key_row(a, key, sh.ld.head());
        row_[tile & 1][tid] = row;
        const unsigned mask = __ballot_sync(0xffffffffu, row != ~0u);
        if (lane == 0) there[tile % (kStages + 1)][warp] = mask;
      }
    };
    auto load = [&]() {
      if (sh.loading()) {
        constexpr int kChunks = HD / 8, kPer = kWarps * 32 / kChunks;  // of a row; rows of one copy of the CTA
        const int sub = tid / kChunks, c = tid % kChunks;
        const uint32_t dst = ring + (tile % kStages) * 2 * kTileB;
#pragma unroll
        for (int i = 0; i < kKeys / kPer; ++i) {
          const int r = i * kPer + sub;
          const uint32_t to = dst + at<HD>(r, c);
          copy_kv<HD>(a, to, to + kTileB, row_[tile & 1][r], c, policy);
        }
        sh.loaded(line);
        if (sh.loading()) key = next_key();
      }
      ++tile;
      cp_commit();
    };
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) {
      name();
      __syncthreads();
      load();
    }
    const float sl2 = a.scale * kLog2e;
    Rows<HD, SHARED, false> rows;
    bool fresh = true, first = false;
    for (int t = 0;; ++t) {
      if (fresh) {
        first = sh.cc.k == 0;
        rows.begin(w, sh.cc, line.hpg, (sh.cc.seg - sh.cc.head() * sh.cc.mt) * kRows + warp * 16);
      }
      name();
      cp_wait<kStages - 2>();
      __syncthreads();
      load();
      const uint32_t K = ring + (t % kStages) * 2 * kTileB;
      const int key0 = sh.cc.k * kKeys;
      if (rows.base < rows.R) {
#pragma unroll 1
        for (int i = 0; i < kKeys / 32; ++i) {  // two groups of 16 keys: one's latencies pass under the other's
          const uint32_t mask = there[t % (kStages + 1)][i];
          if (mask) rows.template keys<2, false>(sl2, K, K + kTileB, i * 32, key0 + i * 32, mask);
        }
      }
      const bool last = sh.last(), more = sh.more(line);
      fresh = last || !more;
      if (fresh && rows.base < rows.R)
        rows.end(w, sh.cc, line.hpg, first && last && !SHARED && a.shared_len == 0, first, (size_t)worker * kRows + warp * 16);
      if (!more) break;
      sh.cc.next(line);
    }
    cp_wait<0>();
  }
};

template <int HD, bool SHARED, template <int, bool> class W>
__global__ void __launch_bounds__(kWarps * 32) paged_attn_kernel(const __grid_constant__ PagedWork w) {
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ int64_t starts[SHARED ? 1 : kMaxSeqs + 1];
  using Worker = W<HD, SHARED>;
  const Line line = make_line(w.a.p, w.a.shared_len, !SHARED, Worker::kRows, Worker::kKeys, SHARED ? 0 : kSetup, starts);
  // The first kernel of a call waits for what ran before it.  An own part that
  // follows a shared one has been let go by it after such a wait, so what ran before
  // is complete and in memory, but only a grid's own wait is promised to show it to
  // that grid: here a fence drops what L1 may hold from earlier.  It needs nothing of
  // the shared part, but the join waits for this kernel alone, so it ends after the
  // other.
  const bool first = SHARED || w.a.shared_len == 0;
  if (first) pdl_wait();
  else __threadfence();
  pdl_trigger();
  int64_t total;
  if (SHARED) {
    total = line.units(line.seq(0));
  } else {
    plan_starts<kWarps * 32>(w.a, line, starts, blockIdx.x == 0);
    total = starts[w.a.p.n_seqs];
  }
  const int worker = Worker::kPerCta == 1 ? blockIdx.x : blockIdx.x * Worker::kPerCta + (threadIdx.x >> 5);
  int64_t x0, x1;
  if (SHARED) {
    x0 = (int64_t)worker * w.shared_per;
    x1 = x0 + w.shared_per;
  } else {
    const Shares shares = deal(total, w.own_workers, w.own_early, w.own_each);
    x0 = shares.begin(worker);
    x1 = shares.begin(worker + 1);
    if (blockIdx.x == 0) {
      for (int i = threadIdx.x; i <= w.a.p.n_seqs; i += kWarps * 32) w.starts[i] = starts[i];
      if (threadIdx.x == 0) *w.shares = shares;
    }
  }
  x1 = min(x1, total);
  if (x0 < x1) Worker::run(w, line, smem, worker, x0, x1);
  if (!first) pdl_wait();
}

// Joins the pieces of each (row, q head), an item.  `parts` warps share an item
// where there are few (1, 8 and 32 rows of 32 heads on about 1500 positions: 9.8,
// 15.7 and 27.4 us in all, 12.1, 20.7 and 28.6 without); else a warp has several, 32
// in its lanes: where their pieces are (a search, divisions) is found by all lanes
// together, mostly before the pieces are written, and what is left of an item then
// is one L2 latency for eight pieces.  128 rows of 32 heads with 11 pieces each
// (25 MB of L2 reads): 10 us from the last piece to the last row.
template <int HD>
__global__ void __launch_bounds__(128) paged_join_kernel(const __grid_constant__ PagedWork w, int parts) {
  __shared__ float sm[4], sl[4];
  __shared__ float so[4][HD];
  constexpr int E = HD / 32;
  const PagedAttnArgs& a = w.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();
  __threadfence();  // the batch is in memory, as for the own part; the pieces only after the wait
  const int hpg = a.p.n_q / a.p.n_kv, items = a.p.n_rows * a.p.n_q;
  const int part = warp % parts, stride = gridDim.x * (4 / parts);
  const Line own = make_line(a.p, a.shared_len, true, w.own_mt, w.own_keys, kSetup, w.starts);
  const Line all = make_line(a.p, a.shared_len, false, w.shared_mt, w.shared_keys, 0, nullptr);
  bool waited = false;
  for (int first = blockIdx.x * (4 / parts) + warp / parts; first < items; first += 32 * stride) {
    // ---- lane j: item first + j * stride
    const int64_t item64 = (int64_t)first + (int64_t)lane * stride;
    int item = item64 < items ? (int)item64 : -1;
    const int row = item < 0 ? 0 : item / a.p.n_q, hq = item < 0 ? 0 : item - row * a.p.n_q;
    const int h = hq / hpg, g = hq - h * hpg;
    int seq = 0, n = a.p.n_seqs;  // the first sequence that ends behind the row
    while (n > 0) {
      const int mid = n >> 1;
      if (a.p.indptr[seq + mid + 1] > row) n = mid;
      else seq += mid + 1, n -= mid + 1;
    }
    SeqInfo s{0, 0, 0, false};
    if (seq >= a.p.n_seqs || row < a.p.indptr[seq]) item = -1;  // behind the last sequence: left as it was
    else s = own.seq(seq);
    const bool ok = item >= 0 && s.ok;
    // pieces of the row's segment in each part, and the slot of its second worker's
    int n_all = 0, n_own = 0;
    uint32_t slot_all = 0, slot_own = 0;
    if (ok && a.shared_len > 0) {
      const SeqInfo every = all.seq(0);
      const int kt = all.key_tiles(every), r = row * hpg + g, tile = share_of(r, w.shared_mt);
      // with workers of their own, shared segments are as long as those workers' shares
      const int64_t each = w.shared_split ? (int64_t)w.shared_split * w.shared_per : kt;
      const int64_t x0 = ((int64_t)h * all.row_tiles(every) + tile) * each;
      const int c0 = share_of(x0, w.shared_per), c1 = share_of(x0 + kt - 1, w.shared_per);
      slot_all = (uint32_t)((c0 + 1) * w.shared_mt + r - tile * w.shared_mt);
      n_all = c1 - c0 + 1;
    }
    const int r_own = ok ? (row - s.row0) * hpg + g : 0, tile_own = share_of(r_own, w.own_mt);
    const int kt_own = ok ? own.key_tiles(s) : 1;
    const int64_t x_own = ok ? ((int64_t)h * own.row_tiles(s) + tile_own) * (kt_own + kSetup) + kSetup : 0;
    if (!waited) pdl_wait();
    waited = true;
    if (ok) {
      const Shares shares = *w.shares;
      const int64_t x0 = w.starts[seq] + x_own;
      const int c0 = shares.of(x0), c1 = shares.of(x0 + kt_own - 1);
      slot_own = (uint32_t)((c0 + 1) * w.own_mt + r_own - tile_own * w.own_mt);
      n_own = c1 - c0 + 1;
      if (a.shared_len == 0 && n_own == 1) item = -1;  // one worker had the segment whole and wrote it
    }
    // ---- item by item
    const int many = min(32, (items - first + stride - 1) / stride);
    for (int j = 0; j < many; ++j) {
      const int it = __shfl_sync(0xffffffffu, item, j);
      const int na = __shfl_sync(0xffffffffu, n_all, j), np = na + __shfl_sync(0xffffffffu, n_own, j);
      const uint32_t sa = __shfl_sync(0xffffffffu, slot_all, j), sw = __shfl_sync(0xffffffffu, slot_own, j);
      if (it < 0 && parts == 1) continue;
      float o[E], m = -INFINITY, l = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = 0.f;
      // piece z: the shared part's first slot and further workers', then the own part's; this warp's are part, part + parts, ...
      auto slot_of = [&](int z, bool& own_part, bool& is_first) {
        own_part = z >= na;
        const int y = own_part ? z - na : z;
        is_first = y == 0;
        return is_first ? (size_t)it : (size_t)(own_part ? sw : sa) + (size_t)(y - 1) * (own_part ? w.own_mt : w.shared_mt);
      };
      for (int z0 = part; it >= 0 && z0 < np; z0 += 32 * parts) {
        const int z = z0 + parts * lane;  // this lane's (max, sum)
        float2 ml = make_float2(-INFINITY, 0.f);
        if (z < np) {
          bool op, fs;
          const size_t at = slot_of(z, op, fs);
          ml = (op ? (fs ? w.own.first_ml : w.own.more_ml) : (fs ? w.shared.first_ml : w.shared.more_ml))[at];
        }
        constexpr int U = 8;  // pieces in flight
        const int here = min(32, (np - z0 + parts - 1) / parts);
        float wx = 0.f;
        for (int y = 0; y < here; y += U) {
          float v[U][E];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const bool on = y + u < here;
            bool op, fs;
            const size_t at = slot_of(on ? z0 + parts * (y + u) : 0, op, fs);
            const float* p = (op ? (fs ? w.own.first_o : w.own.more_o) : (fs ? w.shared.first_o : w.shared.more_o)) + at * HD + lane * E;
            if constexpr (E == 4) {
              const float4 f = on ? *reinterpret_cast<const float4*>(p) : make_float4(0.f, 0.f, 0.f, 0.f);
              v[u][0] = f.x, v[u][1] = f.y, v[u][2] = f.z, v[u][3] = f.w;
            } else {
              const float2 f = on ? *reinterpret_cast<const float2*>(p) : make_float2(0.f, 0.f);
              v[u][0] = f.x, v[u][1] = f.y;
            }
          }
          if (y == 0) {  // with the first loads on their way
            const float to = fmaxf(m, warp_max(ml.x)), base = to == -INFINITY ? 0.f : to;
            const float was = ex2f(m - base);
            wx = ex2f(ml.x - base);
            l = l * was + warp_sum(ml.y * wx);  // a NaN among the sums stays one
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= was;
            m = to;
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const float wu = __shfl_sync(0xffffffffu, wx, (y + u) & 31);
            if (y + u < here)
#pragma unroll
              for (int e = 0; e < E; ++e) o[e] = fmaf(v[u][e], wu, o[e]);
          }
        }
      }
      if (parts > 1) {  // one item a warp: every warp of the CTA comes here once
#pragma unroll
        for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
        if (lane == 0) {
          sm[warp] = m;
          sl[warp] = l;
        }
        __syncthreads();
        if (part > 0 || it < 0) break;
        for (int k = warp + 1; k < warp + parts; ++k) {
          const float to = fmaxf(m, sm[k]), base = to == -INFINITY ? 0.f : to;
          const float x = ex2f(m - base), y = ex2f(sm[k] - base);
          l = l * x + sl[k] * y;
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] = o[e] * x + so[k][lane * E + e] * y;
          m = to;
        }
      }
      const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // no key seen: zeros; NaN stays
      bf16* dst = a.out + (size_t)it * HD + lane * E;
      uint32_t u[E / 2];
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        const __nv_bfloat162 two = __floats2bfloat162_rn(o[2 * e] * inv, o[2 * e + 1] * inv);
        u[e] = *reinterpret_cast<const uint32_t*>(&two);
      }
      if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(u[0], u[1]);
      else *reinterpret_cast<uint32_t*>(dst) = u[0];
    }
  }
  if (!waited) pdl_wait();  // every CTA waits, so that what follows this kernel follows the ones before it
}

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

// The workspace's parts; returns its size (base may be null).
size_t lay_out(PagedWork& w, int num_sms, unsigned char* base) {
  const PagedArgs& p = w.a.p;
  const size_t heads = (size_t)p.n_rows * p.n_q;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    void* q = base ? base + off : nullptr;
    off += up(bytes);
    return q;
  };
  w.starts = static_cast<int64_t*>(take(sizeof(int64_t) * (kMaxSeqs + 1)));
  w.shares = static_cast<Shares*>(take(sizeof(Shares)));
  auto pieces = [&](Pieces& pc, size_t rows) {
    pc.first_o = static_cast<float*>(take(heads * p.head_dim * sizeof(float)));
    pc.first_ml = static_cast<float2*>(take(heads * sizeof(float2)));
    pc.more_o = static_cast<float*>(take(rows * p.head_dim * sizeof(float)));
    pc.more_ml = static_cast<float2*>(take(rows * sizeof(float2)));
  };
  // slots of every kind of worker's rows: warps of 16, CTAs of 64, tcgen05 CTAs of 256
  static_assert(kWarps * 16 == 64, "");
  const size_t rows = (size_t)num_sms * kCtasPerSm * 64, tc = (size_t)num_sms * kTcRows;
  pieces(w.own, rows);
  if (w.a.shared_len > 0) pieces(w.shared, rows > tc ? rows : tc);
  return off;
}

template <int HD, bool SHARED, template <int, bool> class W>
cudaError_t launch_part(const PagedWork& w, int ctas, cudaStream_t st) {
  constexpr int smem = W<HD, SHARED>::kSmem;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = attribute(done, paged_attn_kernel<HD, SHARED, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute at;
  overlapped(cfg, at, (unsigned)ctas, kWarps * 32, smem, st);
  return cudaLaunchKernelEx(&cfg, paged_attn_kernel<HD, SHARED, W>, w);
}

template <int HD>
cudaError_t launch(PagedWork& w, int num_sms, cudaStream_t st) {
  using Few = WarpWorker<HD, false>;
  using Many = CtaWorker<HD, false>;
  const PagedArgs& p = w.a.p;
  const int64_t rows = (int64_t)p.n_rows * (p.n_q / p.n_kv);  // of a KV head
  const int ctas = num_sms * kCtasPerSm;
  // The own part by warps up to 32 rows a sequence and KV head, on average;
  // beyond that a warp's 16 keys are loaded once too often, again for every 16
  // rows (32 sequences of 500 to 2500 positions, 32 heads on 4: 8, 24 and 32 rows
  // 28, 47 and 49 us, by CTAs 44, 51 and 51; 64 rows 85 us, by CTAs 56).
  const bool by_warp = rows <= 2 * Few::kRows * (int64_t)p.n_seqs;
  w.own_mt = by_warp ? Few::kRows : Many::kRows;
  w.own_keys = by_warp ? Few::kKeys : Many::kKeys;
  const int own_per_sm = kCtasPerSm * (by_warp ? Few::kPerCta : 1);
  w.own_workers = num_sms * own_per_sm;
  cudaError_t e = cudaSuccess;
  if (w.a.shared_len > 0) {
    // tcgen05 where it takes the pages and the prefix is more than two of a CTA's
    // 64 x 64 tiles to each of those (592): below, its start and end cost more than
    // its tiles save (8 KV heads of 8 rows: 512 positions, 64 tiles, 16.1 us against
    // 11.8; 4096, 512 tiles, 18.4 against 17.3; 8192, 1024 tiles, 22.3 against 22.4.
    // 4 heads of 512 rows: 1024 positions, 512 tiles, 27.6 against 24.9; 2048, 1024
    // tiles, 29.4 against 31.0; 8192 36.4 against 61.6).  Near the border the tiles
    // alone do not tell: 4 heads of 64 rows on 8192, 512 tiles, take 23.2 us by CTAs
    // and would take 21.1; 8 heads of one row on 8192, 1024 tiles, 21.4 and 20.2.
    const int64_t tiles = (int64_t)p.n_kv * ceil_div(rows, Many::kRows) * ceil_div(w.a.shared_len, Many::kKeys);
    const bool tc = paged_shared_tc_takes(p) && tiles > 2 * ctas;
    w.shared_mt = tc ? kTcRows : Many::kRows;
    w.shared_keys = tc ? kTcKeys : Many::kKeys;
    const int workers = tc ? num_sms : ctas;
    const int kt = ceil_div(w.a.shared_len, w.shared_keys);
    const int64_t segments = (int64_t)p.n_kv * ceil_div(rows, w.shared_mt);
    w.shared_per = ceil_div(segments * kt, workers);
    if (tc) {
      if (segments <= workers) {
        // A worker that goes from one segment to the next stores one's rows and
        // loads the other's Q with nothing to compute meanwhile: about four
        // tiles' time.  Whole workers to a segment where that is not fewer tiles
        // than it costs (40 and 60 segments of 64 to 256 rows: 3 tiles more than even
        // shares have take 0.90 to 1.00 of their time, 4 tiles 0.97 to 1.03, 6 tiles
        // 1.01 to 1.07).
        const int split = (int)(workers / segments), per = ceil_div(kt, split);
        if (per <= w.shared_per + 4) {
          w.shared_split = split;
          w.shared_per = per;
        }
      }
      // SMs without a share go to the own part's first workers, for as long as the others have theirs.
      const int used = w.shared_split ? ceil_div(kt, w.shared_per) * (int)segments : ceil_div(segments * kt, w.shared_per);
      w.own_early = (num_sms - used) * own_per_sm;
      w.own_each = share_of((int64_t)w.shared_per * (rows > kTcRows / 2 ? kPairNs : kHalfNs), by_warp ? kWarpNs : kCtaNs);
    }
    e = tc ? paged_shared_tc_launch(w, num_sms, st) : launch_part<HD, true, CtaWorker>(w, ctas, st);
    if (e != cudaSuccess) return e;
  }
  e = by_warp ? launch_part<HD, false, WarpWorker>(w, ctas, st) : launch_part<HD, false, CtaWorker>(w, ctas, st);
  if (e != cudaSuccess) return e;
  // five CTAs an SM fit beside what the own part's have not left yet; fewer
  // items than their warps are shared by two or four
  const int64_t items = (int64_t)p.n_rows * p.n_q, warps = (int64_t)num_sms * 20;
  const int parts = items * 4 <= warps ? 4 : items * 2 <= warps ? 2 : 1;
  const int64_t grid = (items * parts + 3) / 4;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute at;
  overlapped(cfg, at, (unsigned)(grid < warps / 4 ? grid : warps / 4), 128, 0, st);
  return cudaLaunchKernelEx(&cfg, paged_join_kernel<HD>, static_cast<const PagedWork>(w), parts);
}

}  // namespace

size_t paged_attn_workspace(int n_rows, int n_q, int n_kv, int head_dim, int shared_len, int num_sms) {
  PagedWork w = {};
  w.a.p.n_rows = n_rows;
  w.a.p.n_q = n_q;
  w.a.p.n_kv = n_kv;
  w.a.p.head_dim = head_dim;
  w.a.shared_len = shared_len;
  return lay_out(w, num_sms, nullptr);
}

cudaError_t paged_attn_launch(const PagedAttnArgs& a, int num_sms, cudaStream_t st) {
  PagedWork w = {};
  w.a = a;
  lay_out(w, num_sms, static_cast<unsigned char*>(a.workspace));
  return a.p.head_dim == 128 ? launch<128>(w, num_sms, st) : launch<64>(w, num_sms, st);
}

}  // namespace emx
