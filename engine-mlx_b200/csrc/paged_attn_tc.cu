// paged_attn_tc.cu — the shared prefix of emx_sdpa_paged for a batch of many
// rows, on tcgen05.
//
// All rows of the batch that use one KV head (n_rows * n_q / n_kv of them)
// attend the same S keys without a mask, so the prefix is two dense products
// around a softmax: S = Q K^T, O = P V, rows in tiles of 128, keys in tiles of
// 128.  K and V are read from HBM once per KV head and 256 rows; with up to
// 128 rows a head that stream (64 KB a tile) bounds the kernel, with more the
// exponentials (128 x 128 a tile, 16 an SM and clock) and the tensor pipe.
//
// One CTA an SM, each with an even share of the (KV head, 256 rows, 128 keys)
// tiles in line order; twelve warps:
//   warps 0-7   two softmax groups of 128 threads, a thread a row: S from
//               tensor memory, the running maximum and sum, P back over S;
//   warp 8      one thread issues every MMA;
//   warps 9-11  the keys' rows from their pages into a ring of five 128-row
//               slots (K, V, K, V, ...) by 16-byte asynchronous copies, so a
//               page may have any size and end anywhere in a tile.
// Each group is a stream of its own — S, P and O in tensor memory, its Q tile
// in shared memory: two row tiles against the same keys where the segment has
// more than 128 rows, else the same rows against alternate key tiles (then the
// two halves join at the segment's end).  While one group takes exponentials
// the tensor pipe works for the other.
//
// The maximum that the exponentials use moves only when a tile's exceeds it by
// more than 2^8 (then O and l are rescaled); O / l does not depend on it.  P is
// rounded to bf16 for its product (off by at most 2^-9 of each weight).
#include "paged_attn.cuh"
#include "tc_attn.cuh"

namespace emx {

namespace {

constexpr int kThreads = 384;
constexpr int kSlots = 5;
constexpr int kMmaWarp = 8, kLoadWarp = 9, kLoadWarps = 3;
constexpr float kRescale = 8.0f;
constexpr uint32_t kCols = 512;  // S of the groups at 0 and 128 (P over its upper half), O at 256 and 384
constexpr int kLag = 3;          // most slots whose copies a loader leaves in flight
constexpr int kValid = 4;        // tiles whose key masks are kept: a tile's V slot is free before the ring holds 3 later ones

template <int HD>
struct Smem {
  static constexpr int kTile = HD / 64 * kBlk;  // 128 rows of HD
  static constexpr int kQ = 0;                  // [2]
  static constexpr int kRing = 2 * kTile;       // [kSlots]
  static constexpr int kBar = kRing + kSlots * kTile;
  static constexpr int kBytes = kBar + 512 + 1024;  // barriers; 1 KB to align
  static_assert(kBytes <= 227 * 1024, "");
};

struct Bars {
  uint64_t full[kSlots], empty[kSlots];
  uint64_t q_full[2], s_full[2], p_full[2], o_done[2];
  uint32_t tmem;
  alignas(16) unsigned char valid[kValid][16];  // by tile of the share, bit j: key j is there
};
static_assert(sizeof(Bars) <= 512, "");

constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// 16-byte chunk c of row r of a tile (64-column blocks, 128-byte swizzle).
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  return (uint32_t)((c >> 3) * kBlk + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ void tst16u(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Waits for this thread's tensor-memory loads; what they loaded into v may be used after it only.
__device__ __forceinline__ void wait_ld(float (&v)[32]) {
  tmem_wait_ld_();
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(v[i]));
}

// A share's tiles, segment by segment, the same for every role.
struct Walk {
  Cursor c;
  int left;  // tiles of the share not yet entered
  int n;     // tiles of this segment in the share
  int rows;  // rows of this segment's 256
  bool whole_first;  // its first tile is in the share
  __device__ __forceinline__ bool begin(const Line& line, int64_t total, int worker, int64_t per) {
    const int64_t x0 = worker * per;
    if (x0 >= total) return false;
    left = (int)min(per, total - x0);
    c.seek(line, x0);
    enter(line);
    return true;
  }
  __device__ __forceinline__ void enter(const Line& line) {
    n = min(left, c.kt - c.k);
    left -= n;
    rows = min(line.mt, line.n_rows * line.hpg - (c.seg - c.head() * c.mt) * line.mt);
    whole_first = c.k == 0;
  }
  __device__ __forceinline__ bool next(const Line& line) {
    if (left == 0) return false;
    c.k = 0;
    ++c.seg;
    enter(line);
    return true;
  }
  __device__ __forceinline__ bool pair() const { return rows > 128; }
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) paged_shared_tc_kernel(const __grid_constant__ PagedWork w) {
  using L = Smem<HD>;
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  Bars& B = *reinterpret_cast<Bars*>(smem + L::kBar);
  const PagedAttnArgs& a = w.a;
  int* status = a.p.status;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&B.full[s], kLoadWarps);
      mbar_init(&B.empty[s], 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&B.q_full[g], 128);
      mbar_init(&B.s_full[g], 2);
      mbar_init(&B.p_full[g], 128);
      mbar_init(&B.o_done[g], 1);
    }
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&B.tmem)), "r"(kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tfence_before();
  __syncthreads();
  tfence_after();
  const uint32_t tmem = B.tmem;
  const Line line = make_line(a.p, a.shared_len, false, kTcRows, kTcKeys, nullptr);
  const int64_t total = line.tiles(line.seq(0)), per = share_size(total, w.shared_workers, 1);
  const int worker = blockIdx.x;
  Walk wk;
  const bool any = wk.begin(line, total, worker, per);
  // a wait that gave up leaves `ok` false: later waits are skipped, the work runs out on whatever is there
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) { ok = ok && mbar_wait_bounded(bar, parity, status); };

  if (any && warp >= kLoadWarp) {
    // ---- loaders: warp p has rows 8g .. 8g + 7 of a tile for g = p, p + 3, ... < 16
    const int p = warp - kLoadWarp;
    constexpr int kChunks = HD / 8;
    constexpr int kPerGroup = 8 * kChunks / 32;
    int slot = 0, tile = 0;
    int loaded = 0, done = 0;            // slots begun, slots handed over
    uint32_t parity = 1;                 // of `empty` for the next use of `slot`: the first round waits for nothing
    auto hand_over = [&]() {
      fence_proxy_async();  // the copies were generic writes; the MMAs read through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.full[done % kSlots]);
      ++done;
    };
    do {
      for (int t = 0; t < wk.n; ++t) {
        // cache rows of this warp's keys: groups 0-3 of the warp in id[0] (lane = 8 * group + row), 4-5 in id[1]
        uint32_t id[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int g = p + 3 * (b * 4 + (lane >> 3));
          const int pos = (wk.c.k + t) * kTcKeys + g * 8 + (lane & 7);
          id[b] = ~0u;
          if (g < 16 && pos < a.shared_len) {
            const int pg = pos / a.p.page_size, page = a.shared_pages[pg];
            if (page >= 0 && page < a.p.n_pages)
              id[b] = cache_row(page, a.p.n_kv, wk.c.head(), a.p.page_size, pos - pg * a.p.page_size);
            else
              report_status(status, kDevBadPage);
          }
        }
        const unsigned there[2] = {__ballot_sync(0xffffffffu, id[0] != ~0u), __ballot_sync(0xffffffffu, id[1] != ~0u)};
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          // while the slot is not free, what has been begun goes over as it lands
          while (loaded > done && !__all_sync(0xffffffffu, mbar_test_wait(&B.empty[slot], parity))) {
            switch (loaded - done) {
              case 1: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
              case 2: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
              default: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
            }
            hand_over();
          }
          wait(&B.empty[slot], parity);
          const bf16* src = kv ? a.p.v : a.p.k;
          const uint32_t dst = smem_u32(smem + L::kRing + slot * L::kTile);
#pragma unroll
          for (int y = 0; y < 6; ++y) {
            const int g = p + 3 * y;
            if (g >= 16) break;
#pragma unroll
            for (int i = 0; i < kPerGroup; ++i) {
              const int e = i * 32 + lane, r = e / kChunks, c = e % kChunks;
              const uint32_t row = __shfl_sync(0xffffffffu, id[y >> 2], (y & 3) * 8 + r);
              const bool on = row != ~0u;
              cp16(dst + tile_at(g * 8 + r, c), src + (on ? (size_t)row * HD + c * 8 : 0), on);
            }
            if (kv == 0 && lane == 0) B.valid[tile % kValid][g] = (unsigned char)(there[y >> 2] >> ((y & 3) * 8));
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
          ++loaded;
          if (loaded - done > kLag) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
            hand_over();
          }
          if (++slot == kSlots) {
            slot = 0;
            parity ^= 1;
          }
        }
        ++tile;
      }
    } while (wk.next(line));
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    while (done < loaded) hand_over();
  } else if (any && warp == kMmaWarp) {
    if (lane == 0) {
      // ---- MMA issuer.  A group's QK^T of a tile follows its PV of the one before (P lies over S; MMAs run in order).
      constexpr uint32_t id_s = idesc(128, false), id_pv = idesc(HD, true);
      int slot = 0;             // of the next K tile
      uint32_t full_parity[kSlots];
#pragma unroll
      for (int s = 0; s < kSlots; ++s) full_parity[s] = 0;
      uint32_t p_parity[2] = {0, 0};
      uint32_t seg_parity = 0;
      int pend[2] = {-1, -1};   // V slot that a group's P waits for
      bool first[2] = {true, true}, frees[2] = {true, true};  // its PV begins O / is the slot's last use
      // the ring's slots in order: wait for each once
      uint32_t waited = 0;      // bit s: slot s' current contents are there
      auto need = [&](int s) {
        if (waited >> s & 1) return;
        uint32_t par = 0;
#pragma unroll
        for (int x = 0; x < kSlots; ++x)
          if (x == s) {
            par = full_parity[x];
            full_parity[x] ^= 1;
          }
        wait(&B.full[s], par);
        waited |= 1u << s;
      };
      auto release = [&](int s) {
        umma_commit(&B.empty[s]);
        waited &= ~(1u << s);
      };
      auto pv = [&](int g) {
        if (pend[g] < 0) return;
        wait(&B.p_full[g], p_parity[g]);
        p_parity[g] ^= 1;
        need(pend[g]);
        tfence_after();
        const unsigned char* V = smem + L::kRing + pend[g] * L::kTile;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_ta(tmem + 256 + 128 * g, tmem + 128 * g + 64 + 8 * k, desc_mnmajor(V + k * 2048), id_pv, (k > 0 || !first[g]) ? 1u : 0u);
        if (frees[g]) release(pend[g]);
        umma_commit(&B.o_done[g]);
        pend[g] = -1;
        first[g] = false;
      };
      do {
        const bool pair = wk.pair();
        for (int g = 0; g < 2; ++g) {
          wait(&B.q_full[g], seg_parity);
          first[g] = true;
        }
        seg_parity ^= 1;
        for (int t = 0; t < wk.n; ++t) {
          const int ks = slot, vs = slot + 1 == kSlots ? 0 : slot + 1;
          slot = vs + 1 == kSlots ? 0 : vs + 1;
          for (int g = pair ? 0 : t & 1; g < (pair ? 2 : (t & 1) + 1); ++g) {
            pv(g);
            need(ks);
            tfence_after();
            const unsigned char* Q = smem + L::kQ + g * L::kTile;
            const unsigned char* K = smem + L::kRing + ks * L::kTile;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
              umma(tmem + 128 * g, desc_kmajor(Q + (k >> 2) * kBlk) + 2 * (k & 3), desc_kmajor(K + (k >> 2) * kBlk) + 2 * (k & 3),
                   id_s, k > 0 ? 1u : 0u);
            umma_commit(&B.s_full[g]);
            mbar_arrive(&B.s_full[g]);  // and the key masks that `need` has seen
            pend[g] = vs;
            frees[g] = !pair || g == 1;
          }
          release(ks);
        }
        // the segment's last products, in the order that their tiles were begun
        const int g0 = pair ? 0 : wk.n & 1;
        pv(g0);
        pv(g0 ^ 1);
      } while (wk.next(line));
    }
  } else if (any && warp < kMmaWarp) {
    // ---- softmax: group g, row r of its tile
    const int g = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + 128 * g;
    const float sl2 = fabsf(a.scale) * kLog2e;
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
    uint32_t s_parity = 0;
    uint32_t tiles = 0;   // of this group so far
    int tile = -1;        // of the share
    uint32_t other = 0;   // tiles of the other group so far
    do {
      const bool pair = wk.pair();
      const int h = wk.c.head();
      const int base = (wk.c.seg - h * wk.c.mt) * kTcRows + (pair ? 128 * g : 0);
      const int R = line.n_rows * line.hpg;
      const bool mine = base + r < R;
      const int tok = mine ? (base + r) / line.hpg : 0;
      const size_t head = (size_t)tok * a.p.n_q + h * line.hpg + (mine ? base + r - tok * line.hpg : 0);
      const bool busy = base + (r & ~31) < R;  // some row of this warp is there
      {
        unsigned char* Q = smem + L::kQ + g * L::kTile;
        const uint4* src = reinterpret_cast<const uint4*>(a.q + head * HD);
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
          uint4 v = mine ? src[c] : make_uint4(0u, 0u, 0u, 0u);
          v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
          *reinterpret_cast<uint4*>(Q + tile_at(r, c)) = v;
        }
        fence_proxy_async();
        mbar_arrive(&B.q_full[g]);
      }
      float m = -INFINITY, l = 0.f;
      int mine_n = 0;  // tiles of this group in the segment
      for (int t = 0; t < wk.n; ++t) {
        ++tile;
        if (!pair && (t & 1) != g) {
          ++other;
          continue;
        }
        if (pair) ++other;
        wait(&B.s_full[g], s_parity);
        s_parity ^= 1;
        tfence_after();
        if (busy) {
          // keys 64-127 stay in registers between the maximum and the
          // exponentials, keys 0-63 are read twice (128 floats would spill)
          float sa[32], sb[32];
          const uint4 there = *reinterpret_cast<const uint4*>(B.valid[tile % kValid]);
          const bool all = (there.x & there.y & there.z & there.w) == 0xffffffffu;
          auto get = [&](int c) {  // 32 c .. 32 c + 63
            tld32(tS + 32 * c, sa);
            tld32(tS + 32 * c + 32, sb);
            wait_ld(sa);
            wait_ld(sb);
            if (!all) {
              const uint32_t ba = c ? there.z : there.x, bb = c ? there.w : there.y;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                if (!(ba >> i & 1u)) sa[i] = -INFINITY;
                if (!(bb >> i & 1u)) sb[i] = -INFINITY;
              }
            }
          };
          float mx0 = -INFINITY, mx1 = -INFINITY;
          auto most = [&]() {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              mx0 = fmaxf(mx0, sa[i]);
              mx1 = fmaxf(mx1, sb[i]);
            }
          };
          get(0);
          most();
          get(2);
          most();
          float mx = fmaxf(mx0, mx1) * sl2;
          if (sl2 == 0.f) mx = 0.f;
          const bool up = mx > m + kRescale || (m == -INFINITY && mx > m);
          if (__any_sync(0xffffffffu, up)) {
            const float alpha = up ? ex2f(m - mx) : 1.f;  // 0 at the first tile
            if (mine_n > 0) {
              wait(&B.o_done[g], (tiles - 1) & 1);  // the products so far are in O
              tfence_after();
#pragma unroll
              for (int c = 0; c < HD / 32; ++c) {
                float v[32];
                tld32(tS + 256 + 32 * c, v);
                wait_ld(v);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] *= alpha;
                tst32(tS + 256 + 32 * c, v);
              }
            }
            l *= alpha;
            if (up) m = mx;
          }
          const float nb = m == -INFINITY ? 0.f : -m;
          float sum0 = 0.f, sum1 = 0.f;
          auto put = [&](int c, const float(&s)[32]) {  // P of keys 32 c .. 32 c + 31
            uint32_t u[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float p0 = ex2f(fmaf(s[2 * e], sl2, nb)), p1 = ex2f(fmaf(s[2 * e + 1], sl2, nb));
              sum0 += p0;
              sum1 += p1;
              const __nv_bfloat162 two = __floats2bfloat162_rn(p0, p1);
              u[e] = *reinterpret_cast<const uint32_t*>(&two);
            }
            tst16u(tS + 64 + 16 * c, u);
          };
          put(2, sa);
          put(3, sb);
          get(0);
          put(0, sa);
          put(1, sb);
          l += sum0 + sum1;
          tmem_wait_st_();
        }
        tfence_before();
        mbar_arrive(&B.p_full[g]);
        ++tiles;
        ++mine_n;
      }
      // ---- the segment's pieces
      float* dst;
      const bool first = wk.whole_first;
      const size_t at = first ? head : (size_t)worker * kTcRows + (pair ? 128 * g : 0) + r;
      dst = (first ? w.shared.first_o : w.shared.more_o) + at * HD;
      float2* ml = (first ? w.shared.first_ml : w.shared.more_ml) + at;
      if (pair) {
        wait(&B.o_done[g], (tiles - 1) & 1);
        tfence_after();
        if (busy) {
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) {
            float v[32];
            tld32(tS + 256 + 32 * c, v);
            wait_ld(v);
            if (mine) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                reinterpret_cast<float4*>(dst + 32 * c)[e] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
            }
          }
          if (mine) *ml = make_float2(m, l);
        }
        tfence_before();
      } else {
        // both groups have these rows: each joins one half of the columns
        // (maxima and sums meet where the Q tiles were: their last S is done)
        auto mls = [&](int x) { return reinterpret_cast<float2*>(smem + L::kQ + x * L::kTile) + r; };
        *mls(g) = make_float2(m, l);
        if (mine_n > 0) wait(&B.o_done[g], (tiles - 1) & 1);
        const int other_n = wk.n - mine_n;
        if (other_n > 0) wait(&B.o_done[g ^ 1], (other - 1) & 1);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        tfence_after();
        if (busy) {
          const float2 x = *mls(0), y = *mls(1);
          const int n0 = g == 0 ? mine_n : other_n, n1 = wk.n - n0;
          const float to = fmaxf(x.x, y.x), b = to == -INFINITY ? 0.f : to;
          const float wx = ex2f(x.x - b), wy = ex2f(y.x - b);
          const uint32_t tO = tmem + lanes + 256 + g * (HD / 2);
#pragma unroll
          for (int c = 0; c < HD / 64; ++c) {
            float u[32], v[32];
            tld32(tO + 32 * c, u);
            tld32(tO + 128 + 32 * c, v);
            wait_ld(u);
            wait_ld(v);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float z = n0 > 0 ? u[i] * wx : 0.f;  // a group without tiles: its O is not defined
              if (n1 > 0) z = fmaf(v[i], wy, z);
              u[i] = z;
            }
            if (mine) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                reinterpret_cast<float4*>(dst + g * (HD / 2) + 32 * c)[e] =
                    make_float4(u[4 * e], u[4 * e + 1], u[4 * e + 2], u[4 * e + 3]);
            }
          }
          if (mine && g == 0) *ml = make_float2(to, x.y * wx + y.y * wy);
        }
        tfence_before();
        asm volatile("bar.sync 1, 256;" ::: "memory");  // both have read both
      }
    } while (wk.next(line));
  }
  tfence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tfence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
  }
}

template <int HD>
cudaError_t launch(const PagedWork& w, int num_sms, cudaStream_t st) {
  static cudaError_t once = cudaFuncSetAttribute(paged_shared_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 Smem<HD>::kBytes);
  if (once != cudaSuccess) return once;
  paged_shared_tc_kernel<HD><<<num_sms, kThreads, Smem<HD>::kBytes, st>>>(w);
  return cudaGetLastError();
}

}  // namespace

cudaError_t paged_shared_tc_launch(const PagedWork& w, int num_sms, cudaStream_t st) {
  return w.a.p.head_dim == 128 ? launch<128>(w, num_sms, st) : launch<64>(w, num_sms, st);
}

}  // namespace emx
