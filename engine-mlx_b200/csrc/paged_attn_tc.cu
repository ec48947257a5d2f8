// paged_attn_tc.cu — the shared prefix of emx_sdpa_paged for a batch of many
// rows, on tcgen05.
//
// All rows of the batch that use one KV head (n_rows * n_q / n_kv of them)
// attend the same S keys without a mask, so the prefix is two dense products
// around a softmax: S = Q K^T, O = P V, rows in tiles of 128, keys in tiles of
// 128.  K and V are read from HBM once per KV head and 256 rows.  A tile of 256
// rows and 128 keys takes 2.48 us (2.13 with K and V in L2): 10.1 TFLOP/s of MMAs an
// SM, of the 11.4 that the library's measured rate comes to; the exponentials alone
// (128 x 128 twice, 16 an SM and clock) 1.1.  A tile of up to 128 rows takes 1.61 us,
// its 64 KB on all SMs 1.35 (7 TB/s out of L2 and HBM together).  A worker's start
// (barriers, Q, the first keys) takes 4 us, the end (pieces to memory) 4.
//
// One CTA an SM, each with an even share of the (KV head, 256 rows, 128 keys)
// tiles in line order; twelve warps:
//   warps 0-7  two softmax groups of 128 threads, a thread a row: S from
//              tensor memory, the running maximum and sum, P back over S;
//   warps 8-9  one thread each issues the MMAs of a group;
//   warp 11    one thread waits for the slots that a half's products and the
//              next scores read, and arrives with their P: each wait costs an
//              issuing thread some 200 cycles of the tensor pipe;
//   warp 10    TMA: a lane for each run of keys in one page (a box of 8 to 128
//              rows, the largest power of two that divides the page size),
//              into a ring of five 128-row slots (K, V, K, V, ...).  Boxes
//              behind the prefix and pages outside the cache start beyond the
//              tensor and read as zeros.  A copy takes 20 to 30 ns of the SM's copy
//              engine, so it brings whole rows: with two for the two 64-column
//              blocks a tile of 16-position pages took 2.2 us.  (16-byte
//              asynchronous copies by two or three warps, which take any page size,
//              reached 30 KB/us an SM.)
// Each group is a stream of its own — S, P and O in tensor memory, its Q tile
// in shared memory: two row tiles against the same keys where the segment has
// more than 128 rows, else the same rows against alternate key tiles (then the
// two halves join at the segment's end).  A tile's S comes in two halves of 64
// keys: while a group takes one half's exponentials the tensor pipe adds the
// other's products to O and computes that half of the next tile's S in its
// place, so the group finds its next S ready.
//
// The maximum that the exponentials use moves only when a tile's exceeds it by
// more than 2^8 (then O and l are rescaled); O / l does not depend on it.  P goes
// to its product as the sum of two bf16 (off by at most 2^-14 of each weight, see
// split_weights), which takes another half of the two products' MMAs: with one
// bf16, off by 2^-8, a tile took 1.8 us, and the output's error was 1.4 times its own
// rounding.
#include <cudaTypedefs.h>

#include <mutex>

#include "paged_attn.cuh"
#include "tc_attn.cuh"

namespace emx {

namespace {

constexpr int kThreads = 384;
constexpr int kSlots = 5;
constexpr int kMmaWarp = 8, kLoadWarp = 10, kKeyWarp = 11;
constexpr float kRescale = 8.0f;
constexpr uint32_t kCols = 512;  // S of the groups at 0 and 128 (P of a half over it, high parts and low parts 32 columns each), O at 256 and 384
constexpr int kValid = 4;        // tiles whose key masks are kept: a tile's V slot is free before the ring holds 3 later ones

template <int HD>
struct Smem {
  static constexpr int kTile = HD / 64 * kBlk;  // 128 rows of HD
  // K and V lie in groups of 8 rows, a group's 64-column blocks (8 rows of 128 bytes, swizzled) one after another, so
  // that one copy brings whole rows.
  static constexpr int kGroup = HD / 64 * 1024;
  static constexpr int kQ = 0;                  // [2]
  static constexpr int kRing = 2 * kTile;       // [kSlots]
  static constexpr int kBar = kRing + kSlots * kTile;
  static constexpr int kBytes = kBar + 512 + 1024;  // barriers; 1 KB to align
  static_assert(kBytes <= 227 * 1024, "");
};

struct Bars {
  uint64_t full[kSlots], empty[kSlots];
  uint64_t q_full[2];
  uint64_t s_full[2][2], p_full[2][2];  // by group and half
  uint64_t pv_done[2][2];               // a half's products (and all before) are in O
  uint64_t all_done[2];                 // all of a group's products and commits
  uint32_t tmem;
  alignas(16) unsigned char valid[kValid][16];  // by tile of the share, bit j: key j is there
};
static_assert(sizeof(Bars) <= 512, "");

constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}

// A box of 8-row groups from group `y` of the cache on.
__device__ __forceinline__ void tma_groups(uint32_t dst, const CUtensorMap* map, int y, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %2, %2, %3}], [%4], %5;" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(y), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

__device__ __forceinline__ uint64_t l2_evict_normal_policy() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}

// A place in the ring, and the parity of the mbarrier phase that its next use completes.
struct Slot {
  int s;
  uint32_t parity;
  __device__ __forceinline__ void step(int n) {
    s += n;
    if (s >= kSlots) {
      s -= kSlots;
      parity ^= 1;
    }
  }
};

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

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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
  __device__ __forceinline__ bool begin(const Line& line, int worker, int per, int split) {
    c.seq = 0;
    c.enter(line);
    const int segments = c.mt * line.n_kv;
    if (split) {  // this many workers to a segment
      c.seg = worker / split;
      c.k = (worker - c.seg * split) * per;
      left = min(per, c.kt - c.k);
      if (c.seg >= segments || left <= 0) return false;
    } else {
      const int64_t x0 = (int64_t)worker * per, total = (int64_t)segments * c.kt;
      if (x0 >= total) return false;
      left = (int)min((int64_t)per, total - x0);
      c.seg = share_of(x0, c.kt);
      c.k = (int)(x0 - (int64_t)c.seg * c.kt);
    }
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
__global__ void __launch_bounds__(kThreads, 1)
    paged_shared_tc_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                           const __grid_constant__ PagedWork w, int box) {
  using L = Smem<HD>;
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  Bars& B = *reinterpret_cast<Bars*>(smem + L::kBar);
  const PagedAttnArgs& a = w.a;
  int* status = a.p.status;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // The loader sets the barriers up and begins: it needs no tensor memory.
  if (warp == kLoadWarp) {
    if (lane == 0) {
      for (int s = 0; s < kSlots; ++s) {
        mbar_init(&B.full[s], 1);
        mbar_init(&B.empty[s], 2);
      }
      for (int g = 0; g < 2; ++g) {
        mbar_init(&B.q_full[g], 128);
        mbar_init(&B.all_done[g], 1);
        for (int x = 0; x < 2; ++x) {
          mbar_init(&B.s_full[g][x], 2);
          mbar_init(&B.p_full[g][x], x == 0 ? 129 : 128);  // the first half's with its keys
          mbar_init(&B.pv_done[g][x], 1);
        }
      }
      fence_mbar_init();
    }
    __syncwarp();
    asm volatile("bar.arrive 4, %0;" ::"n"(kThreads) : "memory");
  } else {
    if (warp == kMmaWarp) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&B.tmem)), "r"(kCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tfence_before();
    asm volatile("bar.sync 4, %0;" ::"n"(kThreads) : "memory");
    tfence_after();
  }
  pdl_wait();     // what ran before has written q, the cache and the batch
  pdl_trigger();  // the own part does not read what this one writes (it only ends after it)
  const uint32_t tmem = warp == kLoadWarp ? 0u : B.tmem;
  const Line line = make_line(a.p, a.shared_len, false, kTcRows, kTcKeys, 0, nullptr);
  const int worker = blockIdx.x;
  Walk wk;
  const bool any = wk.begin(line, worker, w.shared_per, w.shared_split);
  // a wait that gave up leaves `ok` false: later waits are skipped and no more copies and MMAs are begun
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) { ok = ok && mbar_wait_bounded(bar, parity, status); };

  if (any && warp == kLoadWarp) {
    // ---- loader: lane b has box b of a tile
    const int boxes = kTcKeys / box;
    // keys that one row tile reads are first out of L2; more row tiles read them again
    const uint64_t policy = wk.c.mt == 1 ? l2_evict_first_policy() : l2_evict_normal_policy();
    const int64_t beyond = (int64_t)a.p.n_pages * a.p.n_kv * a.p.page_size;
    // the page is loaded a tile ahead and not looked at here: a look would wait for it
    auto look_up = [&](int k) {
      const int pos = k * kTcKeys + lane * box;
      return lane < boxes && pos < a.shared_len ? a.shared_pages[pos / a.p.page_size] : -1;
    };
    Slot at{0, 1};  // `empty`: the first round waits for nothing
    int page = look_up(wk.c.k), tile = 0, copies = 0;  // `copies`: slots filled
    bool more = true;
    for (int t = 0; more;) {
      const int pos = (wk.c.k + t) * kTcKeys + lane * box;
      bool on = lane < boxes && pos < a.shared_len;
      if (on && (page < 0 || page >= a.p.n_pages)) {
        report_status(status, kDevBadPage);
        on = false;
      }
      const int row = on ? (int)cache_row(page, a.p.n_kv, wk.c.head(), a.p.page_size, pos % a.p.page_size) : (int)beyond;
      if (++t == wk.n) {
        more = wk.next(line);
        t = 0;
      }
      if (more) page = look_up(wk.c.k + t);
#pragma unroll 1
      for (int kv = 0; kv < 2; ++kv) {
        wait(&B.empty[at.s], at.parity);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (kv == 0 && lane < boxes)
          for (int g = 0; g < box / 8; ++g) B.valid[tile % kValid][lane * (box / 8) + g] = on ? 0xff : 0;
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&B.full[at.s], (uint32_t)L::kTile);
        __syncwarp();
        if (lane < boxes) {
          const uint32_t dst = smem_u32(smem + L::kRing + at.s * L::kTile) + (uint32_t)(lane * (box / 8) * L::kGroup);
          tma_groups(dst, kv ? &tv : &tk, row / 8, &B.full[at.s], policy);
        }
        at.step(1);
        ++copies;
      }
      if (!ok) break;
      ++tile;
    }
    // copies still on their way (after a wait that gave up) have landed before the CTA ends
    for (int i = copies; i-- > 0 && i >= copies - kSlots;) mbar_wait_bounded(&B.full[i % kSlots], (i / kSlots) & 1, status);
  } else if (any && warp == kKeyWarp) {
    if (lane == 0) {
      Slot ks{0, 0}, vs{1, 0};
      uint32_t p_parity[2] = {0, 0};
      auto there = [&](int g) { mbar_arrive(&B.p_full[g][0]); };
      auto passed = [&](int g) {  // before the next arrival
        wait(&B.p_full[g][0], p_parity[g]);
        p_parity[g] ^= 1;
      };
      do {
        for (int t = 0; t < wk.n; ++t) {
          ks.step(2);
          wait(&B.full[vs.s], vs.parity);
          if (wk.pair()) {
            if (t + 1 < wk.n) wait(&B.full[ks.s], ks.parity);
            there(0);
            there(1);
            passed(0);
            passed(1);
          } else if (t & 1) {
            there(1);
            passed(1);
          } else {
            there(0);
            passed(0);
          }
          vs.step(2);
        }
      } while (wk.next(line));
    }
  } else if (any && warp >= kMmaWarp) {
    if (lane == 0) {
      // ---- MMA issuer of group g.  S of a half follows the products of that half of the group's tile before (P lies
      // over S; the MMAs of a thread run in the order of their issue).
      const int g = warp - kMmaWarp;
      constexpr uint32_t id_s = idesc(64, false), id_pv = idesc(HD, true);
      // operand descriptors: the low word holds the address in 16-byte units, the high word is the same for all tiles
      const uint64_t q0 = desc_kmajor(smem), k0 = desc_kmajor(smem, L::kGroup), v0 = desc_mnmajor(smem, 1024, L::kGroup);
      auto at16 = [](uint64_t d, uint32_t bytes) {
        return (d & 0xffffffff00000000ull) | (uint32_t)((uint32_t)d + (bytes >> 4));
      };
      auto soon = [&](uint64_t* bar, uint32_t parity) {  // polls closely before the bounded wait's longer steps
        for (int i = 0; i < 2000 && ok; ++i)
          if (mbar_test_wait(bar, parity)) return;
        wait(bar, parity);
      };
      const uint64_t Q = at16(q0, L::kQ + g * L::kTile);
      const uint32_t tS = tmem + 128 * g, tO = tmem + 256 + 128 * g;
      auto qk = [&](int s, int half) {
        const uint64_t K = at16(k0, L::kRing + s * L::kTile + half * 8 * L::kGroup);  // its 64 rows
        if (ok) {
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)  // 16 head dims a step: 32 bytes along the rows of a 64-column block
            umma(tS + 64 * half, at16(Q, (k >> 2) * kBlk + 32 * (k & 3)), at16(K, (k >> 2) * 1024 + 32 * (k & 3)), id_s,
                 k > 0 ? 1u : 0u);
        }
        umma_commit(&B.s_full[g][half]);
        mbar_arrive(&B.s_full[g][half]);  // and the key masks, which the wait for K has seen
      };
      uint32_t p_parity = 0, seg_parity = 0;
      auto pv = [&](int s, int half, bool first) {
        soon(&B.p_full[g][half], p_parity);
        tfence_after();
        const uint64_t V = at16(v0, L::kRing + s * L::kTile + half * 8 * L::kGroup);
        if (ok) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // 16 keys a step: 8 columns of P, high and low parts, 16 rows of V
            umma_ta(tO, tS + 64 * half + 8 * k, at16(V, k * 2 * L::kGroup), id_pv, (k > 0 || half > 0 || !first) ? 1u : 0u);
            umma_ta(tO, tS + 64 * half + 32 + 8 * k, at16(V, k * 2 * L::kGroup), id_pv, 1u);
          }
        }
        umma_commit(&B.pv_done[g][half]);
      };
      Slot ks{0, 0}, vs{1, 0};
      do {
        wait(&B.q_full[g], seg_parity);
        seg_parity ^= 1;
        if (wk.pair()) {
          soon(&B.full[ks.s], ks.parity);
          tfence_after();
          qk(ks.s, 0);
          qk(ks.s, 1);
          umma_commit(&B.empty[ks.s]);
          ks.step(2);
          for (int t = 0; t < wk.n; ++t) {
            const bool next = t + 1 < wk.n;
            pv(vs.s, 0, t == 0);
            if (next) qk(ks.s, 0);
            pv(vs.s, 1, false);
            umma_commit(&B.empty[vs.s]);
            if (next) {
              qk(ks.s, 1);
              umma_commit(&B.empty[ks.s]);
              ks.step(2);
            }
            p_parity ^= 1;
            vs.step(2);
          }
        } else {
          // alternate tiles: nothing waits for a later tile's keys, so that its V slot can be filled again soon
          for (int t = 0; t < wk.n; ++t) {
            soon(&B.full[ks.s], ks.parity);
            if ((t & 1) == g) {
              tfence_after();
              qk(ks.s, 0);
              qk(ks.s, 1);
              umma_commit(&B.empty[ks.s]);
              pv(vs.s, 0, t < 2);
              pv(vs.s, 1, false);
              umma_commit(&B.empty[vs.s]);
              p_parity ^= 1;
            } else {
              mbar_arrive(&B.empty[ks.s]);  // the other group's: free of this one
              soon(&B.full[vs.s], vs.parity);
              mbar_arrive(&B.empty[vs.s]);
            }
            ks.step(2);
            vs.step(2);
          }
        }
      } while (wk.next(line));
      // nothing of this thread's is on its way when the CTA ends, whatever waits gave up
      umma_commit(&B.all_done[g]);
      mbar_wait_bounded(&B.all_done[g], 0, status);
    }
  } else if (any) {
    // ---- softmax: group g, row r of its tile
    const int g = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + 128 * g;
    const float sl2 = fabsf(a.scale) * kLog2e;
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
    uint32_t s_parity = 0;
    uint32_t tiles = 0;     // of this group so far
    int tile = -1;          // of the share
    // The groups of a pair take their exponentials in turn: in step (which they fall into) both want that unit at the same
    // time and leave it idle while both load, take maxima and wait.
    auto my_turn = [&](bool pair) {
      if (pair) asm volatile("bar.sync %0, 256;" ::"r"(5 + g) : "memory");
    };
    auto your_turn = [&](bool pair) {
      if (pair) asm volatile("bar.arrive %0, 256;" ::"r"(5 + (g ^ 1)) : "memory");
    };
    bool begun = false;  // group 1 gives the first turn, once
    do {
      const bool pair = wk.pair();
      if (pair && g == 1 && !begun) {
        your_turn(true);
        begun = true;
      }
      const int h = wk.c.head();
      const int base = (wk.c.seg - h * wk.c.mt) * kTcRows + (pair ? 128 * g : 0);
      const int R = line.n_rows * line.hpg;
      const bool mine = base + r < R;
      const int tok = mine ? (base + r) / line.hpg : 0;
      const size_t head = (size_t)tok * a.p.n_q + h * line.hpg + (mine ? base + r - tok * line.hpg : 0);
      const bool busy = base + (r & ~31) < R;  // some row of this warp is there
      const unsigned rows_here = __ballot_sync(0xffffffffu, mine);
      {
        // this warp's 32 rows of q, two (at D = 64 four) at a time
        unsigned char* Q = smem + L::kQ + g * L::kTile;
        constexpr int kLanes = HD / 8;  // of a row
        const int c = lane % kLanes;
        uint4 v[kLanes];
#pragma unroll
        for (int i = 0; i < kLanes; ++i) {
          const int x = i * (32 / kLanes) + lane / kLanes;
          const size_t from = __shfl_sync(0xffffffffu, (unsigned long long)head, x);
          v[i] = rows_here >> x & 1u ? *reinterpret_cast<const uint4*>(a.q + from * HD + c * 8) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < kLanes; ++i) {
          const int x = i * (32 / kLanes) + lane / kLanes;
          v[i].x ^= flip, v[i].y ^= flip, v[i].z ^= flip, v[i].w ^= flip;
          *reinterpret_cast<uint4*>(Q + tile_at((warp & 3) * 32 + x, c)) = v[i];
        }
        fence_proxy_async();
        mbar_arrive(&B.q_full[g]);
      }
      float m = -INFINITY, l = 0.f;
      int mine_n = 0;  // tiles of this group in the segment
      for (int t = 0; t < wk.n; ++t) {
        ++tile;
        if (!pair && (t & 1) != g) continue;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          wait(&B.s_full[g][half], s_parity);
          tfence_after();
          if (busy) {
            float sa[32], sb[32];
            tld32(tS + 64 * half, sa);
            tld32(tS + 64 * half + 32, sb);
            wait_ld(sa);
            wait_ld(sb);
            const uint2 there = *reinterpret_cast<const uint2*>(&B.valid[tile % kValid][8 * half]);
            const uint32_t ba = there.x, bb = there.y;
            if ((ba & bb) != 0xffffffffu) {
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                if (!(ba >> i & 1u)) sa[i] = -INFINITY;
                if (!(bb >> i & 1u)) sb[i] = -INFINITY;
              }
            }
            float mx0 = max3(sa[0], sa[1], sa[2]), mx1 = max3(sa[16], sa[17], sa[18]);
            float mx2 = max3(sb[0], sb[1], sb[2]), mx3 = max3(sb[16], sb[17], sb[18]);
#pragma unroll
            for (int i = 3; i < 15; i += 2) {
              mx0 = max3(mx0, sa[i], sa[i + 1]);
              mx1 = max3(mx1, sa[16 + i], sa[17 + i]);
              mx2 = max3(mx2, sb[i], sb[i + 1]);
              mx3 = max3(mx3, sb[16 + i], sb[17 + i]);
            }
            mx0 = max3(mx0, sa[15], sa[31]);
            mx1 = max3(mx1, sb[15], sb[31]);
            const float mx = fmaxf(max3(mx0, mx1, mx2), mx3) * sl2;
            const bool up = mx > m + kRescale || (m == -INFINITY && mx > m);
            if (__any_sync(0xffffffffu, up)) {
              const float alpha = up ? ex2f(m - mx) : 1.f;  // 0 at the first tile
              if (mine_n > 0 || half > 0) {
                // O holds all products so far: the half before's (those before it are done, S came after them)
                wait(&B.pv_done[g][half ^ 1], half ? tiles & 1 : (tiles - 1) & 1);
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
            const uint64_t scale2 = pair32(sl2, sl2), base2 = pair32(nb, nb);
            uint64_t sum0 = 0, sum1 = 0;  // pairs of sums
            auto put = [&](int c, const float(&s)[32]) {  // P of keys 32 c .. 32 c + 31 of the half
              uint32_t hi[16], lo[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                float p0, p1;
                split32(fma2(pair32(s[2 * e], s[2 * e + 1]), scale2, base2), p0, p1);
                p0 = ex2f(p0);
                p1 = ex2f(p1);
                uint64_t& sum = e & 1 ? sum1 : sum0;
                sum = add2(sum, pair32(p0, p1));
                split_weights(p0, p1, hi[e], lo[e]);
              }
              tst16u(tS + 64 * half + 16 * c, hi);
              tst16u(tS + 64 * half + 32 + 16 * c, lo);
            };
            my_turn(pair);
            put(0, sa);
            put(1, sb);
            your_turn(pair);
            float l0, l1;
            split32(add2(sum0, sum1), l0, l1);
            l += l0 + l1;
            tmem_wait_st_();
          } else {
            my_turn(pair);
            your_turn(pair);
          }
          tfence_before();
          mbar_arrive(&B.p_full[g][half]);
        }
        s_parity ^= 1;
        ++tiles;
        ++mine_n;
      }
      // ---- the segment's pieces.  A thread has a row, and 32 rows 512 bytes apart would make 32 separate stores of 16
      // bytes of one instruction: a warp turns its 32 rows x 64 columns in shared memory (where its rows of Q were) and
      // stores two rows' 256 bytes at a time.
      const bool first = wk.whole_first;
      const size_t at = first ? head : (size_t)worker * kTcRows + (pair ? 128 * g : 0) + r;
      float* const pieces = first ? w.shared.first_o : w.shared.more_o;
      float2* const ml = (first ? w.shared.first_ml : w.shared.more_ml) + at;
      float* const turn = reinterpret_cast<float*>(smem + L::kQ + g * L::kTile) + (warp & 3) * 32 * (HD / 2);
      auto put_columns = [&](const float(&v)[32], int part) {  // 32 of the HD / 2 columns staged at once
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<float4*>(turn + lane * (HD / 2) + (((part * 8 + e) ^ (lane & (HD / 8 - 1))) << 2)) =
              make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
      };
      auto store_columns = [&](int c0) {  // columns c0 .. c0 + HD / 2 of this warp's rows
        constexpr int kLanes = HD / 8;    // of a row
        __syncwarp();
#pragma unroll 4
        for (int i = 0; i < kLanes; ++i) {
          const int x = i * (32 / kLanes) + lane / kLanes, c = lane % kLanes;
          const size_t to = __shfl_sync(0xffffffffu, (unsigned long long)at, x);
          const float4 v = *reinterpret_cast<const float4*>(turn + x * (HD / 2) + ((c ^ (x & (HD / 8 - 1))) << 2));
          if (rows_here >> x & 1u) *reinterpret_cast<float4*>(pieces + to * HD + c0 + 4 * c) = v;
        }
        __syncwarp();
      };
      if (pair) {
        wait(&B.pv_done[g][1], (tiles - 1) & 1);
        tfence_after();
        if (busy) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
              float v[32];
              tld32(tS + 256 + half * (HD / 2) + 32 * c, v);
              wait_ld(v);
              put_columns(v, c);
            }
            store_columns(half * (HD / 2));
          }
          if (mine) *ml = make_float2(m, l);
        }
        tfence_before();
        asm volatile("bar.sync %0, 128;" ::"r"(2 + g) : "memory");  // the group's next Q comes where the rows were turned
      } else {
        // both groups have these rows: each joins one half of the columns
        // (maxima and sums meet where the Q tiles were: a group's last S is done, so all of its Q has been written and read)
        auto mls = [&](int x) { return reinterpret_cast<float2*>(smem + L::kQ + x * L::kTile) + r; };
        if (mine_n > 0) {
          *mls(g) = make_float2(m, l);
          wait(&B.pv_done[g][1], (tiles - 1) & 1);
        }
        tfence_before();
        asm volatile("bar.sync 1, 256;" ::: "memory");  // both groups' O are done
        const float2 x = *mls(0), y = wk.n > 1 ? *mls(1) : make_float2(-INFINITY, 0.f);
        asm volatile("bar.sync 1, 256;" ::: "memory");  // both have read them: the places may be used again
        tfence_after();
        if (busy) {
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
              u[i] *= wx;
              if (wk.n > 1) u[i] = fmaf(v[i], wy, u[i]);  // group 1 without a tile: its O is not defined
            }
            put_columns(u, c);
          }
          store_columns(g * (HD / 2));
          if (mine && g == 0) *ml = make_float2(to, x.y * wx + y.y * wy);
        }
        tfence_before();
        asm volatile("bar.sync 1, 256;" ::: "memory");  // both have read both O
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

PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;

// The cache's rows [n_pages * n_kv * page_size][head_dim] as [8-row groups][64-column blocks][8][64], in boxes of `box`
// rows, 128-byte swizzle.
cudaError_t encode(CUtensorMap* map, const PagedArgs& p, const void* base, int box) {
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  if (!g_encode) return cudaErrorNotSupported;
  const cuuint64_t row = (cuuint64_t)p.head_dim * 2, blocks = p.head_dim / 64;
  const cuuint64_t dims[4] = {64, 8, blocks, (cuuint64_t)p.n_pages * p.n_kv * p.page_size / 8};
  const cuuint64_t strides[3] = {row, 128, 8 * row};
  const cuuint32_t size[4] = {64, 8, (cuuint32_t)blocks, (cuuint32_t)box / 8}, one[4] = {1, 1, 1, 1};
  return g_encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, size, one,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? cudaSuccess
             : cudaErrorInvalidValue;
}

template <int HD>
cudaError_t launch(const PagedWork& w, int num_sms, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  cudaError_t e = attribute(done, paged_shared_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD>::kBytes);
  if (e != cudaSuccess) return e;
  int box = kTcKeys;
  while (w.a.p.page_size % box) box /= 2;
  CUtensorMap tk, tv;
  e = encode(&tk, w.a.p, w.a.p.k, box);
  if (e == cudaSuccess) e = encode(&tv, w.a.p, w.a.p.v, box);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute at;
  overlapped(cfg, at, (unsigned)num_sms, kThreads, Smem<HD>::kBytes, st);
  return cudaLaunchKernelEx(&cfg, paged_shared_tc_kernel<HD>, tk, tv, w, box);
}

}  // namespace

bool paged_shared_tc_takes(const PagedArgs& p) {
  return p.page_size % 8 == 0 && p.n_pages > 0;
}

cudaError_t paged_shared_tc_launch(const PagedWork& w, int num_sms, cudaStream_t st) {
  return w.a.p.head_dim == 128 ? launch<128>(w, num_sms, st) : launch<64>(w, num_sms, st);
}

}  // namespace emx
