// paged_plan.h — the index arithmetic of the batched operators over a paged
// K/V cache: which rows, positions and pages belong to a sequence, and how
// the key tiles of all (sequence, KV head, row tile) segments are dealt out
// to a fixed grid.  Plain integer functions, shared by the kernels and by a
// host test that walks every index for whole batches.
#pragma once
#include <stdint.h>

#include <atomic>

#ifdef __CUDACC__
#define EMX_HD __host__ __device__ __forceinline__
#else
#define EMX_HD inline
#endif

namespace emx {

// One sequence of a batch: rows [row0, row0 + rows) of the batch are its last
// `rows` positions, of `len` in all.  !ok: the batch names rows, or a length,
// that cannot be (see seq_info).
struct SeqInfo {
  int row0, rows, len;
  bool ok;
};

// rows [a, b) of a batch of n_rows, `len` positions of which the first
// `shared` belong to the common prefix, `room` positions in the page table.
// A sequence without rows is always in order (nothing of it is looked at).
EMX_HD SeqInfo seq_info(int a, int b, int len, int n_rows, int shared, int64_t room) {
  SeqInfo s;
  s.ok = true;
  if (a < 0 || b < a || b > n_rows) {
    s.row0 = s.rows = s.len = 0;
    s.ok = false;
    return s;
  }
  s.row0 = a;
  s.rows = b - a;
  s.len = len;
  if (s.rows > 0 && (len < 0 || (int64_t)len < (int64_t)shared + s.rows || (int64_t)len > room)) s.ok = false;
  return s;
}

// What `set` sets (a kernel's attributes: 0 or an error) holds for one device,
// so it is called until it has gone well on each; `done` has a bit for a device.
template <typename F>
inline auto once_a_device(std::atomic<uint64_t>& done, int device, F set) -> decltype(set()) {
  const uint64_t bit = device >= 0 && device < 64 ? 1ull << device : 0;  // a 65th is set every time
  if (done.load(std::memory_order_acquire) & bit) return {};
  const auto e = set();
  if (e == decltype(e){}) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// x / per, by the short 32-bit division wherever both fit it.
EMX_HD int share_of(int64_t x, int64_t per) {
  return (x | per) >> 32 ? (int)(x / per) : (int)((uint32_t)x / (uint32_t)per);
}
EMX_HD int ceil_div(int64_t a, int b) { return share_of(a + b - 1, b); }

// Row (in units of head_dim elements) of the cache [n_pages, n_kv, page_size]
// that holds position `off` of page `page` for KV head h; the host refuses a
// cache of 2^31 rows or more.
EMX_HD uint32_t cache_row(int page, int n_kv, int h, int page_size, int off) {
  return ((uint32_t)page * (uint32_t)n_kv + (uint32_t)h) * (uint32_t)page_size + (uint32_t)off;
}

// Segments: (KV head, row tile) pairs of one sequence, row tiles innermost,
// each of `kt` key tiles and, before them, `setup` units for what a segment
// costs its worker besides its tiles.  Units of sequence i are [start_i,
// start_{i+1}) of the batch's T.  Workers take the units in order, so those of a
// segment's tiles follow one another: the first `early` workers early_per units
// each up to unit `cut`, the others late_per each from there on.
struct Shares {
  int64_t cut, early_per, late_per;
  int early;
  EMX_HD int64_t begin(int worker) const {
    if (worker >= early) return cut + (int64_t)(worker - early) * late_per;
    const int64_t x = (int64_t)worker * early_per;
    return x < cut ? x : cut;
  }
  // the worker of a unit
  EMX_HD int of(int64_t x) const { return x < cut ? share_of(x, early_per) : early + share_of(x - cut, late_per); }
};

// Even shares of a line of `units`, but for the first `early` workers, where they
// have time for more than that, `each` units, before the others begin.
EMX_HD Shares deal(int64_t units, int workers, int early, int each) {
  Shares s;
  s.early = (int64_t)each * workers > units ? early : 0;
  s.cut = (int64_t)s.early * each;
  s.early_per = each;
  if (s.early > 0 && s.cut >= units) {  // they have time for all
    s.cut = units;
    s.early_per = share_of(units + early - 1, early);
  }
  s.late_per = share_of(units - s.cut + workers - s.early - 1, workers - s.early);
  return s;
}

// The line of key tiles of one part of a batch's positions: the common prefix
// [0, shared_len), as one sequence with every row of the batch, or (own) each
// sequence's positions from shared_len on.  Row tiles hold `mt` rows (a row
// being one q head of one new token), key tiles `keys` positions.
struct Line {
  bool own;
  int n_seqs, n_rows, n_kv, hpg, shared_len, mt, keys, setup;
  int64_t room;          // positions of a page table
  const int* indptr;
  const int* lengths;
  const int64_t* starts;  // own: units before each sequence

  EMX_HD SeqInfo seq(int i) const {
    if (own) return seq_info(indptr[i], indptr[i + 1], lengths[i], n_rows, shared_len, room);
    SeqInfo s;
    s.row0 = 0;
    s.rows = n_rows;
    s.len = shared_len;
    s.ok = true;
    return s;
  }
  EMX_HD int row_tiles(const SeqInfo& s) const { return ceil_div((int64_t)s.rows * hpg, mt); }
  EMX_HD int key_tiles(const SeqInfo& s) const { return ceil_div(own ? s.len - shared_len : s.len, keys); }
  EMX_HD int64_t units(const SeqInfo& s) const {
    if (!s.ok || s.rows == 0) return 0;
    return (int64_t)n_kv * row_tiles(s) * (key_tiles(s) + setup);
  }
};

// Where a worker stands in a line: at a tile, or behind the last one.
struct Cursor {
  int seq, seg, k;  // sequence, segment within it, key tile within that
  int mt, kt;       // row tiles a KV head, key tiles a segment
  int64_t x;        // the tile's unit
  SeqInfo s;

  EMX_HD void enter(const Line& line) {
    s = line.seq(seq);
    mt = line.row_tiles(s);
    kt = line.key_tiles(s);
  }
  // To the first tile at or behind unit `to` < T.
  EMX_HD void seek(const Line& line, int64_t to) {
    seq = 0;
    int64_t at = 0;
    if (line.own) {
      int lo = 0, hi = line.n_seqs - 1;  // the last sequence that begins at or before it
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (line.starts[mid] <= to) lo = mid;
        else hi = mid - 1;
      }
      seq = lo;
      at = line.starts[lo];
    }
    enter(line);
    const int each = kt + line.setup;
    seg = share_of(to - at, each);
    at += (int64_t)seg * each;
    k = (int)(to - at) - line.setup;
    if (k < 0) k = 0;
    x = at + line.setup + k;
  }
  // To the next tile; the caller does not go on from the last one's unit T - 1.
  EMX_HD void next(const Line& line) {
    ++x;
    if (++k < kt) return;
    k = 0;
    x += line.setup;
    if (++seg < mt * line.n_kv || !line.own) return;
    seg = 0;
    do ++seq;
    while (seq < line.n_seqs - 1 && line.starts[seq + 1] == line.starts[seq]);
    if (seq < line.n_seqs) enter(line);
  }
  EMX_HD int head() const { return seg / mt; }
};

}  // namespace emx
