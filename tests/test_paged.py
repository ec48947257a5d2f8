"""The batched operators without a GPU: what they refuse, and the arithmetic that deals a batch's key tiles out to
workers, walked index by index on the host."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import emx

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # an address that nothing reads: every refusal comes before any device work


def kv(**k):
    d = dict(k=P, v=P, n_pages=8, page_size=16, n_kv=2, head_dim=128)
    d.update(k)
    return emx.PagedKVStruct(*[d[n] for n, _ in emx.PagedKVStruct._fields_])


def batch(**k):
    d = dict(n_seqs=2, n_rows=3, max_pages=4, indptr=P, lengths=P, table=P)
    d.update(k)
    return emx.PagedBatchStruct(*[d[n] for n, _ in emx.PagedBatchStruct._fields_])


def refused(rc, word):
    msg = emx.lib().emx_last_error().decode()
    assert rc == emx.ERR_INVALID and word in msg, (rc, msg)


def append(kv_=None, b=None, qkv=P, qn=P, kn=P, eps=1e-6, theta=1e6, n_q=4, out=P, ctx=None):
    return emx.lib().emx_paged_append(ctx, qkv, qn, kn, eps, theta, n_q, kv_ or kv(), b or batch(), out)


def attend(kv_=None, b=None, q=P, n_q=4, scale=0.1, shared=0, pages=None, out=P, ws=P, nbytes=1 << 40, ctx=None):
    return emx.lib().emx_sdpa_paged(ctx, q, kv_ or kv(), b or batch(), n_q, scale, shared, pages, out, ws, nbytes)


def check(target=P, draft=P, dtype=emx.F32, tokens=P, counts=None, u=P, n=2, m=3, v=100, out=P, acc=P, ctx=None):
    return emx.lib().emx_verify_draft(ctx, target, draft, dtype, tokens, counts, u, n, m, v, out, acc)


def test_a_call_in_order_wants_only_its_context():
    for rc in (append(), append(qn=None, kn=None, theta=0.0), attend(), attend(shared=32, pages=P), check(),
               check(draft=None), check(m=0, tokens=None, draft=None)):
        refused(rc, "null context")


BAD_SHAPES = [(dict(kv_=kv(head_dim=96)), "head_dim"), (dict(kv_=kv(n_kv=3)), "multiple"), (dict(kv_=kv(n_kv=0)), "multiple"),
              (dict(n_q=0), "multiple"), (dict(n_q=2048, kv_=kv(n_kv=2)), "1024"), (dict(kv_=kv(page_size=0)), "bad cache"),
              (dict(kv_=kv(n_pages=-1)), "bad cache"), (dict(kv_=kv(n_pages=1 << 30, page_size=64)), "too large"),
              (dict(b=batch(n_seqs=-1)), "n_seqs"), (dict(b=batch(n_seqs=1025)), "n_seqs"), (dict(b=batch(n_rows=-1)), "n_rows"),
              (dict(b=batch(n_rows=1 << 30)), "n_rows"), (dict(b=batch(max_pages=0)), "max_pages"),
              (dict(b=batch(max_pages=1 << 28)), "max_pages"), (dict(kv_=kv(k=None)), "null"), (dict(kv_=kv(v=None)), "null"),
              (dict(b=batch(indptr=None)), "null"), (dict(b=batch(lengths=None)), "null"), (dict(b=batch(table=None)), "null"),
              (dict(kv_=kv(k=P + 8)), "aligned"), (dict(b=batch(table=P + 2)), "misaligned"), (dict(out=None), "null")]


@pytest.mark.parametrize("call", [append, attend])
@pytest.mark.parametrize("args,word", BAD_SHAPES)
def test_bad_shapes_are_refused(call, args, word):
    refused(call(**args), word)


@pytest.mark.parametrize("args,word", [(dict(qkv=None), "null"), (dict(theta=-1.0), "rope_theta"), (dict(theta=float("inf")), "rope_theta"),
                                       (dict(theta=float("nan")), "rope_theta"), (dict(qkv=P + 4), "aligned"), (dict(qn=P + 2), "aligned"),
                                       (dict(out=P + 4), "aligned")])
def test_append_refuses(args, word):
    refused(append(**args), word)


@pytest.mark.parametrize("args,word", [(dict(q=None), "null"), (dict(ws=None), "null"), (dict(shared=-16, pages=P), "whole pages"),
                                       (dict(shared=24, pages=P), "whole pages"), (dict(shared=32), "shared_pages"),
                                       (dict(shared=80, pages=P), "exceeds"), (dict(q=P + 8), "aligned"), (dict(out=P + 8), "aligned"),
                                       (dict(ws=P + 16), "aligned"), (dict(shared=32, pages=P + 1), "misaligned")])
def test_attend_refuses(args, word):
    refused(attend(**args), word)


@pytest.mark.parametrize("args,word", [(dict(target=None), "null"), (dict(tokens=None), "null"), (dict(u=None), "null"),
                                       (dict(out=None), "null"), (dict(acc=None), "null"), (dict(dtype=emx.U32), "f32 or bf16"),
                                       (dict(n=-1), "shape"), (dict(n=1 << 20), "shape"), (dict(m=-1), "shape"), (dict(v=0), "shape"),
                                       (dict(target=P + 2), "misaligned"), (dict(u=P + 2), "misaligned"), (dict(counts=P + 1), "misaligned")])
def test_verify_refuses(args, word):
    refused(check(**args), word)


def test_workspace_query_refuses():
    n = C.c_size_t()
    f = emx.lib().emx_sdpa_paged_workspace
    refused(f(None, kv(), batch(), 4, 0, None), "null")
    refused(f(None, kv(head_dim=32), batch(), 4, 0, C.byref(n)), "head_dim")
    refused(f(None, kv(), batch(), 4, -16, C.byref(n)), "shared_len")
    refused(f(None, kv(k=None, v=None), batch(indptr=None, lengths=None, table=None), 4, 0, C.byref(n)), "null context")


@pytest.mark.parametrize("page_size,max_pages,fits", [(32767, 65538, False), (1, 2**31 - 1, False), (1, 2**31 - 255, False),
                                                      (1, 2**31 - 256, True), (256, 2**23 - 1, True)])
def test_the_last_key_tile_of_a_table_ends_in_int32(page_size, max_pages, fits):
    """A tile of 64 positions behind a prefix that is no multiple of it may end beyond the table; its positions are int32."""
    for call in (append, attend):
        refused(call(kv_=kv(page_size=page_size), b=batch(max_pages=max_pages)), "null context" if fits else "max_pages")
    refused(emx.lib().emx_sdpa_paged_workspace(None, kv(page_size=page_size), batch(max_pages=max_pages), 4, 0, C.byref(C.c_size_t())),
            "null context" if fits else "max_pages")


class Tensor:
    """What the binding looks at of a torch tensor."""

    def __init__(self, dtype, device=0, contiguous=True):
        self.dtype, self.device, self.contiguous = dtype, device, contiguous

    def get_device(self):
        return self.device

    def is_contiguous(self):
        return self.contiguous

    def data_ptr(self):
        return P


def test_tensors_that_the_kernels_cannot_read_are_refused():
    """On the host, on another GPU, strided, or of another type than the operator's."""
    torch = pytest.importorskip("torch")
    bf, i32, cpu = torch.bfloat16, torch.int32, torch.zeros
    emx.PagedKV(Tensor(bf), Tensor(bf), 1, 1, 1, 64)
    emx.PagedBatch(Tensor(i32), Tensor(i32), Tensor(i32), 1, 1, 1)
    for bad, word in ((cpu(64, dtype=bf), "host"), (Tensor(bf, contiguous=False), "strided"), (Tensor(torch.float16), "float16"),
                      (Tensor(bf, device=1), "several GPUs")):
        for pair in ((bad, Tensor(bf)), (Tensor(bf), bad)):
            with pytest.raises(emx.EmxError, match=word) as e:
                emx.PagedKV(*pair, 1, 1, 1, 64)
            assert e.value.code == emx.ERR_INVALID
    for bad, word in ((cpu(2, dtype=i32), "host"), (Tensor(torch.int64), "int64"), (Tensor(i32, contiguous=False), "strided")):
        for at in range(3):
            arrays = [Tensor(i32) for _ in range(3)]
            arrays[at] = bad
            with pytest.raises(emx.EmxError, match=word):
                emx.PagedBatch(*arrays, 1, 1, 1)
    for _ in range(2):
        for bad in (Tensor(torch.float32, device=1), Tensor(torch.float32, contiguous=False), cpu(3), Tensor(torch.int32)):
            with pytest.raises(emx.EmxError, match="float32 tensor on GPU 0 is wanted, not a"):
                emx._ptr(bad, emx._F32, 0)
        assert emx._ptr(Tensor(torch.float32, device=1), emx._F32, 1) == P and emx._ptr(None, emx._F32, 1) is None


# ------------------------------------------------------------------------------------ the deal of tiles to workers
HARNESS = r"""
#include "paged_plan.h"
#include <stdio.h>
using namespace emx;
// The calls that once_a_device makes of `set`, which fails the first `fails` times, for devices[0..n).
extern "C" int once(const int* devices, int n, int fails, int* made) {
  std::atomic<uint64_t> done{0};
  int errors = 0;
  for (int i = 0; i < n; ++i)
    errors += once_a_device(done, devices[i], [&] { ++made[i]; return fails-- > 0 ? 7 : 0; }) != 0;
  return errors;
}
// Walks every worker's share of the line the way the kernel does.  `choice` units are the first workers' shares; seen[] counts the tiles in line order, pieces[] (at a
// segment's first tile) the pieces written of it; returns 0, or where an index left its range.
extern "C" int walk(int own, int n_seqs, int n_rows, int n_kv, int hpg, int shared, int mt, int keys, int setup, long room,
                    const int* indptr, const int* lengths, int64_t* starts, int workers, int choice, int* seen, long n_seen,
                    int* pieces) {
  Line line{own != 0, n_seqs, n_rows, n_kv, hpg, shared, mt, keys, setup, room, indptr, lengths, starts};
  int64_t T = 0, tiles = 0;
  for (int i = 0; i < (own ? n_seqs : 1); ++i) {
    const SeqInfo s = line.seq(i);
    if (own) starts[i] = T;
    const int64_t u = line.units(s);
    T += u;
    if (u) tiles += u / (line.key_tiles(s) + setup) * line.key_tiles(s);
  }
  if (own) starts[n_seqs] = T;
  if (tiles != n_seen) return 1;
  if (T == 0) return 0;
  const int early = choice > 0 ? choice * workers / 40 : 0;
  const Shares sh = deal(T, workers, early, choice);
  if (sh.begin(0) != 0 || sh.begin(workers) < T || sh.begin(sh.early) != sh.cut) return 13;
  if (sh.early && (sh.early != early || sh.early_per > choice || (sh.cut < T && sh.early_per != choice))) return 16;
  if (!sh.early && sh.late_per > (T + workers - 1) / workers) return 17;
  int64_t at = 0;  // tiles seen: workers follow the line
  for (int c = 0; c < workers; ++c) {
    const int64_t x0 = sh.begin(c), x1 = sh.begin(c + 1) < T ? sh.begin(c + 1) : T;
    if (x0 >= T) continue;
    Cursor cur;
    cur.seek(line, x0);
    if (cur.x >= x1) continue;
    bool fresh = true, whole = false;
    int more_pieces = 0;
    for (;;) {
      if (cur.seq < 0 || (own && cur.seq >= n_seqs)) return 2;
      if (!cur.s.ok || cur.s.rows <= 0 || cur.s.row0 < 0 || cur.s.row0 + cur.s.rows > n_rows) return 3;
      if (cur.k < 0 || cur.k >= cur.kt || cur.seg < 0 || cur.seg >= cur.mt * n_kv) return 4;
      if (cur.head() < 0 || cur.head() >= n_kv) return 5;
      const int row = (cur.seg - cur.head() * cur.mt) * mt;
      if (row >= cur.s.rows * hpg) return 6;
      const int64_t seg0 = (own ? starts[cur.seq] : 0) + (int64_t)cur.seg * (cur.kt + setup) + setup;
      if (seg0 + cur.k != cur.x || cur.x < x0 || cur.x >= x1) return 7;
      const int first_pos = (own ? shared : 0) + cur.k * keys;
      if (first_pos >= cur.s.len) return 8;  // every tile has a position
      if (at >= n_seen) return 14;
      seen[at]++;
      if (fresh) { fresh = false; whole = cur.k == 0; }
      const bool last = cur.k + 1 == cur.kt, more = cur.x + 1 + (last ? setup : 0) < x1;
      if (last || !more) {
        // what the join will look for: the worker of the segment's first tile has the first piece
        const int c0 = sh.of(seg0), c1 = sh.of(seg0 + cur.kt - 1);
        if (whole ? c != c0 : !(c > c0 && c <= c1)) return 9;
        if (!whole && ++more_pieces > 1) return 10;  // one slot a worker
        pieces[at - cur.k] += 1;
        if (last && pieces[at - cur.k] != c1 - c0 + 1) return 12;
        fresh = true;
      }
      ++at;
      if (!more) break;
      cur.next(line);
    }
  }
  return at == n_seen ? 0 : 15;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    src, lib = d / "walk.cc", d / "walk.so"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "engine-mlx_b200", "csrc"),
                    str(src), "-o", str(lib)], check=True)
    return C.CDLL(str(lib))


@pytest.mark.parametrize("devices,fails,made", [([0, 0, 0], 0, [1, 0, 0]), ([0, 1, 0, 1, 7], 0, [1, 1, 0, 0, 1]),
                                                ([3, 3, 3], 1, [1, 1, 0]), ([63, 64, 64, 63], 0, [1, 1, 1, 0])])
def test_attributes_are_set_on_every_device(plan, devices, fails, made):
    got = (C.c_int * len(devices))()
    assert plan.once((C.c_int * len(devices))(*devices), len(devices), fails, got) == fails
    assert list(got) == made


@pytest.fixture(scope="module")
def walk(plan):
    f = plan.walk
    f.restype = C.c_int
    f.argtypes = [C.c_int] * 9 + [C.c_long] + [C.c_void_p] * 3 + [C.c_int, C.c_int, C.c_void_p, C.c_long, C.c_void_p]

    def run(own, indptr, lengths, n_rows, n_kv, hpg, shared, mt, keys, room, workers, choice=0, setup=0):
        indptr, lengths = np.asarray(indptr, np.int32), np.asarray(lengths, np.int32)
        n = len(lengths)
        total = 0
        if own:
            for i in range(n):
                a, b = int(indptr[i]), int(indptr[i + 1])
                if a < 0 or b < a or b > n_rows or a == b or not shared + b - a <= lengths[i] <= room:
                    continue
                total += n_kv * -(-(b - a) * hpg // mt) * -(-(int(lengths[i]) - shared) // keys)
        elif shared:
            total = n_kv * -(-n_rows * hpg // mt) * -(-shared // keys)
        seen, pieces = np.zeros(total + 1, np.int32), np.zeros(total + 1, np.int32)
        starts = np.zeros(n + 1, np.int64)
        rc = f(own, n, n_rows, n_kv, hpg, shared, mt, keys, setup, room, indptr.ctypes.data, lengths.ctypes.data, starts.ctypes.data,
               workers, choice, seen.ctypes.data, total, pieces.ctypes.data)
        assert rc == 0, rc
        assert (seen[:total] == 1).all()
        return total

    return run


@pytest.mark.parametrize("seed", range(60))
def test_every_tile_has_one_worker_and_every_piece_is_joined(walk, seed):
    r = np.random.default_rng(seed)
    n = int(r.choice([1, 2, 5, 33, 200]))
    rows = r.choice([0, 1, 1, 1, 2, 5, 40], n)
    shared = int(r.choice([0, 16, 160, 4096]))
    lens = shared + rows + np.where(r.random(n) < 0.2, 0, r.integers(0, 900, n))
    indptr = np.concatenate([[0], np.cumsum(rows)])
    hpg, n_kv = int(r.choice([1, 2, 3, 8])), int(r.choice([1, 2, 8]))
    for own in (0, 1):
        if own or (shared and indptr[-1]):
            walk(own, indptr, lens, int(indptr[-1]) + 3, n_kv, hpg, shared, int(r.choice([16, 32, 128])),
                 int(r.choice([16, 64, 128])), 8192, int(r.choice([1, 7, 148, 1184])), int(r.choice([0, 0, 1, 4, 9, 39])), int(r.choice([0, 1, 3])))


@pytest.mark.parametrize("seed", range(40))
def test_batches_out_of_order_stay_in_range(walk, seed):
    """Rows and lengths that cannot be: such sequences have no tiles, and no index leaves its range."""
    r = np.random.default_rng(1000 + seed)
    n = int(r.integers(1, 12))
    indptr = r.integers(-3, 20, n + 1)
    lens = r.choice([-5, 0, 1, 20, 64, 100, 513, 2**31 - 1], n)
    walk(1, indptr, lens, 15, 2, int(r.choice([1, 4])), int(r.choice([0, 64])), 16, 16, 512, int(r.choice([1, 148])), int(r.choice([0, 3])), int(r.choice([0, 1])))
    walk(1, [0] * (n + 1), lens, 15, 2, 1, 0, 16, 16, 512, 148)
