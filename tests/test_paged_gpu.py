"""emx_paged_append and emx_sdpa_paged against their definitions in 64 bits, on an sm_100 GPU.  Rows of the cache that
belong to no position, and pages that belong to nobody, hold NaN throughout."""
import ctypes as C

import numpy as np
import pytest

import emx
from paged_case import NAN, Case

pytestmark = pytest.mark.gpu

H = 2.0 ** -8  # half a step of bf16, relative


@pytest.fixture(scope="module")
def ctx():
    c = emx.Ctx(0)
    yield c
    c.close()


def stream_of(ctx):
    p = C.c_void_p()
    assert emx.lib().emx_ctx_stream(ctx.h, C.byref(p)) == 0
    return p.value


def attend(ctx, c, fill=NAN, ws=None):
    out = ctx.put(np.full((c.n_rows + 1, c.n_q, c.hd), fill, np.uint16))
    ctx.sdpa_paged(c.dq, c.kv, c.batch, c.n_q, c.scale, c.shared, c.d_shared, out=out, workspace=ws)
    c.status = ctx.device_status()  # read and cleared: a copy to the host would raise it
    return out.read(np.uint16, (c.n_rows + 1, c.n_q, c.hd))


def check_attend(c, got, fill=NAN):
    """Bound: the output's rounding, H |o|; the weights' rounding to bf16, which moves o by at most H sum w |v - o| <=
    H (mean |v| + |o|); and the scores' fp32 products and exponentials, whose errors (128 terms of 2^-24, a 2-ulp
    exponential) stay below 2^-12 of a weight each: 2^-11 (mean |v| + |o|)."""
    want, size = c.attend()
    g = emx.f32(got[:c.n]).astype(np.float64)
    tol = H * np.abs(want) + (H + 2.0 ** -11) * (size + np.abs(want))
    bad = ~(np.abs(g - want) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.nanmax(np.abs(g - want) / tol)), np.argwhere(bad)[:4].tolist())
    assert (got[c.n:] == fill).all()  # rows behind the last sequence


HEADS = [(4, 2), (8, 8), (16, 2), (5, 1), (32, 1)]


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("n_q,n_kv", HEADS)
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 131])
def test_one_sequence_one_row(ctx, length, n_q, n_kv, hd):
    c = Case(length, [1], [length], n_q, n_kv, hd).device(ctx)
    check_attend(c, attend(ctx, c))
    assert c.status == 0


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("page", [1, 7, 16, 24, 64, 100])
@pytest.mark.parametrize("pages_shared", [0, 1, 3])
def test_pages_of_any_size(ctx, page, pages_shared, hd):
    shared = page * pages_shared
    rows = [1, 3, 0, 1, 2]
    c = Case(page, rows, [shared + t for t in (1, 3, 0, 200, 77)], 4, 2, hd, page, shared, pad=2).device(ctx)
    check_attend(c, attend(ctx, c))
    assert c.status == 0


@pytest.mark.parametrize("n_q,n_kv", HEADS)
@pytest.mark.parametrize("rows", [1, 2, 5, 16, 33, 130])
def test_several_rows_see_no_later_ones(ctx, rows, n_q, n_kv):
    c = Case(rows, [rows, 0, rows, 1], [rows, 0, rows + 61, 150], n_q, n_kv, pad=1).device(ctx)
    check_attend(c, attend(ctx, c))


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("n_q,n_kv", HEADS)
@pytest.mark.parametrize("seqs,shared", [(1, 128), (3, 48), (9, 512), (40, 272), (140, 1040), (300, 144)])
def test_a_shared_prefix(ctx, seqs, shared, n_q, n_kv, hd):
    r = np.random.default_rng(seqs)
    rows = r.choice([0, 1, 1, 1, 3], seqs)
    rows[0] = 1
    c = Case(seqs, rows, shared + rows + r.integers(0, 60, seqs), n_q, n_kv, hd, 16, shared, pad=3).device(ctx)
    check_attend(c, attend(ctx, c))
    assert c.status == 0


def test_long_and_short_together(ctx):
    lens = [9000, 1, 17, 5000, 64, 1, 3, 700]
    c = Case(5, [1, 1, 2, 1, 8, 1, 3, 1], lens, 8, 2, page=32).device(ctx)
    check_attend(c, attend(ctx, c))


def test_a_long_prefix_and_far_pages(ctx):
    c = Case(6, [1] * 20, [6000 + 64 + i for i in range(20)], 8, 2, page=48, shared=6000, spare=50).device(ctx)
    check_attend(c, attend(ctx, c))


def test_all_slots_idle(ctx):
    c = Case(7, [0, 0, 0], [0, 5, 0], pad=4).device(ctx)
    got = attend(ctx, c, fill=7)
    assert (got == 7).all() and c.status == 0


def test_what_a_row_does_not_see_may_be_anything(ctx):
    """NaN and infinities in the K and V of later rows leave earlier rows as they are, and reach the rows that see
    them; a row of q that is NaN spoils no other."""
    c = Case(8, [6, 2, 1], [70, 40, 30], 4, 2)
    at = c.table[0, 67 // 16], 67 % 16
    for x, bad in ((c.v, 0x7F80), (c.k, 0x7FC0)):
        d = Case(8, [6, 2, 1], [70, 40, 30], 4, 2)
        (d.v if x is c.v else d.k)[at[0], :, at[1], 3] = bad  # seen by rows 3, 4, 5 (positions 67, 68, 69)
        d.device(ctx)
        got = attend(ctx, d)
        g = emx.f32(got[:d.n])
        assert not np.isfinite(g[3:6, :, 3]).any()
        want, size = c.attend()
        ok = [0, 1, 2, 6, 7, 8]
        assert (np.abs(g[ok] - want[ok]) <= (2 * H + 2.0 ** -11) * (size[ok] + np.abs(want[ok]))).all()
        if x is c.v:  # only that dimension
            rest = np.delete(np.arange(128), 3)
            assert np.isfinite(g[3:6][..., rest]).all()
    d = Case(8, [6, 2, 1], [70, 40, 30], 4, 2)
    d.q[1, 2] = NAN
    g = emx.f32(attend(ctx, d.device(ctx))[:d.n])
    assert np.isnan(g[1, 2]).all() and np.isnan(g).sum() == 128


def test_scores_of_any_size(ctx):
    """Huge scores (weights of 0 and 1), and a maximum that keeps moving."""
    c = Case(9, [2, 1], [300, 160], 4, 2, shared=0)
    k = emx.f32(c.k)
    c.k = emx.bf16(k * 60)
    c.q = emx.bf16(emx.f32(c.q) * 30)
    c.device(ctx)
    want, size = c.attend()
    g = emx.f32(attend(ctx, c)[:c.n]).astype(np.float64)
    # scores of ~2e4 carry fp32 errors of 128 * 2^-24 * sum |q k| scale ~ 0.25 in the exponent at the worst; the two
    # largest scores of a row are farther apart than 20 here for nearly all rows, so most rows equal one row of V
    s = np.abs(g - want)
    assert np.isfinite(g).all() and np.median(s) <= 2 * H * np.median(size) and (s <= 2 * size.max()).all()


def test_bad_pages_are_left_out_and_reported(ctx):
    c = Case(10, [1, 2], [100, 50], 4, 2)
    c.table[0, 2] = c.n_pages  # positions 32..47
    c.table[1, 1] = -1  # positions 16..31
    c.device(ctx)
    g = emx.f32(attend(ctx, c)[:c.n]).astype(np.float64)
    assert c.status == 5
    for i, hole in ((0, range(32, 48)), (1, range(16, 32))):
        keep = np.array([p for p in range(c.lens[i]) if p not in hole])
        k, v = (emx.f32(x[c.table[i, keep // 16], :, keep % 16]).astype(np.float64) for x in (c.k, c.v))
        for j, p in enumerate(c.positions(i)):
            row, m = c.indptr[i] + j, keep <= p
            q = emx.f32(c.q[row]).astype(np.float64).reshape(2, 2, 128)
            w = np.exp(np.einsum("hgd,shd->hgs", q, k[m]) * c.scale)
            w /= w.sum(-1, keepdims=True)
            want = np.einsum("hgs,shd->hgd", w, v[m]).reshape(4, 128)
            size = np.einsum("hgs,shd->hgd", w, np.abs(v[m])).reshape(4, 128)
            assert (np.abs(g[row] - want) <= (2 * H + 2.0 ** -11) * (size + np.abs(want))).all()
    # no page at all: zeros
    c = Case(11, [1, 1], [30, 30], 4, 2)
    c.table[1] = 1 << 30
    g = attend(ctx, c.device(ctx))
    assert (g[1] == 0).all() and (g[0] != 0).any() and c.status == 5


@pytest.mark.parametrize("shared", [0, 32])
def test_sequences_out_of_order_give_zeros_and_a_status(ctx, shared):
    c = Case(12, [1, 3, 1, 2], [shared + 40, shared + 60, shared + 50, shared + 8], 4, 2, shared=shared).device(ctx)
    c.d_lens.write(np.array([shared + 40, shared + 2, shared + 50, c.max_pages * 16 + 1], np.int32))
    got = attend(ctx, c)
    assert c.status in (4, 6)
    assert (got[1:4] == 0).all() and (got[5:7] == 0).all()
    want, size = c.attend()
    g = emx.f32(got[:c.n])
    for r in (0, 4):
        assert (np.abs(g[r] - want[r]) <= (2 * H + 2.0 ** -11) * (size[r] + np.abs(want[r]))).all()
    # rows that cannot be
    for bad in ([0, 9, 5, 6, 7], [-2, 1, 2, 3, 4], [0, 1, 4, 5, 100]):
        c.d_indptr.write(np.array(bad, np.int32))
        attend(ctx, c)
        assert c.status in (4, 6)
    c.d_indptr.write(c.indptr)
    c.d_lens.write(np.array(c.lens, np.int32))
    check_attend(c, attend(ctx, c))
    assert c.status == 0


@pytest.mark.parametrize("seqs,n_q,n_kv,shared", [(32, 8, 2, 256), (300, 8, 8, 144), (300, 8, 8, 128), (70, 64, 8, 2080),
                                                  (40, 32, 4, 8192)])
def test_the_same_call_gives_the_same_bits(ctx, seqs, n_q, n_kv, shared):
    r = np.random.default_rng(seqs)
    rows = r.choice([0, 1, 1, 2], seqs)
    c = Case(13, rows, shared + rows + r.integers(0, 300, seqs), n_q, n_kv, shared=shared).device(ctx)
    first = attend(ctx, c)
    for _ in range(20):
        assert (attend(ctx, c) == first).all()


@pytest.mark.parametrize("scale", [0.0, -0.1])
@pytest.mark.parametrize("seqs", [3, 40])
def test_scales_that_are_not_positive(ctx, scale, seqs):
    c = Case(26, [1, 2] + [1] * seqs, [200, 90] + [130] * seqs, 8, 2, shared=64)
    c.scale = scale
    check_attend(c, attend(ctx, c.device(ctx)))


def test_one_sequence_equals_the_static_cache(ctx):
    """The same rows through emx_sdpa_decode."""
    c = Case(14, [1], [333], 16, 8).device(ctx)
    k, v = (np.ascontiguousarray(x[c.table[0, np.arange(333) // 16], :, np.arange(333) % 16].transpose(1, 0, 2)) for x in (c.k, c.v))
    ref = emx.f32(ctx.sdpa_decode(c.dq, ctx.put(k), ctx.put(v), 16, 8, 333, 128, 333, c.scale).read(np.uint16, (16, 128)))
    g = emx.f32(attend(ctx, c)[0])
    _, size = c.attend()
    assert (np.abs(g - ref) <= 4 * H * (size[0] + np.abs(ref))).all()


def test_workspace_is_checked_and_not_overrun(ctx):
    c = Case(15, [1, 4, 1], [300, 200, 40], 8, 2, shared=32).device(ctx)
    need = ctx.sdpa_paged_workspace(c.kv, c.batch, 8, 32)
    ws = ctx.put(np.full(need + 4096, 0xA5, np.uint8))
    whole = ws.nbytes
    ws.nbytes = need - 1
    with pytest.raises(emx.EmxError, match="workspace"):
        attend(ctx, c, ws=ws)
    ws.nbytes = need
    check_attend(c, attend(ctx, c, ws=ws))
    ws.nbytes = whole
    assert (ws.read(np.uint8, whole)[need:] == 0xA5).all()


def test_captured_and_replayed_as_the_batch_changes(ctx):
    """One graph of append and attention, replayed with other lengths, rows and tables; a second one with a workspace of
    its own runs at the same time on another stream."""
    torch = pytest.importorskip("torch")
    other = emx.Ctx(0)
    a = Case(16, [1, 1, 2, 1], [100, 37, 90, 64], 8, 2, shared=32).device(ctx)
    e = Case(18, [1] * 6, [900 + i for i in range(6)], 8, 2, shared=64).device(other)
    graphs = []
    for cx, c in ((ctx, a), (other, e)):
        out = cx.put(np.zeros((c.n_rows, 8, 128), np.uint16))
        ws = cx.alloc(cx.sdpa_paged_workspace(c.kv, c.batch, 8, c.shared))
        cx.sdpa_paged(c.dq, c.kv, c.batch, 8, c.scale, c.shared, c.d_shared, out=out, workspace=ws)
        cx.synchronize()
        st, g = torch.cuda.ExternalStream(stream_of(cx)), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st, capture_error_mode="thread_local"):
            cx.sdpa_paged(c.dq, c.kv, c.batch, 8, c.scale, c.shared, c.d_shared, out=out, workspace=ws)
        graphs.append((g, st, out))

    def replay():
        for _ in range(5):
            for g, st, _ in graphs:
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()

    replay()
    check_attend(a, graphs[0][2].read(np.uint16, (a.n_rows, 8, 128)))
    check_attend(e, graphs[1][2].read(np.uint16, (6, 8, 128)))
    # lengths shorter by some positions, rows moved between sequences
    a.lens, a.rows = [70, 36, 33, 64], [2, 1, 1, 1]
    a.indptr = np.concatenate([[0], np.cumsum(a.rows)]).astype(np.int32)
    a.d_lens.write(np.array(a.lens, np.int32))
    a.d_indptr.write(a.indptr)
    ctx.synchronize()
    replay()
    check_attend(a, graphs[0][2].read(np.uint16, (a.n_rows, 8, 128)))
    del graphs
    other.close()


# ------------------------------------------------------------------------------------------------------------ append
def check_append(ctx, c, norm=True, theta=1e6, eps=1e-6):
    r = c.rng
    wq, wk = (emx.bf16(1 + 0.2 * r.normal(size=c.hd)) if norm else None for _ in range(2))
    out = ctx.put(np.full((c.n_rows + 1, c.n_q, c.hd), NAN, np.uint16))
    ctx.paged_append(c.dqkv, c.kv, c.batch, c.n_q, None if wq is None else ctx.put(wq), None if wk is None else ctx.put(wk),
                     eps, theta, out=out)
    got = out.read(np.uint16, (c.n_rows + 1, c.n_q, c.hd))
    k, v = (x.read(np.uint16, c.k.shape) for x in (c.dk, c.dv))
    q_, k_, v_ = c.append(wq, wk, eps, theta)
    half = c.hd // 2

    def near(g, want):
        # one rounding to bf16, and fp32 steps (a mean of squares, a root, two products) of the pair that is rotated:
        # 16 of them at 2^-24 of its length
        pair = np.sqrt(want[..., :half] ** 2 + want[..., half:] ** 2)
        tol = H * np.abs(want) + 2.0 ** -20 * np.concatenate([pair, pair], -1)
        err = np.abs(emx.f32(g).astype(np.float64) - want)
        assert (err <= tol).all(), float((err / np.maximum(tol, 1e-30)).max())

    near(got[:c.n], q_)
    assert (got[c.n:] == NAN).all()
    wk_, wv_ = c.k.copy(), c.v.copy()
    for i in range(c.n_seqs):
        p = c.positions(i)
        at = c.table[i, p // c.page], slice(None), p % c.page
        rows = slice(c.indptr[i], c.indptr[i + 1])
        if c.rows[i]:
            near(k[at], k_[rows])
            assert (emx.f32(v[at]) == v_[rows]).all()
            wk_[at], wv_[at] = k[at], v[at]
    assert (k == wk_).all() and (v == wv_).all()  # and nothing else was written
    return got


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("n_q,n_kv", HEADS + [(64, 8)])
@pytest.mark.parametrize("rows", [[1], [1] * 70, [3, 0, 17, 1, 40], [300]])
def test_append(ctx, rows, n_q, n_kv, hd):
    r = np.random.default_rng(len(rows))
    c = Case(len(rows), rows, [k + int(r.integers(0, 200)) for k in rows], n_q, n_kv, hd, pad=3).device(ctx)
    check_append(ctx, c)
    assert ctx.device_status() == 0


@pytest.mark.parametrize("norm,theta", [(False, 1e6), (True, 0.0), (False, 0.0), (True, 1e4)])
def test_append_without_norm_or_rotation(ctx, norm, theta):
    check_append(ctx, Case(21, [2, 1, 5], [20, 1, 300], 8, 2, page=24).device(ctx), norm, theta)


def test_append_far_positions(ctx):
    """Angles of a million radians: the pages of the last positions alone are there."""
    c = Case(22, [1, 2], [5, 9], 4, 2)
    far = 1_000_003
    c.max_pages = far // 16 + 1
    c.lens = [far, far - 700]
    table = np.full((2, c.max_pages), -1, np.int32)
    for i, (n, t) in enumerate(zip(c.rows, c.lens)):
        for p in range(t - n, t):
            table[i, p // 16] = i
    c.table = table
    c.device(ctx)
    check_append(ctx, c)
    assert ctx.device_status() == 0


def test_append_many_rows(ctx):
    """More rows than the grid has warps."""
    c = Case(23, [9000, 1, 2500], [9000, 50, 2600], 3, 1, 64, 32).device(ctx)
    check_append(ctx, c)


def test_append_skips_what_is_out_of_order(ctx):
    c = Case(24, [1, 2, 1, 1], [10, 20, 30, 31], 4, 2)
    c.table[2, 1] = c.n_pages + 3
    c.device(ctx)
    c.d_lens.write(np.array([10, 1, 30, c.max_pages * 16 + 1], np.int32))
    out = ctx.put(np.full((c.n_rows, 4, 128), NAN, np.uint16))
    ctx.paged_append(c.dqkv, c.kv, c.batch, 4, out=out)
    assert ctx.device_status() in (4, 5, 6)
    got = out.read(np.uint16, (c.n_rows, 4, 128))
    q_, k_, v_ = c.append()
    for r in (0, 3):  # rows of sequences 0 and 2: q is there
        assert np.allclose(emx.f32(got[r]), q_[r], rtol=H, atol=1e-4)
    assert (got[1:3] == NAN).all() and (got[4] == NAN).all()
    k, v = (x.read(np.uint16, c.k.shape) for x in (c.dk, c.dv))
    wv = c.v.copy()
    p = c.positions(0)
    wv[c.table[0, p // 16], :, p % 16] = v[c.table[0, p // 16], :, p % 16]
    assert (v == wv).all()  # sequence 0's row alone was written
    assert np.allclose(emx.f32(k[c.table[0, p // 16], :, p % 16]), k_[:1], rtol=H, atol=1e-4)


def test_append_norm_of_large_and_zero_heads(ctx):
    c = Case(25, [2, 1], [40, 9], 4, 2)
    x = c.qkv.reshape(c.n_rows, 8, 128)
    x[0, 0] = 0  # a head of zeros: eps keeps it
    x[1, 1] = emx.bf16(np.full(128, 1e18, np.float32))  # squares near fp32's end
    x[1, 4] = emx.bf16(np.full(128, 1e-18, np.float32))
    check_append(ctx, c.device(ctx))


# ------------------------------------------------------------------------------------------- sizes and uses at the ends
def want_without(c, hole):
    """The definition where the positions in hole[i] of sequence i are in no page of the cache."""
    want, size = np.zeros((c.n, c.n_q, c.hd)), np.zeros((c.n, c.n_q, c.hd))
    each = c.n_q // c.n_kv
    for i in range(c.n_seqs):
        keep = np.array([p for p in range(c.lens[i]) if p not in hole[i]], int)
        k, v = (emx.f32(x[c.table[i, keep // c.page], :, keep % c.page]).astype(np.float64) for x in (c.k, c.v))
        for j, p in enumerate(c.positions(i)):
            row, m = c.indptr[i] + j, keep <= p
            if not m.any():
                continue
            q = emx.f32(c.q[row]).astype(np.float64).reshape(c.n_kv, each, c.hd)
            s = np.einsum("hgd,shd->hgs", q, k[m]) * c.scale
            w = np.exp(s - s.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            want[row] = np.einsum("hgs,shd->hgd", w, v[m]).reshape(c.n_q, c.hd)
            size[row] = np.einsum("hgs,shd->hgd", w, np.abs(v[m])).reshape(c.n_q, c.hd)
    return want, size


def near(got, want, size):
    return np.abs(emx.f32(got).astype(np.float64) - want) <= H * np.abs(want) + (H + 2.0 ** -11) * (size + np.abs(want))


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("page", [1, 5, 8, 20, 24, 40, 128, 256])
@pytest.mark.parametrize("seqs", [20, 45])
def test_many_rows_over_a_prefix_of_any_pages(ctx, page, hd, seqs):
    """80 and 180 rows a KV head (one and two row tiles), with pages that the tiles' copies take and others."""
    r = np.random.default_rng(page)
    shared = page * max(1, round(400 / page))
    rows = np.ones(seqs, int)
    c = Case(page, rows, shared + rows + r.integers(0, 50, seqs), 8, 2, hd, page, shared, pad=1).device(ctx)
    check_attend(c, attend(ctx, c))
    assert c.status == 0


@pytest.mark.parametrize("shared", [128, 320, 1040])
def test_more_segments_than_workers(ctx, shared):
    """64 KV heads of three row tiles: a worker goes from tiles of two rows' groups to those of one and back."""
    r = np.random.default_rng(3)
    c = Case(30, [1] * 300, shared + 1 + r.integers(0, 20, 300), 128, 64, 64, shared=shared).device(ctx)
    check_attend(c, attend(ctx, c))


@pytest.mark.parametrize("shared", [0, 48])
def test_as_many_sequences_as_there_may_be(ctx, shared):
    r = np.random.default_rng(4)
    rows = r.choice([0, 1, 1, 2, 20], 1024, p=[0.2, 0.4, 0.2, 0.19, 0.01])
    c = Case(31, rows, shared + rows + r.integers(0, 90, 1024), 4, 2, shared=shared, pad=5).device(ctx)
    check_attend(c, attend(ctx, c))
    assert c.status == 0


@pytest.mark.parametrize("shared", [0, 32])
@pytest.mark.parametrize("n_q,n_kv", [(1024, 1), (1024, 1024), (1023, 11)])
def test_as_many_heads_as_there_may_be(ctx, n_q, n_kv, shared):
    c = Case(32, [2, 0, 1], [shared + 40, 0, shared + 3], n_q, n_kv, 64, shared=shared, pad=1).device(ctx)
    check_attend(c, attend(ctx, c))
    check_append(ctx, c)


@pytest.mark.parametrize("seqs", [1, 12, 60])
def test_a_page_may_stand_for_several(ctx, seqs):
    """The same page twice in a table, and twice in the prefix."""
    c = Case(33, [1] * seqs, [200 + i for i in range(seqs)], 8, 2, shared=64)
    c.shared_pages[2] = c.shared_pages[0]
    c.table[:, 2] = c.shared_pages[0]
    c.table[0, 6] = c.table[0, 5]
    c.device(ctx)
    check_attend(c, attend(ctx, c))


@pytest.mark.parametrize("shared", [0, 32])
def test_rows_before_the_first_sequence(ctx, shared):
    """indptr may begin behind row 0."""
    c = Case(34, [3, 2, 1], [shared + 40, shared + 21, shared + 9], 4, 2, shared=shared).device(ctx)
    every = attend(ctx, c)
    b = emx.PagedBatch(ctx.put(c.indptr[1:].copy()), ctx.put(np.array(c.lens[1:], np.int32)), ctx.put(c.table[1:].copy()), 2,
                       c.n_rows, c.max_pages)
    out = ctx.put(np.full((c.n_rows, 4, 128), 9, np.uint16))
    ctx.sdpa_paged(c.dq, c.kv, b, 4, c.scale, shared, c.d_shared, out=out)
    got = out.read(np.uint16, (c.n_rows, 4, 128))
    assert ctx.device_status() == 0 and (got[:3] == 9).all()
    assert near(got[3:], *(x[3:] for x in c.attend())).all() and near(every[:c.n], *c.attend()).all()
    q = ctx.put(np.full((c.n_rows, 4, 128), 9, np.uint16))
    ctx.paged_append(c.dqkv, c.kv, b, 4, out=q)
    got = q.read(np.uint16, (c.n_rows, 4, 128))
    assert ctx.device_status() == 0 and (got[:3] == 9).all()
    assert np.allclose(emx.f32(got[3:]), c.append()[0][3:], rtol=H, atol=1e-4)


@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("seqs", [3, 20, 45])
def test_bad_pages_of_the_prefix(ctx, seqs, page):
    """A page of the prefix outside the cache is left out; a prefix, and then a whole batch, without a page gives zeros."""
    c = Case(35, [1] * seqs, [20 * page + 1 + i for i in range(seqs)], 8, 2, page=page, shared=20 * page).device(ctx)
    pages = c.shared_pages.copy()
    pages[7], pages[19] = c.n_pages, -1
    c.d_shared.write(pages)
    hole = set(range(7 * page, 8 * page)) | set(range(19 * page, 20 * page))
    got = attend(ctx, c)
    assert c.status == 5 and near(got[:c.n], *want_without(c, [hole] * seqs)).all()
    c.d_shared.write(np.full(20, 1 << 30, np.int32))
    got = attend(ctx, c)
    assert c.status == 5 and near(got[:c.n], *want_without(c, [set(range(20 * page))] * seqs)).all()
    c.kv.c.n_pages = 0
    got = attend(ctx, c)
    assert c.status == 5 and (got[:c.n] == 0).all()


def test_output_over_q(ctx):
    for seqs, shared in ((1, 0), (40, 0), (5, 64), (40, 64)):
        c = Case(36, [1] * seqs, [shared + 30 + 9 * i for i in range(seqs)], 8, 2, shared=shared).device(ctx)
        want = attend(ctx, c)[:c.n]
        ctx.sdpa_paged(c.dq, c.kv, c.batch, 8, c.scale, shared, c.d_shared, out=c.dq)
        assert (c.dq.read(np.uint16, want.shape) == want).all()


def test_calls_of_all_kinds_one_after_another(ctx):
    """Nothing waits between them and one workspace serves them all: each call's kernels begin while the last one's end."""
    cases = [Case(37, [1] * 45, [400 + i for i in range(45)], 8, 2, shared=320), Case(38, [1], [3000], 8, 2),
             Case(39, [40, 1, 70], [60, 700, 90], 8, 2), Case(40, [1] * 3, [600, 300, 290], 8, 2, shared=256),
             Case(41, [1] * 20, [130] * 20, 8, 2, page=20, shared=120)]
    for c in cases:
        c.device(ctx)
    ws = ctx.alloc(max(ctx.sdpa_paged_workspace(c.kv, c.batch, 8, c.shared) for c in cases))
    want = [attend(ctx, c, ws=ws) for c in cases]
    for c, w in zip(cases, want):
        check_attend(c, w)
    outs = [[ctx.put(np.full(w.shape, NAN, np.uint16)) for w in want] for _ in range(6)]
    for turn, out in enumerate(outs):
        for i in np.random.default_rng(turn).permutation(len(cases)):
            c = cases[i]
            ctx.sdpa_paged(c.dq, c.kv, c.batch, 8, c.scale, c.shared, c.d_shared, out=out[i], workspace=ws)
    for out in outs:
        for o, w in zip(out, want):
            assert (o.read(np.uint16, w.shape) == w).all()


def test_two_contexts_in_two_threads(ctx):
    import threading
    other = emx.Ctx(0)
    made, wrong = [], []
    for cx, seed in ((ctx, 42), (other, 43)):
        c = Case(seed, [1] * 40, [300 + 7 * i for i in range(40)], 16, 4, shared=160).device(cx)
        made.append((cx, c, attend(cx, c)))

    def work(cx, c, want):
        for _ in range(30):
            if not (attend(cx, c) == want).all():
                wrong.append(c)

    threads = [threading.Thread(target=work, args=m) for m in made]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    other.close()


def test_offsets_past_32_bits(ctx):
    """A cache of more than 2^32 elements, of which only some pages at both ends and in between hold anything."""
    c = Case(44, [1, 3] + [1] * 20, [300, 90] + [70 + i for i in range(20)], 8, 2, page=128, shared=0)
    s = Case(45, [1] * 24, [400 + i for i in range(24)], 8, 2, page=128, shared=256)
    pages = (2 ** 32) // (2 * 128 * 128) + 64  # of 2 x 128 x 128 elements
    k, v = (ctx.alloc(pages * 2 * 128 * 128 * 2) for _ in range(2))
    for x in (c, s):
        x.device(ctx)
        assert x.n_pages <= 64
        far = np.concatenate([np.arange(pages - 40, pages), pages // 2 + np.arange(24)])[:x.n_pages]  # page j of the case
        for j, to in enumerate(far):
            k.write(x.k[j], int(to) * 65536)
            v.write(x.v[j], int(to) * 65536)
        move = lambda t: np.where((t >= 0) & (t < x.n_pages), far[np.clip(t, 0, x.n_pages - 1)], -7).astype(np.int32)  # noqa: E731
        x.kv = emx.PagedKV(k, v, pages, 128, 2, 128)
        x.batch = emx.PagedBatch(x.d_indptr, x.d_lens, ctx.put(move(x.table)), x.n_seqs, x.n_rows, x.max_pages)
        if x.shared:
            x.d_shared = ctx.put(move(x.shared_pages))
        check_attend(x, attend(ctx, x))
        assert x.status == 0
        # appended rows arrive there too
        q = ctx.paged_append(x.dqkv, x.kv, x.batch, 8)
        _, k_, v_ = x.append()
        i, p = 1, x.positions(1)
        at = far[x.table[1, p // 128]]
        for row, pg, off in zip(range(x.indptr[1], x.indptr[2]), at, p % 128):
            import ctypes
            page = np.empty((2, 128, 128), np.uint16)
            for buf, w in ((k, k_), (v, v_)):
                assert emx.lib().emx_memcpy_d2h(ctx.h, page.ctypes.data_as(ctypes.c_void_p), buf.ptr + int(pg) * 65536, page.nbytes) == 0
                assert np.allclose(emx.f32(page[:, off]), w[row], rtol=H, atol=1e-4)
        q.free()
    k.free()
    v.free()


def test_a_graph_keeps_the_default_workspace(ctx):
    """A call without a workspace is captured; a larger one then makes the context's grow; the graph is replayed."""
    torch = pytest.importorskip("torch")
    own = emx.Ctx(0)
    a = Case(46, [1] * 3, [300, 200, 100], 8, 2, shared=64).device(own)
    b = Case(47, [1] * 200, [100] * 200, 32, 2, shared=64).device(own)
    want = attend(own, a)
    out = own.put(np.zeros(want.shape, np.uint16))
    st, g = torch.cuda.ExternalStream(stream_of(own)), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st, capture_error_mode="thread_local"):
        own.sdpa_paged(a.dq, a.kv, a.batch, 8, a.scale, 64, a.d_shared, out=out)
    first = attend(own, b)
    for _ in range(3):
        with torch.cuda.stream(st):
            g.replay()
        assert (attend(own, b) == first).all()
    own.synchronize()
    assert (out.read(np.uint16, want.shape)[:a.n] == want[:a.n]).all()
    del g
    own.close()


FIRST_IN_A_GRAPH = """
import sys
sys.path[:0] = sys.argv[1:]
import ctypes as C, numpy as np, torch, emx
from paged_case import Case, verify
from test_verify_gpu import inputs
ctx = emx.Ctx(0)
c = Case(50, [2] * 30, [300 + i for i in range(30)], 8, 2, shared=64).device(ctx)
t, d, x, u = inputs(51, 4, 3, 1000)
buf = [ctx.put(y) for y in (t, d, x, u)]
q = ctx.put(np.zeros((c.n, 8, 128), np.uint16))
o = ctx.put(np.zeros((c.n, 8, 128), np.uint16))
ws = ctx.alloc(ctx.sdpa_paged_workspace(c.kv, c.batch, 8, 64))
out, acc = ctx.put(np.zeros((4, 4), np.int32)), ctx.put(np.zeros(4, np.int32))
ctx.synchronize()
def step():
    ctx.paged_append(c.dqkv, c.kv, c.batch, 8, out=q)
    ctx.sdpa_paged(q, c.kv, c.batch, 8, c.scale, 64, c.d_shared, out=o, workspace=ws)
    ctx.verify_draft(*buf, 4, 3, 1000, out=out, accepted=acc)
p = C.c_void_p()
assert emx.lib().emx_ctx_stream(ctx.h, C.byref(p)) == 0
st, g = torch.cuda.ExternalStream(p.value), torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=st, capture_error_mode="thread_local"):
    step()
read = lambda: (q.read(np.uint16, c.n * 1024), o.read(np.uint16, c.n * 1024), out.read(np.int32, (4, 4)), acc.read(np.int32, 4))
for turn in range(3):
    if turn:
        r = np.random.default_rng(turn)
        c.lens = [int(k) for k in r.integers(70, 300, 30)]
        x, u = r.integers(0, 1000, (4, 3)).astype(np.int32), r.random((4, 4)).astype(np.float32)
        c.d_lens.write(np.array(c.lens, np.int32)), buf[2].write(x), buf[3].write(u)
        c.dqkv.write(c.qkv[::-1].copy() if turn == 2 else c.qkv)
        ctx.synchronize()
    with torch.cuda.stream(st):
        g.replay()
    got = read()
    assert ctx.device_status() == 0
    step()
    assert all((a == b).all() for a, b in zip(got, read())) and got[1].any()
    want = verify(t, d, x, u)
    assert (got[2] == want[0]).all() and (got[3] == want[1]).all()
del g
print("as eager")
"""


def test_a_step_whose_first_calls_are_captured():
    """In a process of its own, where no kernel has been launched before; then replayed as lengths, rows, drafts and
    uniform numbers change, and compared with the same calls outside of the graph."""
    pytest.importorskip("torch")
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FIRST_IN_A_GRAPH, here, os.path.join(os.path.dirname(here), "engine-mlx_b200")],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as eager" in r.stdout, r.stdout + r.stderr


# ------------------------------------------------------------------- a prefix long enough for the tensor-memory kernel
def long_prefix(seed, page, hd, seqs, n_q=64, n_kv=8, **k):
    """More than 592 tiles of 64 rows and 64 positions: 12, 20 and 45 sequences have one half, one and two row tiles."""
    r = np.random.default_rng(seed)
    shared = page * -(-2500 // page)
    rows = np.ones(seqs, int)
    assert n_kv * -(-seqs * (n_q // n_kv) // 64) * (shared // 64) > 592
    return Case(seed, rows, shared + rows + r.integers(0, 50, seqs), n_q, n_kv, hd, page, shared, **k)


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 128, 256, 20])
@pytest.mark.parametrize("seqs", [12, 20, 45])
def test_a_long_prefix(ctx, seqs, page, hd):
    c = long_prefix(page, page, hd, seqs, pad=1).device(ctx)
    check_attend(c, attend(ctx, c))
    assert c.status == 0


@pytest.mark.parametrize("seqs", [3, 12, 45])
def test_a_long_prefix_of_large_scores(ctx, seqs):
    """Scores of a standard deviation of six: maxima move, and few weights count.  Their fp32 errors (128 products, 2^-24 of
    scores up to 40) stay below the 2^-11 that the bound has for them."""
    c = long_prefix(50, 16, 128, seqs) if seqs > 3 else Case(50, [1] * 3, [5000] * 3, 64, 8, shared=4992)
    c.q = emx.bf16(emx.f32(c.q) * 6)
    ramp = np.linspace(0.2, 1.0, c.shared // 16)  # later pages have larger keys
    for j, p in enumerate(c.shared_pages):
        c.k[p] = emx.bf16(emx.f32(c.k[p]) * ramp[j])
    check_attend(c, attend(ctx, c.device(ctx)))


@pytest.mark.parametrize("scale", [0.0, -0.1])
@pytest.mark.parametrize("seqs", [12, 45])
def test_a_long_prefix_and_scales_that_are_not_positive(ctx, scale, seqs):
    c = long_prefix(51, 16, 128, seqs)
    c.scale = scale
    check_attend(c, attend(ctx, c.device(ctx)))


@pytest.mark.parametrize("seqs", [12, 45])
def test_bad_pages_of_a_long_prefix(ctx, seqs):
    c = long_prefix(52, 16, 128, seqs).device(ctx)
    pages = c.shared_pages.copy()
    pages[7], pages[20], pages[-1] = c.n_pages, -1, 1 << 30
    c.d_shared.write(pages)
    hole = {p * 16 + x for p in (7, 20, len(pages) - 1) for x in range(16)}
    got = attend(ctx, c)
    assert c.status == 5 and near(got[:c.n], *want_without(c, [hole] * seqs)).all()
    c.d_shared.write(np.full(len(pages), -1, np.int32))
    got = attend(ctx, c)
    assert c.status == 5 and near(got[:c.n], *want_without(c, [set(range(c.shared))] * seqs)).all()


@pytest.mark.parametrize("seqs", [12, 45])
def test_what_is_not_finite_in_a_long_prefix(ctx, seqs):
    """A row of q that is NaN spoils no other; NaN in one dimension of V reaches that dimension of all rows."""
    c = long_prefix(53, 16, 128, seqs)
    want, size = c.attend()
    q = c.q.copy()
    q[5, 9] = NAN
    d = long_prefix(53, 16, 128, seqs)
    d.q = q
    got = attend(ctx, d.device(ctx))
    g = emx.f32(got[:c.n])
    assert np.isnan(g[5, 9]).all() and np.isnan(g).sum() == 128
    g[5, 9] = want[5, 9]
    assert near(emx.bf16(g), want, size).all()
    d = long_prefix(53, 16, 128, seqs)
    d.v[d.shared_pages[3], 2, 7, 11] = NAN
    g = emx.f32(attend(ctx, d.device(ctx))[:c.n])
    assert np.isnan(g[:, 16:24, 11]).all() and np.isnan(g).sum() == c.n * 8


@pytest.mark.parametrize("seqs,n_q,n_kv", [(12, 64, 8), (20, 64, 8), (45, 64, 8), (135, 64, 8)])
def test_a_long_prefix_gives_the_same_bits(ctx, seqs, n_q, n_kv):
    c = long_prefix(54, 16, 128, seqs, n_q, n_kv).device(ctx)
    first = attend(ctx, c)
    for _ in range(20):
        assert (attend(ctx, c) == first).all()
    ctx.sdpa_paged(c.dq, c.kv, c.batch, n_q, c.scale, c.shared, c.d_shared, out=c.dq)  # over q
    assert (c.dq.read(np.uint16, c.q.shape) == first[:c.n_rows]).all()


def test_long_and_short_prefixes_one_after_another(ctx):
    cases = [long_prefix(55, 16, 128, 45), Case(56, [1] * 45, [400 + i for i in range(45)], 64, 8, shared=320),
             long_prefix(57, 64, 128, 12), long_prefix(58, 20, 128, 12), Case(59, [1] * 30, [70] * 30, 64, 8)]
    for c in cases:
        c.device(ctx)
    ws = ctx.alloc(max(ctx.sdpa_paged_workspace(c.kv, c.batch, 64, c.shared) for c in cases))
    want = [attend(ctx, c, ws=ws) for c in cases]
    outs = [[ctx.put(np.full(w.shape, NAN, np.uint16)) for w in want] for _ in range(4)]
    for turn, out in enumerate(outs):
        for i in np.random.default_rng(turn).permutation(len(cases)):
            c = cases[i]
            ctx.sdpa_paged(c.dq, c.kv, c.batch, 64, c.scale, c.shared, c.d_shared, out=out[i], workspace=ws)
    for out in outs:
        for o, w in zip(out, want):
            assert (o.read(np.uint16, w.shape) == w).all()


# ------------------------------------------------------------------------------------------------- the weights' precision
@pytest.mark.parametrize("rows,n_q,n_kv,hd", [(1, 32, 4, 128), (1, 16, 8, 64), (40, 8, 2, 128), (40, 8, 2, 64)])
def test_the_output_is_rounded_once(ctx, rows, n_q, n_kv, hd):
    """Own parts by warps (one row a sequence) and by CTAs: the error's root mean square is that of one rounding to bf16.
    What else there is of it: weights off by at most 2^-14, scores by 2^-13 of a weight (128 products of 2^-24, of sums
    |q k| scale up to 8), and as V is drawn apart from q and k, an error e of every weight moves the output by e |o| in
    the mean square; the sum of the weights adds as much again.  2^-11 in all, against 0.0016 |o| for the rounding."""
    c = Case(61, [rows] * 6, [500 + 100 * i for i in range(6)], n_q, n_kv, hd).device(ctx)
    want, _ = c.attend()
    g = emx.f32(attend(ctx, c)[:c.n]).astype(np.float64)
    rms = lambda x: np.sqrt((x * x).mean())  # noqa: E731
    extra = 2.0 ** -11 * rms(want)
    assert rms(g - want) <= np.hypot(rms(emx.f32(emx.bf16(want)) - want), extra)


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("seqs", [12, 20, 45])
def test_the_output_over_a_long_prefix_is_rounded_once(ctx, seqs, hd):
    c = long_prefix(62, 16, hd, seqs).device(ctx)
    want, _ = c.attend()
    g = emx.f32(attend(ctx, c)[:c.n]).astype(np.float64)
    rms = lambda x: np.sqrt((x * x).mean())  # noqa: E731
    extra = 2.0 ** -11 * rms(want)
    assert rms(g - want) <= np.hypot(rms(emx.f32(emx.bf16(want)) - want), extra)


@pytest.mark.parametrize("seqs,prefix", [(1, 0), (3, 64), (12, 2560), (45, 2560)])
def test_a_constant_v_comes_out_as_it_is(ctx, seqs, prefix):
    """Keys of one score below that of a single key, so that all their weights round the same way: the weights of the
    products and those of the sum are the same to 2^-14 of each, well below the half step of 2^-9 that would show."""
    for below in (0.3, 0.69, 1.1, 2.6):
        c = Case(63, [1] * seqs, [prefix + 300] * seqs, 64, 8, page=16, shared=prefix)
        c.q = emx.bf16(np.ones(c.q.shape))
        c.k = emx.bf16(np.zeros(c.k.shape))
        top = (c.shared_pages if prefix else c.table[0])[1]
        c.k[top, :, 3] = emx.bf16(np.full((8, 128), below / (128 * c.scale)))
        c.v = emx.bf16(np.broadcast_to(np.linspace(0.7, 1.4, 128), c.v.shape))
        got = attend(ctx, c.device(ctx))
        assert (got[:c.n] == c.v[0, 0, 0]).all()


@pytest.mark.parametrize("seqs,prefix", [(1, 0), (12, 2560), (45, 2560)])
def test_an_infinite_v_stays_infinite(ctx, seqs, prefix):
    c = Case(64, [1] * seqs, [prefix + 40] * seqs, 64, 8, page=16, shared=prefix)
    page = (c.shared_pages if prefix else c.table[0])[1]
    c.v[page, 2, 7, 11], c.v[page, 2, 7, 12] = 0x7F80, 0xFF80
    g = emx.f32(attend(ctx, c.device(ctx))[:c.n])
    assert (g[:, 16:24, 11] == np.inf).all() and (g[:, 16:24, 12] == -np.inf).all()
    g[:, 16:24, 11:13] = 0
    assert np.isfinite(g).all()


# ------------------------------------------------------------------------------------------ on a stream of the caller's
def tensor(torch, bits):
    return torch.from_numpy(np.ascontiguousarray(bits).view(np.int16)).cuda().view(torch.bfloat16)


@pytest.mark.parametrize("side", [False, True])
def test_a_context_on_a_torch_stream(ctx, side):
    """Inputs that are written behind long products, outputs that are read, and memory that is used again, all without a
    wait: one stream orders them."""
    torch = pytest.importorskip("torch")
    c = Case(65, [1] * 40, [300 + 7 * i for i in range(40)], 16, 4, shared=160).device(ctx)
    want = attend(ctx, c)[:c.n]
    q0 = tensor(torch, c.q)
    torch.cuda.synchronize()
    st = torch.cuda.Stream() if side else torch.cuda.default_stream()
    on = emx.Ctx(0, stream=st)
    assert stream_of(on) == (st.cuda_stream or None)
    with torch.cuda.stream(st):
        got = []
        for _ in range(10):
            x = torch.randn(4096, 4096, device="cuda")
            for _ in range(6):
                x = torch.tanh(x @ x)
            q, out = torch.full_like(q0, float("nan")), torch.empty(c.n, 16, 128, dtype=torch.bfloat16, device="cuda")
            q.copy_(torch.where(x[0, 0] > 2, q, q0))  # tanh: never
            on.sdpa_paged(q, c.kv, c.batch, 16, c.scale, c.shared, c.d_shared, out=out)
            del q
            torch.full_like(q0, float("nan"))  # where q was
            got.append(out.clone())
            out.zero_()
        torch.cuda.synchronize()
    assert on.device_status() == 0
    for g in got:
        assert (g.cpu().view(torch.int16).numpy().view(np.uint16) == want).all()
    on.close()
    with torch.cuda.stream(st):  # still the caller's
        assert float(torch.ones(8, device="cuda").sum()) == 8


def test_a_context_on_a_torch_stream_is_captured_with_it(ctx):
    torch = pytest.importorskip("torch")
    c = Case(66, [1] * 20, [200 + 5 * i for i in range(20)], 8, 2, shared=64).device(ctx)
    want = attend(ctx, c)[:c.n]
    ctx.synchronize()
    q0, st = tensor(torch, c.q), torch.cuda.Stream()
    torch.cuda.synchronize()
    on = emx.Ctx(0, stream=st)
    ws = on.alloc(on.sdpa_paged_workspace(c.kv, c.batch, 8, 64))
    x = torch.zeros_like(q0)
    out = torch.empty(c.n, 8, 128, dtype=torch.bfloat16, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st, capture_error_mode="thread_local"):
        q = x * 0.5
        on.sdpa_paged(q, c.kv, c.batch, 8, c.scale, 64, c.d_shared, out=out, workspace=ws)
        twice = out * 2
    with torch.cuda.stream(st):
        x.copy_(q0 * 2)  # halved and doubled without rounding
        g.replay()
        x.zero_()
        got = twice.clone()
        g.replay()
    torch.cuda.synchronize()
    assert on.device_status() == 0
    assert ((got * 0.5).cpu().view(torch.int16).numpy().view(np.uint16) == want).all()
    del g
    on.close()


def test_a_context_is_not_made_on_a_stream_that_is_captured(ctx):
    torch = pytest.importorskip("torch")
    st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    x = torch.ones(4, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st, capture_error_mode="thread_local"):
        y = x + 1
        with pytest.raises(emx.EmxError, match="captured") as e:
            emx.Ctx(0, stream=st)
        assert e.value.code == emx.ERR_STATE
    g.replay()
    torch.cuda.synchronize()
    assert (y == 2).all()
    on = emx.Ctx(0, stream=st)
    assert on.device_status() == 0
    on.close()


def test_tensors_of_other_types_and_places_are_refused(ctx):
    """Before anything is launched."""
    torch = pytest.importorskip("torch")
    c = Case(72, [1, 2], [30, 20], 4, 2).device(ctx)
    q, out = (torch.zeros(3, 4, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    qkv = torch.zeros(3, 8 * 128, dtype=torch.bfloat16, device="cuda")
    t, u = torch.rand(2, 3, 50, device="cuda"), torch.rand(2, 3, device="cuda")
    x = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    for bad in (q.cpu(), q.half(), q.transpose(0, 1)):
        for call in (lambda: ctx.sdpa_paged(bad, c.kv, c.batch, 4, c.scale, out=out), lambda: ctx.sdpa_paged(q, c.kv, c.batch, 4, c.scale, out=bad),
                     lambda: ctx.paged_append(qkv, c.kv, c.batch, 4, out=bad)):
            with pytest.raises(emx.EmxError, match="is wanted"):
                call()
    for args in ((t.double(), None, x, u), (t.cpu(), None, x, u), (t, t[:, :2], x, u), (t, None, x.long(), u), (t, None, x, u.bfloat16())):
        with pytest.raises(emx.EmxError, match="is wanted"):
            ctx.verify_draft(*args, 2, 2, 50)
    with pytest.raises(emx.EmxError, match="is wanted"):
        ctx.verify_draft(t, None, x, u, 2, 2, 50, dtype=emx.BF16)
    ctx.verify_draft(t, t[:, :2].contiguous(), x, u, 2, 2, 50)
    assert ctx.device_status() == 0


# ------------------------------------------------------------------------- each thing that can be out of order, by itself
OUT_OF_ORDER = [("lengths", 2, 1, 6), ("lengths", 1, 0, 6), ("lengths", 3, -1, 6), ("lengths", 0, -2**31, 6), ("lengths", 1, "room", 4),
                ("lengths", 3, 2**31 - 1, 4), ("indptr", 4, 100, 6), ("indptr", 0, -1, 6), ("indptr", 2, 9, 6), ("indptr", 2, 0, 6),
                ("table", (2, 1), "pages", 5), ("table", (0, 0), -1, 5), ("table", (3, 2), 2**31 - 1, 5), ("table", (1, 1), -2**31, 5)]


@pytest.mark.parametrize("call", ["attend", "append"])
@pytest.mark.parametrize("array,at,value,status", OUT_OF_ORDER)
def test_each_input_out_of_order_has_its_status(ctx, array, at, value, status, call):
    c = Case(67, [1, 2, 3, 1], [10, 20, 30, 48], 4, 2, pad=2)
    c.max_pages = c.table.shape[1]
    indptr, lens, table = c.indptr.copy(), np.array(c.lens, np.int32), c.table.copy()
    {"indptr": indptr, "lengths": lens, "table": table}[array][at] = {"room": c.max_pages * 16 + 1, "pages": c.n_pages}.get(value, value)
    c.device(ctx)
    b = emx.PagedBatch(ctx.put(indptr), ctx.put(lens), ctx.put(table), 4, c.n_rows, c.max_pages)
    out = ctx.alloc(c.n_rows * 4 * 128 * 2)
    if call == "attend":
        ctx.sdpa_paged(c.dq, c.kv, b, 4, c.scale, out=out)
    else:
        if array == "table":  # the page of a new row
            row_page = {(2, 1): (27, 29), (0, 0): (9, 9), (3, 2): (47, 47), (1, 1): (18, 19)}[at]
            assert row_page[0] // 16 == at[1] == row_page[1] // 16
        ctx.paged_append(c.dqkv, c.kv, b, 4, out=out)
    assert ctx.device_status() == status
    attend(ctx, c)
    assert c.status == 0


@pytest.mark.parametrize("seqs,prefix", [(3, 64), (12, 2560)])
@pytest.mark.parametrize("value", [-1, 1 << 30, "pages"])
def test_a_bad_page_of_a_prefix_has_its_status(ctx, seqs, prefix, value):
    c = Case(68, [1] * seqs, [prefix + 20] * seqs, 64, 8, page=16, shared=prefix).device(ctx)
    attend(ctx, c)
    assert c.status == 0
    pages = c.shared_pages.copy()
    pages[-1] = c.n_pages if value == "pages" else value
    c.d_shared.write(pages)
    attend(ctx, c)
    assert c.status == 5


def test_scores_of_any_size_where_one_key_decides(ctx):
    """Scores of some thousands.  Their fp32 products are off by at most 130 * 2^-24 of sum |q k| scale: where the largest is
    ahead of the next by that twice and 20 more, the others' weights come to less than 300 e^-20 = 2^-20."""
    c = Case(9, [2, 1], [300, 160], 4, 2)
    c.k, c.q = emx.bf16(emx.f32(c.k) * 60), emx.bf16(emx.f32(c.q) * 30)
    want, size = c.attend()
    ok = np.zeros((c.n, 4), bool)
    for i in range(2):
        k = c.keys(i)
        for j, p in enumerate(c.positions(i)):
            q = emx.f32(c.q[c.indptr[i] + j]).astype(np.float64).reshape(2, 2, 128)
            s = np.sort(np.einsum("hgd,shd->hgs", q, k[:p + 1]).reshape(4, -1) * c.scale, -1)
            off = np.einsum("hgd,shd->hgs", np.abs(q), np.abs(k[:p + 1])).reshape(4, -1).max(-1) * c.scale * 130 * 2.0 ** -24
            ok[c.indptr[i] + j] = s[:, -1] - s[:, -2] > 20 + 2 * off
    assert ok.mean() > 0.7
    assert near(attend(ctx, c.device(ctx))[:c.n], want, size)[ok].all()


# ----------------------------------------------------------------- the tensor-memory kernel by the arithmetic of its choice
def takes_tensor_memory(ctx, c):
    """Whether the prefix has more than two 64 x 64 tiles to each of two CTAs an SM, in pages of whole 8-row groups."""
    return c.page % 8 == 0 and c.n_kv * -(-c.n_rows * (c.n_q // c.n_kv) // 64) * -(-c.shared // 64) > 4 * ctx.num_sms


def attend_64(c):
    """Case.attend on the device; the pages are looked up on the host."""
    torch = pytest.importorskip("torch")
    out, size = (np.zeros((c.n, c.n_q, c.hd)) for _ in range(2))
    for i in range(c.n_seqs):
        if not c.rows[i]:
            continue
        ks, vs = (torch.from_numpy(c.keys(i, x)).cuda() for x in (c.k, c.v))
        q = torch.from_numpy(emx.f32(c.q[c.indptr[i]:c.indptr[i + 1]])).cuda().double()
        for j, pos in enumerate(c.positions(i)):
            s = torch.einsum("hgd,shd->hgs", q[j].view(c.n_kv, -1, c.hd), ks[:pos + 1]) * c.scale
            w = torch.softmax(s, -1)
            row = c.indptr[i] + j
            out[row] = torch.einsum("hgs,shd->hgd", w, vs[:pos + 1]).reshape(c.n_q, c.hd).cpu().numpy()
            size[row] = torch.einsum("hgs,shd->hgd", w, vs[:pos + 1].abs()).reshape(c.n_q, c.hd).cpu().numpy()
    return out, size


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("seqs,n_q,n_kv,shared", [(300, 128, 64, 128), (300, 128, 64, 1040), (15, 1000, 50, 2080), (17, 960, 48, 2048)])
def test_workers_go_from_segment_to_segment(ctx, seqs, n_q, n_kv, shared, hd):
    """More segments than SMs, and fewer where whole workers to each would take too long: a worker goes from tiles of two
    groups' rows to those of one and back."""
    r = np.random.default_rng(69)
    c = Case(69, [1] * seqs, shared + 1 + r.integers(0, 20, seqs), n_q, n_kv, hd, shared=shared)
    rows, kt = seqs * n_q // n_kv, -(-shared // 128)
    segments = n_kv * -(-rows // 256)
    per = -(-segments * kt // ctx.num_sms)
    assert takes_tensor_memory(ctx, c) and (segments > ctx.num_sms or -(-kt // (ctx.num_sms // segments)) > per + 4)
    got = attend(ctx, c.device(ctx))
    assert c.status == 0 and near(got[:c.n], *attend_64(c)).all()


@pytest.mark.parametrize("seqs", [12, 45])
def test_a_page_may_stand_for_several_of_a_long_prefix(ctx, seqs):
    c = long_prefix(70, 16, 128, seqs)
    for a, b in ((2, 0), (9, 8), (40, 0)):
        c.shared_pages[a] = c.shared_pages[b]
    c.table[:, :len(c.shared_pages)] = c.shared_pages
    assert takes_tensor_memory(ctx, c)
    got = attend(ctx, c.device(ctx))
    assert c.status == 0 and near(got[:c.n], *attend_64(c)).all()


@pytest.mark.parametrize("seqs", [12, 45])
def test_a_long_prefix_past_32_bits(ctx, seqs):
    """Its pages at both ends and in the middle of a cache of more than 2^32 elements."""
    c = long_prefix(71, 128, 128, seqs)
    assert takes_tensor_memory(ctx, c)
    page = 8 * 128 * 128
    pages = 2 ** 32 // page + 128
    want = attend_64(c)
    k, v = (ctx.alloc(pages * page * 2) for _ in range(2))
    assert c.n_pages <= 90
    far = np.concatenate([np.arange(30), pages // 2 + np.arange(20), np.arange(pages - 40, pages)])[:c.n_pages]
    far = np.random.default_rng(71).permutation(far).astype(np.int32)
    c.device(ctx)
    for j, to in enumerate(far):
        k.write(c.k[j], int(to) * page * 2)
        v.write(c.v[j], int(to) * page * 2)
    move = lambda t: np.where((t >= 0) & (t < c.n_pages), far[np.clip(t, 0, c.n_pages - 1)], -7).astype(np.int32)  # noqa: E731
    c.kv = emx.PagedKV(k, v, pages, 128, 8, 128)
    c.batch = emx.PagedBatch(c.d_indptr, c.d_lens, ctx.put(move(c.table)), c.n_seqs, c.n_rows, c.max_pages)
    c.d_shared = ctx.put(move(c.shared_pages))
    got = attend(ctx, c)
    k.free()
    v.free()
    assert c.status == 0 and near(got[:c.n], *want).all()
