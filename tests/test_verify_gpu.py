"""emx_verify_draft against its definition in 64 bits, on an sm_100 GPU, and the batched operators together, as a
speculative decoding step uses them."""
import numpy as np
import pytest

import emx
from paged_case import NAN, Case, verify

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = emx.Ctx(0)
    yield c
    c.close()


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


def inputs(seed, n, m, v, near=0.7, spread=2.0):
    r = np.random.default_rng(seed)
    x = r.normal(size=(n, m + 1, v)) * spread
    target = softmax(x).astype(np.float32)
    draft = softmax(x[:, :m] + near * r.normal(size=(n, m, v))).astype(np.float32)
    tokens = np.zeros((n, m), np.int32)
    for i in range(n):
        for j in range(m):
            tokens[i, j] = min(v - 1, np.searchsorted(np.cumsum(draft[i, j].astype(np.float64)), r.random()))
    return target, draft, tokens, r.random((n, m + 1)).astype(np.float32)


def run(ctx, target, draft, tokens, u, counts=None, kind=emx.F32):
    """(tokens, accepted, status) of the operator, and the definition's on the same values."""
    n, m1, v = target.shape
    as_kind = (lambda x: emx.bf16(x)) if kind == emx.BF16 else (lambda x: x)
    seen = (lambda x: emx.f32(emx.bf16(x))) if kind == emx.BF16 else (lambda x: x)
    put = lambda x: ctx.put(x if x.size else np.zeros(4, np.int32))  # noqa: E731
    out, acc = ctx.put(np.full((n + 1, m1), 77, np.int32)), ctx.put(np.full(n + 1, 77, np.int32))
    ctx.verify_draft(put(as_kind(target)), None if draft is None else put(as_kind(draft)), put(tokens), put(u), n, m1 - 1, v,
                     dtype=kind, counts=None if counts is None else put(counts), out=out, accepted=acc)
    status = ctx.device_status()
    got = out.read(np.int32, (n + 1, m1)), acc.read(np.int32, n + 1)
    assert (got[0][n:] == 77).all() and got[1][n] == 77
    want = verify(seen(target), None if draft is None else seen(draft), tokens, u, counts)
    return got[0][:n], got[1][:n], status, want


def same(ctx, *a, **k):
    out, acc, status, want = run(ctx, *a, **k)
    assert (acc == want[1]).all(), (acc, want[1])
    assert (out == want[0]).all(), np.argwhere(out != want[0])[:5]
    assert status == 0
    return out, acc


@pytest.mark.parametrize("kind", [emx.F32, emx.BF16])
@pytest.mark.parametrize("v", [1, 2, 31, 127, 128, 1000, 1003, 4104, 32000, 151936])
@pytest.mark.parametrize("n,m", [(1, 1), (2, 4), (19, 3)])
def test_verify(ctx, n, m, v, kind):
    same(ctx, *inputs(v + n, n, m, v), kind=kind)


@pytest.mark.parametrize("kind", [emx.F32, emx.BF16])
@pytest.mark.parametrize("m", [0, 1, 33, 70])
def test_numbers_of_drafts(ctx, m, kind):
    t, d, x, u = inputs(m, 5, m, 200, near=0.05)
    same(ctx, t, d if m else None, x, u, kind=kind)
    counts = np.array([m, 0, m // 2, -1, m + 9], np.int32)
    out, acc = same(ctx, t, d if m else None, x, u, counts, kind=kind)
    assert (out[3] == -1).all() and acc[3] == 0


@pytest.mark.parametrize("kind", [emx.F32, emx.BF16])
def test_drafts_without_probabilities(ctx, kind):
    t, _, x, u = inputs(3, 40, 4, 1000, spread=4.0)
    x[::2] = t[::2, :4].argmax(-1)
    _, acc = same(ctx, t, None, x, u, kind=kind)
    assert 0 < acc.sum() < acc.size * 4


def test_a_draft_like_its_target_is_always_accepted(ctx):
    t, _, _, u = inputs(4, 8, 3, 500)
    _, acc = same(ctx, t, t[:, :3].copy(), inputs(4, 8, 3, 500, near=0.0)[2], u)
    assert (acc == 3).all()


def test_ends_of_the_uniform_numbers(ctx):
    """0 takes the first index with mass, the largest number below 1 the last it reaches; 0 accepts anything that the
    target can say, and nothing that it cannot."""
    t, d, x, u = inputs(5, 4, 2, 300)
    t[:, :, :7] = 0
    t[:, :, -9:] = 0
    u[:2] = 0.0
    u[2:] = np.float32(1 - 2.0 ** -24)
    out, _ = same(ctx, t, d, x, u)
    x[0, 0] = 3  # no mass in the target
    _, acc = same(ctx, t, d, x, u)
    assert acc[0] == 0


def test_rows_without_mass(ctx):
    t, d, x, u = inputs(6, 6, 2, 260)
    t[0] = 0  # nothing at all: no token
    t[1, 0] = d[1, 0] * np.float32(0.5)  # below the draft everywhere: refused, and nothing left of p - q
    u[1, 0] = 0.9
    t[2, :, 5] = np.nan
    t[3, :, 6] = np.inf
    t[4, :, 7] = -1.0
    d[5, :, 8] = np.nan
    for y in (x, ):
        y[:, :] = np.where(np.isin(y, [5, 6, 7, 8]), 20, y)
    out, acc = same(ctx, t, d, x, u)
    assert out[0, 0] == -1 and acc[0] == 0 and acc[1] == 0 and out[1, 0] >= 0


def test_only_one_entry_has_mass(ctx):
    for at in (0, 1, 511, 512, 99_999, 151_935):
        t = np.zeros((2, 2, 151936), np.float32)
        t[:, :, at] = 1e-30
        d = np.full((2, 1, 151936), 1 / 151936, np.float32)
        out, acc = same(ctx, t, d, np.full((2, 1), 700, np.int32), np.array([[0.5, 0.0], [0.5, 0.999]], np.float32))
        assert (out[:, 0] == at).all() and (acc == 0).all()


def test_drafts_outside_the_vocabulary(ctx):
    t, d, x, u = inputs(7, 4, 3, 100, near=0.01)
    x[0, 0], x[1, 2], x[2, 1] = 100, -1, 1 << 30
    out, acc, status, want = run(ctx, t, d, x, u)
    assert status == 3 and (out == want[0]).all() and (acc == want[1]).all()
    out, acc, status, want = run(ctx, t, None, x, u)
    assert status == 3 and (out == want[0]).all() and (acc == want[1]).all()


def test_misaligned_rows(ctx):
    """Probabilities that begin between 16-byte borders."""
    t, d, x, u = inputs(8, 3, 2, 400)
    want = verify(t, d, x, u)
    dev = []
    for y in (t, d):
        b = ctx.alloc(y.nbytes + 4)
        b.write(y, 4)

        class At:  # anything with an address
            def __init__(self, p):
                self.p = p

            def data_ptr(self):
                return self.p

        dev.append(At(b.ptr + 4))
    out, acc = ctx.verify_draft(dev[0], dev[1], ctx.put(x), ctx.put(u), 3, 2, 400)
    assert (out.read(np.int32, (3, 3)) == want[0]).all() and (acc.read(np.int32, 3) == want[1]).all()


def test_tokens_are_distributed_as_the_target(ctx):
    """Speculative sampling's promise: the first token of each sequence is a draw of the target's first row, whatever the
    draft proposed.  20,000 sequences of one distribution over six tokens; a share's standard deviation is
    sqrt(p (1 - p) / 20000) <= 0.0036, five of which bound it."""
    n, r = 20000, np.random.default_rng(9)
    p = np.array([0.4, 0.05, 0.25, 0.0, 0.2, 0.1], np.float32)
    q = np.array([0.1, 0.5, 0.2, 0.1, 0.05, 0.05], np.float32)
    t = np.broadcast_to(p, (n, 2, 6)).copy()
    d = np.broadcast_to(q, (n, 1, 6)).copy()
    x = r.choice(6, (n, 1), p=q.astype(np.float64) / q.astype(np.float64).sum()).astype(np.int32)
    out, _ = same(ctx, t, d, x, r.random((n, 2)).astype(np.float32))
    share = np.bincount(out[:, 0], minlength=6) / n
    assert (np.abs(share - p) <= 0.018).all() and share[3] == 0


@pytest.mark.parametrize("kind", [emx.F32, emx.BF16])
@pytest.mark.parametrize("n,m,v", [(65535, 1, 5), (2, 4096, 7), (1, 0, 1), (600, 2, 1000)])
def test_as_many_sequences_and_drafts_as_there_may_be(ctx, n, m, v, kind):
    t, d, x, u = inputs(n + m, n, m, v, near=0.0 if m > 100 else 0.7)
    same(ctx, t, d if m else None, x, u, kind=kind)


def test_rows_past_32_bits(ctx):
    """A vocabulary of 2^30: rows of 2 GB that begin beyond 2^31 elements."""
    torch = pytest.importorskip("torch")
    V = 1 << 30
    t, d = (torch.zeros(2, k, V, dtype=torch.bfloat16, device="cuda") for k in (2, 1))
    # sequence 0: refused, and of p - q one index is left; sequence 1: accepted, and two have mass
    t[0, 0, V // 2], t[0, 0, V - 3], d[0, 0, V // 2], d[0, 0, 5] = 0.5, 0.5, 0.5, 0.5
    t[1, 0, V - 1], d[1, 0, V - 1], t[1, 1, V - 7], t[1, 1, V - 2] = 0.5, 0.5, 0.5, 0.5
    x, u = torch.tensor([[5], [V - 1]], dtype=torch.int32, device="cuda"), torch.tensor([[0.1, 0.9], [0.3, 0.6]], device="cuda")
    torch.cuda.synchronize()
    out, acc = ctx.verify_draft(t, d, x, u, 2, 1, V, dtype=emx.BF16)
    assert ctx.device_status() == 0
    assert out.read(np.int32, (2, 2)).tolist() == [[V - 3, -1], [V - 1, V - 2]] and acc.read(np.int32, 2).tolist() == [0, 1]


def test_two_contexts_verify_at_once(ctx):
    other = emx.Ctx(0)
    runs = []
    for cx, seed in ((ctx, 11), (other, 12)):
        t, d, x, u = inputs(seed, 40, 3, 20000)
        runs.append((cx, [cx.put(y) for y in (t, d, x, u)], verify(t, d, x, u)))
    outs = [[cx.verify_draft(*b, 40, 3, 20000) for cx, b, _ in runs] for _ in range(20)]
    for pair in outs:
        for (out, acc), (_, _, want) in zip(pair, runs):
            assert (out.read(np.int32, (40, 4)) == want[0]).all() and (acc.read(np.int32, 40) == want[1]).all()
    other.close()


def test_a_status_reported_after_another_was_cleared_is_kept(ctx):
    """Clearing is ordered with what follows on the context's stream."""
    t, d, x, u = (ctx.put(y) for y in inputs(12, 1, 1, 8))
    bad = ctx.put(np.array([[8]], np.int32))
    out, acc = ctx.put(np.zeros((1, 2), np.int32)), ctx.put(np.zeros(1, np.int32))
    for _ in range(300):
        ctx.verify_draft(t, d, bad, u, 1, 1, 8, out=out, accepted=acc)
        assert ctx.device_status() == 3
    ctx.verify_draft(t, d, x, u, 1, 1, 8, out=out, accepted=acc)
    assert ctx.device_status() == 0


# ------------------------------------------------------------------------------------------- a step, all of it together
def test_speculative_steps_over_a_shared_prompt(ctx):
    """Three sequences with a common prompt take four steps of speculative decoding: the drafted rows are appended
    together, attend, and are verified; refused rows are overwritten by the next step.  A toy model (embedding, one
    attention layer, unembedding) gives the target's probabilities from the attention's output on the host, so every
    step's output depends on all of the cache before it.  The attention of every step is compared with the definition
    in 64 bits over the accepted tokens' own K and V, which are computed again from those tokens alone."""
    r = np.random.default_rng(10)
    V, n_q, n_kv, hd, page, S, m = 96, 4, 2, 128, 16, 64, 3
    heads = n_q + 2 * n_kv
    embed = r.normal(size=(V, heads * hd)).astype(np.float32)  # token -> its q | k | v
    unembed = (r.normal(size=(n_q * hd, V)) * 0.3).astype(np.float32)
    prompt = r.integers(0, V, S)
    history = [list(prompt) + [int(r.integers(0, V))] for _ in range(3)]  # the last token is not in the cache yet
    n_pages, max_pages = 32, 8
    perm = r.permutation(n_pages).astype(np.int32)
    table = np.full((3, max_pages), -1, np.int32)
    table[:, :S // page] = perm[:S // page]
    for i in range(3):
        table[i, S // page:] = perm[4 + 4 * i:8 + 4 * i]
    k, v = (ctx.put(np.full((n_pages, n_kv, page, hd), NAN, np.uint16)) for _ in range(2))
    kv = emx.PagedKV(k, v, n_pages, page, n_kv, hd)
    d_table, d_shared = ctx.put(table), ctx.put(perm[:S // page].copy())
    d_indptr, d_lens = ctx.put(np.zeros(4, np.int32)), ctx.put(np.zeros(3, np.int32))
    # the prompt once, through sequence 0
    d_indptr.write(np.array([0, S, S, S], np.int32))
    d_lens.write(np.array([S, 0, 0], np.int32))
    ctx.paged_append(ctx.put(emx.bf16(embed[prompt])), kv, emx.PagedBatch(d_indptr, d_lens, d_table, 3, S, max_pages), n_q)
    total = 0
    for step in range(4):
        drafts = r.integers(0, V, (3, m)).astype(np.int32)
        drafts[:, 0] = [(h[-1] * 7 + 3) % V for h in history]
        counts = np.array([m, 1, 2], np.int32)
        toks = [[h[-1]] + drafts[i, :counts[i]].tolist() for i, h in enumerate(history)]
        rows = [len(t) for t in toks]
        indptr = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        n = int(indptr[-1])
        lens = np.array([len(h) - 1 + c for h, c in zip(history, rows)], np.int32)
        d_indptr.write(indptr)
        d_lens.write(lens)
        batch = emx.PagedBatch(d_indptr, d_lens, d_table, 3, n, max_pages)
        q = ctx.paged_append(ctx.put(emx.bf16(embed[sum(toks, [])])), kv, batch, n_q)
        o = ctx.sdpa_paged(q, kv, batch, n_q, hd ** -0.5, S, d_shared)
        plain = ctx.sdpa_paged(q, kv, batch, n_q, hd ** -0.5)
        o, plain = (emx.f32(x.read(np.uint16, (n, n_q, hd))) for x in (o, plain))
        for i in range(3):
            # the sequence's tokens alone, all of them again
            c = Case(0, [rows[i]], [int(lens[i])], n_q, n_kv, hd, page)
            every = np.array(history[i][:-1] + toks[i])
            a = Case(0, [len(every)], [len(every)], n_q, n_kv, hd, page)
            a.qkv = emx.bf16(embed[every])
            qa, ka, va = a.append()
            c.k, c.v = (np.full(c.k.shape, NAN, np.uint16) for _ in range(2))
            p = np.arange(len(every))
            c.k[c.table[0, p // page], :, p % page] = emx.bf16(ka)
            c.v[c.table[0, p // page], :, p % page] = emx.bf16(va)
            c.q = emx.bf16(qa[-rows[i]:])
            want, size = c.attend()
            at = slice(indptr[i], indptr[i + 1])
            # K and q may round to the other neighbour of a value that fp32 and fp64 put on either side of a half step:
            # a score moves by 2^-8 |q k| scale of that one dimension, below 2^-6 in all
            for g in (o[at], plain[at]):
                assert (np.abs(g - want) <= 2.0 ** -6 * (size + np.abs(want))).all()
        # the rows' logits on the host; then the drafts against them
        probs = softmax((o.reshape(n, -1) @ unembed) * 2).astype(np.float32)
        target = np.zeros((3, m + 1, V), np.float32)
        for i in range(3):
            target[i, :rows[i]] = probs[indptr[i]:indptr[i + 1]]
        u = r.random((3, m + 1)).astype(np.float32)
        out, acc, status, want = run(ctx, target, None, drafts, u, counts)
        assert status == 0 and (out == want[0]).all() and (acc == want[1]).all()
        for i in range(3):
            new = out[i][:acc[i] + 1].tolist()
            assert -1 not in new and acc[i] <= counts[i]
            history[i] += new
            total += len(new)
    assert total >= 12
