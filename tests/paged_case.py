"""Batches over a paged K/V cache for the tests: random ones, and the operators' definitions in 64 bits."""
import numpy as np

import emx

NAN = np.uint16(0x7FC0)


class Case:
    """A batch of sequences with rows[i] new rows and lens[i] positions (the first `shared` common to all), over a
    cache whose rows that belong to no position hold NaN."""

    def __init__(self, seed, rows, lens, n_q=4, n_kv=2, hd=128, page=16, shared=0, pad=0, spare=2):
        r = self.rng = np.random.default_rng(seed)
        assert shared % page == 0
        self.rows, self.lens = list(rows), list(lens)
        self.n_q, self.n_kv, self.hd, self.page, self.shared = n_q, n_kv, hd, page, shared
        self.n_seqs, self.n = len(rows), sum(rows)
        self.n_rows = self.n + pad
        self.indptr = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        ns = shared // page
        own = [max(0, -(-t // page) - ns) if k else 0 for t, k in zip(lens, rows)]
        self.max_pages = max(1, ns, max((-(-t // page) for t in lens), default=1))
        self.n_pages = ns + sum(own) + spare
        perm = r.permutation(self.n_pages).astype(np.int32)
        self.shared_pages = perm[:ns].copy()
        self.table = np.full((self.n_seqs, self.max_pages), -7, np.int32)  # no page: must not be read
        at = ns
        for i, k in enumerate(own):
            self.table[i, :ns] = self.shared_pages
            self.table[i, ns:ns + k] = perm[at:at + k]
            at += k
        shape = (self.n_pages, n_kv, page, hd)
        self.k, self.v = emx.bf16(r.normal(size=shape)), emx.bf16(r.normal(size=shape))
        used = np.zeros((self.n_pages, page), bool)
        for i in range(self.n_seqs):
            if rows[i]:
                p = np.arange(lens[i])
                used[self.table[i, p // page], p % page] = True
        for x in (self.k, self.v):
            x.transpose(0, 2, 1, 3)[~used] = NAN
        self.scale = hd ** -0.5
        self.q = emx.bf16(r.normal(size=(self.n_rows, n_q, hd)))
        self.qkv = emx.bf16(r.normal(size=(self.n_rows, (n_q + 2 * n_kv) * hd)) * 2)

    def device(self, ctx):
        d = lambda x: ctx.put(x if x.size else np.zeros(4, np.int32))  # noqa: E731
        self.dk, self.dv = d(self.k), d(self.v)
        self.kv = emx.PagedKV(self.dk, self.dv, self.n_pages, self.page, self.n_kv, self.hd)
        self.d_indptr, self.d_lens = d(self.indptr), d(np.array(self.lens, np.int32))
        self.batch = emx.PagedBatch(self.d_indptr, self.d_lens, d(self.table), self.n_seqs, self.n_rows, self.max_pages)
        self.d_shared = d(self.shared_pages) if self.shared else None
        self.dq, self.dqkv = d(self.q), d(self.qkv)
        return self

    def positions(self, i):
        return np.arange(self.lens[i] - self.rows[i], self.lens[i])

    def keys(self, i, x=None):
        """K (or x) of sequence i, f64 [positions, n_kv, hd]."""
        p = np.arange(self.lens[i])
        return emx.f32((self.k if x is None else x)[self.table[i, p // self.page], :, p % self.page]).astype(np.float64)

    def attend(self):
        """(output, weighted mean of |v|) in f64, [n, n_q, hd]."""
        out, size = np.zeros((self.n, self.n_q, self.hd)), np.zeros((self.n, self.n_q, self.hd))
        each = self.n_q // self.n_kv
        for i in range(self.n_seqs):
            if not self.rows[i]:
                continue
            k, v = self.keys(i), self.keys(i, self.v)
            for j, p in enumerate(self.positions(i)):
                row = self.indptr[i] + j
                q = emx.f32(self.q[row]).astype(np.float64).reshape(self.n_kv, each, self.hd)
                s = np.einsum("hgd,shd->hgs", q, k[:p + 1]) * self.scale
                w = np.exp(s - s.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                out[row] = np.einsum("hgs,shd->hgd", w, v[:p + 1]).reshape(self.n_q, self.hd)
                size[row] = np.einsum("hgs,shd->hgd", w, np.abs(v[:p + 1])).reshape(self.n_q, self.hd)
        return out, size

    def append(self, wq=None, wk=None, eps=1e-6, theta=1e6):
        """(q [n, n_q, hd], k, v [n, n_kv, hd]) in f64."""
        x = emx.f32(self.qkv[:self.n]).astype(np.float64).reshape(self.n, -1, self.hd)
        q, k, v = np.split(x, [self.n_q, self.n_q + self.n_kv], axis=1)
        pos = np.concatenate([self.positions(i) for i in range(self.n_seqs)]).astype(np.float64) if self.n else np.zeros(0)
        half = self.hd // 2

        def head(t, w):
            if w is not None:
                t = t / np.sqrt((t * t).mean(-1, keepdims=True) + eps) * emx.f32(w).astype(np.float64)
            if theta:
                a = pos[:, None, None] * theta ** (-np.arange(half) / half)
                c, s = np.cos(a), np.sin(a)
                t = np.concatenate([t[..., :half] * c - t[..., half:] * s, t[..., :half] * s + t[..., half:] * c], -1)
            return t

        return head(q, wq), head(k, wk), v


def verify(target, draft, tokens, uniforms, counts=None):
    """Acceptance and the next token by their definition, in f64; arrays as the operator takes them (floats)."""
    n, m1, _ = target.shape
    out, acc = np.full((n, m1), -1, np.int32), np.zeros(n, np.int32)
    for i in range(n):
        count = m1 - 1 if counts is None else min(int(counts[i]), m1 - 1)
        if count < 0:
            continue
        j = 0
        while j < count:
            x = tokens[i, j]
            if not 0 <= x < target.shape[2]:
                break
            q = 1.0 if draft is None else float(draft[i, j, x])
            if not float(uniforms[i, j]) * q < float(target[i, j, x]):
                break
            out[i, j] = x
            j += 1
        acc[i] = j

        def mass(r):
            r = r.astype(np.float64)
            return np.where(np.isfinite(r) & (r > 0), r, 0.0)

        p = mass(target[i, j])
        if j < count:
            q = np.zeros_like(p)
            if draft is None:
                if 0 <= tokens[i, j] < p.size:
                    q[tokens[i, j]] = 1
            else:
                q = mass(draft[i, j])
            rest = np.maximum(p - q, 0)
            if rest.sum() > 0:
                p = rest
        c = np.cumsum(p)
        if c[-1] > 0:
            hit = np.nonzero(c > float(uniforms[i, -1]) * c[-1])[0]
            out[i, j] = hit[0] if hit.size else np.nonzero(p)[0][-1]
    return out, acc
