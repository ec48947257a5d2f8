"""The operators of one step of batched, speculative serving over a paged K/V cache, as cases to be timed and compared:

append  the rows of a batch (a token each) leave the q|k|v projection: q and k are normalised per head, rotated to
        their positions, k and v go to their pages of the cache (emx.Ctx.paged_append);
attend  every new row attends the cache of its sequence, whose first `shared` positions are pages that all
        sequences have in common (emx.Ctx.sdpa_paged);
verify  the drafted tokens of each sequence are accepted or replaced against the target's probabilities, from given
        random numbers (emx.Ctx.verify_draft).

Where `own` is false, run() computes them in elementary torch operations in 32 bits (angles, sums over a vocabulary
and comparisons at a border in 64), rounded once at the end; where it is true, run() calls the framework."""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
THETA = 1e6


# --------------------------------------------------------------------------------------------------------- the cases
def _attn(name, op, seqs, rows, past, shared, heads, page, hd=128, idle=0, pad=0, norm=True):
    """A batch of `seqs` sequences with rows[0]..rows[1] new rows each, past[0]..past[1] positions of their own before
    those, `shared` common ones before these; `idle` empty slots and `pad` rows behind the last sequence."""
    return {"name": name, "op": op, "seqs": seqs, "rows_min": rows[0], "rows_max": rows[1], "past_min": past[0],
            "past_max": past[1], "shared": shared, "n_q": heads[0], "n_kv": heads[1], "page": page, "hd": hd,
            "idle": idle, "pad": pad, "norm": norm}


def _verify(name, seqs, drafts, vocab, kind, draft_probs=True, ragged=False, near=0.5):
    """`near`: how far the draft's logits are from the target's (their differences' standard deviation)."""
    return {"name": name, "op": "verify", "seqs": seqs, "drafts": drafts, "vocab": vocab, "kind": kind,
            "draft_probs": draft_probs, "ragged": ragged, "near": near}


def listed():
    return [
        # one sequence decodes: a single row, nothing but latency
        _attn("append 1 row", "append", 1, (1, 1), (131, 131), 0, (16, 8), 16),
        # a decode batch of static size, eight of its slots unused, sequences of all ages
        _attn("append 64 rows", "append", 64, (1, 1), (1, 4000), 4096, (32, 4), 16, idle=8, pad=8),
        # prompts of several users prefilled together, ragged, with rows to spare behind them
        _attn("append prompts", "append", 6, (64, 2666), (0, 500), 0, (16, 8), 64, pad=33),
        # one short sequence decodes: latency again
        _attn("attend 1 at 132", "attend", 1, (1, 1), (131, 131), 0, (16, 8), 16),
        # a decode batch that shares nothing, 17 to 8192 positions
        _attn("attend 32 ragged", "attend", 32, (1, 1), (16, 8191), 0, (32, 4), 16, idle=2),
        # 64 users of one long document
        _attn("attend 64 on 32768", "attend", 64, (1, 1), (0, 1023), 32768, (16, 8), 64),
        # a verification step: one to eight drafted rows a sequence, a long instruction before all of them
        _attn("attend 24 drafts on 8192", "attend", 24, (2, 9), (5, 700), 8192, (64, 8), 16, pad=3),
        # many users of one system prompt
        _attn("attend 128 on 16384", "attend", 128, (1, 1), (1, 520), 16384, (32, 4), 32),
        # one sequence's drafts
        _verify("verify 1 x 4", 1, 4, 151936, "float32"),
        # a full batch
        _verify("verify 64 x 4", 64, 4, 151936, "float32"),
        # bf16 probabilities (what the framework's softmax gives), a smaller vocabulary, ragged drafts
        _verify("verify 48 x 7 ragged", 48, 7, 32000, "bfloat16", ragged=True),
        # drafts without probabilities (copied from the prompt), which count as certain
        _verify("verify 16 x 3 copied", 16, 3, 151936, "bfloat16", draft_probs=False, near=2.0),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "attend", "attend", "verify"])
    if op == "verify":
        seqs, drafts = log(1, 96), rng.randint(1, 8)
        vocab = log(1000, 152000)
        while seqs * (drafts + 1) * vocab > 48_000_000:
            seqs = max(1, seqs // 2)
        c = _verify("", seqs, drafts, vocab, rng.choice(["float32", "float32", "bfloat16"]), rng.random() < 0.75,
                    rng.random() < 0.5, round(rng.uniform(0.1, 2.0), 2))
    else:
        heads = rng.choice([(16, 8), (32, 4), (64, 8), (8, 2), (8, 8), (12, 4), (5, 1)])
        page = rng.choice([8, 16, 16, 24, 32, 64, 128])
        hd = rng.choice([128, 128, 128, 64])
        if op == "append":
            seqs = log(1, 128)
            most = max(1, 7000 // seqs)
            rows = rng.choice([(1, 1), (1, log(1, most)), (0, log(1, most))])
            past = (0, log(1, 4096))
            shared = 0
        else:
            seqs = log(1, 128)
            rows = rng.choice([(1, 1), (1, 1), (1, log(1, 8)), (0, log(1, 32))])
            if seqs * rows[1] > 512:
                rows = (1, 1)
            past = (0, log(1, min(8192, max(64, 200000 // seqs))))
            shared = rng.choice([0, 1, 1]) * page * max(1, log(256, 24000) // page)
        c = _attn("", op, seqs, rows, past, shared, heads, page, hd, rng.choice([0, 0, 1, 5]), rng.choice([0, 0, 1, 17]),
                  rng.random() < 0.8)
    del c["name"]
    return c


def _batch(case):
    """New rows, positions of their own (new rows among them) of each sequence, before the seed puts them in order."""
    n = case["seqs"]

    def spread(lo, hi):
        return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]

    rows, past = spread(case["rows_min"], case["rows_max"]), spread(case["past_min"], case["past_max"])
    return rows, [r + p for r, p in zip(rows, past)]


def work(case):
    if case["op"] == "verify":
        size = 4 if case["kind"] == "float32" else 2
        # the row that the last token is drawn from, of the target and (where the draft was refused) of the draft
        each = case["seqs"] * case["vocab"]
        return {"bytes": each * size * (2 if case["draft_probs"] else 1), "flops": 4 * each}
    rows, lens = _batch(case)
    n, hd, n_q, n_kv = sum(rows), case["hd"], case["n_q"], case["n_kv"]
    if case["op"] == "append":
        each = n * (n_q + 2 * n_kv) * hd
        return {"bytes": 4 * each, "flops": 8 * each}
    keys = case["shared"] + sum(t for t, r in zip(lens, rows) if r)
    pairs = sum(r * (case["shared"] + t) - r * (r - 1) // 2 for r, t in zip(rows, lens))
    return {"bytes": 4 * keys * n_kv * hd + 4 * n * n_q * hd, "flops": 4 * hd * n_q * pairs}


# -------------------------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "verify":
        return _prepare_verify(case, g)
    rows, lens = _batch(case)
    n_seqs = case["seqs"] + case["idle"]
    order = torch.randperm(n_seqs, generator=g, device="cuda").cpu().tolist()
    rows, lens = rows + [0] * case["idle"], [t + case["shared"] for t in lens] + [0] * case["idle"]
    rows, lens = [rows[i] for i in order], [lens[i] for i in order]
    n, page, hd, n_q, n_kv = sum(rows), case["page"], case["hd"], case["n_q"], case["n_kv"]
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    i32 = {"dtype": torch.int32, "device": "cuda"}
    n_shared = case["shared"] // page
    max_pages = max(1, max(-(-t // page) for t in lens))
    each = [max(0, -(-t // page) - n_shared) for t in lens]
    n_pages = n_shared + sum(each) + 3  # a few belong to nobody
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.full((n_seqs, max_pages), -1, dtype=torch.int32)  # -1: no page there
    at = n_shared
    for i, k in enumerate(each):
        if lens[i]:
            table[i, :n_shared] = perm[:n_shared]
        table[i, n_shared:n_shared + k] = perm[at:at + k]
        at += k
    n_rows = n + case["pad"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)

    s = {"op": case["op"], "n_seqs": n_seqs, "n_rows": n_rows, "n": n, "most": max(rows), "longest": max(lens),
         "max_pages": max_pages, "n_pages": n_pages, "page": page, "hd": hd, "n_q": n_q, "n_kv": n_kv,
         "shared": case["shared"], "indptr": torch.tensor(starts, **i32), "lengths": torch.tensor(lens, **i32),
         "table": table.cuda(), "shared_pages": perm[:max(1, n_shared)].cuda(),
         "k": normal(n_pages, n_kv, page, hd), "v": normal(n_pages, n_kv, page, hd),
         "out": torch.zeros(n_rows, n_q, hd, dtype=torch.bfloat16, device="cuda")}
    if case["op"] == "append":
        s["qkv"] = normal(n_rows, (n_q + 2 * n_kv) * hd)
        s["q_norm"] = (1 + 0.1 * normal(hd).float()).bfloat16() if case["norm"] else None
        s["k_norm"] = (1 + 0.1 * normal(hd).float()).bfloat16() if case["norm"] else None
    else:
        s["q"] = normal(n_rows, n_q, hd)  # normalised heads have about this length
        s["scale"] = hd ** -0.5
    return s


def _prepare_verify(case, g):
    n, m, v = case["seqs"], case["drafts"], case["vocab"]
    kind = torch.float32 if case["kind"] == "float32" else torch.bfloat16
    logits = 3 * torch.randn(n, m + 1, v, generator=g, device="cuda")
    target = torch.softmax(logits, -1)
    logits = logits[:, :m] + case["near"] * torch.randn(n, m, v, generator=g, device="cuda")
    draft = torch.softmax(logits, -1)
    tokens = torch.multinomial(draft.reshape(n * m, v), 1, generator=g).reshape(n, m)
    if not case["draft_probs"]:
        # a copied draft is often the likeliest token, and else any
        best = target[:, :m].argmax(-1)
        tokens = torch.where(torch.rand(n, m, generator=g, device="cuda") < 0.5, best, tokens)
    counts = None
    if case["ragged"]:
        counts = torch.randint(0, m + 1, (n,), generator=g, device="cuda").to(torch.int32)
    return {"op": "verify", "n_seqs": n, "drafts": m, "vocab": v, "target": target.to(kind).contiguous(),
            "draft": draft.to(kind).contiguous() if case["draft_probs"] else None,
            "tokens": tokens.to(torch.int32).contiguous(), "counts": counts,
            "uniforms": torch.rand(n, m + 1, generator=g, device="cuda"),
            "out": torch.zeros(n, m + 1, dtype=torch.int32, device="cuda"),
            "accepted": torch.zeros(n, dtype=torch.int32, device="cuda")}


# ---------------------------------------------------------------------------------------------------- the framework's
_ctx = {}


def _framework():
    """The package and the program's context on the current device and stream, where the inputs are made and the outputs
    used; made once for each."""
    at = torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream
    if at not in _ctx:
        if not _ctx:
            sys.path.insert(0, os.path.join(os.getcwd(), "engine-mlx_b200"))
        import emx

        _ctx[at] = emx, emx.Ctx(at[0], stream=at[1])
    return _ctx[at]


def _run_own(s):
    if "on" not in s:  # a program keeps its context, as it keeps to its stream
        s["on"] = _framework()
    emx, ctx = s["on"]
    if s["op"] == "verify":
        return ctx.verify_draft(s["target"], s["draft"], s["tokens"], s["uniforms"], s["n_seqs"], s["drafts"], s["vocab"],
                                dtype=emx.F32 if s["target"].dtype == torch.float32 else emx.BF16, counts=s["counts"],
                                out=s["out"], accepted=s["accepted"])
    if "kv" not in s:  # the descriptions of the cache and of the batch, which a program keeps beside their buffers
        s["kv"] = emx.PagedKV(s["k"], s["v"], s["n_pages"], s["page"], s["n_kv"], s["hd"])
        s["batch"] = emx.PagedBatch(s["indptr"], s["lengths"], s["table"], s["n_seqs"], s["n_rows"], s["max_pages"])
    if s["op"] == "append":
        ctx.paged_append(s["qkv"], s["kv"], s["batch"], s["n_q"], s["q_norm"], s["k_norm"], EPS, THETA, out=s["out"])
        return s["out"], s["k"], s["v"]
    return ctx.sdpa_paged(s["q"], s["kv"], s["batch"], s["n_q"], s["scale"], s["shared"], s["shared_pages"], out=s["out"])


# ----------------------------------------------------------------------------------------------------- the plain forms
def run(state):
    if own:
        return _run_own(state)
    return {"append": _append, "attend": _attend, "verify": _verify_plain}[state["op"]](state)


def _rows_of(s):
    """Sequence, place in it and position of each new row."""
    r = torch.arange(s["n"], device="cuda")
    seq = torch.searchsorted(s["indptr"][1:].long(), r, right=True)
    j = r - s["indptr"].long()[seq]
    new = s["indptr"].long()[seq + 1] - s["indptr"].long()[seq]
    return seq, j, s["lengths"].long()[seq] - new + j


def _append(s):
    n, n_q, n_kv, hd, page = s["n"], s["n_q"], s["n_kv"], s["hd"], s["page"]
    seq, _, pos = _rows_of(s)
    x = s["qkv"][:n].float().view(n, n_q + 2 * n_kv, hd)
    q, k, v = x[:, :n_q], x[:, n_q:n_q + n_kv], x[:, n_q + n_kv:]
    if s["q_norm"] is not None:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * s["q_norm"].float()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * s["k_norm"].float()
    half = hd // 2
    i = torch.arange(half, device="cuda", dtype=torch.float64)
    angle = pos.double()[:, None] * THETA ** (-i / half)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotate(t):
        a, b = t[..., :half], t[..., half:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    s["out"][:n] = rotate(q).bfloat16()
    where = s["table"].long()[seq, pos // page], slice(None), pos % page
    s["k"][where] = rotate(k).bfloat16()
    s["v"][where] = v.bfloat16()
    return s["out"], s["k"], s["v"]


def _attend(s):
    n, n_q, n_kv, hd, page, shared = s["n"], s["n_q"], s["n_kv"], s["hd"], s["page"], s["shared"]
    each = n_q // n_kv
    seq, j, pos = _rows_of(s)
    q = s["q"][:n].float().view(n, n_kv, each, hd) * s["scale"]
    # the sequences' own keys, as wide as the longest; the rows likewise
    wide = max(1, s["longest"] - shared)
    at = shared + torch.arange(wide, device="cuda")
    pages = s["table"].long()[:, (at // page).clamp(max=s["max_pages"] - 1)].clamp(min=0)
    slot = (at % page)[None].expand_as(pages)
    k = s["k"][pages, :, slot].float()  # [sequences, wide, n_kv, hd]
    v = s["v"][pages, :, slot].float()
    padded = torch.zeros(s["n_seqs"], max(1, s["most"]), n_kv, each, hd, device="cuda")
    padded[seq, j] = q
    at_rows = torch.full((s["n_seqs"], max(1, s["most"])), -1, dtype=torch.long, device="cuda")
    at_rows[seq, j] = pos
    x = torch.einsum("bjhgd,bshd->bhjgs", padded, k)
    x = x.masked_fill((at[None, None] > at_rows[:, :, None])[:, None, :, None], -math.inf)
    x = x.permute(0, 2, 1, 3, 4)[seq, j]  # [n, n_kv, each, wide]
    if shared:
        first = s["shared_pages"].long()
        ks = s["k"][first].permute(1, 0, 2, 3).reshape(n_kv, shared, hd).float()
        vs = s["v"][first].permute(1, 0, 2, 3).reshape(n_kv, shared, hd).float()
        y = torch.matmul(q.permute(1, 0, 2, 3).reshape(n_kv, n * each, hd), ks.transpose(1, 2))
        y = y.view(n_kv, n, each, shared)
        y = y.masked_fill((torch.arange(shared, device="cuda") > pos[:, None])[None, :, None], -math.inf)
        y = y.permute(1, 0, 2, 3)
    else:
        y = x[..., :0]
    top = torch.maximum(x.amax(-1), y.amax(-1) if shared else x.amax(-1))
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))[..., None]
    x, y = torch.exp(x - top), torch.exp(y - top)
    total = (x.sum(-1) + y.sum(-1))[..., None]
    padded = torch.zeros(s["n_seqs"], max(1, s["most"]), n_kv, each, wide, device="cuda")
    padded[seq, j] = x
    o = torch.einsum("bjhgs,bshd->bjhgd", padded, v)[seq, j]
    if shared:
        o = o + torch.matmul(y.permute(1, 0, 2, 3).reshape(n_kv, n * each, shared), vs).view(n_kv, n, each, hd).permute(1, 0, 2, 3)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    s["out"][:n] = o.reshape(n, n_q, hd).bfloat16()
    return s["out"]


def _verify_plain(s):
    n, m, v = s["n_seqs"], s["drafts"], s["vocab"]
    counts = s["counts"].long() if s["counts"] is not None else torch.full((n,), m, device="cuda")
    tokens = s["tokens"].long()
    p = s["target"][:, :m].gather(-1, tokens[..., None])[..., 0].double()
    q = torch.ones_like(p) if s["draft"] is None else s["draft"].gather(-1, tokens[..., None])[..., 0].double()
    j = torch.arange(m, device="cuda")
    fine = (s["uniforms"][:, :m].double() * q < p) & (j < counts[:, None])
    accepted = fine.long().cumprod(-1).sum(-1)
    refused = accepted < counts
    i, at = torch.arange(n, device="cuda"), accepted.clamp(max=max(0, m - 1))
    row = s["target"][i, accepted].double()
    if s["draft"] is None:
        other = torch.zeros_like(row).scatter_(1, tokens[i, at][:, None], 1.0)
    else:
        other = s["draft"][i, at].double()
    rest = torch.where(refused[:, None], (row - other).clamp(min=0), row)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, row)
    total = rest.cumsum(-1)
    last = torch.searchsorted(total, (s["uniforms"][:, m].double() * total[:, -1])[:, None], right=True)[:, 0]
    j = torch.arange(m + 1, device="cuda")
    out = torch.where(j < accepted[:, None], torch.nn.functional.pad(tokens, (0, 1)), -1)
    out = torch.where(j == accepted[:, None], last[:, None], out)
    s["out"].copy_(out)
    s["accepted"].copy_(accepted)
    return s["out"], s["accepted"]


# -------------------------------------------------------------------------------------------------- in 64 bits, apart
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "verify":
        return _exact_verify(s)
    starts, lens, table = s["indptr"].tolist(), s["lengths"].tolist(), s["table"].tolist()
    hd, page, n_q, n_kv = s["hd"], s["page"], s["n_q"], s["n_kv"]
    each = n_q // n_kv
    out = torch.zeros(s["n_rows"], n_q, hd, dtype=torch.float64, device="cuda")
    kc, vc = s["k"].double(), s["v"].double()
    for i, (a, b, length) in enumerate(zip(starts, starts[1:], lens)):
        if a == b:
            continue
        pos = torch.arange(length - (b - a), length, device="cuda")
        pages = torch.tensor(table[i], device="cuda")
        if s["op"] == "append":
            x = s["qkv"][a:b].double().reshape(b - a, -1, hd)
            parts = []
            for part, w in ((x[:, :n_q], s["q_norm"]), (x[:, n_q:n_q + n_kv], s["k_norm"])):
                if w is not None:
                    part = part / (part.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
                z = torch.complex(part[..., :hd // 2], part[..., hd // 2:])
                turn = pos.double()[:, None] * torch.exp(torch.arange(hd // 2, device="cuda").double() * (-2 * math.log(THETA) / hd))
                z = z * torch.polar(torch.ones_like(turn), turn)[:, None]
                parts.append(torch.cat([z.real, z.imag], -1))
            out[a:b] = parts[0]
            kc[pages[pos // page], :, pos % page] = parts[1]
            vc[pages[pos // page], :, pos % page] = x[:, n_q + n_kv:]
        else:
            every = torch.arange(length, device="cuda")
            k = kc[pages[every // page], :, every % page]
            v = vc[pages[every // page], :, every % page]
            q = s["q"][a:b].double().view(b - a, n_kv, each, hd)
            x = torch.einsum("jhgd,shd->hgjs", q, k) * s["scale"]
            x = torch.where(every <= pos[:, None], x, -math.inf)
            out[a:b] = torch.einsum("hgjs,shd->jhgd", torch.softmax(x, -1), v).reshape(b - a, n_q, hd)
    return (out, kc, vc) if s["op"] == "append" else out


def _exact_verify(s):
    out = torch.full_like(s["out"], -1).cpu()
    accepted = torch.zeros_like(s["accepted"]).cpu()
    tokens, u = s["tokens"].tolist(), s["uniforms"].double().tolist()
    for i in range(s["n_seqs"]):
        count = s["drafts"] if s["counts"] is None else int(s["counts"][i])
        j = 0
        while j < count:
            t = tokens[i][j]
            if not u[i][j] * (1.0 if s["draft"] is None else float(s["draft"][i, j, t])) < float(s["target"][i, j, t]):
                break
            out[i, j] = t
            j += 1
        p = s["target"][i, j].double()
        if j < count:
            less = torch.zeros_like(p)
            if s["draft"] is None:
                less[tokens[i][j]] = 1.0
            else:
                less = s["draft"][i, j].double()
            rest = (p - less).clamp(min=0)
            p = rest if float(rest.sum()) > 0 else p
        c = torch.cumsum(p, 0)
        out[i, j] = int((c <= u[i][-1] * c[-1]).sum())
        accepted[i] = j
    return out, accepted
