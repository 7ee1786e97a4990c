"""Serving a batch from a paged bf16 cache, and scoring what it answers: prompts of different lengths written into pages and
attended in one launch, the attention of new tokens over the pages (with the weights each cached token has received), the
eviction of the least attended ones, and log probabilities of given tokens.

Head layouts are those of the Llama shapes the repository serves (1B, 8B, 70B heads) and two generic ones; contexts, vocabularies
and batches are those of its decoding and generation paths.
"""

import math
import os
import sys

import torch

own = False  # False: the plain forms below; True: the framework's kernels

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F32, F64, I32, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# q heads, kv heads, head_dim
SHAPES = {"1b": (32, 8, 64), "8b": (32, 8, 128), "70b": (64, 8, 128), "thirds": (15, 5, 128), "single": (16, 16, 64)}
PAGE = 64


# ------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # One long prompt into an empty cache.
        dict(name="prompt_8b", kind="prompt", shape="8b", seqs=1, rows=4096, past=0),
        # A batch of prompts of different lengths, packed.
        dict(name="prompts_8b", kind="prompt", shape="8b", seqs=16, rows=1500, past=0),
        # Further pieces of long prompts, behind what is cached of them.
        dict(name="pieces_70b", kind="prompt", shape="70b", seqs=3, rows=511, past=6000),
        # Short questions to the small model: latency.
        dict(name="prompts_1b", kind="prompt", shape="1b", seqs=5, rows=70, past=0),
        # One autoregressive token of the small model: latency.
        dict(name="step_1b", kind="step", shape="1b", seqs=1, rows=1, context=512, idle=0, weights=False),
        # A decode step of a batch of sequences of different lengths, some places of it idle.
        dict(name="step_batch_8b", kind="step", shape="8b", seqs=32, rows=1, context=8192, idle=3, weights=False),
        # One token of one very long document.
        dict(name="step_long_8b", kind="step", shape="8b", seqs=1, rows=1, context=131000, idle=0, weights=False),
        # A batch's step that keeps count of the weight each cached token receives; heads in threes.
        dict(name="step_weights", kind="step", shape="thirds", seqs=24, rows=1, context=4000, idle=0, weights=True),
        # The last rows of each prompt weigh its cache before some of it is dropped.
        dict(name="window_8b", kind="step", shape="8b", seqs=6, rows=16, context=4001, idle=0, weights=True),
        # The caches of a batch cut to a quarter, two layers.
        dict(name="evict_8b", kind="evict", shape="8b", layers=2, seqs=16, context=4096, keep=1024, recent=256, first=4),
        # What a server returns beside each token: one decode step of a batch.
        dict(name="logprobs_step", kind="logprobs", vocab=128256, rows=25, dtype="bf16", top=5),
        # A document scored: every row of it, odd row length.
        dict(name="logprobs_document", kind="logprobs", vocab=50257, rows=1800, dtype="fp32", top=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "step", "step", "step", "evict", "logprobs", "logprobs"])
    if kind == "logprobs":
        vocab = rng.choice([32000, 128256, rng.randint(1000, 150000)])
        dtype = rng.choice(sorted(TYPES))
        most = 90_000_000 * (4 if dtype == "fp32" else 8) // 4  # as many bytes as the largest listed one
        return dict(kind=kind, vocab=vocab, rows=_log(rng, 1, min(4096, most // vocab)), dtype=dtype,
                    top=rng.choice([0, 1, 5, rng.randint(2, 20)]))
    shape = rng.choice(["1b", "8b", "8b", "70b", "thirds", "single"])
    wide = 2 if shape == "70b" else 1
    if kind == "prompt":
        seqs = _log(rng, 1, 32)
        past = rng.choice([0, 0, _log(rng, 1, 8000)])
        rows = _log(rng, 1, 4096)
        while seqs * rows * (past + rows / 2) * wide > 4096 * 4096 / 2:
            rows = max(1, rows * 3 // 4)
            past, seqs = (past, seqs) if rows > 1 else (past // 2, seqs)
        return dict(kind=kind, shape=shape, seqs=seqs, rows=rows, past=past)
    if kind == "evict":
        seqs, context = _log(rng, 1, 16 // wide), _log(rng, 64, 4096)
        keep = rng.randint(min(16, context), context)
        recent = rng.randint(0, keep // 2)
        return dict(kind=kind, shape=shape, layers=2, seqs=seqs, context=context, keep=keep, recent=recent,
                    first=min(rng.choice([0, 1, 4]), keep - recent))
    weights = rng.random() < 0.4
    if rng.random() < 0.3:  # one long sequence
        return dict(kind=kind, shape=shape, seqs=1, rows=rng.choice([1, 1, rng.randint(2, 8)]), idle=0, weights=weights,
                    context=_log(rng, 2000, 60000))
    seqs = _log(rng, 1, 48)
    return dict(kind=kind, shape=shape, seqs=seqs, rows=rng.choice([1, 1, rng.randint(2, 16)]),
                context=_log(rng, 16, min(8192, 200000 // seqs)), idle=rng.randint(0, seqs // 4), weights=weights)


# ------------------------------------------------------------------------------------------------- inputs
def _spread(s, lo, hi):
    """A value in [lo, hi] for sequence s: the first has hi, the others are spread evenly over the range."""
    return hi if s == 0 else lo + int((hi - lo + 1) * (s * 0.6180339887 % 1.0))


def _sizes(case):
    """(new rows, cached slots before them or in all, rows kept) of every sequence."""
    S = range(case["seqs"])
    if case["kind"] == "prompt":
        rows = [_spread(s, max(1, case["rows"] // 8), case["rows"]) for s in S]
        return rows, [_spread(s + 2 if s else 0, 0, case["past"]) for s in S], None
    ctx = case["context"]
    if case["kind"] == "evict":
        lens = [_spread(s, max(1, ctx // 4), ctx) for s in S]
        if len(lens) > 2:
            lens[2] = max(1, min(ctx, case["keep"]) // 2)  # one that keeps everything
        return None, lens, [min(n, case["keep"]) for n in lens]
    n, idle = case["rows"], set(range(1, 1 + 2 * case["idle"], 2)) if case["idle"] else set()
    lens = [0 if s in idle else _spread(s, max(1, ctx // 2), ctx) for s in S]
    # between half the rows and all of them; an idle place has one row that attends nothing
    return [1 if s in idle else min(n - s * 5 % (n // 2 + 1), max(1, lens[s])) for s in S], lens, None


class _Rand:
    """Tensors of one case, each from its own seeded generator on the GPU; orders of pages from ``host``."""

    def __init__(self, seed):
        self.seed, self.n = seed, 0
        self.host = torch.Generator().manual_seed(seed * 6151 + 29)

    def gen(self):
        self.n += 1
        return torch.Generator(device="cuda").manual_seed(self.seed * 2003 + self.n)

    def normal(self, *size, dtype=BF16):
        return torch.randn(*size, generator=self.gen(), device="cuda", dtype=dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.host)


def _i32(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def _sums(x):
    return [sum(x[:i]) for i in range(len(x) + 1)]


def _projected(r, rows, heads, kv, hd):
    """q, k, v of a fused projection's output rows: column ranges of one matrix, some channels larger as in trained models."""
    x = r.normal(rows, (heads + 2 * kv) * hd)
    gain = torch.ones(hd, device="cuda")
    gain[::17] = 4.0
    x = (x.view(rows, -1, hd) * gain.to(BF16)).view(rows, -1)
    return x[:, :heads * hd], x[:, heads * hd:(heads + kv) * hd], x[:, (heads + kv) * hd:]


def _cached(r, lens, kv, hd):
    """K and V rows of every sequence, one behind the other: [sum of lens, kv * hd]."""
    k, v = r.normal(sum(lens), kv, hd), r.normal(sum(lens), kv, hd)
    k[..., ::17] *= 4.0
    return k.flatten(1), v.flatten(1)


def _package():
    pkg = os.path.join(REPO, "subnetwork-speculative-decoding_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)


def _tables(r, sets):
    """Page tables of several sets of sequences (their lengths), pages handed out in no order: (tables, pages in all)."""
    counts = [[(n + PAGE - 1) // PAGE for n in lens] for lens in sets]
    total = sum(map(sum, counts))
    ids, at, tables = r.order(max(total, 1)).tolist(), 0, []
    for cs in counts:
        rows = []
        for c in cs:
            rows.append(ids[at:at + c] + [0] * (max(max(cs), 1) - c))
            at += c
        tables.append(_i32(rows))
    return tables, max(total, 1)


def prepare(case, seed):
    r = _Rand(seed)
    st = {"case": case}
    if case["kind"] == "logprobs":
        return _prepare_logprobs(case, r, st)
    heads, kv, hd = SHAPES[case["shape"]]
    S = case["seqs"]
    if case["kind"] == "evict":
        return _prepare_evict(case, r, st, kv, hd)
    if case["kind"] == "prompt":
        rows, past, _ = _sizes(case)
        st["q"], st["k"], st["v"] = _projected(r, sum(rows), heads, kv, hd)
        lens = [a + b for a, b in zip(rows, past)]
        old = _cached(r, past, kv, hd)
        st["past"] = past
    else:
        rows, lens, _ = _sizes(case)
        st["q"] = r.normal(sum(rows), heads * hd) * 1.5
        old = _cached(r, lens, kv, hd)
        past = lens
        cap = (max(lens) + PAGE - 1) // PAGE * PAGE
        if case["weights"]:
            st["weights"] = torch.zeros(S, kv, cap, device="cuda")
    st["rows"], st["lens"] = rows, lens
    (table,), pages = _tables(r, [lens])
    lengths, begin = _i32(lens), _i32(_sums(rows))
    if own:
        _package()
        from ssd.engine.kv_cache import PagedBatch, PagedKVCache

        cache = st["cache"] = PagedKVCache(1, pages, kv, hd, "cuda")
        cache.write(0, *old, PagedBatch(table, _i32(past), _i32(_sums(past)), max(past)))
        st["batch"] = PagedBatch(table, lengths, begin, max(rows))
        st["l_max"] = max(lens)
        if case["kind"] == "step":
            st["ws"] = torch.empty(cache.attend_floats(sum(rows), heads, st["batch"], st["l_max"], case["weights"]),
                                   dtype=F32, device="cuda")
    else:
        st["old"], st["lengths"], st["begin"] = old, lengths, begin
    return st


def _prepare_evict(case, r, st, kv, hd):
    S = case["seqs"]
    _, lens, kept = _sizes(case)
    cap = (max(lens) + PAGE - 1) // PAGE * PAGE
    # accumulated weights: few large ones, many small, some never attended
    w = torch.exp(r.normal(case["layers"], S, kv, cap, dtype=F32) * 2.0 - 4.0)
    st["weights"] = torch.where(w < 0.004, torch.zeros_like(w), w)
    olds = [_cached(r, lens, kv, hd) for _ in range(case["layers"])]
    (table, new), pages = _tables(r, [lens, kept])
    st["lens"], st["lengths"] = lens, _i32(lens)
    at = torch.tensor([(s, j) for s in range(S) for j in range(kept[s])], device="cuda")
    st["row_seq"], st["row_at"] = at[:, 0].contiguous(), at[:, 1].contiguous()  # of each row that is read back
    if own:
        _package()
        from ssd.engine.kv_cache import PagedBatch, PagedKVCache

        cache = st["cache"] = PagedKVCache(case["layers"], pages, kv, hd, "cuda")
        whole = PagedBatch(table, st["lengths"], _i32(_sums(lens)), max(lens))
        for i, (k, v) in enumerate(olds):
            cache.write(i, k, v, whole)
        st["batch"] = whole
        st["after"] = PagedBatch(new, torch.zeros_like(st["lengths"]), _i32(_sums(kept)), max(kept))
    else:
        st["olds"] = olds
        st["start"] = torch.tensor(_sums(lens)[:-1], device="cuda")
    return st


def _prepare_logprobs(case, r, st):
    M, V = case["rows"], case["vocab"]
    x = r.normal(M, V, dtype=F32).mul_(3.0)
    u = torch.rand(M, V, generator=r.gen(), device="cuda")
    x.masked_fill_(u[:1] < 0.02, float("-inf"))  # columns that no answer may hold
    st["tokens"] = (x - torch.log(-torch.log(u.clamp(1e-7, 1 - 1e-7)))).argmax(1)  # drawn from the rows
    if M > 4:
        st["tokens"][M // 3] = -1  # a place without a token
    st["logits"] = x.to(TYPES[case["dtype"]])
    return st


# ------------------------------------------------------------------------------------------------- plain forms
def _plain_prompt(st, heads, kv, hd):
    """A product per sequence: a padded batch would cost the plain form more than the loop does."""
    out, rep = [], heads // kv
    a = b = 0
    for n, past in zip(st["rows"], st["past"]):
        k, v = (torch.cat([o[a:a + past], x[b:b + n]]).float().view(past + n, kv, hd).transpose(0, 1)
                for o, x in zip(st["old"], (st["k"], st["v"])))
        q = st["q"][b:b + n].float().view(n, kv, rep, hd).permute(1, 2, 0, 3).reshape(kv, rep * n, hd)
        score = torch.matmul(q, k.transpose(1, 2).contiguous()).view(kv, rep, n, past + n) * hd ** -0.5
        ahead = torch.arange(past + n, device="cuda") > torch.arange(past, past + n, device="cuda")[:, None]
        score.masked_fill_(ahead, float("-inf"))
        w = torch.exp(score - score.amax(-1, keepdim=True))
        o = torch.matmul(w.view(kv, rep * n, past + n), v.contiguous()).view(kv, rep, n, hd) / w.sum(-1, keepdim=True)
        out.append(o.permute(2, 0, 1, 3).reshape(n, heads * hd).to(BF16))
        a, b = a + past, b + n
    return torch.cat(out)


def _plain_step(st, heads, kv, hd):
    case, rep = st["case"], heads // kv
    S, R, L, M = case["seqs"], max(st["rows"]), max(st["lens"]), st["q"].shape[0]
    begin, lengths = st["begin"].long(), st["lengths"].long()
    here = torch.arange(L, device="cuda") < lengths[:, None]
    k, v = (torch.zeros(S, L, kv, hd, device="cuda") for _ in range(2))
    k[here], v[here] = (x.float().view(-1, kv, hd) for x in st["old"])
    k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    seq = torch.repeat_interleave(torch.arange(S, device="cuda"), begin.diff(), output_size=M)
    place = torch.arange(M, device="cuda") - begin[seq]
    q = torch.zeros(S, R, heads, hd, device="cuda")
    q[seq, place] = st["q"].float().view(M, heads, hd)
    q = q.view(S, R, kv, rep, hd).permute(0, 2, 1, 3, 4).reshape(S, kv, R * rep, hd)
    last = torch.full((S, R), -1, device="cuda")  # the last slot that a row attends; -1: none
    last[seq, place] = lengths[seq] - begin.diff()[seq] + place
    see = torch.arange(L, device="cuda") <= last[..., None]
    see = see[:, None, :, None].expand(S, kv, R, rep, L).reshape(S, kv, R * rep, L)
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(hd ** -0.5).masked_fill_(~see, float("-inf"))
    w = torch.exp(score - score.amax(-1, keepdim=True).clamp_min(-1e30))
    w = w / w.sum(-1, keepdim=True).clamp_min(1e-30)
    out = torch.matmul(w, v).view(S, kv, R, rep, hd).transpose(1, 2)[seq, place].reshape(M, heads * hd).to(BF16)
    if not case["weights"]:
        return out
    got = torch.zeros_like(st["weights"])
    got[..., :L] = w.sum(2)
    return out, got


def _rank_keys(x):
    """int64 keys [..., n] in the order of x, of equal values the lowest index first."""
    bits = x.float().add(0.0).view(I32).to(I64)  # -0 is 0
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF) - 1, bits)
    return (bits << 32) - torch.arange(x.shape[-1], device=x.device)


def _plain_evict(st, kv, hd):
    case, w = st["case"], st["weights"]
    keep, recent, first = case["keep"], case["recent"], case["first"]
    slot = torch.arange(w.shape[-1], device="cuda")
    n = st["lengths"].long()[:, None, None]
    # what must stay ranks first, what is not there last
    stay = (slot < first) | (slot >= n - recent)
    lead = torch.where(slot >= n, -1.0, torch.where(stay, float("inf"), w))
    width = min(keep, w.shape[-1])
    pick = _rank_keys(lead).topk(width, -1).indices
    have = torch.arange(width, device="cuda") < n
    kept = torch.where(have, pick, slot.numel()).sort(-1).values
    at = torch.where(have, kept, 0)
    weights = torch.zeros_like(w)
    weights[..., :width] = torch.where(have, w.gather(-1, at), 0.0)
    res = torch.full((*w.shape[:3], keep), -1, dtype=I32, device="cuda")
    res[..., :width] = torch.where(have, kept, -1).to(I32)
    out = [res, st["lengths"].clamp_max(keep), weights]
    s, j = st["row_seq"], st["row_at"]
    src = st["start"][s][None, :, None] + at[:, s, :, j].transpose(0, 1)  # [layers, rows, kv]
    head = torch.arange(kv, device="cuda")
    for i, kept_rows in enumerate(src):
        out += [x.view(-1, kv, hd)[kept_rows, head].flatten(1) for x in st["olds"][i]]
    return out


def _plain_logprobs(st):
    x, t, top = st["logits"].float(), st["tokens"], st["case"]["top"]
    there = t >= 0
    xt = x.gather(1, t.clamp_min(0)[:, None])
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    z = e.sum(1, dtype=F64)
    lse = torch.log(z)
    ent = lse - torch.where(e > 0, e * d, 0.0).sum(1, dtype=F64) / z
    logprob = torch.where(there, (xt - m)[:, 0].double() - lse, 0.0)
    col = torch.arange(x.shape[1], device="cuda")
    rank = ((x > xt) | ((x == xt) & (col < t[:, None]))).sum(1)
    out = [logprob.to(F32), ent.to(F32), torch.where(there, rank, -1).to(I32)]
    if top:
        ids = _rank_keys(x).topk(top, 1).indices
        out += [ids.to(I32), (d.gather(1, ids).double() - lse[:, None]).to(F32)]
    return out


def run(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "logprobs":
        if not own:
            return _plain_logprobs(st)
        from ssd.engine.scoring import token_logprobs

        got = token_logprobs(st["logits"], st["tokens"], top=case["top"])
        out = [got.logprobs, got.entropy, got.rank]
        return out + [got.top_ids, got.top_logprobs] if case["top"] else out
    heads, kv, hd = SHAPES[case["shape"]]
    if kind == "prompt":
        if not own:
            return _plain_prompt(st, heads, kv, hd)
        st["cache"].write(0, st["k"], st["v"], st["batch"])
        return st["cache"].attend_prompt(0, st["q"], st["batch"], st["l_max"])
    if kind == "step":
        if not own:
            return _plain_step(st, heads, kv, hd)
        if not case["weights"]:
            return st["cache"].attend(0, st["q"], st["batch"], st["l_max"], ws=st["ws"])
        out = st["cache"].attend(0, st["q"], st["batch"], st["l_max"], ws=st["ws"], weights=st["weights"], decay=0.0)
        return out, st["weights"]
    if not own:
        return _plain_evict(st, kv, hd)
    kept, weights = st["cache"].evict(st["batch"], st["after"], st["weights"], case["keep"], case["recent"], case["first"])
    out = [kept, st["after"].lengths, weights]
    for i in range(case["layers"]):
        out += st["cache"].read(i, st["after"], st["row_seq"].numel())
    return out


# ------------------------------------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        M, V = case["rows"], case["vocab"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": M * (V * size + 20 + 8 * case["top"]), "flops": 5 * M * V}
    heads, kv, hd = SHAPES[case["shape"]]
    row = 2 * kv * hd * 2  # K and V of one slot
    rows, lens, kept = _sizes(case)
    if kind == "prompt":  # new K and V read and written into the cache, cached ones read
        pairs = sum(n * past + n * (n + 1) // 2 for n, past in zip(rows, lens))
        return {"bytes": sum(rows) * (4 * heads * hd + 2 * row) + sum(lens) * row, "flops": 4 * heads * hd * pairs}
    if kind == "step":
        pairs = sum(n * length - n * (n - 1) // 2 for n, length in zip(rows, lens) if length)
        count = 4 * kv * sum(lens) if case["weights"] else 0
        return {"bytes": row * sum(lens) + 4 * heads * hd * sum(rows) + count, "flops": 4 * heads * hd * pairs}
    # weights read; kept rows read, written, and read back into plain rows; kept weights and slots written
    keys = sum(lens)
    return {"bytes": case["layers"] * (4 * kv * keys + sum(kept) * (4 * row + 8 * kv)), "flops": case["layers"] * kv * keys}


# ------------------------------------------------------------------------------------------------- definitions in 64 bits
def _exact_rows(q, k, v, last):
    """softmax(q k / sqrt(hd)) v and the weights: q [n, kv, rep, hd], k, v [L, kv, hd], row i sees slots [0, last[i]]."""
    n, kv, rep, hd = q.shape
    outs, sums = [], []
    for h in range(kv):
        kk, vv = k[:, h].double(), v[:, h].double()
        s = (q[:, h].double().reshape(n * rep, hd) @ kk.T.contiguous()).view(n, rep, -1) / math.sqrt(hd)
        hidden = torch.arange(kk.shape[0], device="cuda")[None, None, :] > last[:, None, None]
        w = torch.softmax(s.masked_fill(hidden, -1e300), -1).masked_fill(hidden, 0.0)
        outs.append((w.view(n * rep, -1) @ vv).view(n, rep, hd))
        sums.append(w.sum((0, 1)))
    return torch.stack(outs, 1), torch.stack(sums)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    kind = case["kind"]
    if kind == "logprobs":
        return _exact_logprobs(st)
    heads, kv, hd = SHAPES[case["shape"]]
    if kind == "evict":
        return _exact_evict(st, kv, hd)
    out = torch.zeros(sum(st["rows"]), heads, hd, dtype=F64, device="cuda")
    total = torch.zeros(st["weights"].shape, dtype=F64, device="cuda") if case.get("weights") else None
    a = b = 0
    for s, (n, length) in enumerate(zip(st["rows"], st["lens"])):
        cached = st["past"][s] if kind == "prompt" else length
        k, v = (x[a:a + cached].view(-1, kv, hd) for x in st["old"])
        if kind == "prompt":
            k, v = (torch.cat([o, st[x][b:b + n].reshape(n, kv, hd)]) for o, x in ((k, "k"), (v, "v")))
        for i in range(0, n if length else 0, 1024):
            j = min(n, i + 1024)
            last = torch.arange(length - n + i, length - n + j, device="cuda")
            q = st["q"][b + i:b + j].reshape(j - i, kv, heads // kv, hd)
            o, w = _exact_rows(q, k, v, last)
            out[b + i:b + j] = o.reshape(j - i, heads, hd)
            if total is not None:
                total[s, :, :length] += w
        a, b = a + cached, b + n
    out = out.flatten(1)
    return out if total is None else (out, total)


def _exact_evict(st, kv, hd):
    case = st["case"]
    keep, recent, first = case["keep"], case["recent"], case["first"]
    w = st["weights"].double().cpu()
    kept = torch.full((*w.shape[:3], keep), -1, dtype=I32)
    weights = torch.zeros_like(w)
    for i in range(w.shape[0]):
        for s, n in enumerate(st["lens"]):
            for h in range(kv):
                if n <= keep:
                    take = list(range(n))
                else:
                    mid = torch.arange(first, n - recent)
                    best = torch.sort(w[i, s, h, first:n - recent], stable=True, descending=True).indices
                    take = sorted(list(range(first)) + mid[best[:keep - first - recent]].tolist() + list(range(n - recent, n)))
                kept[i, s, h, :len(take)] = torch.tensor(take, dtype=I32)
                weights[i, s, h, :len(take)] = w[i, s, h, take]
    out = [kept.cuda(), _i32([min(n, keep) for n in st["lens"]]), weights.cuda()]
    for i, (k, v) in enumerate(st["olds"]):
        for x in (k, v):
            parts, a = [], 0
            for s, n in enumerate(st["lens"]):
                at = kept[i, s, :, :min(n, keep)].long().cuda()  # [kv, kept]
                rows = x[a:a + n].view(n, kv, hd).double().transpose(0, 1)
                parts.append(torch.stack([rows[h][at[h]] for h in range(kv)], 1).flatten(1))
                a += n
            out.append(torch.cat(parts))
    return out


def _exact_logprobs(st):
    top, t = st["case"]["top"], st["tokens"]
    parts = []
    for i in range(0, t.numel(), 128):
        x = st["logits"][i:i + 128].double()
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        order = torch.sort(x, stable=True, dim=1, descending=True).indices
        tok = t[i:i + 128]
        here = tok >= 0
        mine = torch.where(here, lp.gather(1, tok.clamp_min(0)[:, None])[:, 0], 0.0)
        ent = -torch.xlogy(torch.exp(lp), torch.exp(lp)).sum(1)
        rank = (order == tok[:, None]).long().argmax(1)
        ids = order[:, :top]
        parts.append([mine, ent, torch.where(here, rank, -1).to(I32)] + ([ids.to(I32), lp.gather(1, ids)] if top else []))
    return [torch.cat(p) for p in zip(*parts)]
