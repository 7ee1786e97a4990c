"""The operators of a batched speculative round over an 8-bit KV cache, as a decoding program calls them: rotation and the
quantising cache write with its read-back, the commit of accepted slots, tree attention over the cache, and the verification
of drafted chains.

Sizes are those of the Llama shapes the repository serves (1B, 8B, 70B heads), its trees (24 nodes and the root),
contexts and vocabularies.
"""

import math
import os
import sys

import torch

own = False  # False: the plain forms below; True: the framework's kernels

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
# q heads, kv heads, head_dim
SHAPES = {"1b": (32, 8, 64), "8b": (32, 8, 128), "70b": (64, 8, 128)}
THETA = 500000.0
MAX_DEPTH = 32  # ancestor slots a row may name
SCALING = {
    "none": None,
    "linear": {"rope_type": "linear", "factor": 4.0},
    "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": 8192},
    "yarn": {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 8192},
}


# ------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # One decode step of a batch: a row of each of 32 sequences, rotated, quantised into its cache and read back.
        dict(name="write_step_8b", kind="write", shape="8b", seqs=32, rows=32, context=4096, rot=128, interleaved=False,
             scaling="llama3"),
        # A long prompt's rows entering one sequence's cache.
        dict(name="write_prompt_8b", kind="write", shape="8b", seqs=1, rows=4096, context=4096, rot=128,
             interleaved=False, scaling="none"),
        # A short prompt of odd length, interleaved rotation of half the head, positions interpolated.
        dict(name="write_partial_1b", kind="write", shape="1b", seqs=1, rows=301, context=1000, rot=32,
             interleaved=True, scaling="linear"),
        # The cache work of a verified batch of trees: two layers' rows written, the accepted ones moved, read back.
        dict(name="commit_8b", kind="commit", shape="8b", layers=2, seqs=16, rows=25, context=2048, keep=5),
        # One autoregressive token of the small model: latency.
        dict(name="attend_step_1b", kind="attend", shape="1b", seqs=1, rows=1, context=512, idle=0),
        # The verify rows of a 24-node tree, at an ordinary context and at a long one.
        dict(name="attend_tree_8b", kind="attend", shape="8b", seqs=1, rows=25, context=4096, idle=0),
        dict(name="attend_tree_70b_16k", kind="attend", shape="70b", seqs=1, rows=25, context=16384, idle=0),
        # A batch of sequences of different lengths: one row each, and a small tree each with some idle places.
        dict(name="attend_batch_8b", kind="attend", shape="8b", seqs=32, rows=1, context=8192, idle=0),
        dict(name="attend_trees_8b", kind="attend", shape="8b", seqs=12, rows=9, context=1900, idle=2),
        # One token of one very long document.
        dict(name="attend_long_8b", kind="attend", shape="8b", seqs=1, rows=1, context=131000, idle=0),
        # Chains of drafted tokens verified: one sequence, and a batch with chains of different lengths.
        dict(name="verify_one", kind="verify", vocab=128256, seqs=1, drafts=4),
        dict(name="verify_batch", kind="verify", vocab=128256, seqs=48, drafts=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "commit", "attend", "attend", "attend", "verify"])
    if kind == "verify":
        return dict(kind=kind, vocab=rng.choice([32768, 128256, rng.randint(1000, 128000)]), seqs=_log(rng, 1, 48),
                    drafts=rng.randint(1, 5))
    shape = rng.choice(["1b", "8b", "8b", "70b"])
    hd = SHAPES[shape][2]
    if kind == "write":
        prompt = rng.random() < 0.5
        rows = _log(rng, 1, 2000 if shape == "70b" else 4000) if prompt else _log(rng, 1, 64)
        return dict(kind=kind, shape=shape, seqs=1 if prompt else rows, rows=rows,
                    context=rows + _log(rng, 1, 3000), rot=rng.choice([hd, hd, hd // 2, hd // 4]),
                    interleaved=rng.random() < 0.5, scaling=rng.choice(sorted(SCALING)))
    if kind == "commit":
        return dict(kind=kind, shape=shape, layers=2, seqs=_log(rng, 1, 16), rows=rng.randint(2, 25),
                    context=_log(rng, 16, 2048), keep=rng.randint(1, 6))
    if rng.random() < 0.3:  # one long sequence
        return dict(kind=kind, shape=shape, seqs=1, rows=rng.choice([1, rng.randint(2, 32)]), idle=0,
                    context=_log(rng, 2000, 40000))
    seqs, rows = _log(rng, 1, 32), _log(rng, 1, 40)
    return dict(kind=kind, shape=shape, seqs=seqs, rows=rows, context=_log(rng, 3, min(8192, 150000 // seqs)),
                idle=rng.randint(0, seqs // 4))


# ------------------------------------------------------------------------------------------------- inputs
class _Rand:
    """Tensors of one case, each from its own seeded generator on the GPU; host numbers from ``host``."""

    def __init__(self, seed):
        self.seed, self.n = seed, 0
        self.host = torch.Generator().manual_seed(seed * 7919 + 17)

    def gen(self):
        self.n += 1
        return torch.Generator(device="cuda").manual_seed(self.seed * 1009 + self.n)

    def normal(self, *size, dtype=BF16):
        return torch.randn(*size, generator=self.gen(), device="cuda", dtype=dtype)

    def uniform(self, *size):
        return torch.rand(*size, generator=self.gen(), device="cuda", dtype=F32)

    def between(self, lo, hi):
        return int(torch.randint(lo, hi + 1, (1,), generator=self.host))


def _projected(r, rows, heads, kv, hd):
    """q, k, v of a fused projection's output rows: column ranges of one matrix, some channels larger as in trained models."""
    x = r.normal(rows, (heads + 2 * kv) * hd)
    gain = torch.ones(hd, device="cuda")
    gain[::17] = 6.0
    x = (x.view(rows, -1, hd) * gain.to(BF16)).view(rows, -1)
    return x[:, :heads * hd], x[:, heads * hd:(heads + kv) * hd], x[:, (heads + kv) * hd:]


def _inv_freq(rot, scaling):
    """(frequencies of the rotated pairs, factor on cos and sin) of the model's rotary embedding, in 64 bits."""
    base = [THETA ** (-2.0 * i / rot) for i in range(rot // 2)]
    s = SCALING[scaling]
    if s is None:
        return base, 1.0
    f = s["factor"]
    if s["rope_type"] == "linear":
        return [b / f for b in base], 1.0
    ctx = s["original_max_position_embeddings"]
    if s["rope_type"] == "llama3":
        lo, hi, out = s["low_freq_factor"], s["high_freq_factor"], []
        for b in base:
            t = min(1.0, max(0.0, (ctx * b / (2 * math.pi) - lo) / (hi - lo)))  # 0: all slowed, 1: as it was
            out.append((1 - t) * b / f + t * b)
        return out, 1.0
    dim = [rot * math.log(ctx / (n * 2 * math.pi)) / (2 * math.log(THETA)) for n in (32.0, 1.0)]  # turns 32 and 1
    lo, hi = max(math.floor(dim[0]), 0), min(math.ceil(dim[1]), rot - 1)
    ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3))) for i in range(rot // 2)]
    return [b * (1 - t) + b / f * t for b, t in zip(base, ramp)], 0.1 * math.log(f) + 1.0


def _cuda_i32(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def _tree_paths(r, rows):
    """Ancestor node numbers of each row, itself last; row 0 is the root, later rows hang on one of the eight before."""
    paths = [[]]
    for i in range(1, rows):
        ok = [j for j in range(max(0, i - 8), i) if len(paths[j]) < 6]
        paths.append(paths[ok[r.between(0, len(ok) - 1)] if ok else 0] + [i])
    return paths


def _package():
    pkg = os.path.join(REPO, "subnetwork-speculative-decoding_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)


def _cache(case, layers, seqs, capacity):
    _package()
    from ssd.engine.kv_cache import KVCacheQ8

    _, kv, hd = SHAPES[case["shape"]]
    return KVCacheQ8(layers, capacity, kv, hd, "cuda", sequences=seqs)


def prepare(case, seed):
    r = _Rand(seed)
    st = {"case": case}
    if case["kind"] == "verify":
        V, S, K = case["vocab"], case["seqs"], case["drafts"]
        # warped distributions: a peaked draft, the target near it, the tails cut away
        lq = r.normal(S, K + 1, V, dtype=F32).mul_(3.0)
        lp = r.normal(S, K + 1, V, dtype=F32).mul_(0.7).add_(lq)
        for name, x in (("p", lp), ("q", lq)):
            w = torch.exp(x - x.amax(-1, keepdim=True))
            w = torch.where(w < 1e-3, torch.zeros_like(w), w)
            st[name] = w / w.sum(-1, keepdim=True)
        st["q"] = st["q"][:, :K]
        noise = -torch.log(r.uniform(S, K, V).clamp_min(1e-30))
        st["draft"] = (st["q"] / noise).argmax(-1).to(I32)  # drawn from q
        st["u"], st["u_next"] = r.uniform(S, K), r.uniform(S)
        st["n_draft"] = _cuda_i32([K if S == 1 else r.between(0, K) for _ in range(S)])
        return st
    heads, kv, hd = SHAPES[case["shape"]]
    if case["kind"] == "attend":
        return _prepare_attend(case, r, st, heads, kv, hd)
    rows, ctx, S = case["rows"], case["context"], case["seqs"]
    if case["kind"] == "write":
        if S == 1:
            first = ctx - rows
            seq, slot = [0] * rows, list(range(first, ctx))
        else:
            seq, slot = list(range(S)), [r.between(ctx // 2, ctx - 1) for _ in range(S)]
        st["q"], st["k"], st["v"] = _projected(r, rows, heads, kv, hd)
        st["pos"] = _cuda_i32(slot)
        freq, st["factor"] = _inv_freq(case["rot"], case["scaling"])
        st["freq"] = torch.tensor(freq, dtype=F64, device="cuda")
        if own:
            st["cache"] = _cache(case, 1, S, ctx)
            from ssd.models.llama import rope_tables_f32

            st["rope"] = rope_tables_f32(ctx, case["rot"], THETA, "cuda", SCALING[case["scaling"]])
    else:
        lens = [ctx] + [r.between(ctx // 2, ctx) for _ in range(S - 1)]
        seq = [s for s in range(S) for _ in range(rows)]
        slot = [n + i for n in lens for i in range(rows)]
        keeps = []
        for s, n in enumerate(lens):  # the root and the accepted path: increasing slots behind the committed ones
            want = min(rows, 1 + s % case["keep"]) if S > 1 else min(rows, case["keep"])
            pick = sorted(torch.randperm(rows - 1, generator=r.host)[:want - 1].tolist()) if rows > 1 else []
            keeps.append([n] + [n + 1 + i for i in pick])
        most = min(rows, case["keep"])
        st["start"], st["n_keep"] = _cuda_i32(lens), _cuda_i32([len(k) for k in keeps])
        st["src"] = _cuda_i32([k + [0] * (most - len(k)) for k in keeps])
        kept = [(s, n + j, j) for s, (n, k) in enumerate(zip(lens, keeps)) for j in range(len(k))]
        st["back_seq"], st["back_slot"] = _cuda_i32([s for s, _, _ in kept]), _cuda_i32([t for _, t, _ in kept])
        # the written row that ends up in each committed slot
        st["back_row"] = torch.tensor([s * rows + keeps[s][j] - lens[s] for s, _, j in kept], device="cuda")
        st["kvs"] = [_projected(r, S * rows, 0, kv, hd)[1:] for _ in range(case["layers"])]
        if own:
            st["cache"] = _cache(case, case["layers"], S, ctx + rows)
    st["seq"], st["slot"] = _cuda_i32(seq), _cuda_i32(slot)
    return st


def _prepare_attend(case, r, st, heads, kv, hd):
    S, R, ctx = case["seqs"], case["rows"], case["context"]
    idle = set(range(1, 1 + 2 * case["idle"], 2)) if case["idle"] else set()
    lens = [0 if s in idle else ctx if s == 0 else r.between(max(1, ctx // 2), ctx) for s in range(S)]
    begin, prefix, depth, anc = [0], [], [], []
    for s, n in enumerate(lens):
        if s in idle:  # a place no sequence uses: one row that attends nothing
            prefix, depth, anc = prefix + [0], depth + [0], anc + [[0] * MAX_DEPTH]
        else:
            for path in _tree_paths(r, R - s * 5 % (R // 2 + 1)):  # between half the rows and all of them
                prefix.append(n + 1)
                depth.append(len(path))
                anc.append([n + i for i in path] + [0] * (MAX_DEPTH - len(path)))
        begin.append(len(prefix))
    M, cap = len(prefix), (ctx + R + 63) // 64 * 64
    st["q"] = r.normal(M, heads * hd) * 1.5
    st["begin"], st["prefix"], st["depth"], st["anc"] = (_cuda_i32(x) for x in (begin, prefix, depth, anc))
    st["lens"] = [n + 1 if n else 0 for n in lens]
    st["rows_of"] = [b - a for a, b in zip(begin, begin[1:])]
    k, v = r.normal(S, kv, cap, hd), r.normal(S, kv, cap, hd)
    k[..., ::17] *= 4.0
    if own:
        cache = st["cache"] = _cache(case, 1, S, cap)
        slots = torch.arange(cap, dtype=I32, device="cuda")
        for s in range(S):
            cache.write(0, k[s].transpose(0, 1).reshape(cap, -1), v[s].transpose(0, 1).reshape(cap, -1),
                        torch.full_like(slots, s), slots)
        st["rows_max"] = max(st["rows_of"])
        st["l_max"] = max(p + d for p, d in zip(prefix, depth))
        st["ws"] = torch.empty(cache.attend_floats(M, heads, st["l_max"]), dtype=F32, device="cuda")
    else:
        st["k"], st["v"] = _codes(k.float()), _codes(v.float())
    return st


# ------------------------------------------------------------------------------------------------- plain forms
def _exponent(amax):
    """The least e with amax <= 448 * 2^e, at least -100; 448 = 0.875 * 2^9."""
    m, e = torch.frexp(amax)
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp_min(-100)
    return torch.where(amax > 0, e, torch.full_like(e, -100))


def _codes(x):
    """8-bit values of rows [..., hd] and the rows' power-of-two scales."""
    e = _exponent(x.abs().amax(-1))
    return torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn), torch.ldexp(torch.ones_like(x[..., 0]), e)


def _values(codes, scale):
    return codes.to(F32) * scale[..., None]


def _rotated(x, st, hd):
    """Rows [M, n * hd] rotated by their positions, [M, n, hd] fp32 (angles in 64 bits)."""
    case = st["case"]
    x = x.float().view(x.shape[0], -1, hd)
    ang = st["pos"].to(F64)[:, None] * st["freq"]
    c, s = ((f(ang) * st["factor"]).to(F32)[:, None] for f in (torch.cos, torch.sin))
    rot = case["rot"]
    y = x.clone()
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return y


def _stored(x, hd):
    """Rows as the cache holds them, [M, n * hd] bf16 (every stored value is a bf16 value)."""
    return _values(*_codes(x.float().view(x.shape[0], -1, hd))).to(BF16).flatten(1)


def _plain_attend(st, heads, kv, hd):
    case = st["case"]
    S, R, rep = len(st["lens"]), max(st["rows_of"]), heads // kv
    k, v = _values(*st["k"]), _values(*st["v"])
    L, M = k.shape[2], st["q"].shape[0]
    seq = torch.repeat_interleave(torch.arange(S, device="cuda"), st["begin"].diff().long(), output_size=M)
    place = torch.arange(M, device="cuda") - st["begin"].long()[seq]
    q = torch.zeros(S, R, heads, hd, dtype=F32, device="cuda")
    q[seq, place] = st["q"].float().view(M, heads, hd)
    see = torch.arange(L, device="cuda") < st["prefix"][:, None]
    used = torch.arange(MAX_DEPTH, device="cuda") < st["depth"][:, None]
    line = torch.arange(M, device="cuda")[:, None].expand(M, MAX_DEPTH)
    see[line[used], st["anc"].long()[used]] = True
    mask = torch.zeros(S, R, L, dtype=torch.bool, device="cuda")
    mask[seq, place] = see
    q = q.view(S, R, kv, rep, hd).transpose(1, 2).reshape(S, kv, R * rep, hd)
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) * hd ** -0.5
    mask = mask[:, None, :, None].expand(S, kv, R, rep, L).reshape(S, kv, R * rep, L)
    score = score.masked_fill(~mask, float("-inf"))
    top = score.amax(-1, keepdim=True).clamp_min(-1e30)
    w = torch.exp(score - top)
    out = torch.matmul(w, v) / w.sum(-1, keepdim=True).clamp_min(1e-30)
    out = out.view(S, kv, R, rep, hd).transpose(1, 2)[seq, place]
    return out.reshape(M, heads * hd).to(BF16)


def _plain_verify(st):
    p, q, draft = st["p"], st["q"], st["draft"].long()
    S, K, V = q.shape
    px, qx = (x[:, :K].gather(2, draft[..., None])[..., 0].to(F64) for x in (p, q))
    ok = (st["u"].to(F64) * qx < px) & (torch.arange(K, device="cuda") < st["n_draft"][:, None])
    n = ok.long().cumprod(1).sum(1)
    s = torch.arange(S, device="cuda")
    row = p[s, n].to(F64)
    left = (row - q[s, n.clamp_max(K - 1)].to(F64)).clamp_min(0)
    use = (n < st["n_draft"]) & (left.sum(1) > 0)
    left = torch.where(use[:, None], left, row)
    cum = left.cumsum(1)
    nxt = (cum <= (st["u_next"].to(F64) * cum[:, -1])[:, None]).sum(1)
    last = V - 1 - (left > 0).flip(1).long().argmax(1)
    out = torch.full((S, K + 1), -1, dtype=I32, device="cuda")
    out[:, :K] = torch.where(torch.arange(K, device="cuda") < n[:, None], st["draft"], out[:, :K])
    out[s, n] = torch.minimum(nxt, last).to(I32)
    return n.to(I32), out


def run(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "verify":
        if not own:
            return _plain_verify(st)
        from ssd.engine.verify import verify_chain

        return verify_chain(st["p"], st["q"], st["draft"], st["u"], st["u_next"], st["n_draft"])
    heads, kv, hd = SHAPES[case["shape"]]
    if kind == "attend":
        if not own:
            return _plain_attend(st, heads, kv, hd)
        return st["cache"].attend(0, st["q"], st["begin"], st["prefix"], st["depth"], st["anc"], st["rows_max"],
                                  st["l_max"], ws=st["ws"])
    if kind == "write":
        if not own:
            k = _rotated(st["k"], st, hd).flatten(1)
            return _rotated(st["q"], st, hd).to(BF16).flatten(1), _stored(k, hd), _stored(st["v"], hd)
        q = st["cache"].write(0, st["k"], st["v"], st["seq"], st["slot"], rope=st["rope"], pos=st["pos"], q=st["q"],
                              interleaved=case["interleaved"])
        return (q, *st["cache"].read(0, st["seq"], st["slot"]))
    out = []
    if not own:
        for k, v in st["kvs"]:
            out += [_stored(k[st["back_row"]], hd), _stored(v[st["back_row"]], hd)]
        return out
    cache = st["cache"]
    for i, (k, v) in enumerate(st["kvs"]):
        cache.write(i, k, v, st["seq"], st["slot"])
    cache.compact_device(st["start"], st["src"], st["n_keep"])
    for i in range(case["layers"]):
        out += cache.read(i, st["back_seq"], st["back_slot"])
    return out


# ------------------------------------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    if kind == "verify":  # one target and one draft row of each sequence
        return {"bytes": case["seqs"] * (8 * case["vocab"] + 16 * case["drafts"]), "flops": 3 * case["seqs"] * case["vocab"]}
    heads, kv, hd = SHAPES[case["shape"]]
    if kind == "attend":
        S, R, ctx = case["seqs"], case["rows"], case["context"]
        live = S - case["idle"]
        keys = ctx + 0.75 * ctx * (live - 1)  # the first sequence is full, the others' lengths average three quarters
        rows = R + max(1.0, 0.75 * R) * (live - 1)
        per = rows / live
        return {"bytes": int(2 * kv * (hd + 1) * (keys + rows) + 4 * heads * hd * rows),
                "flops": int(4 * heads * hd * keys * per)}
    rows = case["rows"]
    back = 2 * kv * hd * 2  # K and V read back in bf16
    if kind == "write":
        one = (2 * heads + 2 * kv) * hd * 2 + 2 * 2 * kv * (hd + 1) + back + 8 * (case["rot"] // 2)
        return {"bytes": rows * one, "flops": rows * 3 * case["rot"] * (heads + kv)}
    kept = case["seqs"] * min(rows, (1 + case["keep"]) / 2)
    one = 2 * kv * hd * 2 + 2 * kv * (hd + 1)
    return {"bytes": int(case["layers"] * (case["seqs"] * rows * one + kept * (3 * 2 * kv * (hd + 1) + back))),
            "flops": case["layers"] * case["seqs"] * rows * 4 * kv * hd}


# ------------------------------------------------------------------------------------------------- definitions in 64 bits
def _exact_round(x):
    """[..., hd] doubles -> the values an 8-bit row stands for: four significant bits, steps of 2^(e - 9) at the least."""
    big = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(big.clamp_min(1e-300) / 448))
    e = e + (big > 448 * torch.exp2(e)).to(F64) - (big <= 224 * torch.exp2(e)).to(F64)  # log2's own rounding
    e = e.clamp_min(-100)
    _, b = torch.frexp(x)
    step = torch.exp2(torch.maximum(b.to(F64) - 4, e - 9))
    return torch.round(x / step) * step


def _exact_turn(x, st, hd):
    case, x = st["case"], x.double().view(x.shape[0], -1, hd)
    half = case["rot"] // 2
    ang = torch.outer(st["pos"].double(), st["freq"])
    turn = torch.polar(torch.full_like(ang, st["factor"]), ang)[:, None]
    part, rest = x[..., :2 * half], x[..., 2 * half:]
    if case["interleaved"]:
        z = torch.view_as_complex(part.reshape(*part.shape[:-1], half, 2).contiguous()) * turn
        done = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(part[..., :half].contiguous(), part[..., half:].contiguous()) * turn
        done = torch.cat([z.real, z.imag], -1)
    return torch.cat([done, rest], -1)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    kind = case["kind"]
    if kind == "verify":
        return _exact_verify(st)
    heads, kv, hd = SHAPES[case["shape"]]
    if kind == "attend":
        out = torch.zeros(st["q"].shape[0], heads, hd, dtype=F64, device="cuda")
        begin, prefix, depth, anc = (st[n].tolist() for n in ("begin", "prefix", "depth", "anc"))
        for s in range(len(begin) - 1):
            n = st["lens"][s]
            if not n:
                continue
            end = n + max(st["rows_of"]) if n else 0
            kk, vv = (st[x][0][s][:, :end].double() * st[x][1][s][:, :end].double()[..., None] for x in ("k", "v"))
            kk, vv = (t.repeat_interleave(heads // kv, 0) for t in (kk, vv))
            for t in range(begin[s], begin[s + 1]):
                at = torch.tensor(list(range(prefix[t])) + anc[t][:depth[t]], device="cuda")
                if not len(at):
                    continue
                w = (kk[:, at] * st["q"][t].double().view(heads, 1, hd)).sum(-1) / math.sqrt(hd)
                w = torch.softmax(w, -1)
                out[t] = (w[..., None] * vv[:, at]).sum(1)
        return out.flatten(1)
    if kind == "write":
        k, v = _exact_turn(st["k"], st, hd), st["v"].double().view(case["rows"], kv, hd)
        return _exact_turn(st["q"], st, hd).flatten(1), _exact_round(k).flatten(1), _exact_round(v).flatten(1)
    out = []
    for k, v in st["kvs"]:
        out += [_exact_round(x.double().view(-1, kv, hd)).flatten(1)[st["back_row"]] for x in (k, v)]
    return out


def _exact_verify(st):
    counts, tokens = [], []
    draft, u, last, n_draft = (st[x].tolist() for x in ("draft", "u", "u_next", "n_draft"))
    K = len(u[0])
    for s, todo in enumerate(n_draft):
        n = 0
        while n < todo and u[s][n] * float(st["q"][s, n, draft[s][n]]) < float(st["p"][s, n, draft[s][n]]):
            n += 1
        w = st["p"][s, n].double().cpu()
        if n < todo:
            left = torch.relu(w - st["q"][s, n].double().cpu())
            w = left if float(left.max()) > 0 else w
        cum = torch.cumsum(w, 0)
        nxt = int(torch.searchsorted(cum, last[s] * cum[-1:], right=True))
        counts.append(n)
        tokens.append(draft[s][:n] + [min(nxt, int(torch.nonzero(w)[-1]))] + [-1] * (K - n))
    return _cuda_i32(counts), _cuda_i32(tokens)
