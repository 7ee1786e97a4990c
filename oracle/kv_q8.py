"""Plain 64-bit (CPU) forms of the batched round's operators over the 8-bit KV cache, written from their definitions:
quantisation, the cache's element order, rotary positions, tree attention and chain verification."""

from __future__ import annotations

import math

import torch


# ------------------------------------------------------------------------------------------------- quantisation
def exponent(x: torch.Tensor) -> torch.Tensor:
    """Least e >= -100 with max|x| <= 448 * 2^e over the finite values of the last dim."""
    amax = torch.where(torch.isfinite(x), x.double().abs(), torch.zeros((), dtype=torch.float64)).amax(-1)
    out = torch.empty(amax.shape, dtype=torch.int64)
    for i, a in enumerate(amax.flatten().tolist()):
        e = -100
        if a > 0:
            e = max(-100, math.frexp(a)[1] - 10)
            while a > math.ldexp(448.0, e):
                e += 1
        out.view(-1)[i] = e
    return out


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """Doubles within 448 rounded to e4m3 values: four significant bits, half to even, steps of 2^-9 at the least."""
    _, b = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (b.long() - 4).clamp_min(-9))
    return torch.round(x / step) * step


def stored(x: torch.Tensor) -> torch.Tensor:
    """The values a cache row [..., head_dim] holds, as doubles; NaN where x is not finite."""
    e = exponent(x)[..., None]
    d = torch.where(torch.isfinite(x), x.double(), torch.full((), float("nan"), dtype=torch.float64))
    return torch.ldexp(e4m3(torch.ldexp(d, -e)), e)


# ------------------------------------------------------------------------------------------------- element order
def k_offset(s: int, d: int, hd: int) -> int:
    """Byte of K[slot s][dim d]: the 16 keys of a tile side by side, 16 dims of one key a lane."""
    block, o = divmod(s, 64)
    tile, key = divmod(o, 16)
    part, rest = divmod(d, 64)
    lane = (rest // 16) * 16 + key
    return (((block * 4 + tile) * (hd // 64) + part) * 64 + lane) * 16 + rest % 16


def v_offset(s: int, d: int, hd: int) -> int:
    """Byte of V[slot s][dim d]: one dim and sixteen keys a lane, the keys 16 kt + 4 g + e of lane group g."""
    block, o = divmod(s, 64)
    kt, r = divmod(o, 16)
    g, e = divmod(r, 4)
    return ((block * (hd // 16) + d // 16) * 64 + g * 16 + d % 16) * 16 + kt * 4 + e


def x_offset(s: int) -> int:
    """Byte of slot s's exponent."""
    block, o = divmod(s, 64)
    kt, r = divmod(o, 16)
    return block * 64 + (r // 4) * 16 + kt * 4 + r % 4


# ------------------------------------------------------------------------------------------------- rotation
def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """x [M, heads, hd] (doubles out); cos/sin [rows, rot / 2]; positions outside the table use its nearest row."""
    x = x.double().clone()
    p = pos.long().clamp(0, cos.shape[0] - 1)
    c, s = cos.double()[p][:, None], sin.double()[p][:, None]
    half = cos.shape[1]
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    xa, xb = x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = xa * c - xb * s, xb * c + xa * s
    return x


# ------------------------------------------------------------------------------------------------- attention
def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, row_begin, prefix, depth, anc, scale=None):
    """q [M, heads, hd]; k, v [sequences, kv_heads, slots, hd] (the stored values). Returns (out, sum of
    w |v|), [M, heads, hd] doubles each. NaN rows: those of no sequence."""
    M, heads, hd = q.shape
    rep = heads // k.shape[1]
    scale = hd ** -0.5 if scale is None else scale
    out = torch.full((M, heads, hd), float("nan"), dtype=torch.float64)
    mag = torch.zeros_like(out)
    for s in range(len(row_begin) - 1):
        for t in range(row_begin[s], row_begin[s + 1]):
            at = list(range(prefix[t])) + [int(a) for a in anc[t][:depth[t]]]
            if not at:
                out[t] = 0
                continue
            for h in range(heads):
                kk, vv = k[s, h // rep, at].double(), v[s, h // rep, at].double()
                w = torch.softmax(kk @ q[t, h].double() * scale, 0)
                out[t, h], mag[t, h] = w @ vv, w @ vv.abs()
    return out, mag


# ------------------------------------------------------------------------------------------------- verification
def verify_chain(P, Q, draft, u, u_next, n_draft=None):
    """Lists (accepted counts, tokens [k + 1] per sequence) by the definition, in doubles."""
    counts, tokens = [], []
    B, k1, V = P.shape
    K = k1 - 1
    for s in range(B):
        todo = K if n_draft is None else min(max(int(n_draft[s]), 0), K)
        n = 0
        while n < todo:
            x = int(draft[s, n])
            if not 0 <= x < V or not float(u[s, n]) * float(Q[s, n, x]) < float(P[s, n, x]):
                break
            n += 1
        w = P[s, n].double().clamp_min(0)
        if n < todo:
            r = (P[s, n].double() - Q[s, n].double()).clamp_min(0)
            if float(r.sum()) > 0:
                w = r
        total, want, cum, tok = float(w.sum()), None, 0.0, -1
        want = float(u_next[s]) * total
        for y in torch.nonzero(w)[:, 0].tolist():
            cum += float(w[y])
            tok = y
            if cum > want:
                break
        counts.append(n)
        tokens.append([int(x) for x in draft[s, :n]] + [tok] + [-1] * (K - n))
    return counts, tokens
