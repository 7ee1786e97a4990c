"""64-bit definitions of the operators on a paged cache and of token log probabilities, on plain (unpaged) rows."""

from __future__ import annotations

import math

import torch


def attention(q, k, v, last, scale=None):
    """Rows q [n, heads, hd] over k, v [L, kv, hd]; row i attends slots [0, last[i]] (none below 0). Returns (out [n, heads, hd],
    the same for |v|, weights [n, heads, L], largest sum of |q k| scale of each row and head), in doubles."""
    n, heads, hd = q.shape
    kv = k.shape[1]
    scale = hd ** -0.5 if scale is None else scale
    out = torch.zeros(n, heads, hd, dtype=torch.float64)
    mag = torch.zeros_like(out)
    w_all = torch.zeros(n, heads, k.shape[0], dtype=torch.float64)
    size = torch.zeros(n, heads, dtype=torch.float64)
    for i in range(n):
        end = int(last[i]) + 1
        if end <= 0:
            continue
        for h in range(heads):
            kk, vv = k[:end, h * kv // heads].double(), v[:end, h * kv // heads].double()
            qq = q[i, h].double()
            w = torch.softmax(kk @ qq * scale, 0)
            out[i, h], mag[i, h] = w @ vv, w @ vv.abs()
            w_all[i, h, :end] = w
            size[i, h] = (kk.abs() @ qq.abs()).max() * scale
    return out, mag, w_all, size


def evict(w, length, keep, recent, first):
    """Slots of one (sequence, kv head) that stay, of weights w [>= length]: a sorted list."""
    if length <= keep:
        return list(range(length))
    mid = range(first, length - recent)

    def rank(t):
        x = float(w[t])
        return (1, 0.0, t) if math.isnan(x) else (0, -x, t)

    return sorted([*range(first), *sorted(mid, key=rank)[:keep - first - recent], *range(length - recent, length)])


def token_logprobs(logits, tokens, top):
    """(logprobs, entropy, rank, top ids, top logprobs) of finite or -inf logits [M, V], in doubles."""
    x = logits.double()
    d = x - x.amax(1, keepdim=True)  # first: beside a type's lowest value ln V is nothing, in 64 bits too
    lp = d - d.exp().sum(1, keepdim=True).log()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    have = (tokens >= 0) & (tokens < x.shape[1])
    t = torch.where(have, tokens, 0).long()
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, 0.0).sum(1)
    rank = (order == t[:, None]).long().argmax(1)
    ids = order[:, :top]
    return (torch.where(have, lp.gather(1, t[:, None])[:, 0], 0.0), ent, torch.where(have, rank, -1), ids, lp.gather(1, ids))
