"""Operators of a batched speculative round over the 8-bit KV cache on the GPU, against their 64-bit definitions
(oracle/kv_q8.py): rotation, quantising write, read-back, compaction, tree attention, chain verification, and a round of them."""

import pytest
import torch

from oracle import kv_q8 as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cache(layers, length, kv, hd, seqs=1, span=None):
    from ssd.engine.kv_cache import KVCacheQ8

    return KVCacheQ8(layers, length, kv, hd, DEV, sequences=seqs, span=span)


def _rot32(x, cos, sin, pos, interleaved, hd):
    """Rotation in fp32 with every product and sum rounded (CPU), [M, n, hd]."""
    y = x.float().view(x.shape[0], -1, hd).clone()
    p = pos.long().clamp(0, cos.shape[0] - 1)
    c, s, half = cos[p][:, None], sin[p][:, None], cos.shape[1]
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    xa, xb = y[..., a].clone(), y[..., b].clone()
    y[..., a] = xa * c - xb * s
    y[..., b] = xb * c + xa * s
    return y


def _same(a, b):
    """Equal values, NaN at the same places."""
    a, b = a.double(), b.double()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0))


# ------------------------------------------------------------------------------------------------- write, read
@pytest.mark.parametrize("hd,kv,heads,rows,rot,interleaved", [
    (128, 8, 32, 1, 128, False), (128, 2, 6, 37, 64, True), (64, 8, 32, 19, 64, False), (64, 1, 5, 130, 16, False),
    (128, 3, 3, 65, 96, False), (64, 2, 2, 64, 48, True), (128, 1, 1, 257, None, False)])
def test_write_then_read(hd, kv, heads, rows, rot, interleaved):
    from ssd.models.llama import rope_tables_f32

    g = _gen(rows * 7 + hd)
    x = (torch.randn(rows, (heads + 2 * kv) * hd, generator=g) * torch.logspace(-3, 3, hd).repeat(heads + 2 * kv)).to(BF16)
    q, k, v = x[:, :heads * hd], x[:, heads * hd:(heads + kv) * hd], x[:, (heads + kv) * hd:]
    seqs, length = 3, 300
    places = torch.randperm(seqs * length, generator=g)[:rows]
    seq, slot = (places // length).int(), (places % length).int()
    pos = torch.randint(-2, 90000, (rows,), generator=g, dtype=torch.int32)
    cache = _cache(1, length, kv, hd, seqs)
    xd = x.to(DEV)
    qd, kd, vd = xd[:, :heads * hd], xd[:, heads * hd:(heads + kv) * hd], xd[:, (heads + kv) * hd:]
    args = dict(q=qd)
    if rot:
        cos, sin = rope_tables_f32(80000, rot, 500000.0, "cpu")
        args.update(rope=(cos.to(DEV), sin.to(DEV)), pos=pos.to(DEV), interleaved=interleaved)
    q_out = cache.write(0, kd, vd, seq.to(DEV), slot.to(DEV), **args)
    k2, v2 = cache.read(0, seq.to(DEV), slot.to(DEV))
    kr = _rot32(k, cos, sin, pos, interleaved, hd) if rot else k.float().view(rows, kv, hd)
    qr = _rot32(q, cos, sin, pos, interleaved, hd) if rot else q.float().view(rows, heads, hd)
    assert _same(q_out.cpu(), qr.to(BF16).flatten(1))
    assert _same(k2.cpu(), ref.stored(kr).flatten(1))
    assert _same(v2.cpu(), ref.stored(v.float().view(rows, kv, hd)).flatten(1))
    # the documented places of the bytes
    kb, xb = cache.k.cpu(), cache.k_exp.cpu()
    vb, yb = cache.v.cpu(), cache.v_exp.cpu()
    ks, vs = ref.stored(kr), ref.stored(v.float().view(rows, kv, hd))
    for r in range(0, rows, max(1, rows // 4)):
        s, t = int(seq[r]), int(slot[r])
        for d in (0, 1, 17, hd - 1):
            for arr, ex, off, val in ((kb, xb, ref.k_offset(t, d, hd), ks[r, kv - 1, d]), (vb, yb, ref.v_offset(t, d, hd), vs[r, kv - 1, d])):
                code = arr[0, s, kv - 1, off:off + 1].view(torch.float8_e4m3fn).double()
                assert float(code * 2.0 ** (int(ex[0, s, kv - 1, ref.x_offset(t)]) - 127)) == float(val)


@pytest.mark.parametrize("rows", [4096, 200, 63])
def test_write_consecutive_slots(rows):
    """A prompt's rows: consecutive slots from an odd one, and nothing else changes."""
    hd, kv, first = 128, 2, 37
    g = _gen(rows)
    k, v = (torch.randn(rows, kv * hd, generator=g).to(BF16) for _ in range(2))
    cache = _cache(1, rows + 100, kv, hd, 2)
    for t in (cache.k, cache.v, cache.k_exp, cache.v_exp):
        t.fill_(93)
    slot = torch.arange(first, first + rows, dtype=torch.int32, device=DEV)
    cache.write(0, k.to(DEV), v.to(DEV), torch.ones_like(slot), slot)
    k2, v2 = cache.read(0, torch.ones_like(slot), slot)
    assert _same(k2.cpu(), ref.stored(k.float().view(rows, kv, hd)).flatten(1))
    assert _same(v2.cpu(), ref.stored(v.float().view(rows, kv, hd)).flatten(1))
    cap = cache.capacity
    for t, n in ((cache.k, hd), (cache.v, hd), (cache.k_exp, 1), (cache.v_exp, 1)):
        t = t.view(1, 2, kv, -1).cpu()
        assert (t[:, 0] == 93).all()
        assert int((t[:, 1] != 93).sum()) <= kv * rows * n
    for s in [0, first - 1, first + rows, cap - 1]:
        for d in (0, 63, hd - 1):
            assert int(cache.k[0, 1, 1, ref.k_offset(s, d, hd)]) == 93 and int(cache.v[0, 1, 1, ref.v_offset(s, d, hd)]) == 93
        assert int(cache.k_exp[0, 1, 0, ref.x_offset(s)]) == 93


def test_write_special_values_and_places_outside():
    hd, kv = 64, 2
    inf, nan = float("inf"), float("nan")
    base = torch.randn(9, kv * hd, generator=_gen(3))
    base[0] = 0
    base[1, 5], base[1, 6], base[1, 70] = inf, -inf, nan
    base[2] = nan
    base[3] = 3.0e38
    base[4] = 1e-38
    base[5] = torch.linspace(-448, 448, kv * hd)
    base[6, 0] = 448 * 2.0 ** 9
    k = base.to(BF16)
    seq, slot = _i32([0, 0, 0, 0, 0, 0, 0, 0, 2]), _i32([0, 1, 2, 3, 4, 5, 6, 64, 0])  # the last two: no such slot, no such sequence
    cache = _cache(1, 64, kv, hd, 2)
    cache.k_exp.fill_(11)
    cache.write(0, k.to(DEV), k.flip(1).contiguous().to(DEV), seq, slot)
    k2, v2 = cache.read(0, seq, slot)
    want = ref.stored(k.float().view(9, kv, hd)).flatten(1)
    assert _same(k2[:7].cpu(), want[:7]) and not k2[7:].any() and not v2[7:].any()
    assert _same(v2[:7].cpu(), ref.stored(k.flip(1).float().view(9, kv, hd)).flatten(1)[:7])
    assert int((cache.k_exp != 11).sum()) == 7 * kv  # nothing else was written
    print(cache.read(0, _i32([-1]), _i32([5]))[0].abs().max())


def test_write_takes_no_rows_and_refuses_bad_tensors():
    cache = _cache(2, 64, 2, 64)
    k = torch.zeros(4, 128, dtype=BF16, device=DEV)
    i = _i32([0, 1, 2, 3])
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    cache.write(0, k[:0], k[:0], none, none)
    assert cache.read(1, none, none)[0].shape == (0, 128)
    for bad in (lambda: cache.write(0, k.float(), k, i, i), lambda: cache.write(0, k, k, i.long(), i),
                lambda: cache.write(0, k, k, i[:3], i), lambda: cache.write(0, k[:, :64], k, i, i),
                lambda: cache.write(0, k.cpu(), k, i, i), lambda: cache.write(0, k, k, i, i, pos=i),
                lambda: cache.write(0, k, k, i, i, q=k[:, :96]), lambda: cache.write(0, k, k, i.repeat_interleave(2)[::2], i),
                lambda: cache.compact_device(i[:1], i, i[:1]), lambda: cache.read(0, i, i[:2])):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("hd,heads,rows,rot,interleaved,in_place", [(128, 32, 33, 128, False, True), (64, 3, 1, 32, True, True),
                                                                    (128, 1, 700, 64, False, False), (64, 32, 50, 64, True, False)])
def test_rope(hd, heads, rows, rot, interleaved, in_place):
    from ssd import ops
    from ssd.models.llama import rope_tables_f32

    g = _gen(rows)
    x = torch.randn(rows, heads * hd + 8, generator=g).to(BF16)
    pos = torch.randint(0, 131072, (rows,), generator=g, dtype=torch.int32)
    cos, sin = rope_tables_f32(131072, rot, 1e6, "cpu", {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 16384})
    xd = x.to(DEV)
    out = xd if in_place else torch.zeros_like(xd)
    ops.rope(xd, rows, heads, hd, (cos.to(DEV), sin.to(DEV)), pos.to(DEV), out, interleaved)
    want = _rot32(x[:, :heads * hd], cos, sin, pos, interleaved, hd)
    assert torch.equal(out[:, :heads * hd].cpu(), want.to(BF16).flatten(1))
    exact = ref.rope(x[:, :heads * hd].view(rows, heads, hd), cos, sin, pos, interleaved)
    # the terms' magnitudes |a c| + |b s| (first of a pair: minus a negative sine; second: plus a positive one)
    terms = [ref.rope(x[:, :heads * hd].view(rows, heads, hd).abs(), cos.abs(), t * sin.abs(), pos, interleaved) for t in (-1, 1)]
    # two products off by 2^-24 each, their sum by 2^-24 of at most the terms
    assert ((want - exact).abs() <= torch.maximum(*terms) * 2 ** -23).all()
    assert torch.equal(out[:, heads * hd:].cpu(), x[:, heads * hd:] if in_place else torch.zeros(rows, 8, dtype=BF16))


# ------------------------------------------------------------------------------------------------- compaction
@pytest.mark.parametrize("hd,kv,layers,seqs", [(128, 2, 3, 4), (64, 8, 1, 1), (64, 1, 2, 7)])
def test_compact(hd, kv, layers, seqs):
    g = _gen(hd + seqs)
    length, n_max = 200, 9
    cache = _cache(layers, length, kv, hd, seqs)
    for t in (cache.k, cache.v, cache.k_exp, cache.v_exp):
        t.copy_(torch.randint(30, 120, t.shape, generator=g, dtype=torch.uint8))
    start = torch.randint(0, 150, (seqs,), generator=g)
    n = torch.randint(0, n_max + 1, (seqs,), generator=g)
    n[0] = n_max
    src = torch.stack([s + torch.randperm(40, generator=g)[:n_max] for s in start])  # any order, destinations among them
    src[0, 2] = src[0, 1]       # one source twice
    if seqs > 1:
        src[1, 0], start[2 % seqs] = -3, cache.capacity - 2  # skipped: no such source; destinations past the end
        n[1] = max(int(n[1]), 1)
    every = torch.arange(cache.capacity, dtype=torch.int32, device=DEV)
    before = [[cache.read(i, torch.full_like(every, s), every) for s in range(seqs)] for i in range(layers)]
    cache.compact_device(start.int().to(DEV), src.int().to(DEV), n.int().to(DEV))
    for i in range(layers):
        for s in range(seqs):
            for old, new in zip(before[i][s], cache.read(i, torch.full_like(every, s), every)):
                want = old.clone()
                for j in range(int(n[s])):
                    a, b = int(src[s, j]), int(start[s]) + j
                    if 0 <= a < cache.capacity and b < cache.capacity:
                        want[b] = old[a]
                assert torch.equal(new, want), (i, s)


# ------------------------------------------------------------------------------------------------- attention
def _fill(cache, seed, layer=0, scale=1.0):
    """Random K and V in every slot of the cache; returns the stored values [seqs, kv, capacity, hd] (CPU, bf16)."""
    g = _gen(seed)
    out = []
    cap, kv, hd = cache.capacity, cache.kv_heads, cache.head_dim
    slots = torch.arange(cap, dtype=torch.int32, device=DEV)
    vals = []
    for s in range(cache.sequences):
        k, v = (torch.randn(cap, kv * hd, generator=g) * torch.exp2(torch.randint(-3, 3, (cap, 1), generator=g)) * scale for _ in range(2))
        k, v = k.to(BF16).to(DEV), (3 * v).to(BF16).to(DEV)
        cache.write(layer, k, v, torch.full_like(slots, s), slots)
        vals.append([t.cpu().view(cap, kv, hd).transpose(0, 1) for t in cache.read(layer, torch.full_like(slots, s), slots)])
    return tuple(torch.stack([x[i] for x in vals]) for i in range(2))


def _table(rows):
    """rows: per sequence a list of (prefix, ancestor slots). Returns device tensors and host lists."""
    begin, prefix, depth, anc = [0], [], [], []
    for seq in rows:
        for p, a in seq:
            prefix.append(p), depth.append(len(a)), anc.append(list(a) + [10 ** 6] * (32 - len(a)))
        begin.append(len(prefix))
    return (_i32(begin), _i32(prefix), _i32(depth), torch.tensor(anc, dtype=torch.int32, device=DEV).view(-1, 32)), begin, prefix, depth, anc


def _tolerance(want, mag):
    """A bf16 rounding is off by at most half a step, 2^-8 of the value (a step is 2^-7 of a power of two). Weights
    p (1 + d) over the sum of the same: relative error at most 2 * 2^-8 each, so 2^-7 of mag = sum w |v|; the output's own
    rounding 2^-8 of it; fp32 scores, exp2 and sums together below 2^-12 of mag."""
    return mag * (2 ** -7 + 2 ** -12) + want.abs() * 2 ** -8


def _check_attend(cache, rows, heads, seed, kv_vals, extra=0, ld_pad=0, scale=None, l_max=None):
    tab, begin, prefix, depth, anc = _table(rows)
    hd, M = cache.head_dim, begin[-1]
    q = torch.randn(M + extra, heads * hd + ld_pad, generator=_gen(seed)).to(BF16)
    qd = q.to(DEV)[:, :heads * hd]
    out = torch.full((M + extra, heads * hd + ld_pad), 7.0, dtype=BF16, device=DEV)
    pad = [torch.cat([t, torch.zeros(extra, *t.shape[1:], dtype=t.dtype, device=DEV)]) if extra else t for t in tab[1:]]
    cache.attend(0, qd, tab[0], *pad, max(b - a for a, b in zip(begin, begin[1:])) or 1,
                 l_max or max([p + d for p, d in zip(prefix, depth)] + [1]), out=out[:, :heads * hd], scale=scale)
    assert (out[M:] == 7).all() and (out[:, heads * hd:] == 7).all()
    got = out[:M, :heads * hd].cpu().view(M, heads, hd)
    want, mag = ref.tree_attention(q[:M, :heads * hd].view(M, heads, hd), *kv_vals, begin, prefix, depth, anc, scale)
    err, tol = (got.double() - want).abs(), _tolerance(want, mag)
    assert (err <= tol).all(), (float((err - tol).max()), (err > tol).nonzero()[:4].tolist())
    return got


def _tree(n, first, count, g):
    """A root in the prefix (slots < n) and count - 1 nodes at slots first ..: rows (n, path)."""
    paths = [[]]
    for i in range(1, count):
        p = paths[int(torch.randint(max(0, i - 6), i, (1,), generator=g))]
        paths.append((p if len(p) < 31 else []) + [first + i - 1])
    return [(n, p) for p in paths]


@pytest.mark.parametrize("hd,heads,kv,span", [(128, 8, 2, 256), (64, 4, 4, 64), (64, 16, 1, 128), (128, 20, 1, 128)])
@pytest.mark.parametrize("length", [1, 2, 63, 64, 65, 127, 130, 320])
def test_attend_one_row(hd, heads, kv, span, length):
    cache = _cache(1, 384, kv, hd, 1, span)
    _check_attend(cache, [[(length, [])]], heads, length, _fill(cache, hd + length))


@pytest.mark.parametrize("hd,heads,kv,span,n", [(128, 8, 2, 256, 300), (128, 4, 1, 64, 64), (64, 8, 8, 128, 127), (64, 6, 2, 64, 1),
                                                (128, 8, 1, 128, 200), (64, 24, 1, 64, 97)])
@pytest.mark.parametrize("count", [2, 17, 40])
def test_attend_tree(hd, heads, kv, span, n, count):
    cache = _cache(1, 400, kv, hd, 1, span)
    g = _gen(count + n)
    _check_attend(cache, [_tree(n, n + 3, count, g)], heads, count, _fill(cache, n), extra=2, ld_pad=16)


def test_attend_batch_of_trees_and_empty_places():
    hd, kv, heads = 128, 2, 8
    cache = _cache(1, 640, kv, hd, 7, 128)
    g = _gen(5)
    rows = [_tree(500, 501, 9, g), [], [(0, [])], [(1, [])], [(0, [5, 9, 600])], _tree(64, 70, 64, g),
            [(200, [201]), (0, []), (17, [40, 3]), (600, [])]]  # rows of very different prefixes
    _check_attend(cache, rows, heads, 9, _fill(cache, 11), extra=3)


def test_attend_ancestors_outside_the_cache_are_not_attended():
    hd, kv, heads = 64, 1, 4
    cache = _cache(1, 128, kv, hd, 1, 64)
    vals = _fill(cache, 2)
    tab, *_ = _table([[(70, [-1, 80, 128, 1 << 30, 90]), (0, [-5])]])
    q = torch.randn(2, heads * hd, generator=_gen(4)).to(BF16)
    got = cache.attend(0, q.to(DEV), *tab, 2, 128).cpu().view(2, heads, hd).double()
    want, mag = ref.tree_attention(q.view(2, heads, hd), *vals, [0, 2], [70, 0], [2, 0], [[80, 90], []])
    assert ((got - want).abs() <= _tolerance(want, mag)).all() and not got[1].any()


def test_attend_masked_places_hold_anything():
    """NaN codes and the largest exponents in every slot that is not attended do not reach the output."""
    hd, kv, heads = 128, 1, 4
    cache = _cache(1, 256, kv, hd, 1, 64)
    vals = _fill(cache, 8)
    see = list(range(100)) + [130, 133, 190]
    keep = cache.read(0, _i32([0] * len(see)), _i32(see))
    cache.k.fill_(0x7f), cache.v.fill_(0xff), cache.k_exp.fill_(255), cache.v_exp.fill_(255)
    cache.write(0, *keep, _i32([0] * len(see)), _i32(see))
    _check_attend(cache, [[(100, [130, 133, 190]), (100, []), (0, []), (100, [190])]], heads, 3, vals)


def test_attend_nan_and_extreme_values():
    hd, kv, heads = 64, 1, 2
    cache = _cache(1, 128, kv, hd, 1, 64)
    vals = _fill(cache, 8, scale=1.0)
    q = torch.randn(3, heads * hd, generator=_gen(1)).to(BF16)
    q[1, 3] = float("nan")
    tab, *_ = _table([[(90, []), (90, []), (90, [])]])
    got = cache.attend(0, q.to(DEV), *tab, 3, 90).cpu().view(3, heads, hd)
    assert got[1, 0].isnan().all() and not got[1, 1].isnan().any() and not got[0].isnan().any()
    # a stored NaN reaches the rows that attend it
    k = torch.full((1, hd), float("nan"), dtype=BF16, device=DEV)
    cache.write(0, k, k, _i32([0]), _i32([70]))
    tab, *_ = _table([[(70, []), (71, [])]])
    got = cache.attend(0, q[:2].to(DEV), *tab, 2, 71).cpu()
    assert not got[0].isnan().any() and got[1].isnan().all()
    # huge and tiny rows side by side: scores far apart, values of every size
    k, v = torch.zeros(40, hd), torch.randn(40, hd, generator=_gen(3))
    k[7] = 1e4
    v = v * torch.logspace(-30, 30, 40)[:, None]
    cache.write(0, k.to(BF16).to(DEV), v.to(BF16).to(DEV), _i32([0] * 40), _i32(list(range(40))))
    slots = torch.arange(64, dtype=torch.int32, device=DEV)
    vals = tuple(t.cpu().view(1, 64, 1, hd).transpose(1, 2) for t in cache.read(0, torch.zeros_like(slots), slots))
    q = torch.full((1, heads * hd), -1.0).to(BF16)
    tab, begin, prefix, depth, anc = _table([[(40, [])]])
    got = cache.attend(0, q.to(DEV), *tab, 1, 40).cpu().view(1, heads, hd).double()
    want, mag = ref.tree_attention(q.view(1, heads, hd), *vals, begin, prefix, depth, anc)
    assert ((got - want).abs() <= _tolerance(want, mag)).all()


@pytest.mark.parametrize("hd,heads,kv,span", [(128, 8, 2, 64), (128, 4, 1, 256), (64, 32, 8, 128)])
def test_verify_rows_equal_autoregressive_steps_bit_for_bit(hd, heads, kv, span):
    """A tree row's output is that of the step at its position whose path lies in consecutive slots, alone or in a batch."""
    cache = _cache(1, 640, kv, hd, 3, span)
    _fill(cache, 21)
    g = _gen(hd)
    for n in (1, 63, 64, 250, 255, 256, 300, 511):
        rows = _tree(n, n + 5, 30, g)
        M = len(rows)
        q = torch.randn(M, heads * hd, generator=g).to(BF16).to(DEV)
        other = [(400, [])] * 5
        tab, *_ = _table([other, rows, []])
        l_max = max(n + len(p) for _, p in rows)
        both = torch.cat([torch.randn(5, heads * hd, generator=g).to(BF16).to(DEV), q])
        tree = cache.attend(0, both, *tab, M, max(l_max, 400))[5:]
        committed = torch.arange(n, dtype=torch.int32, device=DEV)
        kv0 = cache.read(0, torch.ones_like(committed), committed)
        cache.write(0, *kv0, torch.full_like(committed, 2), committed)
        for t in range(0, M, 4):
            path = rows[t][1]
            if path:
                src = _i32(path)
                kp = cache.read(0, torch.ones_like(src), src)
                dst = torch.arange(n, n + len(path), dtype=torch.int32, device=DEV)
                cache.write(0, *kp, torch.full_like(dst, 2), dst)
            step, *_ = _table([[], [], [(n + len(path), [])]])
            one = cache.attend(0, q[t:t + 1], *step, 1, n + len(path))
            assert torch.equal(one[0], tree[t]), (n, t, len(path))


@pytest.mark.parametrize("hd,heads,kv,span", [(128, 32, 8, 64), (64, 24, 8, 128), (128, 40, 8, 64), (64, 16, 16, 192)])
def test_a_batch_equals_each_sequence_alone_bit_for_bit(hd, heads, kv, span):
    """Many rows (several of a sequence in one workgroup) against calls of one sequence and of one row: no bit differs."""
    S = 14
    cache = _cache(1, 900, kv, hd, S, span)
    slots = torch.arange(900, dtype=torch.int32, device=DEV)
    for s in range(S):
        k, v = (torch.randn(900, kv * hd, generator=_gen(s * 2 + i)).to(BF16).to(DEV) for i in range(2))
        cache.write(0, k, v, torch.full_like(slots, s), slots)
    g = _gen(hd + heads)
    rows = [_tree(60 * s + 3, 60 * s + 5, 1 + (5 * s) % 11, g) for s in range(S)]
    rows[4] = [(p - 40 * (i % 2), a) for i, (p, a) in enumerate(rows[4])]  # a sequence of two prefixes
    tab, begin, prefix, depth, anc = _table(rows)
    q = torch.randn(begin[-1], heads * hd, generator=g).to(BF16).to(DEV)
    top = max(p + d for p, d in zip(prefix, depth))
    batch = cache.attend(0, q, *tab, 11, top)
    for s in range(S):
        only, *_ = _table([r if i == s else [] for i, r in enumerate(rows)])
        a, b = begin[s], begin[s + 1]
        l_max = max(p + d for p, d in zip(prefix[a:b], depth[a:b]))
        assert torch.equal(cache.attend(0, q[a:b], *only, b - a, l_max), batch[a:b]), s
        t = a + (b - a) // 2
        one, *_ = _table([[rows[s][t - a]] if i == s else [] for i in range(S)])
        assert torch.equal(cache.attend(0, q[t:t + 1], *one, 1, prefix[t] + depth[t])[0], batch[t]), (s, t)


@pytest.mark.parametrize("hd,heads,kv,span", [(128, 32, 8, 64), (64, 24, 8, 64), (64, 12, 12, 128), (128, 40, 8, 64)])
def test_many_short_trees(hd, heads, kv, span):
    """More rows than are resident one a workgroup, all of few keys: the definition, and every row as it is alone."""
    S = 22
    cache = _cache(1, 256, kv, hd, S, span)
    vals = _fill(cache, hd)
    g = _gen(heads)
    rows = [_tree(9 * s + 1, 9 * s + 3, 1 + s % 7, g) for s in range(S)]
    rows[3], rows[8], rows[9] = [], [(0, [])] * 5, [(0, []), (77, [200, 201]), (0, [255]), (128, []), (63, [1, 0])]
    batch = _check_attend(cache, rows, heads, kv, vals, extra=2, ld_pad=8).view(-1, heads * hd)
    tab, begin, prefix, depth, anc = _table(rows)
    q = torch.randn(begin[-1] + 2, heads * hd + 8, generator=_gen(kv)).to(BF16).to(DEV)[:begin[-1], :heads * hd]
    for s in range(S):
        for t in range(begin[s], begin[s + 1], 2):
            one, *_ = _table([[rows[s][t - begin[s]]] if i == s else [] for i in range(S)])
            assert torch.equal(cache.attend(0, q[t:t + 1], *one, 1, max(prefix[t] + depth[t], 1)).cpu()[0], batch[t]), (s, t)


def test_attend_long_and_past_32_bits():
    """Regions past 4 GiB of codes, and a long context of many spans."""
    kv, hd, heads, cap = 8, 128, 8, 1 << 19
    cache = _cache(1, cap, kv, hd, 9, 1024)
    assert cache.k.numel() > 1 << 32
    for s, slots in ((8, range(cap - 70, cap)), (0, range(0, 5000))):
        slots = _i32(list(slots))
        k, v = (torch.randn(slots.numel(), kv * hd, generator=_gen(s + i)).to(BF16).to(DEV) for i in range(2))
        cache.write(0, k, v, torch.full_like(slots, s), slots)
    rows = [[(5000, []), (4990, [4995])]] + [[]] * 7 + [[(0, [cap - 70 + i for i in range(32)]), (0, [cap - 1])]]
    tab, begin, prefix, depth, anc = _table(rows)
    q = torch.randn(4, heads * hd, generator=_gen(77)).to(BF16)
    got = cache.attend(0, q.to(DEV), *tab, 2, 5000).cpu().view(4, heads, hd).double()
    for t, s, at in ((0, 0, list(range(5000))), (1, 0, list(range(4990)) + [4995]), (2, 8, [cap - 70 + i for i in range(32)]), (3, 8, [cap - 1])):
        k, v = (x.cpu().view(-1, kv, hd).transpose(0, 1)[None] for x in cache.read(0, _i32([s] * len(at)), _i32(at)))
        want, mag = ref.tree_attention(q[t:t + 1].view(1, heads, hd), k, v, [0, 1], [len(at)], [0], [[]])
        assert ((got[t] - want[0]).abs() <= _tolerance(want[0], mag[0])).all(), t


def test_attend_refuses_bad_tensors():
    cache = _cache(1, 128, 2, 64, 2)
    tab, *_ = _table([[(5, [])], [(9, [])]])
    q = torch.zeros(2, 256, dtype=BF16, device=DEV)
    assert cache.attend(0, q[:0], *tab, 1, 9).shape == (0, 256)
    small = torch.empty(10, device=DEV)
    for bad in (lambda: cache.attend(0, q[:, :96], *tab, 1, 9), lambda: cache.attend(0, q.float(), *tab, 1, 9),
                lambda: cache.attend(0, q, tab[0][:2], *tab[1:], 1, 9), lambda: cache.attend(0, q, *tab, 1, 9, ws=small),
                lambda: cache.attend(0, q, *tab, 1, 200), lambda: cache.attend(0, q, tab[0], tab[1].long(), *tab[2:], 1, 9),
                lambda: cache.attend(0, q, *tab[:3], tab[3][:, :16], 1, 9), lambda: cache.attend(0, q, *tab, 1, 9, out=q[:1])):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------------------------------- verification
def _dists(B, K, V, seed, cut=True):
    g = _gen(seed)
    lq = torch.randn(B, K + 1, V, generator=g) * 3
    lp = lq + torch.randn(B, K + 1, V, generator=g) * 0.7
    out = []
    for x in (lp, lq):
        w = torch.exp(x - x.amax(-1, keepdim=True))
        if cut:
            w = torch.where(w < 0.01, torch.zeros_like(w), w)
        out.append(w / w.sum(-1, keepdim=True))
    draft = torch.multinomial(out[1].view(-1, V), 1, generator=g).view(B, K + 1)[:, :K].int()
    return out[0], out[1][:, :K], draft, torch.rand(B, K, generator=g), torch.rand(B, generator=g)


def _same_chain(P, Q, draft, u, nxt, nd=None, ld=0):
    from ssd.engine.verify import verify_chain

    dev = [x.to(DEV) for x in (P, Q, draft, u, nxt)]
    if ld:  # rows of a wider, odd stride
        for i in range(2):
            wide = torch.full((*dev[i].shape[:2], P.shape[2] + ld), float("nan"), device=DEV)
            wide[..., :P.shape[2]] = dev[i]
            dev[i] = wide[..., :P.shape[2]]
    n, tok = verify_chain(*dev[:2], dev[2].contiguous(), dev[3].contiguous(), dev[4], None if nd is None else _i32(nd))
    want_n, want_tok = ref.verify_chain(P, Q, draft, u, nxt, nd)
    assert n.tolist() == want_n and tok.tolist() == want_tok
    return want_n


@pytest.mark.parametrize("B,K,V,ld", [(1, 4, 128256, 0), (7, 3, 32768, 0), (5, 1, 1000, 3), (33, 6, 517, 0), (2, 64, 300, 1), (3, 2, 1, 0),
                                      (4, 5, 4096, 0), (4, 5, 4097, 0), (2, 0, 9000, 0), (2, 2, 600001, 0)])
def test_verify_chain(B, K, V, ld):
    P, Q, draft, u, nxt = _dists(B, K, V, B * 31 + K)
    _same_chain(P, Q, draft, u, nxt, None, ld)
    nd = [(5 * i) % (K + 1) for i in range(B)]
    _same_chain(P, Q, draft, u, nxt, nd, ld)


def test_verify_chain_borders():
    """Tests on the border (u q == p is refused), tokens without mass, tokens outside the vocabulary, counts outside their range,
    rows equal to each other, rows without mass, u_next 0 and the largest below 1."""
    V = 12
    top = 1.0 - 2.0 ** -24
    p, q = torch.zeros(9, 3, V), torch.zeros(9, 2, V)
    p[:, :, 3], p[:, :, 7] = 0.25, 0.75
    q[:, :, 3], q[:, :, 5] = 0.5, 0.5
    draft = torch.tensor([[3, 3], [3, 5], [5, 5], [12, 3], [-1, 3], [7, 7], [3, 3], [3, 3], [3, 3]], dtype=torch.int32)
    u = torch.tensor([[0.5, 0.25], [0.25, 0.0], [0.0, 0.0], [0.0, 0.0], [0.0, 0.0], [top, top], [0.4, 0.4], [0.4, 0.4], [0.6, 0.6]])
    nxt = torch.tensor([0.0, top, 0.5, 0.25, 0.2499, top, 0.1, 0.9, 0.5])
    q[5] = p[5, :2]          # equal rows: refused tokens leave nothing, the target row itself is drawn from
    u[5], draft[5] = 1.0, torch.tensor([7, 7])
    p[7] = 0                 # nothing to draw
    p[8, 0], q[8, 0] = 0, 0  # 0 < 0 is refused
    counts = _same_chain(p, q, draft, u, nxt)
    assert counts[0] == 0 and counts[2] == 0 and counts[3] == 0 and counts[6] == 2
    _same_chain(p, q, draft, u, nxt, [-3, 7, 0, 2, 1, 2, 1, 0, 2])


def test_verify_chain_draws_what_the_rule_says():
    """Accepted and drawn tokens are distributed as the target row (the rule's point): 40000 sequences of one draft."""
    from ssd.engine.verify import verify_chain

    V, B = 8, 40000
    p, q = torch.rand(V, generator=_gen(1)), torch.rand(V, generator=_gen(2))
    p, q = p / p.sum(), q / q.sum()
    draft = torch.multinomial(q.expand(1, V), B, True, generator=_gen(3)).view(B, 1).int()
    u, nxt = torch.rand(B, 1, generator=_gen(4)), torch.rand(B, generator=_gen(5))
    n, tok = verify_chain(p.expand(B, 2, V).to(DEV), q.expand(B, 1, V).to(DEV), draft.to(DEV), u.to(DEV), nxt.to(DEV))
    first = torch.bincount(tok[:, 0].cpu().long(), minlength=V) / B
    # five standard deviations of a count
    assert ((first - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all()
    assert verify_chain(p.expand(0, 2, V).to(DEV), q.expand(0, 1, V).to(DEV), draft[:0].to(DEV), u[:0].to(DEV), nxt[:0].to(DEV))[0].shape == (0,)


def test_verify_chain_refuses_bad_tensors():
    from ssd.engine.verify import verify_chain

    P, Q, draft, u, nxt = (x.to(DEV) for x in _dists(3, 2, 50, 1))
    for bad in (lambda: verify_chain(P.double(), Q, draft, u, nxt), lambda: verify_chain(P, Q[:, :1], draft, u, nxt),
                lambda: verify_chain(P, Q, draft.long(), u, nxt), lambda: verify_chain(P, Q, draft, u[:2], nxt),
                lambda: verify_chain(P.transpose(1, 2).contiguous().transpose(1, 2), Q, draft, u, nxt),
                lambda: verify_chain(P, Q, draft, u, nxt, ws=torch.empty(8, dtype=torch.uint8, device=DEV)),
                lambda: verify_chain(P, Q, draft, u, nxt.cpu())):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------------------------------- together
def _round(cache, st):
    """One batched round's cache work: drafted rows written, attended, verified, committed, and the committed rows read."""
    from ssd.engine.verify import verify_chain

    q = cache.write(0, st["k"], st["v"], st["seq"], st["slot"], rope=st["rope"], pos=st["slot"], q=st["q"])
    out = cache.attend(0, q, *st["tab"], st["rows_max"], st["l_max"])
    n, tok = verify_chain(st["P"], st["Q"], st["draft"], st["u"], st["nxt"])
    cache.compact_device(st["start"], st["src"], n + 1)
    return (q, out, n, tok, *cache.read(0, st["seq"], st["slot"]))


def _round_state(cache, seed, heads, B, K, length):
    from ssd.models.llama import rope_tables_f32

    g = _gen(seed)
    kv, hd, V = cache.kv_heads, cache.head_dim, 600
    lens = torch.randint(length // 2, length, (B,), generator=g).tolist()
    x = torch.randn(B * (K + 1), (heads + 2 * kv) * hd, generator=g).to(BF16).to(DEV)
    # a chain's K + 1 rows written at every second slot behind the committed ones
    slot = [n + 2 * i for n in lens for i in range(K + 1)]
    rows = [[(n + 1, [n + 2 * j for j in range(1, i + 1)]) for i in range(K + 1)] for n in lens]
    P, Q, draft, u, nxt = (t.to(DEV) for t in _dists(B, K, V, seed + 1))
    return dict(q=x[:, :heads * hd], k=x[:, heads * hd:(heads + kv) * hd], v=x[:, (heads + kv) * hd:],
                seq=_i32([s for s in range(B) for _ in range(K + 1)]), slot=_i32(slot),
                rope=rope_tables_f32(length + 64, hd, 1e4, DEV), tab=_table(rows)[0], rows_max=K + 1,
                l_max=length + K + 1, P=P, Q=Q, draft=draft.contiguous(), u=u.contiguous(), nxt=nxt, start=_i32(lens),
                src=_i32([[n + 2 * i for i in range(K + 1)] for n in lens]), rows=rows, lens=lens)


def test_a_round_of_them_against_the_definitions():
    heads, B, K, kv, hd, length = 8, 5, 4, 2, 64, 200
    cache = _cache(1, length + 32, kv, hd, B, 128)
    _fill(cache, 30)
    st = _round_state(cache, 40, heads, B, K, length)
    q, out, n, tok, k2, v2 = _round(cache, st)
    cos, sin = (t.cpu() for t in st["rope"])
    pos = st["slot"].cpu()
    assert torch.equal(q.cpu(), _rot32(st["q"].cpu(), cos, sin, pos, False, hd).to(BF16).flatten(1))
    k_in = ref.stored(_rot32(st["k"].cpu(), cos, sin, pos, False, hd))
    want_n, want_tok = ref.verify_chain(*(st[x].cpu() for x in ("P", "Q", "draft", "u", "nxt")))
    assert n.tolist() == want_n and tok.tolist() == want_tok
    # the committed slots hold the accepted path's rows
    for s in range(B):
        at = torch.arange(st["lens"][s], st["lens"][s] + want_n[s] + 1, dtype=torch.int32, device=DEV)
        k, _ = cache.read(0, torch.full_like(at, s), at)
        assert torch.equal(k.cpu().double(), k_in[s * (K + 1):s * (K + 1) + want_n[s] + 1].flatten(1))
    # the attention, over the cache as it was before the commit: write the rows again
    cache.write(0, st["k"], st["v"], st["seq"], st["slot"], rope=st["rope"], pos=st["slot"])
    slots = torch.arange(cache.capacity, dtype=torch.int32, device=DEV)
    vals = [cache.read(0, torch.full_like(slots, s), slots) for s in range(B)]
    kk, vv = (torch.stack([x[i].cpu().view(-1, kv, hd).transpose(0, 1) for x in vals]) for i in range(2))
    # slots the commit moved into hold other rows than they did: drop sequences whose prefix or path they touch
    tab, begin, prefix, depth, anc = _table(st["rows"])
    got = cache.attend(0, q, *tab, K + 1, st["l_max"]).cpu().view(-1, heads, hd).double()
    want, mag = ref.tree_attention(q.cpu().view(-1, heads, hd), kk, vv, begin, prefix, depth, anc)
    assert ((got - want).abs() <= _tolerance(want, mag)).all()


def test_a_captured_round_replays_with_new_inputs():
    """Two rounds captured into graphs of their own, replayed by turns with eager work between, equal the eager ones."""
    heads, B, K, kv, hd, length = 8, 3, 3, 2, 128, 300
    state, graphs, outs, caches = [], [], [], []
    for i in range(2):
        cache = _cache(1, length + 32, kv, hd, B, 128)
        _fill(cache, 50 + i)
        st = _round_state(cache, 60 + i, heads, B, K, length)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _round(cache, st)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _round(cache, st)
        caches.append(cache), state.append(st), graphs.append(graph), outs.append(out)
    for turn in range(4):
        for i in (0, 1):
            st = state[i]
            g = _gen(100 + turn * 2 + i)
            for name in ("q", "k", "v"):
                st[name].copy_(torch.randn(st[name].shape, generator=g).to(BF16))
            st["u"].copy_(torch.rand(st["u"].shape, generator=g))
        graphs[0].replay(), graphs[1].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            held = [t.clone() for t in outs[i]]
            for a, b in zip(held, _round(caches[i], state[i])):
                assert torch.equal(a, b), (turn, i)


def test_two_streams_at_once():
    """Calls on two streams with buffers of their own."""
    heads, kv, hd = 8, 2, 128
    streams = [torch.cuda.Stream() for _ in range(2)]
    caches = [_cache(1, 500, kv, hd, 2, 64) for _ in range(2)]
    for i, c in enumerate(caches):
        _fill(c, i)
    tab, *_ = _table([_tree(400, 401, 9, _gen(1)), [(333, [])]])
    q = torch.randn(10, heads * hd, generator=_gen(2)).to(BF16).to(DEV)
    want = [c.attend(0, q, *tab, 9, 440).clone() for c in caches]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(caches[i].attend(0, q, *tab, 9, 440))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_prompt_from_the_bf16_cache():
    """A prefilled bf16 cache loaded into a sequence of the 8-bit one."""
    from ssd.engine.kv_cache import KVCache

    kv, hd, n = 2, 64, 150
    bf = KVCache(2, 200, kv, hd, DEV)
    k, v = (torch.randn(1, kv, n, hd, generator=_gen(i)).to(BF16).to(DEV) for i in range(2))
    for i in range(2):
        bf.update(i, k + i, v - i)
    cache = _cache(2, 200, kv, hd, 3)
    for i in range(2):
        cache.load(i, bf, n, seq=1)
        at = torch.arange(n, dtype=torch.int32, device=DEV)
        k2, v2 = cache.read(i, torch.ones_like(at), at)
        assert torch.equal(k2.cpu().double(), ref.stored((k + i)[0].transpose(0, 1).float().cpu()).flatten(1))
        assert torch.equal(v2.cpu().double(), ref.stored((v - i)[0].transpose(0, 1).float().cpu()).flatten(1))
    with pytest.raises(ValueError, match="load"):
        cache.load(0, bf, n, seq=3)


def test_values_that_round_past_the_largest_are_infinite():
    cache = _cache(1, 64, 1, 64)
    top = torch.tensor([1.9375, -1.9296875, 1.75]).double() * 2.0 ** 127
    k = top.to(BF16)[:, None].repeat(1, 64)
    assert torch.equal(k[:, 0].double(), top)
    at = _i32([0, 1, 2])
    cache.write(0, k.to(DEV), k.to(DEV), torch.zeros_like(at), at)
    want = torch.tensor([float("inf"), -1.875 * 2.0 ** 127, 1.75 * 2.0 ** 127]).double()
    for got in cache.read(0, torch.zeros_like(at), at):
        assert torch.equal(got.cpu().double(), want[:, None].expand(3, 64))


@pytest.mark.parametrize("hd,heads,kv", [(128, 16, 4), (64, 32, 8)])
@pytest.mark.parametrize("n", [1, 200, 500, 1000, 2000])
def test_a_larger_bound_changes_no_bit(hd, heads, kv, n):
    """l_max chooses the kernels (one launch, lanes or workgroups for the groups' sum), not the result."""
    cache = _cache(1, 4096, kv, hd, 2, 64)
    vals = _fill(cache, hd)
    rows = [_tree(n, n + 2, 7, _gen(n)), [(n // 2, []), (0, [n + 1]), (0, [])]]
    want = _check_attend(cache, rows, heads, n, vals)
    for l_max in (256, 512, 1024, 2048, 2304, 4096):
        if l_max >= n + 8:
            assert torch.equal(_check_attend(cache, rows, heads, n, vals, l_max=l_max), want), l_max


def test_rebuilt_caches_keep_no_device_memory():
    import gc

    from ssd.models.llama import rope_tables_f32

    def use():
        cache = _cache(2, 4096, 8, 128, 4)
        rope = rope_tables_f32(64, 128, 1e4, DEV)
        k, at = torch.ones(3, 1024, dtype=BF16, device=DEV), _i32([0, 1, 2])
        q = cache.write(1, k, k, at, at, rope=rope, pos=at, q=k)
        cache.attend(1, q, _i32([0, 1, 2, 3, 3]), at + 1, at * 0, torch.zeros(3, 32, dtype=torch.int32, device=DEV), 1, 4)
        cache.compact_device(_i32([0] * 4), _i32([[0]] * 4), _i32([1] * 4))
        assert cache.read(1, at, at)[1].eq(1).all()

    use()
    gc.collect(), torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    for _ in range(3):
        use()
    gc.collect(), torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() <= held


def test_slots_up_to_the_capacity_exist():
    """max_length 200: 256 slots are written, read, loaded, attended and moved into; 256 and 257 are not there."""
    from ssd.engine.kv_cache import KVCache

    kv, hd, heads = 2, 64, 4
    cache = _cache(1, 200, kv, hd, 2, 64)
    x = torch.randn(5, kv * hd, generator=_gen(1)).to(BF16)
    at = _i32([199, 200, 255, 256, 257])
    cache.write(0, x.to(DEV), x.to(DEV), torch.ones_like(at), at)
    for got in cache.read(0, torch.ones_like(at), at):
        assert _same(got[:3].cpu(), ref.stored(x[:3].float().view(3, kv, hd)).flatten(1)) and not got[3:].any()
    bf = KVCache(1, 256, kv, hd, DEV)
    k, v = (torch.randn(1, kv, 256, hd, generator=_gen(2 + i)).to(BF16).to(DEV) for i in range(2))
    bf.update(0, k, v)
    cache.load(0, bf, 256)
    every = torch.arange(256, dtype=torch.int32, device=DEV)
    vals = [t.cpu().view(256, kv, hd).transpose(0, 1)[None].expand(2, -1, -1, -1) for t in cache.read(0, torch.zeros_like(every), every)]
    assert _same(vals[0][0], ref.stored(k[0].float().cpu())) and _same(vals[1][0], ref.stored(v[0].float().cpu()))
    _check_attend(cache, [[(256, []), (250, [255]), (0, [200])], []], heads, 5, vals)
    cache.compact_device(_i32([254, 0]), _i32([[3, 4, 5], [0, 0, 0]]), _i32([3, 0]))
    moved = cache.read(0, torch.zeros_like(every), every)[0].cpu().view(256, kv, hd).transpose(0, 1)
    assert torch.equal(moved[:, 254:], vals[0][0][:, 3:5]) and torch.equal(moved[:, :254], vals[0][0][:, :254])


@pytest.mark.parametrize("hd,kv,heads,interleaved,rot", [(128, 8, 32, False, 128), (128, 8, 1, True, 64), (64, 8, 6, False, 32),
                                                         (64, 8, 32, True, 64), (128, 8, 6, False, 96)])
@pytest.mark.parametrize("scattered", [False, True])
def test_long_rotated_writes(hd, kv, heads, interleaved, rot, scattered):
    """Calls of 6144 (row, kv head) pairs and more take four rows and four q heads a unit: a prompt's consecutive slots from an odd
    one on, and rows at any place with some outside the cache; exactly the definition, and nothing else written."""
    from ssd.models.llama import rope_tables_f32

    rows, seqs, first = 803, 2, 37
    g = _gen(hd + heads + scattered)
    x = (torch.randn(rows, (heads + 2 * kv) * hd, generator=g) * torch.logspace(-2, 2, hd).repeat(heads + 2 * kv)).to(BF16)
    q, k, v = x[:, :heads * hd], x[:, heads * hd:(heads + kv) * hd], x[:, (heads + kv) * hd:]
    cache = _cache(1, 900, kv, hd, seqs)
    cap = cache.capacity
    if scattered:
        places = torch.randperm(seqs * cap, generator=g)[:rows]
        seq, slot = (places // cap).int(), (places % cap).int()
        for i, (s, t) in enumerate(((-1, 3), (seqs, 4), (0, -1), (1, cap))):
            seq[200 * i + i], slot[200 * i + i] = s, t
    else:
        seq, slot = torch.ones(rows, dtype=torch.int32), torch.arange(first, first + rows, dtype=torch.int32)
    pos = torch.randint(-2, 4100, (rows,), generator=g, dtype=torch.int32)
    cos, sin = rope_tables_f32(4096, rot, 500000.0, "cpu")
    for t in (cache.k, cache.v, cache.k_exp, cache.v_exp):
        t.fill_(93)
    xd = x.to(DEV)
    qd, kd, vd = xd[:, :heads * hd], xd[:, heads * hd:(heads + kv) * hd], xd[:, (heads + kv) * hd:]
    got_q = cache.write(0, kd, vd, seq.to(DEV), slot.to(DEV), rope=(cos.to(DEV), sin.to(DEV)), pos=pos.to(DEV), interleaved=interleaved, q=qd)
    assert _same(got_q.cpu(), _rot32(q, cos, sin, pos, interleaved, hd).to(BF16).flatten(1))
    there = (seq >= 0) & (seq < seqs) & (slot >= 0) & (slot < cap)
    assert int(there.sum()) == rows - 4 * scattered
    k2, v2 = (t.cpu() for t in cache.read(0, seq.to(DEV), slot.to(DEV)))
    assert _same(k2[there], ref.stored(_rot32(k, cos, sin, pos, interleaved, hd)).flatten(1)[there])
    assert _same(v2[there], ref.stored(v.float().view(rows, kv, hd)).flatten(1)[there])
    assert not k2[~there].any() and not v2[~there].any()
    # the other slots' bytes are as they were, codes and exponents
    every = torch.zeros(seqs, cap, dtype=torch.bool)
    every[seq[there].long(), slot[there].long()] = True
    at = torch.tensor([ref.x_offset(s) for s in range(cap)])
    for t in (cache.k_exp, cache.v_exp):
        assert (t[0].cpu()[:, :, at][~every[:, None].expand(-1, kv, -1)] == 93).all()
    for t, off in ((cache.k, ref.k_offset), (cache.v, ref.v_offset)):
        at_d = torch.tensor([[off(s, d, hd) for d in (0, 31, hd - 1)] for s in range(cap)])
        assert (t[0].cpu()[:, :, at_d][~every[:, None, :, None].expand(-1, kv, -1, 3)] == 93).all()


@pytest.mark.parametrize("hd,heads,interleaved,in_place", [(128, 1, False, False), (64, 6, True, True), (64, 3, False, True), (128, 5, True, False)])
def test_rope_of_many_rows(hd, heads, interleaved, in_place):
    """6144 rows and more: four heads of a row a unit, whatever the head count."""
    from ssd import ops
    from ssd.models.llama import rope_tables_f32

    rows, g = 6147, _gen(heads)
    x = torch.randn(rows, heads * hd + 8, generator=g).to(BF16)
    pos = torch.randint(-5, 9000, (rows,), generator=g, dtype=torch.int32)
    cos, sin = rope_tables_f32(8192, hd // 2, 1e4, "cpu")
    xd = x.to(DEV)
    out = xd if in_place else torch.zeros_like(xd)
    ops.rope(xd, rows, heads, hd, (cos.to(DEV), sin.to(DEV)), pos.to(DEV), out, interleaved)
    assert torch.equal(out[:, :heads * hd].cpu(), _rot32(x[:, :heads * hd], cos, sin, pos, interleaved, hd).to(BF16).flatten(1))
    assert torch.equal(out[:, heads * hd:].cpu(), x[:, heads * hd:] if in_place else torch.zeros(rows, 8, dtype=BF16))


@pytest.mark.parametrize("hd,heads,kv", [(128, 4, 1), (64, 4, 2)])
@pytest.mark.parametrize("n", [16385, 16449, 33100])
def test_attend_more_groups_than_lanes(hd, heads, kv, n):
    """A group is 256 keys at a span of 64: past 64 of them the sum of the groups takes further turns (65, 65 and 130 here)."""
    cache = _cache(1, 33280, kv, hd, 1, 64)
    vals = _fill(cache, n)
    rows = _tree(n, n + 2, 4, _gen(n)) + [(16384, []), (16380, [n + 1, n]), (0, [])]
    got = _check_attend(cache, [rows], heads, n, vals)
    assert torch.equal(_check_attend(cache, [rows], heads, n, vals, l_max=33280), got)


def test_the_attention_inside_a_round():
    """What a round's attention returns, against the definition over the cache as the round's write leaves it, and its bits
    against the same call outside a round."""
    heads, B, K, kv, hd, length = 8, 5, 4, 2, 64, 200
    caches = [_cache(1, length + 32, kv, hd, B, 128) for _ in range(2)]
    for c in caches:
        _fill(c, 30)
    st = _round_state(caches[0], 40, heads, B, K, length)
    q, out, *_ = _round(caches[0], st)
    other = caches[1]
    assert torch.equal(other.write(0, st["k"], st["v"], st["seq"], st["slot"], rope=st["rope"], pos=st["slot"], q=st["q"]), q)
    slots = torch.arange(other.capacity, dtype=torch.int32, device=DEV)
    vals = [other.read(0, torch.full_like(slots, s), slots) for s in range(B)]
    kk, vv = (torch.stack([x[i].cpu().view(-1, kv, hd).transpose(0, 1) for x in vals]) for i in range(2))
    tab, begin, prefix, depth, anc = _table(st["rows"])
    want, mag = ref.tree_attention(q.cpu().view(-1, heads, hd), kk, vv, begin, prefix, depth, anc)
    assert ((out.cpu().view(-1, heads, hd).double() - want).abs() <= _tolerance(want, mag)).all()
    assert torch.equal(other.attend(0, q, *tab, K + 1, st["l_max"]), out)


def test_places_of_no_sequence_read_zeros():
    cache = _cache(1, 64, 2, 64, 2)
    _fill(cache, 6)
    for s, t in ((-1, 5), (2, 5), (1 << 30, 0), (0, -1), (1, 64), (-(1 << 31), -(1 << 31))):
        k, v = cache.read(0, _i32([s, 1]), _i32([t, 3]))
        assert not k[0].any() and not v[0].any() and k[1].any() and v[1].any()
