"""The paged cache's operators on the GPU against 64-bit definitions (oracle.paged)."""

import pytest
import torch

from oracle import paged as ref

pytestmark = pytest.mark.gpu
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
NAN = float("nan")


def i32(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def sums(x):
    return [sum(x[:i]) for i in range(len(x) + 1)]


class Setup:
    """A cache whose pool holds NaN wherever no row has been written, and a batch of sequences on it. lens: slots in use, new rows
    included; rows: new rows of each sequence."""

    def __init__(self, lens, rows, heads, kv, hd, seed=0, cols=None, spare=3, layers=1, span=None, poison=True):
        from ssd.engine.kv_cache import PagedBatch, PagedKVCache

        g = torch.Generator().manual_seed(seed)
        self.lens, self.rows, self.heads, self.kv, self.hd, self.g = lens, rows, heads, kv, hd, g
        need = [(n + 63) // 64 for n in lens]
        cols = cols or max(max(need), 1)
        self.cache = PagedKVCache(layers, sum(need) + spare, kv, hd, "cuda", span=span)
        if poison:
            self.cache.k.fill_(NAN)
            self.cache.v.fill_(NAN)
        ids = torch.randperm(sum(need) + spare, generator=g).tolist()
        self.ids = [[ids.pop() for _ in range(c)] for c in need]
        table = [p + [10 ** 6] * (cols - len(p)) for p in self.ids]
        self.table, self.lengths, self.begin = i32(table), i32(lens), i32(sums(rows))
        self.PB = PagedBatch
        self.batch = PagedBatch(self.table, self.lengths, self.begin, max(max(rows), 0))
        self.all = PagedBatch(self.table, self.lengths, i32(sums(lens)), max(lens))
        self.k = [torch.randn(n, kv, hd, generator=g).to(BF16) for n in lens]
        self.v = [torch.randn(n, kv, hd, generator=g).to(BF16) for n in lens]
        self.q = (torch.randn(sum(rows), heads * hd, generator=g) * 1.5).to(BF16)

    def fill(self, layer=0):
        cat = lambda x: torch.cat([t.flatten(1) for t in x]).cuda() if sum(self.lens) else torch.zeros(0, self.kv * self.hd, dtype=BF16).cuda()  # noqa: E731
        self.cache.write(layer, cat(self.k), cat(self.v), self.all)
        return self

    def last(self, s):
        return [self.lens[s] - self.rows[s] + i for i in range(self.rows[s])]

    def check(self, out, weights=None, start=None, decay=0.0):
        out = out.double().cpu().view(-1, self.heads, self.hd)
        b = sums(self.rows)
        for s, n in enumerate(self.rows):
            q = self.q[b[s]:b[s + 1]].view(n, self.heads, self.hd)
            want, mag, w, size = ref.attention(q, self.k[s], self.v[s], self.last(s))
            got = out[b[s]:b[s + 1]]
            # each weight is rounded to bf16 once (2^-8 of it), the result once; scores are sums of hd products in fp32
            slack = 2.0 ** -24 * (4 * self.hd * size[..., None] + 4 * self.lens[s] + 256)
            tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + slack) * mag * (1 + 2.0 ** -8) + 1e-30
            bad = (got - want).abs() > tol
            assert not bad.any(), (s, int(bad.sum()), float(((got - want).abs() - tol).max()))
            if weights is not None:
                total = w.view(n, self.kv, self.heads // self.kv, self.lens[s]).sum((0, 2))
                old = start[s, :, :self.lens[s]].double().cpu() * decay
                mine = weights[s, :, :self.lens[s]].double().cpu()
                # relative error of each weight: exponent (the score's error), l's sum; then the sum over rows and heads
                rel = 2.0 ** -24 * (4 * self.hd * float(size.max() if size.numel() else 0) + 2 * self.lens[s] + 2 * n * self.heads + 256)
                assert ((mine - (old + total)).abs() <= rel * (total + old) + 1e-30).all(), s
                assert torch.equal(weights[s, :, self.lens[s]:].cpu(), start[s, :, self.lens[s]:].cpu())


SHAPES = [(32, 8, 128), (32, 8, 64), (15, 5, 128), (16, 16, 64), (64, 8, 128), (20, 1, 64), (2, 2, 128)]


# ------------------------------------------------------------------------------------------------- write, read
@pytest.mark.parametrize("kv,hd", [(8, 128), (5, 64), (1, 128)])
def test_write_fills_exactly_its_slots_and_read_gives_them_back(kv, hd):
    from ssd import ops

    lens, rows = [0, 1, 64, 65, 200, 130, 63, 9], [0, 1, 64, 3, 200, 66, 5, 2]
    s = Setup(lens, rows, kv, kv, hd, cols=5)
    wide = torch.randn(sum(rows), 3 * kv * hd, generator=s.g).to(BF16).cuda()
    k, v = wide[:, :kv * hd], wide[:, 2 * kv * hd:]  # column ranges of one matrix
    want_k, want_v = s.cache.k.clone(), s.cache.v.clone()
    ki, vi = ops.kv_block_index(64, hd, "cuda")
    at = 0
    for q, (n, m) in enumerate(zip(lens, rows)):
        for i in range(m):
            t = n - m + i
            want_k[0, s.ids[q][t // 64]][:, ki[t % 64]] = k[at].view(kv, hd)
            want_v[0, s.ids[q][t // 64]][:, vi[t % 64]] = v[at].view(kv, hd)
            at += 1
    s.cache.write(0, k, v, s.batch)
    for a, b in ((s.cache.k, want_k), (s.cache.v, want_v)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    rk, rv = s.cache.read(0, s.batch, sum(rows))
    assert torch.equal(rk, k) and torch.equal(rv, v)
    out = torch.full((sum(rows) + 2, 2 * kv * hd), 7.0, dtype=BF16, device="cuda")
    s.cache.read(0, s.batch, sum(rows), out[:, :kv * hd], out[:, kv * hd:])
    assert torch.equal(out[:-2], torch.cat([k, v], 1)) and (out[-2:] == 7).all()  # rows of no sequence stay


def test_places_that_do_not_exist():
    """Pages outside the pool, slots beyond the table, rows before slot 0."""
    from ssd.engine.kv_cache import PagedBatch, PagedKVCache

    kv, hd = 2, 64
    cache = PagedKVCache(2, 3, kv, hd, "cuda")
    table = i32([[-1, 0], [1, 3], [2, 2 ** 31 - 1], [5, 5]])
    lengths, begin = i32([70, 200, 4, -5]), i32([0, 70, 160, 170, 172])
    b = PagedBatch(table, lengths, begin, 90)
    x = torch.randn(172, kv * hd, device="cuda").to(BF16)
    cache.write(1, x, x + 1, b)
    assert not cache.k[0].any() and not cache.v[0].any()  # the other layer
    k, v = cache.read(1, b, 172)
    want = torch.zeros_like(x)
    want[64:70] = x[64:70]  # sequence 0: slots 64 .. 69 in page 0
    want[166:170] = x[166:170]  # sequence 2: rows 0 .. 5 before slot 0 (sequence 1: slots 110 .. 199, page 3 of 3 and none)
    lost = want.abs().sum(1) == 0
    assert torch.equal(k, want) and not v[lost].any() and torch.equal(v[~lost], (x + 1)[~lost])
    assert not cache.k[1, 1].any()


def test_rows_beyond_rows_max_and_empty_calls():
    s = Setup([5, 3], [5, 3], 2, 2, 64)
    few = s.PB(s.table, s.lengths, s.begin, 2)  # the first two rows of each are taken
    x = torch.randn(8, 128, device="cuda").to(BF16)
    s.cache.write(0, x, x, few)
    k, _ = s.cache.read(0, s.batch, 8)
    assert torch.equal(k[[0, 1, 5, 6]], x[[0, 1, 5, 6]]) and k[[2, 3, 4, 7]].isnan().all()
    before = s.cache.k.clone()
    s.cache.write(0, x[:0], x[:0], s.batch)
    none = s.PB(s.table[:0], s.lengths[:0], s.begin[:1], 4)
    s.cache.write(0, x, x, none)
    assert torch.equal(s.cache.k.view(torch.int16), before.view(torch.int16))
    assert s.cache.attend(0, x[:0], s.batch).shape == (0, 128) and s.cache.attend_prompt(0, x[:0], s.batch).shape == (0, 128)


# ------------------------------------------------------------------------------------------------- attention
LENS = [([1, 2, 63, 64, 65, 128, 129, 0, 300], [1, 1, 1, 1, 1, 1, 1, 1, 1]), ([5, 64, 70, 200, 0, 130], [5, 3, 2, 7, 2, 1]),
        ([700], [1]), ([1030, 257], [4, 16])]


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("lens,rows", LENS)
def test_attend_and_attend_prompt(heads, kv, hd, lens, rows):
    s = Setup(lens, rows, heads, kv, hd, seed=heads + hd).fill()
    s.check(s.cache.attend(0, s.q.cuda(), s.batch, max(lens)))
    s.check(s.cache.attend_prompt(0, s.q.cuda(), s.batch, max(lens)))


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
def test_attend_prompt_of_many_rows(heads, kv, hd):
    lens, rows = [150, 64, 65, 33, 1, 290, 0, 200], [150, 64, 65, 33, 1, 100, 0, 129]
    s = Setup(lens, rows, heads, kv, hd, seed=3).fill()
    s.check(s.cache.attend_prompt(0, s.q.cuda(), s.batch))


def test_attend_prompt_large_tiles_and_many_sequences():
    """Enough rows for the larger tiles, and more sequences than a wave has lanes."""
    lens = [1 + 37 * i % 90 for i in range(150)]
    s = Setup(lens, lens, 16, 2, 64, seed=4).fill()
    s.check(s.cache.attend_prompt(0, s.q.cuda(), s.batch))
    s = Setup([900, 1200], [900, 300], 32, 8, 128, seed=5).fill()
    out = s.cache.attend_prompt(0, s.q.cuda(), s.batch)
    s.rows, s.q, whole = [3, 2], torch.cat([s.q[897:900], s.q[1198:1200]]), out  # the last rows of both against 64 bits
    s.check(torch.cat([whole[897:900], whole[1198:1200]]))


def test_attend_prompt_more_than_64_pages():
    s = Setup([64 * 66 + 5], [70], 4, 1, 128, seed=6).fill()
    s.check(s.cache.attend_prompt(0, s.q.cuda(), s.batch))


@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (15, 5, 128), (16, 16, 64)])
def test_attend_prompt_of_few_rows_behind_a_long_past(heads, kv, hd):
    """The length in parts, which some sequences do not reach."""
    lens, rows = [4400, 900, 64, 3000, 0, 1], [20, 33, 5, 1, 2, 1]
    s = Setup(lens, rows, heads, kv, hd, seed=30).fill()
    ws = torch.full((s.cache.prompt_floats(sum(rows), heads, s.batch),), NAN, device="cuda")
    assert ws.numel()
    s.check(s.cache.attend_prompt(0, s.q.cuda(), s.batch, ws=ws))
    s.table[0, 1:40] = -1  # whole parts without a page
    out = s.cache.attend_prompt(0, s.q.cuda(), s.batch)[:20].double().cpu().view(20, heads, hd)
    keep = [t for t in range(4400) if not 64 <= t < 40 * 64]
    want, mag, _, _ = ref.attention(s.q[:20].view(20, heads, hd), s.k[0][keep], s.v[0][keep], [len(keep) - 20 + i for i in range(20)])
    assert ((out - want).abs() <= 2 ** -8 * want.abs() + 2 ** -7.9 * mag).all()


@pytest.mark.parametrize("span", [64, 192, 1024, 4096])
def test_spans_and_rows_alone_or_in_a_batch(span):
    lens, rows = [1500, 64, 900, 3], [3, 1, 5, 2]
    s = Setup(lens, rows, 32, 8, 128, seed=7, span=span, cols=30).fill()
    out = s.cache.attend(0, s.q.cuda(), s.batch, 1920)
    s.check(out)
    b = sums(rows)
    for q in range(4):
        for i in range(rows[q]):  # a row as a step of its own, its sequence that long
            one = s.PB(s.table[q:q + 1], i32([lens[q] - rows[q] + i + 1]))
            alone = s.cache.attend(0, s.q[b[q] + i:b[q] + i + 1].cuda(), one, lens[q])
            assert torch.equal(alone[0], out[b[q] + i])


def test_attention_of_rows_in_strided_tensors_and_rows_of_no_sequence():
    s = Setup([100, 70], [2, 70], 8, 2, 64, seed=8).fill()
    wide = torch.zeros(74, 1536, dtype=BF16, device="cuda")
    wide[1:73, 512:1024] = s.q.cuda()
    b = s.PB(s.table, s.lengths, i32([1, 3, 73]), 70)
    for f in (s.cache.attend, s.cache.attend_prompt):
        out = torch.full((74, 640), 7.0, dtype=BF16, device="cuda")
        f(0, wide[:, 512:1024], b, out=out[:, 64:576])
        s.check(out[1:73, 64:576])
        assert (out[[0, 73]] == 7).all() and (out[:, :64] == 7).all() and (out[:, 576:] == 7).all()


def test_lengths_beyond_the_bound_are_cut_there():
    s = Setup([200, 130], [1, 2], 8, 2, 64, seed=9).fill()
    for f in (s.cache.attend, s.cache.attend_prompt):
        out = f(0, s.q.cuda(), s.batch, 100)
        short = [ref.attention(s.q[i:i + 1].view(1, 8, 64), s.k[q], s.v[q], [99])[0] for i, q in enumerate((0, 1, 1))]
        assert (out.cpu().double() - torch.cat(short).flatten(1)).abs().max() < 2 ** -6


def test_pages_outside_the_pool_are_not_attended():
    s = Setup([300], [2], 8, 2, 128, seed=10).fill()
    s.table[0, 1], s.table[0, 4] = -7, 99
    keep = [t for t in range(300) if t // 64 not in (1, 4)]
    want, mag, w, _ = ref.attention(s.q.view(2, 8, 128), s.k[0][keep], s.v[0][keep], [len(keep) - 1] * 2)
    weights = torch.full((1, 2, 320), 5.0, device="cuda")
    for out in (s.cache.attend(0, s.q.cuda(), s.batch, weights=weights, decay=0.0), s.cache.attend_prompt(0, s.q.cuda(), s.batch)):
        assert ((out.cpu().double().view_as(want) - want).abs() <= 2 ** -8 * want.abs() + 2 ** -7 * mag).all()
    got = weights[0].cpu().double()
    assert (got[:, keep] - w.view(2, 2, 4, -1).sum((0, 2))).abs().max() < 1e-5 and not got[:, 64:128].any() and not got[:, 256:300].any()
    s.table.fill_(-1)
    for f in (s.cache.attend, s.cache.attend_prompt):
        assert not f(0, s.q.cuda(), s.batch).any()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [NAN, float("inf")])
def test_values_that_are_not_finite_reach_the_rows_that_attend_them(hd, value):
    """V of slot 75, dim 3 and K of slot 85: rows before them keep their results."""
    s = Setup([90], [20], 4, 2, hd, seed=11).fill()  # slots 70 .. 89
    want = [f(0, s.q.cuda(), s.batch).view(20, 4, hd) for f in (s.cache.attend, s.cache.attend_prompt)]
    s.v[0][75, 1, 3] = value
    s.k[0][85, 0] = NAN
    s.fill()
    for f, w in zip((s.cache.attend, s.cache.attend_prompt), want):
        out = f(0, s.q.cuda(), s.batch).view(20, 4, hd)
        assert not out[5:, 2:, 3].isfinite().any() and out[15:, :2].isnan().all()
        out[5:, 2:, 3], w[5:, 2:, 3] = 0, 0
        assert torch.equal(out[:15], w[:15]) and torch.equal(out[:, 2:], w[:, 2:])


def test_large_scores_and_a_given_scale():
    s = Setup([400], [3], 4, 2, 64, seed=12)
    s.q, s.k[0] = s.q * 30, s.k[0] * 8  # weights of one key or two
    s.fill()
    for f in (s.cache.attend, s.cache.attend_prompt):
        s.check(f(0, s.q.cuda(), s.batch))
        out = f(0, s.q.cuda(), s.batch, scale=1e-4).double().cpu().view(3, 4, 64)
        want, mag, _, _ = ref.attention(s.q.view(3, 4, 64), s.k[0], s.v[0], s.last(0), 1e-4)
        assert ((out - want).abs() <= 2 ** -8 * want.abs() + 2 ** -7.9 * mag).all()


def test_places_past_2_to_the_31_elements():
    from ssd.engine.kv_cache import PagedBatch, PagedKVCache

    kv, hd = 8, 128
    cache = PagedKVCache(1, 33000, kv, hd, "cuda")  # 65536 elements a page
    table = i32([[32999, 0, 32900]])
    b = PagedBatch(table, i32([150]), i32([0, 150]), 150)
    x = torch.randn(150, 2 * kv * hd, generator=torch.Generator().manual_seed(13)).to(BF16).cuda()
    k, v = x[:, :kv * hd], x[:, kv * hd:]
    cache.write(0, k, v, b)
    rk, rv = cache.read(0, b, 150)
    assert torch.equal(rk, k) and torch.equal(rv, v)
    q = torch.randn(1, 2 * kv * hd, generator=torch.Generator().manual_seed(14)).to(BF16).cuda()
    want = ref.attention(q.cpu().view(1, 2 * kv, hd), k.cpu().view(-1, kv, hd), v.cpu().view(-1, kv, hd), [149])[0].flatten(1)
    one = PagedBatch(table, i32([150]))
    for f in (cache.attend, cache.attend_prompt):
        assert (f(0, q, one).double().cpu() - want).abs().max() < 2 ** -6
    after = PagedBatch(i32([[32998]]), i32([0]))
    kept, _ = cache.evict(one, after, torch.arange(192.0, device="cuda").expand(1, 1, kv, 192).contiguous(), 20, 5, 3)
    assert torch.equal(cache.read(0, PagedBatch(after.table, after.lengths, i32([0, 20]), 20), 20)[0], k[kept[0, 0, 0].long()])


# ------------------------------------------------------------------------------------------------- received weights
@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (15, 5, 128), (16, 16, 64), (20, 1, 64), (64, 8, 128)])
@pytest.mark.parametrize("decay", [0.0, 0.5, 1.0])
def test_received_weights(heads, kv, hd, decay):
    lens, rows = [1, 700, 0, 130, 64, 1100], [1, 3, 1, 16, 2, 1]
    s = Setup(lens, rows, heads, kv, hd, seed=15).fill()
    store = torch.rand(len(lens), kv + 1, 1200, generator=torch.Generator().manual_seed(1)).cuda()
    if decay == 0.0:
        store.fill_(NAN)  # not read
    weights = store[:, 1:, :1160]
    start = weights.clone()
    out = s.cache.attend(0, s.q.cuda(), s.batch, 1100, weights=weights, decay=decay)
    if decay == 0.0:
        for i, n in enumerate(lens):
            assert not weights[i, :, :n].isnan().any() and weights[i, :, n:].isnan().all()
        start, weights = start.nan_to_num(0.0), weights.nan_to_num(0.0)
    s.check(out, weights, start, decay)
    assert torch.equal(out, s.cache.attend(0, s.q.cuda(), s.batch, 1100))  # with or without
    if decay == 1.0:  # and again: in a fixed order
        again = start.clone()
        s.cache.attend(0, s.q.cuda(), s.batch, 1100, weights=again, decay=1.0)
        assert torch.equal(again, weights)


def test_more_pairs_than_the_weights_kernel_holds_at_once():
    s = Setup([330], [20], 20, 1, 64, seed=16).fill()  # 400 (row, head) pairs of one kv head
    weights = torch.zeros(1, 1, 330, device="cuda")
    s.check(s.cache.attend(0, s.q.cuda(), s.batch, 330, weights=weights), weights, torch.zeros_like(weights))


@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (15, 5, 128), (16, 16, 64), (64, 8, 64)])
@pytest.mark.parametrize("rows", [1, 2, 16, 17])
def test_received_weights_of_a_step_and_of_a_window(heads, kv, hd, rows):
    """Both sides of the number of pairs up to which scores are kept, several groups, and a sequence that takes no part."""
    lens, rows = [600, 333, 70, 2400], [rows, 0, rows, 1]
    s = Setup(lens, rows, heads, kv, hd, seed=31, span=64).fill()
    weights = torch.rand(4, kv, 2500, generator=torch.Generator().manual_seed(2)).cuda()
    start = weights.clone()
    out = s.cache.attend(0, s.q.cuda(), s.batch, 2432, weights=weights, decay=0.75)
    assert torch.equal(weights[1], start[1])  # without rows: as they were
    start[1, :, :333] /= 0.75  # what check expects to have been decayed
    s.check(out, weights, start, 0.75)


def test_weights_where_a_pair_attends_scores_of_minus_infinity_alone():
    s = Setup([40, 100], [1, 20], 4, 1, 64, seed=32).fill()
    s.q[:] = 0
    s.q[:, ::64] = 1.0
    s.k[0][..., 0], s.k[1][..., 0] = float("-inf"), float("-inf")
    s.fill()
    weights = torch.zeros(2, 1, 128, device="cuda")
    for b, q, w in ((s.batch, s.q, weights), (s.PB(s.table[:1], s.lengths[:1]), s.q[:1], weights[:1])):  # from K again, and kept
        out = s.cache.attend(0, q.cuda(), b, weights=w, decay=0.0)
        assert not out.any() and not w.any()


def test_sequences_that_share_pages():
    """A common prefix of two whole pages in one place, and as many copies."""
    s = Setup([200, 170], [9, 3], 32, 8, 128, seed=33).fill()
    s.k[1][:128], s.v[1][:128] = s.k[0][:128], s.v[0][:128]
    s.table[1, :2] = s.table[0, :2]
    weights = torch.zeros(2, 8, 256, device="cuda")
    s.check(s.cache.attend(0, s.q.cuda(), s.batch, weights=weights), weights, torch.zeros_like(weights))
    s.check(s.cache.attend_prompt(0, s.q.cuda(), s.batch))


@pytest.mark.parametrize("rows", [4, 7])
def test_attend_prompt_of_a_round_of_pieces_behind_a_past(rows):
    """As many workgroups as one round and a little more, whose waves take turns, and a bound that ends it."""
    lens = [150 + 37 * i % 400 for i in range(17)]
    s = Setup(lens, [rows] * 17, 32, 32, 128, seed=34).fill()
    s.check(s.cache.attend_prompt(0, s.q.cuda(), s.batch))


# ------------------------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("hd,kv", [(128, 2), (64, 3)])
@pytest.mark.parametrize("keep,recent,first", [(64, 8, 4), (100, 0, 0), (1, 0, 0), (1, 1, 0), (130, 100, 30), (600, 5, 1), (63, 0, 63)])
def test_evict(hd, kv, keep, recent, first):
    lens = [0, 1, 63, 64, 65, 300, 700]
    s = Setup(lens, [1] * 7, kv, kv, hd, seed=17, layers=2, spare=80).fill(0)
    ks, vs = [s.k], [s.v]
    s.k, s.v = [x + 1 for x in s.k], [x - 1 for x in s.v]
    s.fill(1)
    ks.append(s.k), vs.append(s.v)
    w = torch.rand(2, 7, kv, 710, generator=s.g)
    w[:, :, :, ::3] = 0.25  # equal ones
    w[0, 5, 0, 20], w[0, 5, 0, 40], w[1, 5, 0, 30] = NAN, -1.0, -0.0
    w[1, 6, 0] = 0.0
    w[1, 6, 0, 1::2] = -0.0  # all equal
    unused = [p for p in range(s.cache.pages) if p not in sum(s.ids, [])]
    cols = (keep + 63) // 64
    new = i32([[unused.pop() if c * 64 < min(n, keep) else -1 for c in range(cols)] for n in lens])
    after = s.PB(new, i32([9] * 7), i32(sums([min(n, keep) for n in lens])), min(keep, 700))
    old_k = s.cache.k.clone()
    kept, moved = s.cache.evict(s.batch, after, w.cuda(), keep, recent, first)
    assert after.lengths.tolist() == [min(n, keep) for n in lens]
    used = sorted(set(sum(s.ids, [])))
    assert torch.equal(s.cache.k[:, used].view(torch.int16), old_k[:, used].view(torch.int16))  # the old pages stay
    for layer in range(2):
        rk, rv = (x.cpu().view(-1, kv, hd) for x in s.cache.read(layer, after, sum(min(n, keep) for n in lens)))
        at = 0
        for q, n in enumerate(lens):
            for h in range(kv):
                want = ref.evict(w[layer, q, h], n, keep, recent, first)
                assert kept[layer, q, h].tolist() == want + [-1] * (keep - len(want)), (layer, q, h)
                m = moved[layer, q, h].cpu()
                assert torch.equal(m[:len(want)].view(I32), w[layer, q, h, want].view(I32)) and not m[len(want):].any()
                assert torch.equal(rk[at:at + len(want), h], ks[layer][q][want, h]) and torch.equal(rv[at:at + len(want), h], vs[layer][q][want, h])
            at += min(n, keep)


def test_evict_of_long_rows_and_into_the_old_lengths():
    from ssd.engine.kv_cache import PagedBatch, PagedKVCache

    kv, n, keep = 2, 20000, 5000
    cache = PagedKVCache(1, 313 + 79, kv, 64, "cuda")
    g = torch.Generator().manual_seed(18)
    lengths = i32([n])
    batch = PagedBatch(i32([list(range(313))]), lengths, i32([0, n]), n)
    k = torch.randn(n, kv * 64, generator=g).to(BF16).cuda()
    cache.write(0, k, -k, batch)
    w = torch.randint(0, 40, (1, 1, kv, n), generator=g).float().cuda()  # many equal ones
    w[0, 0, 1] = torch.exp(torch.randn(n, generator=g) * 6).cuda()
    kept, _ = cache.evict(batch, PagedBatch(i32([list(range(313, 392))]), lengths), w, keep, 100, 10)
    assert lengths.tolist() == [keep]
    rk, rv = cache.read(0, PagedBatch(i32([list(range(313, 392))]), lengths, i32([0, keep]), keep), keep)
    for h in range(kv):
        want = ref.evict(w[0, 0, h].cpu(), n, keep, 100, 10)
        assert kept[0, 0, h].tolist() == want
        assert torch.equal(rk.view(keep, kv, 64)[:, h], k.view(n, kv, 64)[want, h])
    assert torch.equal(rv, -rk)


# ------------------------------------------------------------------------------------------------- graphs, streams, refusals
def test_captured_step_follows_lengths_tables_and_queries():
    s = Setup([500, 70, 0], [1, 1, 1], 8, 2, 128, seed=19, cols=10, spare=6).fill()
    q, weights, ws = s.q.cuda(), torch.zeros(3, 2, 640, device="cuda"), torch.empty(10 ** 6, device="cuda")
    one = s.PB(s.table, s.lengths)
    k, v = (torch.randn(3, 256, generator=s.g).to(BF16).cuda() for _ in range(2))
    out, prompt = torch.empty_like(q), torch.empty_like(q)

    def step():
        s.cache.write(0, k, v, one)
        s.cache.attend(0, q, one, out=out, ws=ws, weights=weights, decay=0.5)
        s.cache.attend_prompt(0, q, one, out=prompt)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    unused = [p for p in range(s.cache.pages) if p not in sum(s.ids, [])]
    weights.zero_()
    for r in range(4):
        s.lengths += 1
        if r == 2:
            s.table[2, 0] = unused[0]
        q.copy_(torch.randn(q.shape, generator=s.g).to(BF16))
        k.copy_(torch.randn(k.shape, generator=s.g).to(BF16))
        s.cache.k[0, unused[0]] = 0  # what the third sequence has not written
        s.cache.v[0, unused[0]] = 0
        eager_w = weights.clone()
        graph.replay()
        got, got_p, got_w = out.clone(), prompt.clone(), weights.clone()
        s.cache.attend(0, q, one, out=out, ws=ws, weights=eager_w, decay=0.5)
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.equal(got_w, eager_w) and got.any()
        assert torch.equal(got_p, s.cache.attend_prompt(0, q, one))
        assert not got[2].any() if r < 2 else got[2].any()


def test_two_streams_at_once():
    s = Setup([3000, 2500], [1, 1], 32, 8, 128, seed=20).fill()
    p = Setup([800, 700], [800, 700], 32, 8, 128, seed=21).fill()
    want = s.cache.attend(0, s.q.cuda(), s.batch), p.cache.attend_prompt(0, p.q.cuda(), p.batch)
    qs, qp = s.q.cuda(), p.q.cuda()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(a):
            x = s.cache.attend(0, qs, s.batch)
        with torch.cuda.stream(b):
            y = p.cache.attend_prompt(0, qp, p.batch)
        torch.cuda.synchronize()
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_python_refusals():
    from ssd.engine.kv_cache import PagedBatch

    s = Setup([100, 70], [2, 2], 8, 2, 64).fill()
    q, cache = s.q.cuda(), s.cache
    cpu = torch.zeros(2, dtype=I32)
    for args in ((s.table.long(), s.lengths), (s.table, s.lengths.float()), (s.table, cpu), (s.table[0], s.lengths), (s.table, s.lengths[:1]),
                 (s.table.t(), s.lengths), (s.table, s.lengths, s.begin[:2]), (s.table, s.lengths, None, 2), (s.table, s.lengths, s.begin, -1),
                 (s.table[:, :0], s.lengths), (s.table[:1].expand(2, -1), s.lengths)):
        with pytest.raises(ValueError, match="PagedBatch"):
            PagedBatch(*args)
    rows = torch.zeros(4, 128, dtype=BF16, device="cuda")
    bad = [lambda: cache.write(0, rows.float(), rows, s.batch), lambda: cache.write(0, rows, rows[:3], s.batch),
           lambda: cache.write(0, rows[:, :64], rows, s.batch), lambda: cache.write(0, rows.cpu(), rows, s.batch),
           lambda: cache.attend(0, q[:, :200], s.batch), lambda: cache.attend(0, q[:, :192], s.batch), lambda: cache.attend(0, q.half(), s.batch),
           lambda: cache.attend(0, q, s.batch, 129), lambda: cache.attend(0, q, s.batch, 0), lambda: cache.attend(0, q, s.batch, out=q[:3]),
           lambda: cache.attend(0, q, s.batch, ws=torch.empty(8, device="cuda")), lambda: cache.attend(0, q, s.batch, scale=-1.0),
           lambda: cache.attend(0, q, s.batch, weights=torch.zeros(2, 2, 100, device="cuda")),
           lambda: cache.attend(0, q, s.batch, weights=torch.zeros(2, 3, 128, device="cuda")),
           lambda: cache.attend(0, q, s.batch, weights=torch.zeros(2, 2, 128, device="cuda").half()),
           lambda: cache.attend(0, q, s.batch, weights=torch.zeros(1, 2, 128, device="cuda").expand(2, -1, -1)),
           lambda: cache.attend(0, q, s.batch, weights=torch.zeros(2, 2, 128, device="cuda"), decay=2.0),
           lambda: cache.attend_prompt(0, q, s.batch, 129), lambda: cache.attend_prompt(0, q[1:, 1:], s.batch),
           lambda: cache.read(0, s.batch, 4, rows[:2], rows), lambda: cache.evict(s.batch, s.batch, torch.zeros(1, 2, 3, 128, device="cuda"), 8),
           lambda: cache.evict(s.batch, s.batch, torch.zeros(1, 2, 2, 128, device="cuda"), 200),
           lambda: cache.evict(s.batch, s.batch, torch.zeros(1, 2, 2, 128, device="cuda"), 8, 6, 4)]
    before = cache.k.clone()
    for f in bad:
        with pytest.raises(ValueError):
            f()
    w = torch.zeros(1, 2, 2, 128, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        cache.evict(s.batch, s.batch, w, 8, out_weights=w)
    torch.cuda.synchronize()
    assert torch.equal(cache.k.view(torch.int16), before.view(torch.int16))


# ------------------------------------------------------------------------------------------------- a run of them together
def test_a_served_batch():
    """Prompts, steps that count received weights, eviction, further steps and scores, in two layers, against plain rows."""
    from ssd.engine.kv_cache import PagedBatch, PagedKVCache
    from ssd.engine.scoring import token_logprobs

    heads, kv, hd, layers, V = 8, 2, 64, 2, 1000
    g = torch.Generator().manual_seed(22)
    rand = lambda *n: torch.randn(*n, generator=g).to(BF16)  # noqa: E731
    cache = PagedKVCache(layers, 30, kv, hd, "cuda")
    lens = [150, 40, 260]
    pages = [cache.alloc(cache.pages_for(n + 8)) for n in lens]
    cols = max(map(len, pages))
    pad = lambda rows: i32([p + [-1] * (cols - len(p)) for p in rows])  # noqa: E731
    lengths = i32(lens)
    batch = PagedBatch(pad(pages), lengths, i32(sums(lens)), max(lens))
    plain = [[(rand(n, kv, hd), rand(n, kv, hd)) for n in lens] for _ in range(layers)]
    weights = torch.zeros(layers, 3, kv, cols * 64, device="cuda")
    head = rand(heads * hd, V).float()

    def close(out, q, i, at):  # rows q of the sequences, which attend all of plain[i]
        for s in range(3):
            k, v = plain[i][s]
            want, mag, w, _ = ref.attention(q[at[s]:at[s + 1]].view(-1, heads, hd), k, v, range(len(k) - (at[s + 1] - at[s]), len(k)))
            got = out[at[s]:at[s + 1]].double().cpu().view_as(want)
            assert ((got - want).abs() <= 2 ** -8 * want.abs() + 2 ** -7.9 * mag).all()
            yield w.view(len(want), kv, heads // kv, -1).sum((0, 2))

    for i in range(layers):
        q = rand(sum(lens), heads * hd)
        cache.write(i, *(torch.cat([x[j].flatten(1) for x in plain[i]]).cuda() for j in (0, 1)), batch)
        list(close(cache.attend_prompt(i, q.cuda(), batch, max(lens)), q, i, sums(lens)))
    step = PagedBatch(batch.table, lengths)
    total = [[0.0] * 3 for _ in range(layers)]

    def one_step(b, count):
        b.lengths += 1
        for i in range(layers):
            q, k, v = rand(3, heads * hd), rand(3, kv, hd), rand(3, kv, hd)
            plain[i] = [(torch.cat([a, k[s:s + 1]]), torch.cat([c, v[s:s + 1]])) for s, (a, c) in enumerate(plain[i])]
            cache.write(i, k.flatten(1).cuda(), v.flatten(1).cuda(), b)
            out = cache.attend(i, q.cuda(), b, weights=weights[i] if count else None)
            for s, w in enumerate(close(out, q, i, [0, 1, 2, 3])):
                total[i][s] = torch.nn.functional.pad(total[i][s], (0, 1)) + w if count and torch.is_tensor(total[i][s]) else w
        return out

    for _ in range(5):
        out = one_step(step, True)
    for i in range(layers):
        for s in range(3):
            got = weights[i, s, :, :lens[s] + 5].double().cpu()
            assert (got - total[i][s]).abs().max() < 1e-5 and abs(float(got.sum()) - 5 * heads) < 1e-4
    keep = 100
    new = [cache.alloc(cache.pages_for(keep + 8)) for _ in lens]
    after = PagedBatch(pad(new), torch.zeros_like(lengths))
    kept, weights = cache.evict(step, after, weights, keep, recent=10, first=2)
    for p in pages:
        cache.free(p)
    for i in range(layers):
        cut = []
        for s in range(3):
            at = [torch.tensor([t for t in kept[i, s, h].tolist() if t >= 0]) for h in range(kv)]
            cut.append(tuple(torch.stack([x[at[h], h] for h in range(kv)], 1) for x in plain[i][s]))
        plain[i] = cut
    assert after.lengths.tolist() == [100, 45, 100]
    for _ in range(3):
        out = one_step(after, False)
    logits = (out.float() @ head.cuda()).to(BF16)
    tokens = logits.argmax(1)
    got = token_logprobs(logits, tokens, top=4)
    want = ref.token_logprobs(logits.cpu(), tokens.cpu(), 4)
    assert torch.equal(got.top_ids.cpu().long(), want[3]) and not got.rank.any()
    assert (got.logprobs.cpu().double() - want[0]).abs().max() < 1e-4 and (got.entropy.cpu().double() - want[1]).abs().max() < 1e-4
