"""The paged cache's operators at other sizes of a call: a row's bits in the attention of few new rows follow from its query, its keys and
the span alone, whatever the batch, the bound of the lengths and so the number of groups that a call cuts; eviction that keeps all."""

import pytest
import torch

from test_gpu_paged import Setup, i32, sums

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
def test_a_row_alone_in_a_large_batch_and_under_any_bound(hd):
    """66 sequences of 32 heads, of up to 10 groups (the join of a call of few pairs and many groups has four waves a pair, that of
    others one), under bounds of few and many groups."""
    lens = [2500 - 37 * (i % 50) for i in range(65)] + [700]
    s = Setup(lens, [1] * 66, 32, 1, hd, seed=40, span=64, cols=80).fill()
    q = s.q.cuda()
    out = s.cache.attend(0, q, s.batch, 2500)
    assert torch.equal(out, s.cache.attend(0, q, s.batch))  # 20 groups
    for i in (0, 1, 17, 49, 65):
        one = s.PB(s.table[i:i + 1], s.lengths[i:i + 1])
        for bound in (lens[i], 2500, 5120):  # the shortest: 3 groups in all under the first
            assert torch.equal(s.cache.attend(0, q[i:i + 1], one, bound)[0], out[i]), (i, bound)


@pytest.mark.parametrize("groups", [1, 7, 8, 9, 16, 31, 33, 64, 65, 130])
def test_groups_are_added_up_the_same_by_one_wave_and_by_four(groups):
    length = 256 * groups - 3
    s = Setup([length], [1], 4, 1, 64, seed=41, span=64).fill()
    out = s.cache.attend(0, s.q.cuda(), s.batch, length)
    s.check(out)
    n = 520  # pairs past the four waves' bound
    many = s.PB(s.table.expand(n, -1).contiguous(), i32([length] * n), i32(sums([1] * n)), 1)
    assert torch.equal(s.cache.attend(0, s.q.cuda().expand(n, -1).contiguous(), many, length), out.expand(n, -1))


# ------------------------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("keep,cap", [(129, 128), (200, 128), (300, 150), (64, 60)])
def test_eviction_that_keeps_more_than_the_weights_hold_keeps_all(keep, cap):
    """A batch whose sequences are all short: every slot stays, in new pages; slots from the weights' end on count as not there."""
    kv, lens = 2, [100, 0, 128, 37]
    s = Setup(lens, [1] * 4, kv, kv, 64, seed=42, spare=20).fill()
    unused = [p for p in range(s.cache.pages) if p not in sum(s.ids, [])]
    cols = (keep + 63) // 64
    stay = [min(n, cap, keep) for n in lens]
    new = i32([[unused.pop() if c * 64 < n else -1 for c in range(cols)] for n in stay])
    after = s.PB(new, i32([7] * 4), i32(sums(stay)), max(stay))
    w = torch.rand(1, 4, kv, cap, generator=s.g)
    kept, moved = s.cache.evict(s.batch, after, w.cuda(), keep, 5, 3)
    assert after.lengths.tolist() == stay and kept.shape[-1] == keep and moved.shape == w.shape
    k, v = (x.cpu().view(-1, kv, 64) for x in s.cache.read(0, after, sum(stay)))
    at = 0
    for q, n in enumerate(stay):
        for h in range(kv):
            assert kept[0, q, h].tolist() == list(range(n)) + [-1] * (keep - n)
            assert torch.equal(moved[0, q, h].cpu(), torch.cat([w[0, q, h, :n], torch.zeros(cap - n)]))
        assert torch.equal(k[at:at + n], s.k[q][:n]) and torch.equal(v[at:at + n], s.v[q][:n])
        at += n


# ------------------------------------------------------------------------------------------------- prompts
@pytest.mark.parametrize("n,rows,past", [(16, 32, 1200), (7, 32, 700), (3, 64, 1500), (64, 32, 0), (5, 33, 1100)])
def test_prompts_of_one_length_that_fill_their_tiles(n, rows, past):
    """As many tiles as the launch counts, none to spare, with the length whole and in parts."""
    s = Setup([past + rows + i % 3 for i in range(n)], [rows] * n, 4, 1, 64, seed=43).fill()
    ws = torch.full((s.cache.prompt_floats(n * rows, 4, s.batch),), float("nan"), device="cuda")
    s.check(s.cache.attend_prompt(0, s.q.cuda(), s.batch, ws=ws))


@pytest.mark.parametrize("rows", [[130, 1, 1, 2, 0], [1, 1, 40], [64, 0, 0, 0, 0, 0, 0, 64]])
def test_prompts_whose_workspace_is_sized_by_the_rows_alone(rows):
    """Uneven rows, and a bound of them that is far too large."""
    s = Setup([600 + 100 * i + n for i, n in enumerate(rows)], rows, 4, 1, 64, seed=44).fill()
    for most in (max(rows), 4096):
        b = s.PB(s.table, s.lengths, s.begin, most)
        ws = torch.full((s.cache.prompt_floats(sum(rows), 4, b),), float("nan"), device="cuda")
        s.check(s.cache.attend_prompt(0, s.q.cuda(), b, ws=ws))


def test_prompt_rows_of_no_sequence_and_a_tight_bound():
    """More rows than the sequences own."""
    s = Setup([900, 1000], [20, 31], 4, 1, 64, seed=45).fill()
    q = torch.zeros(300, 256, dtype=torch.bfloat16, device="cuda")
    q[100:151] = s.q.cuda()
    out = torch.full_like(q, 7.0)
    b = s.PB(s.table, s.lengths, i32([100, 120, 151]), 31)
    ws = torch.full((s.cache.prompt_floats(300, 4, b),), float("nan"), device="cuda")
    s.cache.attend_prompt(0, q, b, out=out, ws=ws)
    s.check(out[100:151])
    assert (out[:100] == 7).all() and (out[151:] == 7).all()


# ------------------------------------------------------------------------------------------------- the output in q's place
@pytest.mark.parametrize("lens,rows", [([70, 500], [1, 2]), ([3000], [1]), ([200, 90, 64], [150, 90, 3]), ([5000], [20])])
def test_outputs_may_take_the_place_of_q(lens, rows):
    s = Setup(lens, rows, 8, 2, 128, seed=46, span=64).fill()
    for f in (s.cache.attend, s.cache.attend_prompt):
        q = s.q.cuda()
        want = f(0, q, s.batch)
        f(0, q, s.batch, out=q)
        assert torch.equal(q, want)
    if max(rows) * 4 <= 16:  # scores that are kept
        q, w = s.q.cuda(), torch.zeros(2, len(lens), 2, s.batch.capacity, device="cuda")
        want = s.cache.attend(0, q, s.batch, weights=w[0])
        s.cache.attend(0, q, s.batch, weights=w[1], out=q)
        assert torch.equal(q, want) and torch.equal(w[0], w[1])
