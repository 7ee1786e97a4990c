"""A row's bits in the attention of few new rows: they follow from its query, its keys and the span alone, whatever the batch, the
bound of the lengths and so the number of groups that a call cuts."""

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
