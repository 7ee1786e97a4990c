"""Token log probabilities of logits of any size, on the GPU against 64 bits: their error does not grow with the logits, a column that has
all the mass has no positive log probability, and the type's lowest and largest values are numbers like others."""

import pytest
import torch

from oracle import paged as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24


def check(x, tokens, top):
    from ssd.engine.scoring import token_logprobs

    got = token_logprobs(x.cuda(), tokens.cuda(), top)
    lp, ent, rank, ids, tlp = ref.token_logprobs(x, tokens, top)
    V, d = x.shape[1], x.double() - x.double().amax(1, keepdim=True)
    p = torch.softmax(x.double(), 1)
    d = torch.where(p > 0, d, 0.0).abs()
    d1, d2, lnz = (p * d).sum(1), (p * d * d).sum(1), d.neg().exp().where(p > 0, 0.0).sum(1).log()
    # An exponent is a difference, a constant and a product of 24 bits each: off by 3 U |d|, so z by 3 U times the mean of |d|; exp2
    # 2 U. A thread adds up to V / 256 + 32 terms and is rescaled (5 U) up to V / 8192 + 1 times; then 14 sums and 8 rescalings.
    a = 2 + (V / 256 + 32) + 5 * (V / 8192 + 1) + 14 + 40
    z = U * (a + 3 * d1)
    assert torch.equal(got.rank.cpu().long(), rank) and torch.equal(got.top_ids.cpu().long(), ids)
    for mine, want in [(got.logprobs, lp), *((got.top_logprobs[:, i], tlp[:, i]) for i in range(top))]:
        mine, want = mine.cpu().double(), want.float().double()
        there = want > -torch.inf  # a column of -inf
        assert torch.equal(mine > -torch.inf, there) and (mine <= 0).all()
        # ln z is off by z's relative error and 2 U of itself; x - m, the difference and the comparison value are rounded once each
        assert ((mine - want).abs()[there] <= (z + 2 * U * lnz + 3 * U * want.abs())[there]).all()
    # t: its terms' weights as z's and their factors y once more (3 U), z as above; ln z, the product and the difference
    tol = U * (a + 2 * a * d1 + 6 * d2 + 10 * d1 + 3 * lnz + ent.abs())
    assert ((got.entropy.cpu().double() - ent).abs() <= tol).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 60, -60, 1000.7, 3e4, -3e4])
@pytest.mark.parametrize("V", [700, 130001])
def test_the_error_does_not_grow_with_the_logits(dtype, shift, V):
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(5, V, generator=g) * 3 + shift).to(dtype)
    x[:, torch.rand(V, generator=g) < 0.02] = float("-inf")
    check(x, torch.tensor([3, V - 1, int(x[2].argmax()), -1, 77]), 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [300, 140000])
def test_a_column_that_has_the_mass(dtype, V):
    """The others 12 to 40 below it."""
    tops = torch.tensor([10.3, 20.0, 31.7, 50.1, 100.3, 333.3, 1000.7, 30001.0, -50.0, -1000.7])
    g = torch.Generator().manual_seed(V)
    x = (tops[:, None] - 12 - 28 * torch.rand(10, V, generator=g)).to(dtype)
    at = torch.randint(0, V, (10,), generator=g)
    x[torch.arange(10), at] = tops.to(dtype)
    check(x, at, 3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [300, 20000, 140000])
@pytest.mark.parametrize("end", ["min", "max"])
def test_the_lowest_and_the_largest_value_of_the_type(dtype, V, end):
    """Columns that are masked with the lowest value: few, a half, all but one, all; and columns of the largest value."""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(6, V, generator=g) * 3).to(dtype)
    value = getattr(torch.finfo(dtype), end)
    x[0, ::7], x[1, :V // 2], x[2, V // 2:], x[3, torch.arange(V) != V // 3], x[4], x[5, 9] = (value,) * 6
    tokens = torch.tensor([1, 2, V - 1, V // 3, 5, 9])
    if end == "max":
        x[3, V // 3] = value
        x[3, torch.arange(V) != V // 3] = 1.0
    check(x, tokens, 4)
