"""What the attention of few new rows loses: the rounding of its output, and of each weight 16 bits, since a weight goes into the second
product as the sum of two bf16 numbers. One bf16 number a weight would be seen."""

import pytest
import torch

from oracle import paged as ref

BF16 = torch.bfloat16


def tolerance(want, mag, size, keys, hd):
    """A weight is off by 2^-8 of what its first bf16 number leaves, 2^-16 of it; a score by the rounding of sums of hd products, the sums
    over the keys by theirs; the result is rounded to bf16 once."""
    slack = 2.0 ** -24 * (4 * hd * size[..., None] + 4 * keys + 256)
    return 2.0 ** -8 * want.abs() + (2.0 ** -16 + slack) * mag * (1 + 2.0 ** -8) + 1e-30


def inputs(n, keys, heads, kv, hd, seed):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(keys, kv, hd, generator=g).to(BF16) for _ in range(2))
    return (torch.randn(n, heads, hd, generator=g) * 1.5).to(BF16), k, v


CASES = [(1, 60, 8, 2, 64), (3, 700, 16, 2, 128), (2, 300, 15, 5, 128), (16, 1500, 8, 2, 64)]


@pytest.mark.parametrize("n,keys,heads,kv,hd", CASES[:3])  # over 1500 keys the bound of the sums' roundings hides one of the weights
def test_the_tolerance_tells_one_bf16_number_a_weight_from_two(n, keys, heads, kv, hd):
    q, k, v = inputs(n, keys, heads, kv, hd, 70)
    want, mag, w, size = ref.attention(q, k, v, [keys - n + i for i in range(n)])
    tol = tolerance(want, mag, size, keys, hd)
    vv = v.double().repeat_interleave(heads // kv, 1)
    peak = w.amax(-1, keepdim=True)
    p = (w / peak).float()  # as a kernel has them
    hi = p.to(BF16).float()
    one, two = (torch.einsum("nhk,khd->nhd", x.double() * peak, vv) for x in (hi, hi + (p - hi).to(BF16).float()))
    assert ((two.to(BF16).double() - want).abs() <= tol).all()
    assert ((one.to(BF16).double() - want).abs() > tol).any()


@pytest.mark.gpu
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("n,keys,heads,kv,hd", CASES)
def test_attention_of_new_rows_to_its_precision(n, keys, heads, kv, hd, weights):
    from test_gpu_paged import Setup

    s = Setup([keys], [n], heads, kv, hd, seed=71)
    q, s.k[0], s.v[0] = inputs(n, keys, heads, kv, hd, 70)
    s.q = q.flatten(1)
    s.fill()
    got = torch.zeros(1, kv, (keys + 63) // 64 * 64, device="cuda") if weights else None
    out = s.cache.attend(0, s.q.cuda(), s.batch, weights=got).double().cpu().view(n, heads, hd)
    want, mag, _, size = ref.attention(q, s.k[0], s.v[0], s.last(0))
    assert ((out - want).abs() <= tolerance(want, mag, size, keys, hd)).all()
