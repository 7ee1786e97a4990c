"""Token log probabilities on the GPU against 64 bits (oracle.paged.token_logprobs)."""

import pytest
import torch

from oracle import paged as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def check(logits, tokens, top):
    from ssd.engine.scoring import token_logprobs

    got = token_logprobs(logits, tokens, top)
    x = logits.cpu().float()
    lp, ent, rank, ids, tlp = ref.token_logprobs(x, tokens.cpu(), top)
    V = x.shape[1]
    size = float(x[x > -1e30].abs().max())
    # the sum of up to V / 256 terms a thread and the threads' tree, exponents off by roundings of x log2 e, two more roundings
    tol = 2.0 ** -24 * (V / 256 + 64 + 8 * size)
    assert torch.equal(got.rank.cpu().long(), rank) and torch.equal(got.top_ids.cpu().long(), ids)
    mine, there = got.logprobs.cpu().double(), lp > -1e30  # a masked column's is -inf
    assert torch.equal(mine > -1e30, there) and not mine.isnan().any()
    assert ((mine - lp).abs()[there] <= tol + 2.0 ** -23 * lp[there].abs()).all()
    assert (got.entropy.cpu().double() - ent).abs().max() <= tol * (3 + 2 * float(ent.max()))
    if top:
        fine = tlp > -1e30
        assert torch.equal(fine, got.top_logprobs.cpu() > -1e30)
        assert ((got.top_logprobs.cpu().double() - tlp).abs()[fine] <= tol + 2.0 ** -23 * tlp[fine].abs()).all()
    assert got.logprobs.dtype == got.entropy.dtype == got.top_logprobs.dtype == torch.float32 and got.rank.dtype == torch.int32


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,V,top", [(1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 33, 20), (4, 1000, 5), (25, 128256, 5), (1, 128256, 32), (7, 50257, 0),
                                     (600, 4099, 3), (1100, 260, 1), (2, 300001, 17)])
def test_against_64_bits(dtype, M, V, top):
    g = torch.Generator().manual_seed(V + M)
    x = torch.randn(M, V, generator=g) * 3
    if V > 100:
        x[:, torch.rand(V, generator=g) < 0.05] = float("-inf")
    tokens = torch.randint(0, V, (M,), generator=g, dtype=torch.int32 if M % 2 else torch.int64)
    tokens[0] = int(x[0].argmax())
    if M > 2:
        tokens[1], tokens[2] = -1, V  # none
    check(x.to(dtype).cuda(), tokens.cuda(), top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [0, 1, 3, 5])
def test_rows_at_any_alignment(dtype, offset):
    x = (torch.randn(9, 9000, generator=torch.Generator().manual_seed(offset)) * 4).to(dtype).cuda()
    tokens = torch.arange(9, device="cuda") * 7
    check(x[:, offset:offset + 8191 - offset], tokens, 6)
    check(x.flatten()[offset:offset + 9 * 8999].view(9, 8999), tokens, 6)  # odd row stride
    check(x[:, offset:offset + 5], tokens % 5, 2)


@pytest.mark.parametrize("V", [500, 40000])
def test_equal_logits_and_few_with_mass(V):
    """More candidates than the list holds: all equal, two values, nearly all masked; the largest in one thread's columns."""
    x = torch.zeros(6, V, dtype=torch.bfloat16)
    x[1, ::2] = 1.0
    x[2] = float("-inf")
    x[2, [3, V - 1]] = torch.tensor([1.0, 2.0]).bfloat16()
    x[3], x[3, V // 2:] = -0.0, 0.0
    x[4] = torch.arange(V).float().neg().bfloat16()
    x[5, :8 * 40] = 5.0
    check(x.cuda(), torch.tensor([0, V - 1, 3, V - 1, 17, 9], device="cuda"), 20)


def test_logits_far_from_zero():
    g = torch.Generator().manual_seed(5)
    for shift in (-3e4, 3e4):
        x = torch.randn(4, 5000, generator=g) + shift
        check(x.cuda(), torch.tensor([0, 1, 2, 3], device="cuda"), 3)


def test_rows_without_numbers():
    from ssd.engine.scoring import token_logprobs

    for V in (300, 40000):
        x = torch.randn(5, V, generator=torch.Generator().manual_seed(V)).cuda()
        x[1, V - 5], x[2, 10], x[3] = float("nan"), float("inf"), float("-inf")
        got = token_logprobs(x, torch.tensor([1, 1, 1, 1, 1], device="cuda"), top=4)
        assert got.logprobs.isnan().tolist() == got.entropy.isnan().tolist() == [False, True, True, True, False]
        assert got.rank[1] == -1 and got.rank[2] > 0
        best = torch.sort(torch.where(x.isnan(), -torch.inf, x)[[0, 1, 4]], dim=1, descending=True, stable=True).indices[:, :4]
        assert torch.equal(got.top_ids[[0, 1, 4]].long(), best) and got.top_ids[2, 0] == 10


def test_captured_and_given_workspace_and_no_rows():
    from ssd import ops
    from ssd.engine.scoring import token_logprobs

    x = torch.randn(3, 30000, device="cuda").bfloat16()
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    ws = torch.empty(ops.token_logprobs_ws_bytes(3, 30000, x.dtype, 5), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        token_logprobs(x, t, 5, ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = token_logprobs(x, t, 5, ws)
    for i in range(3):
        x.copy_(torch.randn(3, 30000, device="cuda"))
        t.fill_(i + 2)
        graph.replay()
        held = [y.clone() for y in got]
        for a, b in zip(held, token_logprobs(x, t, 5)):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
    assert [y.shape for y in token_logprobs(x[:0], t[:0], 2)] == [(0,), (0,), (0,), (0, 2), (0, 2)]


def test_refusals():
    from ssd.engine.scoring import token_logprobs

    x, t = torch.randn(4, 100, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    for args in ((x.double(), t), (x.cpu(), t), (x[0], t), (x.t(), t), (x, t.float()), (x, t[:3]), (x, t.cpu()), (x, t, 33), (x, t, -1),
                 (x[:, :5], t, 6), (x[:, ::2], t), (x[:1].expand(4, -1), t), (x, torch.zeros(8, dtype=torch.int32, device="cuda")[::2])):
        with pytest.raises((ValueError, RuntimeError)):
            token_logprobs(*args)
    y = torch.randn(1, 128256, device="cuda")
    with pytest.raises(ValueError):
        token_logprobs(y, t[:1], 5, torch.empty(16, dtype=torch.uint8, device="cuda"))
