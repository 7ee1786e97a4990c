"""Workspaces that a caller gives: what is refused, and what their sizes say is accepted."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_token_logprobs_take_their_bytes_in_one_run():
    """Bytes that a view skips or repeats are not its own to write."""
    from ssd import ops
    from ssd.engine.scoring import token_logprobs

    x, t = torch.randn(2, 128256, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    need = ops.token_logprobs_ws_bytes(2, 128256, x.dtype, 3)
    assert need
    buf = torch.full((2 * need + 16,), 7, dtype=torch.uint8, device="cuda")
    for ws in (buf[:2 * need:2], buf[:1].expand(need), buf[:need - 1], buf.view(torch.int8)[:need], buf[:2 * need].view(2, need).t()):
        with pytest.raises(ValueError, match="ws"):
            token_logprobs(x, t, 3, ws)
    torch.cuda.synchronize()
    assert (buf == 7).all()
    got = token_logprobs(x, t, 3, buf[16:16 + need])
    for a, b in zip(got, token_logprobs(x, t, 3)):
        assert torch.equal(a, b)
    assert (buf[:16] == 7).all() and (buf[16 + need:] == 7).all()


def test_workspaces_of_no_floats_are_taken():
    """What prompt_floats and attend_floats give, 0 among it, is enough."""
    from test_gpu_paged import Setup

    s = Setup([70, 30], [70, 30], 4, 2, 64, seed=60).fill()
    q = s.q.cuda()
    assert s.cache.prompt_floats(100, 4, s.batch) == 0 and s.cache.attend_floats(0, 4, s.batch) == 0
    none = torch.empty(0, device="cuda")
    s.check(s.cache.attend_prompt(0, q, s.batch, ws=none))
    assert s.cache.attend(0, q[:0], s.batch, ws=none).shape == (0, 256)
    assert s.cache.attend_prompt(0, q[:0], s.batch, ws=none).shape == (0, 256)
    with pytest.raises(ValueError):
        s.cache.attend(0, q, s.batch, ws=none)


def test_prompt_workspaces_that_are_too_small_or_not_in_one_run_are_refused():
    from test_gpu_paged import Setup

    s = Setup([4000], [20], 4, 2, 64, seed=61).fill()
    q = s.q.cuda()
    need = s.cache.prompt_floats(20, 4, s.batch)
    assert need
    buf = torch.full((2 * need,), 7.0, device="cuda")
    for ws in (buf[::2], buf[:1].expand(need), buf[:need - 1], buf[:0], buf.half()[:need], buf[1:need + 1]):
        with pytest.raises(ValueError):
            s.cache.attend_prompt(0, q, s.batch, ws=ws)
    torch.cuda.synchronize()
    assert (buf == 7).all()
    assert torch.equal(s.cache.attend_prompt(0, q, s.batch, ws=buf[:need]), s.cache.attend_prompt(0, q, s.batch))


@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (15, 5, 128), (16, 16, 64), (20, 1, 64)])
def test_attention_with_weights_stays_in_its_workspace(heads, kv, hd):
    """Windows of more pairs than keep scores, and calls of fewer rows in the same workspace."""
    from test_gpu_paged import Setup, i32

    s = Setup([900, 333, 70], [17, 18, 20], heads, kv, hd, seed=62, span=64).fill()
    q = s.q.cuda()
    need = s.cache.attend_floats(55, heads, s.batch, 960, weights=True)
    buf = torch.full((need + 64,), float("nan"), device="cuda")
    buf[need:] = 7.0
    weights = torch.zeros(3, kv, 960, device="cuda")
    s.check(s.cache.attend(0, q, s.batch, 960, ws=buf[:need], weights=weights), weights, torch.zeros_like(weights))
    for most in (18, 1):  # rows of the first sequence alone, under the same bound and one of its own
        for m in (1, 3, 16):
            if most < m:
                continue
            one = s.PB(s.table[:1], i32([900 - 17 + m]), i32([0, m]), most)
            weights = torch.zeros(1, kv, 960, device="cuda")
            again = torch.zeros_like(weights)
            out = s.cache.attend(0, q[:m], one, 960, ws=buf[:need], weights=weights)
            assert torch.equal(out, s.cache.attend(0, q[:m], one, 960, weights=again)) and torch.equal(weights, again)
    assert (buf[need:] == 7).all()
    if 18 * heads // kv > 16:
        assert need < ws_with_scores(s, heads, hd)
    with pytest.raises(ValueError, match="workspace"):
        s.cache.attend(0, q, s.batch, 960, ws=torch.empty(100, device="cuda"), weights=torch.zeros(3, kv, 960, device="cuda"))


def ws_with_scores(s, heads, hd):
    from ssd import ops

    return ops.paged_attn_ws_floats(55, heads, hd, 960, 64, True)
