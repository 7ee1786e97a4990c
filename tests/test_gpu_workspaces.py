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
