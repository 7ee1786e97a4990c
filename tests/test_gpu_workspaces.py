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
