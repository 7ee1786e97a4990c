"""Scores of given tokens under a model's logits: what a server returns beside an answer, what a document's perplexity or a
drafted token's likelihood is computed from."""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ssd import ops


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # [M] fp32: log softmax at the token (0 for no token)
    entropy: torch.Tensor       # [M] fp32: the row's entropy in nats
    rank: torch.Tensor          # [M] int32: columns that rank before the token (-1 for no token)
    top_ids: torch.Tensor       # [M, top] int32: the most likely columns, best first
    top_logprobs: torch.Tensor  # [M, top] fp32


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, ws: Optional[torch.Tensor] = None) -> TokenLogprobs:
    """Of every row of logits [M, V] (bf16, fp16 or fp32; unit column stride, any row stride): the log probability and rank of
    tokens[m] (int32 or int64; outside [0, V): none, a padded place), the row's entropy, and the ``top`` <= 32 most likely columns
    (equal ones: the lowest first). -inf columns have no mass; a row with a NaN gives NaN and rank -1. Inference only: no
    gradient flows through it. ``ws``: uint8 workspace of ops.token_logprobs_ws_bytes(M, V, dtype, top) bytes (None: allocated
    here)."""
    return TokenLogprobs(*ops.token_logprobs(logits, tokens, top, ws))
