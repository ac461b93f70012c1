"""Log probabilities of given tokens under a model's logits, with the entropy and the likeliest alternatives of
every position, and the logits' gradient (``ccq_token_logprobs_fwd`` / ``_bwd`` of ``libccq_hip.so``).

The reference's models end in HF's cross entropy over the LM head's logits; ``graph.greedy_embed`` is the greedy
pick of a decode step.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._native import ops

__all__ = ["token_logprobs", "TokenLogprobs"]


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor                        # fp32, the shape of ids
    entropy: torch.Tensor                         # fp32, the shape of ids
    top_logprobs: Optional[torch.Tensor] = None   # fp32 [..., top_k] (None without alternatives)
    top_ids: Optional[torch.Tensor] = None        # int64 [..., top_k]


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top_k: int = 0, ignore_index: int = -100) -> TokenLogprobs:
    """Of ``logits [..., V]`` (bf16, fp16 or fp32 on the GPU, V at most 2^30, any stride between rows) and tokens
    ``ids [...]`` (int64 or int32): fp32 ``log_softmax(logits)[ids]`` and the entropy of every position, both
    differentiable (first derivatives, reverse mode), and with ``top_k`` (at most 64) the log probabilities and ids of
    its likeliest tokens, ties to the lowest id (not differentiable).  A position whose id is ``ignore_index`` is
    skipped: its logits are not read, its results are 0 (ids -1) and its gradient is 0.  An id outside the vocabulary
    has the log probability NaN (nothing is read out of bounds); a logit of -inf masks its token.  Positions that do not lie at one stride, such as
    ``logits[:, :-1]`` of ``[B, T, V]``, are copied first and the copy is kept for the backward: of all positions, with
    ``ids`` of ``ignore_index`` at the last ones, nothing is."""
    return TokenLogprobs(*ops().token_logprobs(logits, ids, top_k, ignore_index))
