"""Log probabilities of given tokens under a model's logits, with the entropy and the likeliest alternatives of
every position, and the logits' gradient (``ccq_token_logprobs_fwd`` / ``_bwd`` of ``libccq_hip.so``).

The reference's models end in HF's cross entropy over the LM head's logits; ``graph.greedy_embed`` is the greedy
pick of a decode step.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from ._rows import (DTYPES, address, call, current, needs_grad, require_gpu, require_on, rows_of, stream_on,
                    stride_of)

__all__ = ["token_logprobs", "TokenLogprobs", "TokenLogprobsFunction"]

MAX_TOP = 64


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor                 # fp32, the shape of ids
    entropy: torch.Tensor                  # fp32, the shape of ids
    top_logprobs: Optional[torch.Tensor]   # fp32 [..., top_k] (None without alternatives)
    top_ids: Optional[torch.Tensor]        # int64 [..., top_k]


def _forward(logits, ids, k, ignore, keep):
    """The four results and the logits as rows, the ids as the kernels read them and (with ``keep``) each row's
    maximum and log sum."""
    x2 = rows_of(logits)
    rows, V = x2.shape
    i2 = ids.contiguous()
    logp = x2.new_empty(ids.shape, dtype=torch.float32)
    ent = x2.new_empty(ids.shape, dtype=torch.float32)
    stats = x2.new_empty(2 * rows, dtype=torch.float32) if keep else None
    top = x2.new_empty(*ids.shape, k, dtype=torch.float32) if k else None
    top_ids = x2.new_empty(*ids.shape, k, dtype=torch.int64) if k else None
    call("ccq_token_logprobs_fwd", x2.data_ptr(), stride_of(x2), i2.data_ptr(), logp.data_ptr(), ent.data_ptr(),
         address(stats), address(top), address(top_ids), rows, V, k, ignore, DTYPES[logits.dtype], stream_on(logits))
    return logp, ent, top, top_ids, x2, i2, stats


class TokenLogprobsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, k, ignore):
        logp, ent, top, top_ids, x2, i2, stats = _forward(logits, ids, k, ignore, True)
        ctx.save_for_backward(x2, i2, ent, stats)
        ctx.meta = (logits.shape, ignore)
        ctx.set_materialize_grads(False)
        if k:
            ctx.mark_non_differentiable(top, top_ids)
        return logp, ent, top, top_ids

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp, dent, _top=None, _top_ids=None):
        if dlogp is None and dent is None:
            return None, None, None, None
        saved = ctx.saved_tensors
        if not current(saved[0]):
            with torch.cuda.device(saved[0].device):
                return TokenLogprobsFunction._backward(ctx, *saved, dlogp, dent)
        return TokenLogprobsFunction._backward(ctx, *saved, dlogp, dent)

    @staticmethod
    def _backward(ctx, x2, i2, ent, stats, dlogp, dent):
        shape, ignore = ctx.meta
        dx = x2.new_empty(shape)
        dlogp = dlogp.contiguous() if dlogp is not None else None
        dent = dent.contiguous() if dent is not None else None
        call("ccq_token_logprobs_bwd", x2.data_ptr(), stride_of(x2), i2.data_ptr(), ent.data_ptr(), stats.data_ptr(),
             address(dlogp), address(dent), dx.data_ptr(), x2.shape[0], x2.shape[1], ignore, DTYPES[x2.dtype],
             stream_on(x2))
        return dx, None, None, None


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top_k: int = 0, ignore_index: int = -100) -> TokenLogprobs:
    """Of ``logits [..., V]`` (bf16, fp16 or fp32 on the GPU, any row stride) and tokens ``ids [...]`` (int64 or
    int32): fp32 ``log_softmax(logits)[ids]`` and the entropy of every position, both differentiable, and with
    ``top_k`` (at most 64) the log probabilities and ids of its likeliest tokens, ties to the lowest id (not
    differentiable).  A position whose id is ``ignore_index`` is skipped: its logits are not read, its results are
    0 (ids -1) and its gradient is 0.  An id outside the vocabulary has the log probability NaN (nothing is read
    out of bounds); a logit of -inf masks its token."""
    if logits.dtype not in DTYPES:
        raise TypeError(f"token_logprobs takes bf16, fp16 or fp32 logits (got {logits.dtype})")
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"token_logprobs takes int64 or int32 ids (got {ids.dtype})")
    if logits.dim() < 1 or logits.shape[-1] < 1 or ids.shape != logits.shape[:-1]:
        raise ValueError(f"token_logprobs: ids {tuple(ids.shape)}: expected the positions of logits "
                         f"{tuple(logits.shape)}")
    require_on("token_logprobs", "ids", ids, logits)
    top_k = int(top_k)
    if not 0 <= top_k <= min(MAX_TOP, logits.shape[-1]):
        raise ValueError(f"token_logprobs: top_k={top_k} must lie in [0, {min(MAX_TOP, logits.shape[-1])}]")
    require_gpu("token_logprobs", logits)
    if not current(logits):
        with torch.cuda.device(logits.device):
            return token_logprobs(logits, ids, top_k, ignore_index)
    ids = ids.long()
    if needs_grad(logits):
        return TokenLogprobs(*TokenLogprobsFunction.apply(logits, ids, top_k, int(ignore_index)))
    return TokenLogprobs(*_forward(logits, ids, top_k, int(ignore_index), False)[:4])
