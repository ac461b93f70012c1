"""Block norms: layer norm and RMS norm over the last dimension, with the residual stream's add in the same pass
(``ccq_norm_fwd`` / ``ccq_norm_bwd`` of ``libccq_hip.so``).

The reference's layers (``ccq/gdn/layer.py``, ``ccq/gla/layer.py``) sit in pre-norm blocks whose norms its HF
model classes take from fla; ``prologue.gated_rmsnorm`` is the norm inside the layers.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from ._rows import (DTYPES, address, call, current, entry, like, needs_grad, require_gpu, require_on, rows_of,
                    stream_on, stride_of)

__all__ = ["layer_norm", "rms_norm", "BlockNormFunction"]

MAX_WIDTH = 8192


def _forward(x, residual, weight, bias, layer, eps, keep):
    """``(y, s or None, x as rows, statistics or None)``; the statistics (mean, then 1 / deviation, of every row) only
    with ``keep``."""
    x2 = rows_of(x)
    r2 = rows_of(residual) if residual is not None else None
    rows, D = x2.shape
    y = like(x)
    s = like(x) if r2 is not None else None
    stats = x.new_empty(2 * rows, dtype=torch.float32) if keep else None
    mean = address(stats)
    wdtype = DTYPES[weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype]
    call("ccq_norm_fwd", x2.data_ptr(), stride_of(x2), address(r2), stride_of(r2) if r2 is not None else 0,
         address(weight), address(bias), y.data_ptr(), address(s), mean if layer else 0,
         mean + 4 * rows if keep else 0, rows, D, DTYPES[x.dtype], wdtype, layer, eps, stream_on(x))
    return y, s, x2, stats


class BlockNormFunction(torch.autograd.Function):
    """The norm of ``x`` (``+ residual``); returns ``y`` or ``(y, s)`` with ``s = x + residual``."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, layer, eps):
        y, s, x2, stats = _forward(x, residual, weight, bias, layer, eps, True)
        # the normalised rows: the stream where there is a residual (an output, saved as such), x otherwise
        ctx.save_for_backward(x2 if s is None else s, weight, stats)
        ctx.meta = (layer, x.shape, None if bias is None else bias.dtype)
        ctx.set_materialize_grads(False)
        return y if s is None else (y, s)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds=None):
        if dy is None and ds is None:
            return None, None, None, None, None, None
        rows_in, weight, stats = ctx.saved_tensors
        if not current(rows_in):
            with torch.cuda.device(rows_in.device):
                return BlockNormFunction._backward(ctx, rows_in, weight, stats, dy, ds)
        return BlockNormFunction._backward(ctx, rows_in, weight, stats, dy, ds)

    @staticmethod
    def _backward(ctx, rows_in, weight, stats, dy, ds):
        layer, shape, bdtype = ctx.meta
        need_x, need_r, need_w, need_b = ctx.needs_input_grad[:4]
        x2 = rows_of(rows_in)
        rows, D = x2.shape
        dtype = x2.dtype
        if dy is None:
            dy = x2.new_zeros(shape)  # (only the stream was used)
        d2 = rows_of(dy)
        s2 = rows_of(ds) if ds is not None else None
        wdt = weight.dtype if weight is not None else bdtype if bdtype is not None else dtype
        dx = x2.new_empty(shape) if need_x or need_r else None
        dw = x2.new_empty(D, dtype=wdt) if need_w else None
        db = x2.new_empty(D, dtype=wdt) if need_b else None
        ws = None
        if need_w or need_b:
            ws = x2.new_empty(entry("ccq_norm_bwd_workspace_bytes")(rows, D, DTYPES[dtype]), dtype=torch.uint8)
        mean = stats.data_ptr()
        call("ccq_norm_bwd", x2.data_ptr(), stride_of(x2), address(weight), mean if layer else 0, mean + 4 * rows,
             d2.data_ptr(), stride_of(d2), address(s2), stride_of(s2) if s2 is not None else 0, address(dx),
             address(dw), address(db), address(ws), rows, D, DTYPES[dtype], DTYPES[wdt], layer, stream_on(x2))
        return dx if need_x else None, dx if need_r else None, dw, db, None, None


def _norm(who, x, weight, bias, eps, residual, layer):
    if x.dtype not in DTYPES:
        raise TypeError(f"{who} takes bf16, fp16 or fp32 rows (got {x.dtype})")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"{who}: x {tuple(x.shape)}: needs a last dimension in [1, {MAX_WIDTH}]")
    if not eps >= 0:
        raise ValueError(f"{who}: eps={eps} must not be negative")
    require_on(who, "weight", weight, x)
    require_on(who, "bias", bias, x)
    require_on(who, "residual", residual, x)
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != (x.shape[-1],):
            raise ValueError(f"{who}: {name} {tuple(t.shape)}: expected [{x.shape[-1]}]")
        if t.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{who}: {name} {t.dtype}: expected x's type ({x.dtype}) or fp32")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"{who}: weight {weight.dtype} and bias {bias.dtype}: expected one type")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"{who}: residual {tuple(residual.shape)} {residual.dtype}: expected x's {tuple(x.shape)} "
                         f"{x.dtype}")
    require_gpu(who, x)
    if not current(x):
        with torch.cuda.device(x.device):
            return _norm(who, x, weight, bias, eps, residual, layer)
    weight = weight if weight is None else weight.contiguous()
    bias = bias if bias is None else bias.contiguous()
    eps = float(eps)
    if needs_grad(x, residual, weight, bias):
        return BlockNormFunction.apply(x, residual, weight, bias, layer, eps)
    y, s, _, _ = _forward(x, residual, weight, bias, layer, eps, False)
    return y if s is None else (y, s)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, residual: Optional[torch.Tensor] = None
               ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension (bf16, fp16 or fp32 on the GPU, 1 to
    8192 wide, any row stride); ``weight`` and ``bias`` ``[D]`` in x's type or fp32, each optional.  With
    ``residual`` (x's shape and type) the rows are ``s = x + residual``, rounded to their type as the residual
    stream holds them, and it returns ``(y, s)``.  Statistics and sums in fp32, one rounding of y.  Gradients of x,
    residual, weight and bias."""
    return _norm("layer_norm", x, weight, bias, eps, residual, 1)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
             residual: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension; otherwise as ``layer_norm``."""
    return _norm("rms_norm", x, weight, None, eps, residual, 0)
