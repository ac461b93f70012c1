"""A linear map with bias, activation and residual in its epilogue, for any number of rows, with gradients
(``ccq_linear_fwd`` / ``ccq_linear_bwd`` of ``libccq_hip.so``).

The reference's blocks run their projections and MLPs as ``nn.Linear`` and torch operations (``ccq/gdn/layer.py:
286-316, 408``; its HF models' MLP is fla's); ``prologue.narrow_linear`` is the form for at most 16 outputs and
``graph.decode_linear`` / ``decode_linear_glu`` those for a decode step's rows.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from ._rows import (DTYPES, address, call, current, entry, needs_grad, require_gpu, require_on, rows_of, stream_on,
                    stride_of)

__all__ = ["fused_linear", "FusedLinearFunction", "ACTIVATIONS"]

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "swish": 2, "gelu": 3, "gelu_tanh": 4, "swiglu": 5}  # CCQ_ACT_*
SWIGLU = ACTIVATIONS["swiglu"]
MAX_STRIDE = 1 << 22


def _operand(x2: torch.Tensor) -> torch.Tensor:
    """Rows as the products read them: 16-byte pieces, zeros up to a multiple of 8 columns.  A copy where x2's width,
    stride or address does not allow that."""
    rows, K = x2.shape
    ld = stride_of(x2)
    if K % 8 == 0 and ld % 8 == 0 and ld <= MAX_STRIDE and x2.data_ptr() % 16 == 0:
        return x2
    ldd = -(-K // 8) * 8
    out = x2.new_empty(rows, ldd)
    call("ccq_pad_rows", x2.data_ptr(), ld, out.data_ptr(), ldd, rows, K, stream_on(x2))
    return out


def _forward(x, weight, bias, residual, act, keep_z):
    x2, w2 = rows_of(x), rows_of(weight)
    (M, K), outs = x2.shape, w2.shape[0]
    N = outs // 2 if act == SWIGLU else outs
    r2 = rows_of(residual) if residual is not None else None
    y = x.new_empty(*x.shape[:-1], N)
    # what the activation's backward reads, in 24 bits
    z = x.new_empty(3 * M * (-(-outs // 8) * 8), dtype=torch.uint8) if keep_z and act else None
    xp, wp = _operand(x2), _operand(w2)
    n = entry("ccq_linear_workspace_bytes")(M, N, K, act)
    ws = x.new_empty(n, dtype=torch.uint8) if n else None
    call("ccq_linear_fwd", xp.data_ptr(), stride_of(xp), wp.data_ptr(), stride_of(wp), address(bias),
         DTYPES[bias.dtype if bias is not None else x.dtype], address(r2), stride_of(r2) if r2 is not None else 0,
         y.data_ptr(), address(z), address(ws), M, N, K, act, DTYPES[x.dtype], stream_on(x))
    return y, z, x2, w2


class FusedLinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        y, z, x2, w2 = _forward(x, weight, bias, residual, act, any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x2, w2, z)
        ctx.meta = (x.shape, y.shape[-1], act, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        saved = ctx.saved_tensors
        if not current(saved[0]):
            with torch.cuda.device(saved[0].device):
                return FusedLinearFunction._backward(ctx, *saved, dy)
        return FusedLinearFunction._backward(ctx, *saved, dy)

    @staticmethod
    def _backward(ctx, x2, w2, z, dy):
        shape, N, act, bdtype = ctx.meta
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            (M, K), outs = x2.shape, w2.shape[0]
            dtype = x2.dtype
            d2 = rows_of(dy)
            dx = x2.new_empty(shape) if need_x else None
            dw = x2.new_empty(outs, K) if need_w else None
            db = x2.new_empty(outs, dtype=bdtype) if need_b else None
            xp = _operand(x2) if need_w else None
            wp = _operand(w2) if need_x else None
            ld = -(-K // 8) * 8
            ws = x2.new_empty(entry("ccq_linear_bwd_workspace_bytes")(M, N, K, act), dtype=torch.uint8)
            call("ccq_linear_bwd", address(xp), stride_of(xp) if need_w else ld, address(wp),
                 stride_of(wp) if need_x else ld, address(z), d2.data_ptr(), stride_of(d2), address(dx), address(dw),
                 address(db), DTYPES[bdtype if bdtype is not None else dtype], ws.data_ptr(), M, N, K, act,
                 DTYPES[dtype], stream_on(x2))
        return dx, dw, db, dy if need_r else None, None


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 activation: Optional[str] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` (bf16 or fp16 on the GPU, any number of rows, any widths): the
    activation one of None, "relu", "silu" ("swish"), "gelu" (erf), "gelu_tanh", or "swiglu", where ``weight``
    ``[2 N, K]`` (and ``bias`` ``[2 N]``) hold the gate rows, then the up rows, and ``act(z) = silu(gate) * up``.
    ``bias`` in x's type or fp32; ``residual`` of the output's shape.  Products accumulate in fp32, and bias,
    activation and residual are applied there: one rounding of the output.  Gradients of all four tensors; the
    gradient of ``x @ weight.T + bias`` is rounded to x's type once, where it enters the products.  Rows that are
    not 16-byte aligned or an odd width are copied to padded rows first."""
    if x.dtype not in (torch.bfloat16, torch.float16) or weight.dtype != x.dtype:
        raise TypeError(f"fused_linear takes bf16 or fp16 x and weight of one type (got {x.dtype}, {weight.dtype})")
    if activation not in ACTIVATIONS:
        raise ValueError(f"fused_linear: activation {activation!r} is unknown (expected one of "
                         f"{', '.join(map(repr, ACTIVATIONS))})")
    act = ACTIVATIONS[activation]
    if (x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or not 1 <= x.shape[-1] <= MAX_STRIDE
            or not 1 <= weight.shape[0] <= MAX_STRIDE):
        raise ValueError(f"fused_linear: x {tuple(x.shape)} and weight {tuple(weight.shape)}: expected [..., K] and "
                         f"[outputs, K], both at least 1 wide and at most {MAX_STRIDE}")
    outs = weight.shape[0]
    if act == SWIGLU and outs % 2:
        raise ValueError(f"fused_linear: swiglu needs as many gate as up rows (weight has {outs})")
    require_on("fused_linear", "weight", weight, x)
    require_on("fused_linear", "bias", bias, x)
    require_on("fused_linear", "residual", residual, x)
    if bias is not None:
        if bias.shape != (outs,):
            raise ValueError(f"fused_linear: bias {tuple(bias.shape)}: expected [{outs}]")
        if bias.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"fused_linear: bias {bias.dtype}: expected x's type ({x.dtype}) or fp32")
    N = outs // 2 if act == SWIGLU else outs
    if residual is not None and (residual.shape != (*x.shape[:-1], N) or residual.dtype != x.dtype):
        raise ValueError(f"fused_linear: residual {tuple(residual.shape)} {residual.dtype}: expected "
                         f"{(*x.shape[:-1], N)} {x.dtype}")
    require_gpu("fused_linear", x)
    if not current(x):
        with torch.cuda.device(x.device):
            return fused_linear(x, weight, bias, activation, residual)
    bias = bias if bias is None else bias.contiguous()
    if needs_grad(x, weight, bias, residual):
        return FusedLinearFunction.apply(x, weight, bias, residual, act)
    return _forward(x, weight, bias, residual, act, False)[0]
