"""Serving in 8 bits: rows and weights in e4m3 with a power-of-two scale for each block of 128, the RMS norm that leaves
its rows so, and the linear map over two operands of that form (``ccq_quantize_fp8``, ``ccq_norm_fp8_fwd``,
``ccq_fp8_linear`` of ``libccq_hip.so``).

The reference has no 8-bit path: its projections are ``nn.Linear`` in the activations' type (``ccq/gdn/layer.py:286-316,
408``).  ``fused_linear`` and ``rms_norm`` are the forms that train.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from ._native import ops
from .linear import ACTIVATIONS

__all__ = ["Fp8Rows", "quantize_fp8", "rms_norm_fp8", "fp8_linear"]


class Fp8Rows(NamedTuple):
    """Rows in 8 bits: ``values`` ``[..., D]`` (``float8_e4m3fn``) and ``scales`` ``[..., ceil(D / 128)]``
    (``float8_e8m0fnu``, powers of two); element k of a row stands for ``values[k] * scales[k // 128]``.  The operators
    here lay value rows out at multiples of 16 bytes and scale rows at multiples of 4, as the products read them;
    rows laid out otherwise are taken too, and copied at every call."""

    values: torch.Tensor
    scales: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The numbers that the rows stand for, in ``dtype``."""
        scales = self.scales.to(torch.float32).repeat_interleave(128, -1)[..., :self.values.shape[-1]]
        return (self.values.to(torch.float32) * scales).to(dtype)


def quantize_fp8(x: torch.Tensor) -> Fp8Rows:
    """Rows (bf16, fp16 or fp32 on the GPU, at most 4 Mi wide, any stride between rows) in 8 bits: the scale of a block of 128
    consecutive elements is the least power of two from 2^-126 on that brings its largest magnitude to 448 or below, and
    the values round to the nearest, ties to even.  A block with an infinity or NaN is NaN, its scale too.  A weight
    ``[outputs, K]`` for ``fp8_linear`` is quantised once, when it is loaded.  Inference only."""
    return Fp8Rows(*ops().quantize_fp8(x))


def rms_norm_fp8(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
                 residual: Optional[torch.Tensor] = None) -> Union[Fp8Rows, Tuple[Fp8Rows, torch.Tensor]]:
    """``rms_norm`` with its result in 8 bits (``quantize_fp8`` of the result in fp32: one rounding), for rows of at most 8192 as
    there; wider ones are normed by other means and given to ``quantize_fp8``.  With ``residual`` it returns ``(y, s)``, the
    stream ``s = x + residual`` in x's type.  Inference only: tensors that need gradients are refused while gradients are
    recorded."""
    values, scales, s = ops().rms_norm_fp8(x, weight, eps, residual)
    return Fp8Rows(values, scales) if residual is None else (Fp8Rows(values, scales), s)


def fp8_linear(x: Fp8Rows, weight: Fp8Rows, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
               residual: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16,
               quantize: bool = False) -> Union[torch.Tensor, Fp8Rows]:
    """``act(x @ weight.T + bias) + residual`` over rows in 8 bits: x ``[..., K]``, weight ``[outputs, K]`` (``swiglu``: the gate
    rows, then the up rows), activations as ``fused_linear``'s; ``bias`` in bf16, fp16 or fp32.  Products accumulate in fp32
    on the matrix cores, which apply the scales, and bias, activation and residual are applied there.  The result is rounded
    once, to ``dtype`` (bf16, fp16 or fp32; ``residual`` has the same), or with ``quantize`` to 8 bits, as the next
    ``fp8_linear`` takes it (no residual then).  Sums into fp32 are exact but for fp32's additions; into 16 and 8 bits the
    matrix instruction cuts off, of each eight consecutive products, what lies below 2^-13 of the largest one's power of
    two: 1.5e-5 of a result on normal data (about one 8-bit output in a thousand rounds to its other neighbour), up to 9e-5
    with channels 100 to 1000 times the others, and where such channels cancel in a result 3e-4 to 4e-3 of what is left.
    Where that is too much, call it with ``dtype=torch.float32`` (and the residual in fp32) and round its result: ``.to`` of
    a 16-bit type, or ``quantize_fp8``.  Inference only, as ``rms_norm_fp8``."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"fp8_linear: activation {activation!r} is unknown (expected one of "
                         f"{', '.join(map(repr, ACTIVATIONS))})")
    y, scales = ops().fp8_linear(x[0], x[1], weight[0], weight[1], bias, act, residual, dtype, quantize)
    return Fp8Rows(y, scales) if quantize else y
