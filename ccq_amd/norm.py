"""Block norms: layer norm and RMS norm over the last dimension, with the residual stream's add in the same pass
(``ccq_norm_fwd`` / ``ccq_norm_bwd`` of ``libccq_hip.so``).

The reference's layers (``ccq/gdn/layer.py``, ``ccq/gla/layer.py``) sit in pre-norm blocks whose norms its HF
model classes take from fla; ``prologue.gated_rmsnorm`` is the norm inside the layers.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from ._native import ops

__all__ = ["layer_norm", "rms_norm"]


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, residual: Optional[torch.Tensor] = None
               ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension (bf16, fp16 or fp32 on the GPU, 1 to
    8192 wide, any stride between rows; leading dimensions without one such stride are copied); ``weight`` and ``bias``
    ``[D]`` in x's type or fp32, each optional.  With ``residual`` (x's shape and type) the rows are ``s = x + residual``,
    rounded to their type as the residual stream holds them, and it returns ``(y, s)``.  Statistics and sums in fp32, one
    rounding of y.  Gradients of x, residual, weight and bias (first derivatives, reverse mode)."""
    if residual is None:
        return ops().norm("layer_norm", x, weight, bias, eps, True)
    return ops().norm_residual("layer_norm", x, weight, bias, eps, residual, True)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
             residual: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension; otherwise as ``layer_norm``."""
    if residual is None:
        return ops().norm("rms_norm", x, weight, None, eps, False)
    return ops().norm_residual("rms_norm", x, weight, None, eps, residual, False)
