"""A linear map with bias, activation and residual in its epilogue, for any number of rows, with gradients
(``ccq_linear_fwd`` / ``ccq_linear_bwd`` of ``libccq_hip.so``).

The reference's blocks run their projections and MLPs as ``nn.Linear`` and torch operations (``ccq/gdn/layer.py:
286-316, 408``; its HF models' MLP is fla's); ``prologue.narrow_linear`` is the form for at most 16 outputs and
``graph.decode_linear`` / ``decode_linear_glu`` those for a decode step's rows.
"""

from __future__ import annotations

from typing import Optional

import torch

from ._native import ops

__all__ = ["fused_linear", "ACTIVATIONS"]

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "swish": 2, "gelu": 3, "gelu_tanh": 4, "swiglu": 5}  # CCQ_ACT_*


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 activation: Optional[str] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` (bf16 or fp16 on the GPU, any number of rows, any widths): the
    activation one of None, "relu", "silu" ("swish"), "gelu" (erf), "gelu_tanh", or "swiglu", where ``weight``
    ``[2 N, K]`` (and ``bias`` ``[2 N]``) hold the gate rows, then the up rows, and ``act(z) = silu(gate) * up``.
    ``bias`` in x's type or fp32; ``residual`` of the output's shape.  Products accumulate in fp32, and bias,
    activation and residual are applied there: one rounding of the output.  Gradients of all four tensors (first derivatives,
    reverse mode); the gradient of ``x @ weight.T + bias`` is rounded to x's type once, where it enters the products.  Rows
    that are not 16-byte aligned or an odd width are copied to padded rows first, in each direction; leading dimensions
    whose strides are not those of rows one after the other are copied too."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"fused_linear: activation {activation!r} is unknown (expected one of "
                         f"{', '.join(map(repr, ACTIVATIONS))})")
    return ops().fused_linear(x, weight, bias, act, residual)
