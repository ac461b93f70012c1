"""What the operators over whole rows of several element types share: the types as the C ABI numbers them, views
of tensors as rows, and the device a call runs on."""

from __future__ import annotations

import contextlib

import torch

DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # CCQ_DTYPE_*


def rows_of(x: torch.Tensor) -> torch.Tensor:
    """``x [..., D]`` as ``[rows, D]`` with consecutive elements and rows that do not overlap: a view where the
    strides allow one, a copy otherwise."""
    D = x.shape[-1]
    if x.dim() != 2:
        x = x.reshape(-1, D) if D else x.reshape(0, 0)
    if (x.stride(1) != 1 and D > 1) or (x.stride(0) < D and x.shape[0] > 1):
        x = x.contiguous()
    return x


def stride_of(x: torch.Tensor) -> int:
    """Elements between rows of ``rows_of``'s view, at least the row (the stride of a single row is any number)."""
    return max(x.stride(0), x.shape[1])


def on_device(x: torch.Tensor):
    """A context in which ``x``'s device is the current one, which the C entry points ask for."""
    if x.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(x.device)


def require_gpu(who: str, x: torch.Tensor) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"{who} runs on the GPU only (its input is on the {x.device.type})")


def require_like(who: str, x: torch.Tensor, **tensors) -> None:
    """Tensors that must lie on x's device."""
    for name, t in tensors.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{who}: {name} must be on {x.device} (got {t.device})")


def needs_grad(*xs) -> bool:
    return torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in xs)
