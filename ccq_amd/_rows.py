"""What the operators over whole rows of several element types share: the types as the C ABI numbers them, views
of tensors as rows, and calls of the C entry points with little host time."""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib

DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # CCQ_DTYPE_*

_entries = {}


def entry(name: str):
    """The C entry point of that name."""
    f = _entries.get(name)
    if f is None:
        f = _entries[name] = getattr(_lib.load(), name)
    return f


def call(name: str, *args) -> None:
    """``_lib.call`` with addresses as plain numbers (0 or None for NULL)."""
    status = entry(name)(*args)
    if status:
        _lib.check(status, name)


def address(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def stream_on(x: torch.Tensor) -> int:
    """The current stream of x's device, as the C entry points take it."""
    return torch._C._cuda_getCurrentRawStream(x.device.index)


def rows_of(x: torch.Tensor) -> torch.Tensor:  # (host time counts: the common case first)
    """``x [..., D]`` as ``[rows, D]`` with consecutive elements and rows that do not overlap: a view where the
    strides allow one, a copy otherwise."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.is_contiguous():
        return x
    rows, D = x.shape
    if (x.stride(1) != 1 and D > 1) or (x.stride(0) < D and rows > 1):
        return x.contiguous()
    return x


def stride_of(x: torch.Tensor) -> int:
    """Elements between rows of ``rows_of``'s view, at least the row (the stride of a single row is any number)."""
    return max(x.stride(0), x.shape[1])


def current(x: torch.Tensor) -> bool:
    """Whether x's device is the current one, which the C entry points ask for."""
    return x.device.index == torch.cuda.current_device()


def like(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of x's shape, type and device."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def require_gpu(who: str, x: torch.Tensor) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"{who} runs on the GPU only (its input is on the {x.device.type})")


def require_on(who: str, name: str, t: Optional[torch.Tensor], x: torch.Tensor) -> None:
    """A tensor that must lie on x's device."""
    if t is not None and t.device != x.device:
        raise ValueError(f"{who}: {name} must be on {x.device} (got {t.device})")


def needs_grad(*xs) -> bool:
    if torch.is_grad_enabled():
        for x in xs:
            if x is not None and x.requires_grad:
                return True
    return False
