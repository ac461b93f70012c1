"""The PyTorch side of the operators around the mixers (``csrc/ccq_torch.cpp``), loaded at their first call.

It is built in-tree beside ``libccq_hip.so`` by ``ccq_amd/build.py``; a call fails loudly where it is missing.
"""

from __future__ import annotations

import os

import torch  # noqa: F401  (its libraries have to be loaded first)

PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_ccq_torch.so")

_ops = None


def ops():
    """The module of the compiled entry points."""
    global _ops
    if _ops is None:
        if not os.path.exists(PATH):
            raise RuntimeError(f"{PATH} is missing: build it with `python -m ccq_amd.build` "
                               "(or __graft_entry__.build()); the operators have no fallback")
        from . import _ccq_torch
        _ops = _ccq_torch
    return _ops
