"""Forward-mode differentiation of kernels that have no rule for it."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad


def refuse_tangents(name: str, *tensors: torch.Tensor | None) -> None:
    """Raises if a tensor carries a forward-mode tangent. The kernels write through raw pointers and would drop it: a dual
    tensor has no `requires_grad`, so a call that skips autograd where nothing requires a gradient does not see it, and
    neither does a backward function."""
    if forward_ad._current_level < 0:  # no dual level is open: the usual case
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has no forward-mode derivative")
