"""rmsnorm and fused_residual_add_rmsnorm, the functionals of those names in the reference
(xma/functional/__init__.py:5-16), extended to the norm after a block, the block's gate and the scale of
its residual add; one kernel forward and one (plus a small sum) backward."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _native as N
from ..accelerator import KernelBackend, require_cuda_backend
from ..ops import norm_backward_cuda, norm_forward_cuda
from ._forward_mode import refuse_tangents

GATE_NONE, GATE_CHANNEL, GATE_TOKEN, GATE_FULL = 0, 1, 2, 3
_MAX_HIDDEN = 1 << 24


def _forward(x, residual, weight, post_weight, gate, gate_mode: int, eps: float, multiplier: float, saving: bool):
    """(y, stream or None, contiguous inputs, row statistics of both norms): the forward launch."""
    x = x.contiguous()
    residual = None if residual is None else residual.contiguous()
    weight = None if weight is None else weight.contiguous()
    post_weight = None if post_weight is None else post_weight.contiguous()
    gate = None if gate is None else gate.contiguous()
    y = torch.empty_like(x)
    stream = None if residual is None else torch.empty_like(residual)
    rstd = torch.empty(2, x.numel() // x.size(-1), dtype=torch.float32, device=x.device) if saving else None
    norm_forward_cuda(x, residual, weight, post_weight, gate, gate_mode, eps, multiplier, stream, y, rstd)
    return y, stream, (x, residual, weight, post_weight, gate), rstd


class _Norm(torch.autograd.Function):
    """Rows of any leading shape; returns y, or (y, stream) with a residual."""

    @staticmethod
    def forward(ctx, x, residual, weight, post_weight, gate, gate_mode: int, eps: float, multiplier: float):
        y, stream, (x, residual, weight, post_weight, gate), rstd = _forward(
            x, residual, weight, post_weight, gate, gate_mode, eps, multiplier, True)
        if residual is None:
            base, branch = x, None
        elif post_weight is None and gate is None:
            base, branch = stream, None  # a plain residual add: the stream alone will do
        else:
            base, branch = residual, x  # the stream is computed from them again, before its rounding
        ctx.save_for_backward(base, branch, weight, post_weight, gate, rstd)
        ctx.dtype, ctx.alone = x.dtype, residual is None
        ctx.gate_mode, ctx.multiplier = gate_mode, multiplier
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, stream)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, d_stream=None):
        refuse_tangents("rmsnorm" if ctx.alone else "fused_residual_add_rmsnorm", dy, d_stream)
        base, x, weight, post_weight, gate, rstd = ctx.saved_tensors
        dy = None if dy is None else dy.contiguous()
        d_stream = None if d_stream is None else d_stream.contiguous()
        want_x, want_residual, want_weight, want_post, want_gate = ctx.needs_input_grad[:5]
        empty = base.numel() == 0

        # The norm alone differentiates with respect to its "stream", x. A plain residual add in one type
        # gives x and the residual the same gradient: one tensor.
        shared = not ctx.alone and x is None and ctx.multiplier == 1.0 and base.dtype == ctx.dtype
        want_stream = want_x if ctx.alone else want_residual or (shared and want_x)
        d_residual = torch.empty_like(base) if want_stream else None
        dx = None
        if want_x and not ctx.alone and not shared:
            dx = torch.empty_like(base, dtype=ctx.dtype)
        new = torch.zeros_like if empty else torch.empty_like
        d_weight = new(weight) if want_weight and weight is not None else None
        d_post = new(post_weight) if want_post and post_weight is not None else None
        d_gate = new(gate) if want_gate and gate is not None else None
        if not empty:
            hidden = base.size(-1)
            workspace = torch.empty(N.norm_workspace_floats(base.numel() // hidden, hidden), dtype=torch.float32, device=base.device)
            norm_backward_cuda(
                dy, d_stream, base, x, weight, post_weight, gate, ctx.gate_mode, ctx.dtype, ctx.multiplier, rstd,
                dx, d_residual, d_gate, d_weight, d_post, workspace)
        if ctx.alone:
            return d_residual, None, d_weight, None, None, None, None, None
        if shared:
            dx = d_residual if want_x else None
            d_residual = d_residual if want_residual else None
        return dx, d_residual, d_weight, d_post, d_gate, None, None, None


def _norm(x, residual, weight, post_weight, gate, gate_mode: int, eps: float, multiplier: float):
    refuse_tangents("rmsnorm" if residual is None else "fused_residual_add_rmsnorm", x, residual, weight, post_weight, gate)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight, post_weight, gate)):
        return _Norm.apply(x, residual, weight, post_weight, gate, gate_mode, eps, multiplier)
    y, stream, _, _ = _forward(x, residual, weight, post_weight, gate, gate_mode, eps, multiplier, False)
    return y if residual is None else (y, stream)


def _check_rows(x: torch.Tensor) -> None:
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"x should be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() < 1 or not 1 <= x.size(-1) <= _MAX_HIDDEN:
        raise ValueError(f"x should have a last dimension of 1 to {_MAX_HIDDEN} elements, got shape {tuple(x.shape)}")


def _check_parameter(name: str, t: torch.Tensor | None, x: torch.Tensor) -> None:
    if t is None:
        return
    if t.dim() != 1 or t.size(0) != x.size(-1):
        raise ValueError(f"{name} should have shape {tuple(x.shape[-1:])}, got {tuple(t.shape)}")
    if t.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"{name} should be {x.dtype} or float32, got {t.dtype}")
    if t.device != x.device:
        raise ValueError(f"{name} is on {t.device}, x on {x.device}")


def _eps(eps: float | None, x: torch.Tensor) -> float:
    eps = torch.finfo(x.dtype).eps if eps is None else float(eps)
    if not 0 <= eps < float("inf"):
        raise ValueError(f"eps should be finite and not negative, got {eps}")
    return eps


def rmsnorm(
    x: torch.Tensor, weight: torch.Tensor | None, eps: float | None = None, *, kernel_backend: KernelBackend | None = None
) -> torch.Tensor:
    """`weight * x / sqrt(mean(x^2, -1) + eps)`, computed in float32 and rounded once to the dtype of `x`.

    `weight` is `[H]` in the dtype of `x` or in float32, or None (ones). `eps=None` takes the machine epsilon of
    the dtype of `x`. Forward-mode differentiation is refused."""
    require_cuda_backend(kernel_backend)
    _check_rows(x)
    _check_parameter("weight", weight, x)
    return _norm(x, None, weight, None, None, GATE_NONE, _eps(eps, x), 1.0)


def fused_residual_add_rmsnorm(
    x: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor | None,
    eps: float | None = None,
    multiplier: float | None = None,
    *,
    post_weight: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    kernel_backend: KernelBackend | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Joins the output `x` of a block to the residual stream and norms the result for the next block:

        u = x if post_weight is None else rmsnorm(x, post_weight, eps)
        stream = residual + multiplier * gate * u
        y = rmsnorm(stream, weight, eps)

    and returns `(y, stream)`. All of it runs in float32; `y` is taken before `stream` is rounded.

    `residual` (and with it `stream`) has the shape of `x` and its dtype or float32. `gate` is `[H]` (a
    parameter), one factor per token (the shape of `x` with a last dimension of 1) or has the shape of `x`; a
    gate that is not `[H]` has the dtype of `x`, the parameters that or float32. `weight=None` norms without a
    weight, `multiplier=None` is 1, `eps=None` the machine epsilon of the dtype of `x`. Forward-mode differentiation is
    refused."""
    require_cuda_backend(kernel_backend)
    _check_rows(x)
    if residual.shape != x.shape:
        raise ValueError(f"residual should have the shape of x, {tuple(x.shape)}, got {tuple(residual.shape)}")
    if residual.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"residual should be {x.dtype} or float32, got {residual.dtype}")
    if residual.device != x.device:
        raise ValueError(f"residual is on {residual.device}, x on {x.device}")
    _check_parameter("weight", weight, x)
    _check_parameter("post_weight", post_weight, x)
    gate_mode = GATE_NONE
    if gate is not None:
        if gate.shape == x.shape and gate.dtype == x.dtype:
            gate_mode = GATE_FULL
        elif gate.shape == x.shape[-1:]:
            _check_parameter("gate", gate, x)
            gate_mode = GATE_CHANNEL
        elif gate.shape == x.shape[:-1] + (1,):
            gate_mode = GATE_TOKEN
        else:
            raise ValueError(
                f"gate should have shape {tuple(x.shape[-1:])}, {tuple(x.shape[:-1]) + (1,)} or, in {x.dtype}, {tuple(x.shape)}, "
                f"got {tuple(gate.shape)} {gate.dtype}")
        if gate_mode != GATE_CHANNEL and gate.dtype != x.dtype:
            raise ValueError(f"a gate of every token should be {x.dtype}, got {gate.dtype}")
        if gate.device != x.device:
            raise ValueError(f"gate is on {gate.device}, x on {x.device}")
    return _norm(x, residual, weight, post_weight, gate, gate_mode, _eps(eps, x), 1.0 if multiplier is None else float(multiplier))
