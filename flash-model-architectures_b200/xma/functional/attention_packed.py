"""attention_packed: causal attention with grouped heads over the packed token stream that pack_sequence makes
(the same cu_seqlens), forward and backward on tensor cores (csrc/attention.cu)."""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from .. import _native as N
from ..accelerator import KernelBackend, require_cuda_backend
from ..ops import attention_packed_backward_cuda, attention_packed_forward_cuda
from ._forward_mode import refuse_tangents

MAX_HEAD_DIM = 128
_MAX_TOKENS = 1 << 30
_MAX_SEQUENCES = 1 << 20
_MIN_SCALE = 2.0 ** -149  # float32's smallest number


def _tiled(t: torch.Tensor) -> torch.Tensor:
    """`t` itself where the copy engine can read it in place (heads contiguous, other strides multiples of 16
    bytes), else a contiguous copy: slices of a fused projection are read where they are."""
    (tokens, heads, _), (token, head, inner) = t.shape, t.stride()
    in_place = inner == 1 and (tokens <= 1 or (token > 0 and token % 8 == 0)) and (heads <= 1 or (head > 0 and head % 8 == 0))
    return t if in_place else t.contiguous()


def _forward(q, k, v, cu_seqlens, softmax_scale: float, saving: bool):
    q, k, v, cu_seqlens = _tiled(q), _tiled(k), _tiled(v), cu_seqlens.contiguous()
    total, heads, dim = q.shape
    batch = cu_seqlens.numel() - 1
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = out_rest = None
    if saving:
        out_rest = torch.empty(total, heads, -(-dim // 16) * 16, dtype=torch.uint8, device=q.device)
        lse = torch.empty(heads, N.attention_stat_rows(total, batch), dtype=torch.float32, device=q.device)
    workspace = torch.empty(N.attention_workspace_bytes(total, batch), dtype=torch.uint8, device=q.device)
    attention_packed_forward_cuda(q, k, v, cu_seqlens, softmax_scale, out, lse, out_rest, workspace)
    return out, (q, k, v, cu_seqlens, out, out_rest, lse)


class _AttentionPacked(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, softmax_scale: float):
        out, saved = _forward(q, k, v, cu_seqlens, softmax_scale, True)
        ctx.save_for_backward(*saved)
        ctx.softmax_scale = softmax_scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        refuse_tangents("attention_packed", d_out)
        q, k, v, cu_seqlens, out, out_rest, lse = ctx.saved_tensors
        opts = dict(dtype=q.dtype, device=q.device)
        dq, dk, dv = torch.empty(q.shape, **opts), torch.empty(k.shape, **opts), torch.empty(v.shape, **opts)
        delta = torch.empty_like(lse)
        workspace = torch.empty(N.attention_workspace_bytes(q.size(0), cu_seqlens.numel() - 1), dtype=torch.uint8, device=q.device)
        attention_packed_backward_cuda(
            q, k, v, cu_seqlens, ctx.softmax_scale, out, out_rest, d_out.contiguous(), lse, delta, dq, dk, dv, workspace)
        return dq, dk, dv, None, None


def attention_packed(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: torch.Tensor,
    *,
    softmax_scale: float | None = None,
    kernel_backend: KernelBackend | None = None,
) -> torch.Tensor:
    """Causal attention inside each sequence of a packed stream.

    `q` is `[total_tokens, heads, head_dim]`, `k` and `v` `[total_tokens, kv_heads, head_dim]`, in bfloat16 or
    float16; `heads` is a multiple of `kv_heads` (query head `h` reads head `h // (heads // kv_heads)`), `head_dim` a
    multiple of 8 up to 128. Any strides are taken; slices along the head dimension of one projection are read in
    place. `cu_seqlens` (`[sequences + 1]`, int32 or int64, on the same device) holds ascending offsets: sequence `b` is
    the tokens `cu_seqlens[b] .. cu_seqlens[b + 1] - 1` (none, one or many). `softmax_scale` is positive (a
    float32 number below 1e30) and defaults to `1 / sqrt(head_dim)`.

    Scores and sums are float32; probabilities are rounded to the inputs' dtype before they meet the values (in float16
    times a power of two, so that keys which others outweigh keep their share; in sequences of up to 128 tokens as two
    numbers, so that nothing is lost). For a backward pass the call keeps its inputs, its output, a float32 per row and
    head and, so that gradients do not suffer from the output's rounding, one byte per output element; gradients are
    summed in a fixed order. In float16 probabilities and the gradient of the scores are rounded with powers of two, the
    latter one that the batch's largest finite upstream gradient and value set, so small gradients keep their bits
    without loss scaling.

    Tokens that no sequence owns get zeros, in the output and in the gradients, and what they hold reaches nothing. A
    NaN or an infinity in a value also reaches rows before it in its own sequence, as in a product with probabilities
    that are zero there, and one in a key their gradients. Offsets are read on the device: values that are out of order
    or outside the stream give meaningless outputs, not an error. Forward-mode differentiation is refused."""
    require_cuda_backend(kernel_backend)
    dtype, device = q.dtype, q.device
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"q should be bfloat16 or float16, got {dtype}")
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 3:
            raise ValueError(f"{name} should be [tokens, heads, head_dim], got shape {tuple(t.shape)}")
        if t.dtype != dtype:
            raise ValueError(f"{name} should be {dtype} like q, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, q on {device}")
    total, heads, dim = q.shape
    if k.shape != v.shape:
        raise ValueError(f"k and v should have the same shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.size(0) != total or k.size(2) != dim:
        raise ValueError(f"k and v should be [{total}, kv_heads, {dim}], got {tuple(k.shape)}")
    if not 8 <= dim <= MAX_HEAD_DIM or dim % 8 != 0:
        raise ValueError(f"head_dim should be a multiple of 8 up to {MAX_HEAD_DIM}, got {dim}")
    if heads < 1 or k.size(1) < 1 or heads % k.size(1) != 0 or heads > 4096:
        raise ValueError(f"heads ({heads}) should be a multiple of kv_heads ({k.size(1)}), at most 4096")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"cu_seqlens should be a 1-dimensional int32 or int64 tensor of at least one offset, got "
                         f"{cu_seqlens.dtype} {tuple(cu_seqlens.shape)}")
    if cu_seqlens.device != device:
        raise ValueError(f"cu_seqlens is on {cu_seqlens.device}, q on {device}")
    if total > _MAX_TOKENS or cu_seqlens.numel() > _MAX_SEQUENCES:
        raise ValueError(f"at most {_MAX_TOKENS} tokens and {_MAX_SEQUENCES - 1} sequences are supported")
    scale = 1.0 / math.sqrt(dim) if softmax_scale is None else float(softmax_scale)
    if not _MIN_SCALE <= scale < 1e30:
        raise ValueError(f"softmax_scale should be a positive float32 number below 1e30, got {scale}")
    refuse_tangents("attention_packed", q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _AttentionPacked.apply(q, k, v, cu_seqlens, scale)
    return _forward(q, k, v, cu_seqlens, scale, False)[0]
