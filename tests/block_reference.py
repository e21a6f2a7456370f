"""Plain 64-bit forms of the operators around the expert layer, each value with the magnitude that its rounding
errors scale with (the same sum with absolute values), for the tests' error bounds."""

from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24  # half a step of float32, relative


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def norm_reference(x, residual, weight, post, gate, eps, m, dy=None, dd=None, stream_rounded=None):
    """dict name -> (value, magnitude) in float64. All inputs 2-D rows (gate broadcastable) or [H]; gradients use
    `stream_rounded` (the stream as it was returned), if it is given, where the backward pass reads it (a plain residual add)."""
    f = lambda t: None if t is None else t.detach().double()
    x, residual, weight, post, gate, dy, dd = map(f, (x, residual, weight, post, gate, dy, dd))
    H = x.size(-1)
    one = torch.ones((), dtype=torch.float64, device=x.device)
    w = one if weight is None else weight
    p = one if post is None else post
    g = one if gate is None else gate
    out = {}
    if residual is None:
        rp, branch, s, mag = one, None, x, x.abs()
    else:
        rp = one if post is None else torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)
        branch = m * g * p * x * rp
        s = residual + branch
        mag = residual.abs() + branch.abs()
        out["stream"] = (s, mag)
    rs = torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + eps)
    # rounding of s moves rs by at most the mean of |s| |ds| over the mean square
    spread = (s.abs() * mag).mean(-1, keepdim=True) * rs * rs
    out["y"] = (w * s * rs, (w * rs).abs() * (mag + s.abs() * (1 + spread)))
    if dy is None and dd is None:
        return out
    sr = s if stream_rounded is None else stream_rounded.detach().double()
    dy = torch.zeros_like(x) if dy is None else dy
    a = w * dy
    d = torch.zeros_like(s) if dd is None else dd
    mean_as, mean_as_mag = (a * sr).mean(-1, keepdim=True), (a * sr).abs().mean(-1, keepdim=True)
    ds = rs * (a - sr * rs * rs * mean_as) + d
    ds_mag = (rs * (a.abs() + sr.abs() * rs * rs * mean_as_mag) + d.abs()) * (1 + spread)
    out["d_weight"] = ((dy * sr * rs).sum(0), ((dy * sr * rs).abs() * (1 + spread)).sum(0))
    if residual is None:
        out["d_x"] = (ds, ds_mag)
        return out
    out["d_residual"] = (ds, ds_mag)
    u = p * x * rp
    dz, dz_mag = m * ds, abs(m) * ds_mag
    du, du_mag = dz * g, dz_mag * g.abs()
    if gate is not None:
        dg, dg_mag = dz * u, dz_mag * u.abs()
        if gate.dim() == 1:
            dg, dg_mag = dg.sum(0), dg_mag.sum(0)
        elif gate.size(-1) == 1 and H > 1:
            dg, dg_mag = dg.sum(-1, keepdim=True), dg_mag.sum(-1, keepdim=True)
        out["d_gate"] = (dg, dg_mag)
    if post is not None:
        hat = x * rp
        b, b_mag = du * p, du_mag * p.abs()
        out["d_post_weight"] = ((du * hat).sum(0), (du_mag * hat.abs()).sum(0))
        out["d_x"] = (rp * (b - hat * (b * hat).mean(-1, keepdim=True)),
                      rp * (b_mag + hat.abs() * (b_mag * hat.abs()).mean(-1, keepdim=True)))
    else:
        out["d_x"] = (du, du_mag)
    return out


def assert_within(name: str, got: torch.Tensor, value: torch.Tensor, bound: torch.Tensor) -> None:
    """|got - value| <= bound everywhere, with the worst place in the message."""
    err = (got.detach().double() - value).abs()
    bad = ~(err <= bound)
    if bad.any():
        at = (err / bound.clamp_min(1e-300)).nan_to_num(nan=math.inf).argmax()
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} outside; worst at flat {int(at)}: got "
                             f"{got.flatten()[at].item()}, want {value.flatten()[at].item()}, bound {bound.expand_as(value).flatten()[at].item()}")
