"""What the norms refuse, on the host."""

import pytest
import torch

import xma


def x(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call,match", [
    (lambda: xma.rmsnorm(x(2, 8, dtype=torch.float64), None), "bfloat16, float16 or float32"),
    (lambda: xma.rmsnorm(x(2, 8, dtype=torch.int32), None), "bfloat16, float16 or float32"),
    (lambda: xma.rmsnorm(x(2, 0), None), "last dimension"),
    (lambda: xma.rmsnorm(torch.zeros((), dtype=torch.bfloat16), None), "last dimension"),
    (lambda: xma.rmsnorm(x(2, 8), x(7)), "weight should have shape"),
    (lambda: xma.rmsnorm(x(2, 8), x(1, 8)), "weight should have shape"),
    (lambda: xma.rmsnorm(x(2, 8), x(8, dtype=torch.float16)), "weight should be"),
    (lambda: xma.rmsnorm(x(2, 8), x(8), -1e-5), "eps"),
    (lambda: xma.rmsnorm(x(2, 8), x(8), float("nan")), "eps"),
    (lambda: xma.fused_residual_add_rmsnorm(x(2, 8), x(1, 8), None), "residual should have the shape"),
    (lambda: xma.fused_residual_add_rmsnorm(x(2, 8), x(2, 8, dtype=torch.float16), None), "residual should be"),
    (lambda: xma.fused_residual_add_rmsnorm(x(2, 8), x(2, 8), None, post_weight=x(9)), "post_weight should have shape"),
    (lambda: xma.fused_residual_add_rmsnorm(x(2, 8), x(2, 8), None, gate=x(2)), "gate should have shape"),
    (lambda: xma.fused_residual_add_rmsnorm(x(2, 8), x(2, 8), None, gate=x(1, 8)), "gate should have shape"),
    (lambda: xma.fused_residual_add_rmsnorm(x(2, 8), x(2, 8), None, gate=x(2, 1, dtype=torch.float32)), "gate of every token"),
    (lambda: xma.fused_residual_add_rmsnorm(x(2, 8), x(2, 8), None, gate=x(2, 8, dtype=torch.float32)), "gate should have shape"),
    (lambda: xma.fused_residual_add_rmsnorm(x(2, 8), x(2, 8), None, gate=x(8, dtype=torch.float16)), "gate should be"),
    (lambda: xma.rmsnorm(x(2, 8), x(8), kernel_backend=xma.KernelBackend.triton), "kernel_backend"),
])
def test_refused(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU path"):
        xma.rmsnorm(x(2, 8), x(8))


def test_c_entry_refuses():
    """Bad sizes and pointers come back as a status, before anything is launched."""
    from xma import _native as N

    lib = N.lib()
    forward = lambda x=1 << 20, res=None, w=None, post=None, gate=None, mode=0, dt=0, sdt=0, rows=1, hidden=8, out=None, y=1 << 20: lib.xma_norm_forward(
        x, res, w, post, gate, mode, dt, sdt, 0, rows, hidden, 1e-5, 1.0, out, y, None, None, None, None)
    assert forward(rows=0) == 0
    assert forward(rows=-1) == 1 and forward(hidden=0) == 1 and forward(x=None) == 1 and forward(y=None) == 1
    assert forward(mode=4) == 1 and forward(mode=1) == 1 and forward(res=1 << 20) == 1
    assert forward(post=1 << 20) == 1 and forward(sdt=2) == 1  # a post norm or another stream type without a residual
    assert forward(res=1 << 20, out=1 << 20, dt=0, sdt=1) == 2 and forward(dt=3, sdt=3) == 2
    assert lib.xma_norm_workspace_floats(3, 5) == N.norm_workspace_floats(3, 5)


@pytest.mark.parametrize("which", ["x", "residual", "weight", "post_weight", "gate"])
def test_forward_mode_is_refused(which):
    """A dual tensor has no requires_grad; its tangent is not dropped in silence."""
    from torch.autograd import forward_ad

    t = {"x": x(2, 8), "residual": x(2, 8), "weight": x(8), "post_weight": x(8), "gate": x(2, 1)}
    with forward_ad.dual_level():
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            xma.fused_residual_add_rmsnorm(t["x"], t["residual"], t["weight"], post_weight=t["post_weight"], gate=t["gate"])
        if which in ("x", "weight"):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                xma.rmsnorm(t["x"], t["weight"])
        with pytest.raises(RuntimeError, match="no CPU path"):  # a level that is open is no reason
            xma.rmsnorm(x(2, 8), x(8))
