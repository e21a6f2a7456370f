"""What attention_packed refuses, on the host."""

import pytest
import torch

import xma


def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


CU = torch.tensor([0, 4], dtype=torch.int32)


@pytest.mark.parametrize("q,k,v,cu,options,match", [
    (t(4, 64), t(4, 2, 64), t(4, 2, 64), CU, {}, "q should be \\[tokens"),
    (t(4, 2, 64), t(4, 64), t(4, 64), CU, {}, "k should be \\[tokens"),
    (t(4, 2, 64, dtype=torch.float32), t(4, 2, 64), t(4, 2, 64), CU, {}, "bfloat16 or float16"),
    (t(4, 2, 64), t(4, 2, 64, dtype=torch.float16), t(4, 2, 64), CU, {}, "like q"),
    (t(4, 2, 64), t(4, 2, 64), t(4, 1, 64), CU, {}, "same shape"),
    (t(4, 2, 64), t(5, 2, 64), t(5, 2, 64), CU, {}, "k and v should be"),
    (t(4, 2, 64), t(4, 2, 32), t(4, 2, 32), CU, {}, "k and v should be"),
    (t(4, 2, 60), t(4, 2, 60), t(4, 2, 60), CU, {}, "head_dim"),
    (t(4, 2, 136), t(4, 2, 136), t(4, 2, 136), CU, {}, "head_dim"),
    (t(4, 2, 0), t(4, 2, 0), t(4, 2, 0), CU, {}, "head_dim"),
    (t(4, 3, 64), t(4, 2, 64), t(4, 2, 64), CU, {}, "multiple of kv_heads"),
    (t(4, 2, 64), t(4, 0, 64), t(4, 0, 64), CU, {}, "multiple of kv_heads"),
    (t(4, 0, 64), t(4, 1, 64), t(4, 1, 64), CU, {}, "multiple of kv_heads"),
    (t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), CU.float(), {}, "cu_seqlens"),
    (t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), CU[None], {}, "cu_seqlens"),
    (t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), CU[:0], {}, "cu_seqlens"),
    (t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), CU.to("meta"), {}, "cu_seqlens is on"),
    (t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), CU, {"softmax_scale": 0.0}, "softmax_scale"),
    (t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), CU, {"softmax_scale": -1.0}, "softmax_scale"),
    (t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), CU, {"softmax_scale": float("inf")}, "softmax_scale"),
    (t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), CU, {"kernel_backend": xma.KernelBackend.torch}, "kernel_backend"),
])
def test_refused(q, k, v, cu, options, match):
    with pytest.raises(ValueError, match=match):
        xma.attention_packed(q, k, v, cu, **options)


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU path"):
        xma.attention_packed(t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), CU)


def test_c_entry_refuses():
    from xma import _native as N

    lib, a = N.lib(), 1 << 20
    def forward(q=a, k=a, v=a, strides=(128, 64) * 3, dt=0, cu=a, batch=1, total=4, heads=2, kv=2, dim=64, scale=0.1, out=a, rest=None, ws=a):
        return lib.xma_attention_forward(q, k, v, *strides, dt, cu, 0, batch, total, heads, kv, dim, scale, out, None, rest, ws, None, None)

    assert forward(total=0) == 0
    assert forward(q=None) == 1 and forward(out=None) == 1 and forward(ws=None) == 1 and forward(cu=None) == 1
    assert forward(q=a + 2) == 1 and forward(out=a + 8) == 1 and forward(batch=-1) == 1 and forward(total=-1) == 1
    assert forward(strides=(128, 64, 128, 60, 128, 64)) == 1 and forward(strides=(0, 64) * 3) == 1
    assert forward(scale=0.0) == 1 and forward(scale=float("nan")) == 1
    assert forward(rest=a) == 1  # what the backward pass needs is written as a whole or not at all
    assert forward(dt=2) == 2 and forward(dim=20) == 2 and forward(dim=136) == 2 and forward(heads=3) == 2
    assert forward(batch=1 << 21) == 2 and forward(total=1 << 31) == 2
    for total, batch in ((0, 0), (1, 1), (127, 3), (128, 1), (100000, 77)):
        assert lib.xma_attention_workspace_bytes(total, batch) == N.attention_workspace_bytes(total, batch)
        assert lib.xma_attention_stat_rows(total, batch) == N.attention_stat_rows(total, batch)


def test_settle_selftest_refuses():
    from xma import _native as N

    f, a = N.lib().xma_selftest_settle, 1 << 20
    assert f(None, 1, a, a, 1000, None) == 1 and f(a + 8, 1, a, a, 1000, None) == 1 and f(a, 1, None, a, 1000, None) == 1
    assert f(a, 65, a, a, 1000, None) == 1 and f(a, -1, a, a, 1000, None) == 1 and f(a, 1, a, a, 0, None) == 1
    assert f(a, 1, a, a, 2_000_000_000, None) == 1 and f(a, 1, a, None, 1000, None) == 1


@pytest.mark.parametrize("which", range(3))
def test_forward_mode_is_refused(which):
    """A dual tensor has no requires_grad; its tangent is not dropped in silence."""
    from torch.autograd import forward_ad

    inputs = [t(4, 2, 64), t(4, 2, 64), t(4, 2, 64)]
    with forward_ad.dual_level():
        inputs[which] = forward_ad.make_dual(inputs[which], torch.ones_like(inputs[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            xma.attention_packed(*inputs, CU)
        with pytest.raises(RuntimeError, match="no CPU path"):  # a level that is open is no reason
            xma.attention_packed(t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), CU)


@pytest.mark.parametrize("scale", [1e-50, 3e38, 1e39, float("nan"), float("-inf")])
def test_scales_that_float32_cannot_work_with(scale):
    from xma import _native as N

    with pytest.raises(ValueError, match="softmax_scale"):
        xma.attention_packed(t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), CU, softmax_scale=scale)
    a = 1 << 20
    assert N.lib().xma_attention_forward(a, a, a, *(128, 64) * 3, 0, a, 0, 1, 0, 2, 2, 64, scale, a, None, None, a, None, None) == 1
