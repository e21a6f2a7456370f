"""The operators around the expert layer as they are used together: a padded batch is packed, goes through norm,
attention, norm with gate and residual, the expert layer and the norm after it, and is unpacked; forward and backward
against plain float32 torch on the CPU-side oracle's expert layer.

Bound: the 2-norm of a tensor's error over that of the tensor. Every tensor passes about 20 roundings to bf16 on its way
forward and as many backward, each of 2^-9 / sqrt(3) of the rounded tensor and independent: sqrt(40) * 2^-9.8 = 0.7 %;
a factor of four on top covers the tensors that are differences of larger ones."""

import math

import pytest
import torch

import xma
from gpu_helpers import assert_status_clean
from oracle import moe_oracle as O
from xma.layers.moe.routing import router_topk_softmax

pytestmark = pytest.mark.gpu

LENGTHS, B, S, HEADS, KV, D, H, I, E, K, EPS, M = [37, 200, 1, 129], 4, 200, 8, 2, 64, 512, 256, 8, 2, 1e-5, 0.5


def parameters(dtype):
    g = torch.Generator(device="cuda").manual_seed(0)
    n = lambda *s, scale, shift=0.0: (torch.randn(*s, device="cuda", generator=g) * scale + shift).to(dtype).requires_grad_()
    return {
        "w1": n(H, scale=0.1, shift=1.0), "qkv": n((HEADS + 2 * KV) * D, H, scale=H ** -0.5),
        "out": n(H, HEADS * D, scale=(HEADS * D) ** -0.5), "post1": n(H, scale=0.1, shift=1.0),
        "gate1": n(H, scale=0.1, shift=0.7), "w2": n(H, scale=0.1, shift=1.0), "post2": n(H, scale=0.1, shift=1.0),
        "w3": n(H, scale=0.1, shift=1.0),
    }


def block(x, p, moe, cu):
    (tokens,) = xma.pack_sequence([x], cu, sum(LENGTHS), padding_side="right")
    h = xma.rmsnorm(tokens, p["w1"], EPS)
    qkv = (h @ p["qkv"].t()).view(-1, HEADS + 2 * KV, D)
    a = xma.attention_packed(qkv[:, :HEADS], qkv[:, HEADS: HEADS + KV], qkv[:, HEADS + KV:], cu)
    a = a.reshape(-1, HEADS * D) @ p["out"].t()
    h, stream = xma.fused_residual_add_rmsnorm(a, tokens, p["w2"], EPS, M, post_weight=p["post1"], gate=p["gate1"])
    mlp, logits = moe(h)
    y, stream = xma.fused_residual_add_rmsnorm(mlp, stream, p["w3"], EPS, M, post_weight=p["post2"])
    return xma.unpack_sequence([y, stream], cu, B, S, padding_side="right"), logits


def plain(x, p, moe_weights, selected):
    norm = lambda t, w: t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + EPS) * w
    tokens = torch.cat([x[b, :n] for b, n in enumerate(LENGTHS)])
    h = norm(tokens, p["w1"])
    qkv = (h @ p["qkv"].t()).view(-1, HEADS + 2 * KV, D)
    rows, at = [], 0
    for n in LENGTHS:
        q, k, v = qkv[at: at + n].split([HEADS, KV, KV], 1)
        k, v = k.repeat_interleave(HEADS // KV, 1), v.repeat_interleave(HEADS // KV, 1)
        s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(D)
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), -math.inf)
        rows.append(torch.einsum("hij,jhd->ihd", s.softmax(-1), v))
        at += n
    a = torch.cat(rows).reshape(-1, HEADS * D) @ p["out"].t()
    stream = tokens + M * p["gate1"] * norm(a, p["post1"])
    mlp = O.moe_forward(norm(stream, p["w2"]), *moe_weights, K, selected_experts=selected)[0]
    stream = stream + M * norm(mlp, p["post2"])
    out = []
    for t in (norm(stream, p["w3"]), stream):
        padded, at = torch.zeros_like(x), 0
        for b, n in enumerate(LENGTHS):
            padded[b, :n] = t[at: at + n]
            at += n
        out.append(padded)
    return out


def test_block_forward_and_backward():
    dtype = torch.bfloat16
    torch.manual_seed(0)
    with torch.device("cuda"):
        moe = xma.MoE(E, K, H, I, xma.swiglu_packed, True, False, 0.05).to(dtype)
    with torch.no_grad():
        moe.gate.weight.normal_(0, 0.05)
    p = parameters(dtype)
    x = torch.randn(B, S, H, device="cuda").to(dtype).requires_grad_()
    cu = torch.tensor([0] + LENGTHS, device="cuda").cumsum(0).to(torch.int32)
    upstream = [torch.randn(B, S, H, device="cuda").to(dtype) for _ in range(2)]
    leaves = {"x": x, **p, "moe.gate": moe.gate.weight, "moe.fc": moe.c_fc.weight, "moe.proj": moe.c_proj.weight}

    outputs, logits = block(x, p, moe, cu)
    grads = torch.autograd.grad(outputs, list(leaves.values()), upstream)
    assert_status_clean(x.device)

    selected = router_topk_softmax(logits.detach(), K)[1]
    wide = {k: v.detach().float().requires_grad_() for k, v in leaves.items()}
    want = plain(wide["x"], wide, (wide["moe.gate"], wide["moe.fc"], wide["moe.proj"]), selected)
    want_grads = torch.autograd.grad(want, list(wide.values()), [u.float() for u in upstream])
    for name, got, ref in [*zip(("y", "stream"), outputs, want), *zip(leaves, grads, want_grads)]:
        error = ((got.float() - ref).norm() / ref.norm()).item()
        assert error < 0.028, f"{name}: {error}"
    again, _ = block(x, p, moe, cu)
    for a, b in zip(again, outputs):
        assert torch.equal(a, b)


def test_block_captured():
    """The whole step in one CUDA graph: the replay on other tokens and lengths gives what an eager call gives."""
    torch.manual_seed(1)
    with torch.device("cuda"):
        moe = xma.MoE(E, K, H, I, xma.swiglu_packed, True, False, 0.05).to(torch.bfloat16)
    p = parameters(torch.bfloat16)
    total = sum(LENGTHS)
    tokens = torch.randn(B, S, H, device="cuda").to(torch.bfloat16).requires_grad_()
    cu = torch.tensor([0] + LENGTHS, device="cuda").cumsum(0).to(torch.int32)
    up = [torch.randn(B, S, H, device="cuda").to(torch.bfloat16) for _ in range(2)]
    leaves = [tokens, *p.values(), moe.gate.weight, moe.c_fc.weight, moe.c_proj.weight]

    def step():
        outputs, _ = block(tokens, p, moe, cu)
        return [*outputs, *torch.autograd.grad(outputs, leaves, up)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        tokens.copy_(torch.randn(B, S, H, device="cuda"))
        lengths = [100, 60, S, total - 160 - S]  # a sequence is at most S long
        cu.copy_(torch.tensor([0] + lengths, device="cuda").cumsum(0))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, step()):
        assert torch.equal(a, b)
    assert_status_clean(tokens.device)


def test_second_derivatives_are_refused():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    (dx,) = torch.autograd.grad(xma.rmsnorm(x, None, EPS).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)
    q = torch.randn(9, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    cu = torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    (dq,) = torch.autograd.grad(xma.attention_packed(q, q, q, cu).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), q)


def test_compiled_for_any_length():
    """One compiled graph for all lengths, with and without gradients; checkpointing computes the same again."""
    from torch.utils.checkpoint import checkpoint

    attention = torch.compile(lambda q, k, v, cu: xma.attention_packed(q, k, v, cu), fullgraph=True, dynamic=True)
    norm = torch.compile(lambda x, r, w: xma.fused_residual_add_rmsnorm(x, r, w, EPS, M, gate=w), fullgraph=True, dynamic=True)
    for lengths in ([100, 28], [300], [77, 1, 9, 200]):
        total = sum(lengths)
        q, k, v, up = (torch.randn(total, h, D, device="cuda", dtype=torch.bfloat16) for h in (4, 2, 2, 4))
        cu = torch.tensor([0] + lengths, device="cuda").cumsum(0).to(torch.int32)
        leaves = [t.requires_grad_() for t in (q, k, v)]
        want = xma.attention_packed(*leaves, cu)
        grads = torch.autograd.grad(want, leaves, up, retain_graph=True)
        for call in (lambda: attention(*leaves, cu), lambda: checkpoint(lambda *a: xma.attention_packed(*a, cu), *leaves, use_reentrant=False)):
            got = call()
            assert torch.equal(got, want)
            for a, b in zip(torch.autograd.grad(got, leaves, up), grads):
                assert torch.equal(a, b)
        with torch.no_grad():
            assert torch.equal(attention(q, k, v, cu), want)
            x, w = torch.randn(total, 8 * len(lengths), device="cuda"), torch.randn(8 * len(lengths), device="cuda")
            for a, b in zip(norm(x, x, w), xma.fused_residual_add_rmsnorm(x, x, w, EPS, M, gate=w)):
                assert torch.equal(a, b)


def test_forward_mode_is_refused():
    """A directional derivative through the operators, or through their backward passes, is refused, not wrong."""
    from torch.autograd import forward_ad

    x = torch.randn(9, 64, device="cuda")
    q = torch.randn(9, 2, 64, device="cuda", dtype=torch.bfloat16)
    cu = torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    calls = [(x, lambda t: xma.rmsnorm(t, None, EPS)), (x, lambda t: xma.fused_residual_add_rmsnorm(t, x, None, EPS)[0]),
             (q, lambda t: xma.attention_packed(t, q, q, cu))]
    with forward_ad.dual_level():
        for t, call in calls:
            for leaf in (t, t.clone().requires_grad_()):
                with pytest.raises(NotImplementedError):
                    call(forward_ad.make_dual(leaf, torch.ones_like(leaf)))
            leaf = t.clone().requires_grad_()
            out = call(leaf)
            upstream = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(out, leaf, upstream)
    want = calls[0][1](x)
    with forward_ad.dual_level():
        assert torch.equal(calls[0][1](x), want)
