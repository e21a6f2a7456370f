"""Cases of the operators that stand around the expert layer in a transformer block: causal attention over a packed
token stream, and the norms, gate and residual add that join two sublayers. Each case can be run in a plain form
(elementary torch operations in float32) or through the framework's public calls (`own`), and in 64 bits (`exact`)."""

import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-5


def _xma():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-model-architectures_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import xma

    return xma


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------


def _attention(name, lengths, heads, kv_heads, head_dim, dtype, backward, behind=0):
    """`lengths`: tokens of each packed sequence; `behind`: rows of the stream that no sequence owns."""
    case = {
        "op": "attention", "lengths": ",".join(str(n) for n in lengths), "behind": behind, "heads": heads,
        "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "backward": backward,
    }
    return {"name": name, **case} if name else case


def _norm(name, rows, hidden, dtype, backward, residual="same", post=False, gate="none", multiplier=1.0):
    """`residual`: "none" (norm alone), "same" (stream in the activations' type) or "fp32"; `gate`: "none", "channel"
    ([hidden]), "token" ([rows, 1]) or "full" ([rows, hidden])."""
    case = {
        "op": "norm", "rows": rows, "hidden": hidden, "dtype": dtype, "backward": backward, "residual": residual,
        "post": post, "gate": gate, "multiplier": multiplier,
    }
    return {"name": name, **case} if name else case


def listed():
    return [
        # The first request of a quiet server: three short prompts, one of a single token. Latency counts.
        _attention("attention_short_prompts", [1, 17, 63], 16, 16, 128, "bf16", False),
        # Prefill of one long prompt with grouped heads (hidden size 4096).
        _attention("attention_prefill_8192", [8192], 32, 8, 128, "bf16", False),
        # Prefill of a batch of ragged prompts, an empty one among them, in half precision and with narrow heads.
        _attention("attention_prefill_ragged", [517, 0, 2049, 1, 130, 1023, 255, 4001, 128], 16, 4, 64, "fp16", False),
        # A training step over a packed batch of documents, with rows behind the last one (the padded tail of a buffer).
        _attention("attention_train_packed", [4096, 2048, 2047, 1024, 1025, 1000, 777, 512, 511, 300, 128, 127, 64, 33, 1, 0, 2500], 32, 8, 128,
                   "bf16", True, behind=191),
        # Training on short documents with as many key as query heads and a head size between two powers of two.
        _attention("attention_train_short_docs", [97 + 13 * n for n in range(40)], 16, 16, 80, "fp16", True),
        # Training on one document of the full context length.
        _attention("attention_train_16384", [16384], 32, 8, 128, "bf16", True),
        # One token of a few running requests through a block's norms. Latency counts.
        _norm("norm_tokens", 4, 4096, "bf16", False, post=True),
        # A packed prompt through the norms before and after a block, the stream kept in float32.
        _norm("norm_prompt", 8191, 2048, "bf16", False, residual="fp32", post=True, gate="channel", multiplier=0.5),
        # The training step at the hidden size of the wide expert layer, every part in use.
        _norm("norm_train_4096", 16384, 4096, "bf16", True, post=True, gate="channel", multiplier=0.22),
        # Training with a gate that another projection computed for every token and channel.
        _norm("norm_train_gated", 4097, 7168, "fp16", True, gate="full"),
        # A first norm of a block alone, in float32, at a hidden size that no vector divides.
        _norm("norm_train_odd_fp32", 5001, 1001, "fp32", True, residual="none"),
        # A residual stream in float32 beside bf16 activations, gated for each token.
        _norm("norm_train_token_gate", 8192, 2048, "bf16", True, residual="fp32", gate="token", post=True),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.5:
        backward = rng.random() < 0.5
        heads, kv_heads = rng.choice([(4, 4), (8, 2), (16, 16), (16, 4), (12, 3), (32, 8), (28, 4), (6, 1), (24, 24)])
        head_dim = rng.choice([64, 128, 128, 64, 80, 96, 40, 112, 24])
        longest = _log_uniform(rng, 1, 12000)
        budget = _log_uniform(rng, longest, 16000) if longest < 16000 else longest
        lengths = [longest]
        while sum(lengths) < budget and len(lengths) < 200:
            lengths.append(min(_log_uniform(rng, 1, longest), budget - sum(lengths)))
            if rng.random() < 0.05:
                lengths.append(0)
        rng.shuffle(lengths)
        return _attention(None, lengths, heads, kv_heads, head_dim, rng.choice(["bf16", "fp16"]), backward,
                          rng.choice([0, 0, rng.randint(1, 300)]))
    hidden = _log_uniform(rng, 64, 8192)
    if rng.random() < 0.7:
        hidden = max(64, hidden // 64 * 64)
    rows = _log_uniform(rng, 1, min(16384, 16384 * 4096 // hidden))
    residual = rng.choice(["none", "same", "same", "fp32"])
    alone = residual == "none"
    return _norm(None, rows, hidden, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.6, residual,
                 not alone and rng.random() < 0.5, "none" if alone else rng.choice(["none", "channel", "token", "full"]),
                 1.0 if alone else rng.choice([1.0, 0.25, rng.randint(1, 99) / 100]))


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "attention":
        lengths = _lengths(case)
        total = sum(lengths) + case["behind"]
        pairs = sum(n * (n + 1) // 2 for n in lengths)
        q = total * case["heads"] * case["head_dim"] * size
        kv = total * case["kv_heads"] * case["head_dim"] * size
        # two products forward; five backward (scores and dP again, dQ, dK, dV)
        flops = 4 * case["head_dim"] * case["heads"] * pairs * (3.5 if case["backward"] else 1)
        return {"bytes": (2 * q + 2 * kv) * (2 if case["backward"] else 1), "flops": int(flops)}
    elements = case["rows"] * case["hidden"]
    stream = 4 if case["residual"] == "fp32" else size
    added = case["residual"] != "none"
    gate = {"none": 0, "channel": 0, "token": case["rows"] * size, "full": elements * size}[case["gate"]]
    vectors = case["hidden"] * size * (1 + case["post"] + (case["gate"] == "channel"))
    forward = elements * (2 * size + (2 * stream if added else 0)) + gate + vectors
    # backward: the gradients of both outputs in, those of every input out
    return {"bytes": forward * (2 if case["backward"] else 1),
            "flops": elements * ((8 if added else 4) + (4 if case["post"] else 0)) * (3 if case["backward"] else 1)}


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, to=dtype):
        return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(to)

    state = {"case": case}
    if case["op"] == "attention":
        lengths = _lengths(case)
        total = sum(lengths) + case["behind"]
        offsets = [0]
        for n in lengths:
            offsets.append(offsets[-1] + n)
        # one projection gives queries, keys and values side by side: keys and values are strided views of it, the
        # queries went through a step of their own (a norm or a rotation) since
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
        qkv = normal(total, heads + 2 * kv_heads, dim)
        state["q"] = (qkv[:, :heads] * 1.5).requires_grad_(case["backward"])
        state["k"] = qkv[:, heads: heads + kv_heads].detach().requires_grad_(case["backward"])
        state["v"] = qkv[:, heads + kv_heads:].detach().requires_grad_(case["backward"])
        state["cu_seqlens"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        if case["backward"]:
            state["d_out"] = normal(total, heads, dim, scale=0.02)
        return state
    rows, hidden = case["rows"], case["hidden"]
    stream = torch.float32 if case["residual"] == "fp32" else dtype
    leaf = case["backward"]
    state["x"] = normal(rows, hidden, scale=0.7).requires_grad_(leaf)
    state["weight"] = normal(hidden, scale=0.2, shift=1.0).requires_grad_(leaf)
    if case["residual"] != "none":
        # a residual stream has a few channels far larger than the rest
        channels = torch.exp(torch.randn(hidden, device="cuda", generator=g))
        state["residual"] = (normal(rows, hidden, to=torch.float32) * channels).to(stream).requires_grad_(leaf)
    if case["post"]:
        state["post_weight"] = normal(hidden, scale=0.2, shift=0.8).requires_grad_(leaf)
    if case["gate"] != "none":
        shape = {"channel": (hidden,), "token": (rows, 1), "full": (rows, hidden)}[case["gate"]]
        state["gate"] = normal(*shape, scale=0.5, shift=0.3).requires_grad_(leaf)
    if leaf:
        state["d_y"] = normal(rows, hidden, scale=0.05)
        if case["residual"] != "none":
            state["d_stream"] = normal(rows, hidden, scale=0.05, to=stream)
    return state


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------


def run(state):
    attention = state["case"]["op"] == "attention"
    if own:
        return _own_attention(state) if attention else _own_norm(state)
    with torch.no_grad():
        return _plain_attention(state) if attention else _plain_norm(state)


def _own_attention(state):
    xma = _xma()
    out = xma.attention_packed(state["q"], state["k"], state["v"], state["cu_seqlens"])
    if not state["case"]["backward"]:
        return {"out": out}
    dq, dk, dv = torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["d_out"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


def _own_norm(state):
    xma = _xma()
    case = state["case"]
    if case["residual"] == "none":
        outputs = {"y": xma.rmsnorm(state["x"], state["weight"], _EPS)}
        upstream = [state.get("d_y")]
    else:
        y, stream = xma.fused_residual_add_rmsnorm(
            state["x"], state["residual"], state["weight"], _EPS, case["multiplier"], post_weight=state.get("post_weight"),
            gate=state.get("gate"))
        outputs = {"y": y, "stream": stream}
        upstream = [state.get("d_y"), state.get("d_stream")]
    if not case["backward"]:
        return outputs
    names = [n for n in ("x", "residual", "weight", "post_weight", "gate") if n in state]
    grads = torch.autograd.grad(list(outputs.values()), [state[n] for n in names], upstream)
    return {**{n: t.detach() for n, t in outputs.items()}, **{"d_" + n: t for n, t in zip(names, grads)}}


def _plain_attention(state):
    """One sequence at a time, as many heads at once as keep the score matrices within a few GB."""
    case = state["case"]
    q, k, v = state["q"], state["k"], state["v"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    group = heads // kv_heads
    scale = 1.0 / math.sqrt(dim)
    backward = case["backward"]
    out = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
    dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float32, device=t.device) if backward else None for t in (q, k, v))
    start = 0
    for length in _lengths(case):
        rows = slice(start, start + length)
        start += length
        if length == 0:
            continue
        masked = torch.ones(length, length, dtype=torch.bool, device=q.device).triu(1)
        step = max(1, min(kv_heads, int(2**29 // (group * length * length))))
        for first in range(0, kv_heads, step):
            kv = slice(first, min(first + step, kv_heads))
            count = kv.stop - kv.start
            qh = slice(kv.start * group, kv.stop * group)
            # [kv heads, group, length, dim] and [kv heads, 1, length, dim]
            qs = q[rows, qh].float().transpose(0, 1).reshape(count, group, length, dim)
            ks = k[rows, kv].float().transpose(0, 1).unsqueeze(1)
            vs = v[rows, kv].float().transpose(0, 1).unsqueeze(1)
            p = torch.matmul(qs, ks.transpose(-1, -2)).mul_(scale).masked_fill_(masked, -math.inf)
            p = p.sub_(p.amax(-1, keepdim=True)).exp_()
            p = p.div_(p.sum(-1, keepdim=True))
            o = torch.matmul(p, vs)
            out[rows, qh] = o.reshape(count * group, length, dim).transpose(0, 1)
            if not backward:
                continue
            do = state["d_out"][rows, qh].float().transpose(0, 1).reshape(count, group, length, dim)
            delta = (o * do).sum(-1, keepdim=True)
            dv[rows, kv] = torch.matmul(p.transpose(-1, -2), do).sum(1).transpose(0, 1)
            ds = torch.matmul(do, vs.transpose(-1, -2)).sub_(delta).mul_(p).mul_(scale)
            dq[rows, qh] = torch.matmul(ds, ks).reshape(count * group, length, dim).transpose(0, 1)
            dk[rows, kv] = torch.matmul(ds.transpose(-1, -2), qs).sum(1).transpose(0, 1)
    if not backward:
        return {"out": out.to(q.dtype)}
    return {"out": out.to(q.dtype), "dq": dq.to(q.dtype), "dk": dk.to(k.dtype), "dv": dv.to(v.dtype)}


def _plain_norm(state):
    case = state["case"]
    dtype = state["x"].dtype
    x, w = state["x"].float(), state["weight"].float()
    added = "residual" in state
    multiplier = case["multiplier"]
    if case["post"]:
        pw = state["post_weight"].float()
        rp = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        u = pw * (x * rp)
    else:
        u = x
    gate = state["gate"].float() if "gate" in state else None
    z = u if gate is None else gate * u
    s = state["residual"].float() + multiplier * z if added else x
    rs = torch.rsqrt((s * s).mean(-1, keepdim=True) + _EPS)
    hat = s * rs
    outputs = {"y": (w * hat).to(dtype)}
    if added:
        outputs["stream"] = s.to(state["residual"].dtype)
    if not case["backward"]:
        return outputs
    dy = state["d_y"].float()
    a = dy * w
    ds = rs * (a - hat * (a * hat).mean(-1, keepdim=True))
    d_weight = (dy * hat).sum(0)
    if not added:
        return {**outputs, "d_x": ds.to(dtype), "d_weight": d_weight.to(dtype)}
    ds = ds + state["d_stream"].float()
    dz = multiplier * ds
    du = dz if gate is None else dz * gate
    dx, grads = du, {}
    if case["post"]:
        hat_x = x * rp
        b = du * pw
        dx = rp * (b - hat_x * (b * hat_x).mean(-1, keepdim=True))
        grads["d_post_weight"] = (du * hat_x).sum(0).to(dtype)
    if gate is not None:
        d_gate = dz * u
        if case["gate"] == "channel":
            d_gate = d_gate.sum(0)
        elif case["gate"] == "token":
            d_gate = d_gate.sum(-1, keepdim=True)
        grads["d_gate"] = d_gate.to(dtype)
    return {**outputs, "d_x": dx.to(dtype), "d_residual": ds.to(state["residual"].dtype), "d_weight": d_weight.to(dtype), **grads}


# ---------------------------------------------------------------------------------------------
# 64 bits: the definitions alone, gradients by differentiation
# ---------------------------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_attention(state) if case["op"] == "attention" else _exact_norm(state)


def _exact_attention(state):
    case = state["case"]
    group = case["heads"] // case["kv_heads"]
    names = ("q", "k", "v")
    wide = {n: state[n].detach().double() for n in names}
    out = torch.zeros_like(wide["q"])
    grads = {n: torch.zeros_like(wide[n]) for n in names}
    end = 0
    for length in _lengths(case):
        begin, end = end, end + length
        if length == 0:
            continue
        future = torch.arange(length, device="cuda")[None, :] > torch.arange(length, device="cuda")[:, None]
        for head in range(case["heads"]):
            part = [wide[n][begin:end, head if n == "q" else head // group].clone().requires_grad_(case["backward"]) for n in names]
            scores = torch.einsum("id,jd->ij", part[0], part[1]) / math.sqrt(case["head_dim"])
            o = torch.softmax(torch.where(future, torch.full_like(scores, -math.inf), scores), 1) @ part[2]
            out[begin:end, head] = o.detach()
            if case["backward"]:
                found = torch.autograd.grad(o, part, state["d_out"][begin:end, head].double())
                for n, d in zip(names, found):
                    grads[n][begin:end, head if n == "q" else head // group] += d
    if not case["backward"]:
        return {"out": out}
    return {"out": out, "dq": grads["q"], "dk": grads["k"], "dv": grads["v"]}


def _exact_norm(state):
    case = state["case"]
    names = [n for n in ("x", "residual", "weight", "post_weight", "gate") if n in state]
    part = {n: state[n].detach().double().requires_grad_(case["backward"]) for n in names}

    def normed(t, weight):
        return t / torch.sqrt(t.pow(2).mean(1, keepdim=True) + _EPS) * weight

    branch = part["x"]
    if "post_weight" in part:
        branch = normed(branch, part["post_weight"])
    if "gate" in part:
        branch = branch * part["gate"]
    outputs, upstream = {}, [state.get("d_y")]
    if "residual" in part:
        stream = part["residual"] + branch * case["multiplier"]
        outputs = {"y": normed(stream, part["weight"]), "stream": stream}
        upstream.append(state.get("d_stream"))
    else:
        outputs = {"y": normed(branch, part["weight"])}
    if not case["backward"]:
        return outputs
    grads = torch.autograd.grad(list(outputs.values()), list(part.values()), [t.double() for t in upstream])
    return {**{n: t.detach() for n, t in outputs.items()}, **{"d_" + n: t for n, t in zip(names, grads)}}
