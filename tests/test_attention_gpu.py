"""attention_packed on the GPU against its formula in 64 bits.

Bounds. With u the half step of the inputs' type: p is rounded once (u relative) where it meets v, so
|o - exact| <= u |o| + u sum_j p_ij |v_j| + e sum_j p_ij |v_j|, where e collects what is done in float32: scores are
sums of D products (D 2^-24 sum |q||k| scale, an absolute error of the exponent, the same in nominator and sum), ex2
(2 steps) and the sums over keys. The backward pass adds, per ds, the rounding of ds and that of delta (taken from the
rounded o: u sum_d |o||do|)."""

import math

import pytest
import torch

import xma
from block_reference import F32, assert_within, half_step
from gpu_helpers import assert_status_clean

pytestmark = pytest.mark.gpu


def offsets(lengths, first=0, dtype=torch.int32):
    return torch.tensor([first] + lengths, dtype=torch.int64).cumsum(0).to(dtype).cuda()


def make(lengths, heads, kv_heads, dim, dtype, behind=0, before=0, seed=0, q_scale=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    total = before + sum(lengths) + behind
    n = lambda h, s: (torch.randn(total, h, dim, device="cuda", generator=g) * s).to(dtype)
    return n(heads, q_scale), n(kv_heads, 1.0), n(kv_heads, 1.0), n(heads, 0.05)


def reference(q, k, v, do, lengths, before=0, scale=None):
    """Per output (value, bound) in float64; rows of no sequence are zeros with a bound of zero."""
    u = half_step(q.dtype)
    T, H, D = q.shape
    G = H // k.size(1)
    scale = scale or 1 / math.sqrt(D)
    out = {n: (torch.zeros(t.shape, dtype=torch.float64, device=q.device), torch.zeros(t.shape, dtype=torch.float64, device=q.device))
           for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    at = before
    for L in lengths:
        r = slice(at, at + L)
        at += L
        if L == 0:
            continue
        for h in range(H):
            qq, kk, vv, dd = (t.double() for t in (q[r, h], k[r, h // G], v[r, h // G], do[r, h]))
            mask = torch.ones(L, L, dtype=torch.bool, device=q.device).tril()
            s = (qq @ kk.t() * scale).masked_fill(~mask, -math.inf)
            p = torch.softmax(s, -1)
            o = p @ vv
            # float32: D products a score, their rounding is an absolute error of the exponent; row sums of L terms
            es = ((D + 8) * F32 * (qq.abs() @ kk.abs().t()) * scale).masked_fill(~mask, 0)
            # p's own relative error: exponent, ex2 (2^-22), argument (|s - m| 2^-23, at most 2^-16 for |s| <= 128), sum
            ep = es + es.max(-1, keepdim=True).values + 2 ** -16 + (L / 8 + 64) * F32
            bo = u * o.abs() + (p * (ep + u)) @ vv.abs() + 64 * F32 * (p @ vv.abs())
            out["o"][0][r, h], out["o"][1][r, h] = o, bo
            delta = (o * dd).sum(-1, keepdim=True)
            e_delta = (bo * dd.abs()).sum(-1, keepdim=True) + D * F32 * (o.abs() * dd.abs()).sum(-1, keepdim=True)
            dp = dd @ vv.t()
            e_dp = D * F32 * (dd.abs() @ vv.abs().t())
            ds = p * (dp - delta)
            e_ds = p * (e_dp + e_delta) + ds.abs() * (ep + u + 4 * F32)
            acc = (L * G + 64) * F32
            bq = scale * (e_ds @ kk.abs() + acc * (ds.abs() @ kk.abs()))
            bk = scale * (e_ds.t() @ qq.abs() + acc * (ds.abs().t() @ qq.abs()))
            bv = (p * (ep + u + acc)).t() @ dd.abs()
            dq, dk, dv = scale * ds @ kk, scale * ds.t() @ qq, p.t() @ dd
            out["dq"][0][r, h], out["dq"][1][r, h] = dq, bq
            for name, val, b in (("dk", dk, bk), ("dv", dv, bv)):
                out[name][0][r, h // G] += val
                out[name][1][r, h // G] += b
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    for n in ("dq", "dk", "dv"):
        val, b = out[n]
        out[n] = (val, b + u * (val.abs() + b))
    # a subnormal result steps evenly; zeros of unowned rows are exact
    return {n: (val, torch.where(b > 0, b + tiny, b)) for n, (val, b) in out.items()}


def run(q, k, v, do, cu, scale=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = xma.attention_packed(*leaves, cu, softmax_scale=scale)
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))))


def check(lengths, heads, kv_heads, dim, dtype, behind=0, before=0, seed=0, q_scale=1.5, scale=None, int64=False):
    q, k, v, do = make(lengths, heads, kv_heads, dim, dtype, behind, before, seed, q_scale)
    cu = offsets(lengths, before, torch.int64 if int64 else torch.int32)
    got = run(q, k, v, do, cu, scale)
    assert_status_clean(q.device)
    ref = reference(q, k, v, do, lengths, before, scale)
    for name, value in got.items():
        assert value.dtype == dtype and value.is_contiguous()
        assert_within(name, value, *ref[name])
    with torch.no_grad():
        assert torch.equal(xma.attention_packed(q, k, v, cu, softmax_scale=scale), got["o"])
    return got


LENGTHS = [[1], [2], [127], [128], [129], [255, 1, 0, 257], [0, 0, 5], [300, 77, 512, 1, 1, 130], [1025], [64] * 9, [640, 384]]


def test_first_one_tile():
    """The smallest case, forward only."""
    q, k, v, do = make([128], 1, 1, 64, torch.bfloat16)
    with torch.no_grad():
        o = xma.attention_packed(q, k, v, offsets([128]))
    assert_status_clean(q.device)
    assert_within("o", o, *reference(q, k, v, do, [128])["o"])


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
def test_lengths(lengths, dim):
    check(lengths, 2, 1, dim, torch.bfloat16)
    check(lengths, 2, 2, dim, torch.float16, seed=1)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (8, 2), (5, 1), (12, 3)])
def test_heads(heads, kv_heads):
    check([200, 33], heads, kv_heads, 128, torch.bfloat16)


@pytest.mark.parametrize("dim", [8, 16, 24, 40, 56, 72, 80, 96, 104, 112, 120])
def test_head_dims(dim):
    check([150, 270], 4, 2, dim, torch.bfloat16)
    check([150, 270], 2, 2, dim, torch.float16)


def test_long():
    check([2300, 1], 2, 1, 128, torch.bfloat16)
    check([3001], 1, 1, 64, torch.float16)


@pytest.mark.parametrize("q_scale", [0.0, 1e-3, 20.0])
def test_sharp_and_flat(q_scale):
    """Rows that look at one key alone (the running maximum keeps growing) and rows that look at all alike."""
    check([700], 2, 1, 64, torch.bfloat16, q_scale=q_scale)


def test_growing_scores():
    """Scores rise along the keys by far more than 2^8 a tile: the accumulator is rescaled in every tile."""
    L, D = 900, 64
    q, k, v, do = make([L], 2, 2, D, torch.bfloat16)
    ramp = torch.linspace(0, 60, L, device="cuda")[:, None].to(torch.bfloat16)
    q[..., 0], k[..., 0] = 8.0, ramp
    got, ref = run(q, k, v, do, offsets([L])), reference(q, k, v, do, [L])
    for name, value in got.items():
        assert_within(name, value, *ref[name])


def test_softmax_scale_and_int64_offsets():
    check([100, 60], 2, 1, 64, torch.bfloat16, scale=0.3, int64=True)


@pytest.mark.parametrize("before,behind", [(0, 70), (13, 0), (130, 500)])
def test_rows_of_no_sequence(before, behind):
    """They get zeros, and NaNs in them (in inputs and upstream gradient) reach no row of a sequence."""
    lengths = [77, 128, 200]
    clean = check(lengths, 4, 2, 64, torch.bfloat16, behind, before)
    q, k, v, do = make(lengths, 4, 2, 64, torch.bfloat16, behind, before)
    for t in (q, k, v, do):
        t[:before] = math.nan
        t[before + sum(lengths):] = math.inf
    got = run(q, k, v, do, offsets(lengths, before))
    for name in got:
        assert torch.equal(got[name], clean[name])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_no_leak_between_sequences(dtype):
    """A sequence of NaN and infinity changes no bit of its neighbours, outputs and gradients."""
    lengths = [100, 60, 300, 41]
    q, k, v, do = make(lengths, 4, 2, 128, dtype)
    if dtype == torch.float16:  # the factor ds is rounded with comes from the largest values: keep those
        v[0, 0, 0], do[0, 0, 0] = 60000.0, 60000.0
    clean = run(q, k, v, do, offsets(lengths))
    bad = slice(160, 460)
    for t in (q, k, v, do):
        t[bad, :, ::2] = math.nan
        t[bad, :, 1::2] = math.inf
    got = run(q, k, v, do, offsets(lengths))
    for name in got:
        assert torch.equal(got[name][:160], clean[name][:160]) and torch.equal(got[name][460:], clean[name][460:])
        assert not got[name][bad].isfinite().all()


def test_strided_views():
    """Slices of one projection, heads first, a misaligned slice: the same bits as contiguous copies."""
    g = torch.Generator(device="cuda").manual_seed(5)
    T, H, K, D = 333, 4, 2, 64
    cu = offsets([133, 200])
    qkv = torch.randn(T, H + 2 * K, D, device="cuda", generator=g).to(torch.bfloat16)
    heads_first = torch.randn(H + 2 * K, T, D, device="cuda", generator=g).to(torch.bfloat16).transpose(0, 1)
    odd = torch.randn(T, H + 2 * K, D + 3, device="cuda", generator=g).to(torch.bfloat16)[..., 1: D + 1]
    do = torch.randn(T, H, D, device="cuda", generator=g).to(torch.bfloat16)
    for t in (qkv, heads_first, odd):
        views = t[:, :H], t[:, H: H + K], t[:, H + K:]
        a = run(*views, do, cu)
        b = run(*(x.contiguous() for x in views), do, cu)
        c = run(*views, do.transpose(0, 1).contiguous().transpose(0, 1), cu)
        for name in a:
            assert torch.equal(a[name], b[name]) and torch.equal(a[name], c[name])
    flat = torch.randn(T * H * D + 1, device="cuda", generator=g).to(torch.bfloat16)[1:].view(T, H, D)  # 2 bytes off
    for name, value in run(flat, flat, flat, flat, cu).items():
        assert torch.equal(value, run(flat.clone(), flat.clone(), flat.clone(), flat.clone(), cu)[name])
    one = torch.randn(T, 1, D, device="cuda", generator=g).to(torch.bfloat16)
    shared = one.expand(T, H, D)  # a head shared by expansion: its gradient is the sum over the heads
    leaf = one.clone().requires_grad_()
    o = xma.attention_packed(qkv[:, :H], leaf.expand(T, H, D), shared, cu)
    (d_one,) = torch.autograd.grad(o, leaf, do)
    d_all = run(qkv[:, :H], shared, shared, do, cu)["dk"]
    assert torch.equal(d_one, d_all.sum(1, keepdim=True))


def test_gradients_in_small_numbers_fp16():
    """Upstream gradients as small as a mean over many tokens makes them, where fp16 has few steps left."""
    q, k, v, do = make([500], 2, 1, 64, torch.float16)
    do = (do * 2.0 ** -6).to(torch.float16)
    got, ref = run(q, k, v, do, offsets([500])), reference(q, k, v, do, [500])
    for name, value in got.items():
        assert_within(name, value, *ref[name])


def test_large_values_fp16():
    """Values near the largest fp16: products overflow fp16, not the result."""
    q, k, v, do = make([300], 2, 1, 64, torch.float16, q_scale=1.0)
    v = (v * 8000).clamp(-60000, 60000)
    do = (do * 0.01).to(torch.float16)
    got, ref = run(q, k, v, do, offsets([300])), reference(q, k, v, do, [300])
    for name, value in got.items():
        want, bound = ref[name]
        assert_within(name, value, want, bound)


def test_gradient_against_differences():
    """Directional derivatives: o is rounded to bf16 (2^-9 each, random over 64 000 values), a step moves the scores by
    about h: the difference quotient is off by the roundings' sum over 2h and h^2."""
    L, H, D = 250, 2, 128
    q, k, v, do = make([L], H, H, D, torch.bfloat16)
    got = run(q, k, v, do, offsets([L]))

    def loss(q, k, v):
        with torch.no_grad():
            return (xma.attention_packed(q, k, v, offsets([L])).double() * do.double()).sum().item()

    for i, name in enumerate(("dq", "dk", "dv")):
        direction = torch.sign(got[name]).to(torch.bfloat16)  # along the gradient's signs the slope is its 1-norm
        h = 2.0 ** -4
        up, down = [q, k, v], [q, k, v]
        up[i], down[i] = up[i] + h * direction, down[i] - h * direction
        step = (up[i].double() - down[i].double())
        want = (got[name].double() * step).sum().item()
        assert abs(loss(*up) - loss(*down) - want) <= 0.05 * abs(want), name


def test_same_results_every_time_and_on_a_side_stream():
    lengths = [700, 1, 300, 129]
    q, k, v, do = make(lengths, 8, 2, 128, torch.bfloat16)
    cu = offsets(lengths)
    first = run(q, k, v, do, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(q, k, v, do, cu)
    torch.cuda.current_stream().wait_stream(side)
    for name in first:
        assert torch.equal(first[name], again[name])


def test_two_calls_at_once():
    """Two streams, each with its own workspace."""
    a, b = make([900], 4, 4, 64, torch.bfloat16), make([400, 500], 4, 4, 64, torch.bfloat16, seed=2)
    cu_a, cu_b = offsets([900]), offsets([400, 500])
    want_a, want_b = run(*a, cu_a), run(*b, cu_b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s, args, cu in zip(streams, (a, b), (cu_a, cu_b)):
        with torch.cuda.stream(s):
            got.append(run(*args, cu))
    torch.cuda.synchronize()
    for g, w in zip(got, (want_a, want_b)):
        for name in w:
            assert torch.equal(g[name], w[name])


def test_captured_step():
    """Forward and backward in a CUDA graph, replayed on other values and other sequence lengths."""
    lengths = [200, 56, 144]
    q, k, v, do = make(lengths, 4, 2, 64, torch.bfloat16)
    cu = offsets(lengths)
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        o = xma.attention_packed(*leaves, cu)
        return [o, *torch.autograd.grad(o, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    new = make([1], 4, 2, 64, torch.bfloat16, behind=399, seed=8)
    with torch.no_grad():
        for old, n in zip((q, k, v, do), new):
            old.copy_(n)
        cu.copy_(offsets([1, 390, 3]))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, step()):
        assert torch.equal(a, b)
    assert (captured[0][394:] == 0).all()


def test_compiled():
    lengths = [100, 28]
    q, k, v, do = make(lengths, 4, 2, 64, torch.bfloat16)
    cu = offsets(lengths)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    f = torch.compile(lambda *a: xma.attention_packed(*a), fullgraph=True)
    o = f(*leaves, cu)
    want = run(*(t.detach() for t in leaves), do, cu)
    assert torch.equal(o, want["o"])
    for a, name in zip(torch.autograd.grad(o, leaves, do), ("dq", "dk", "dv")):
        assert torch.equal(a, want[name])


def test_nothing_to_do():
    for shape_k, cu in (((0, 2, 64), offsets([])), ((0, 2, 64), offsets([0, 0])), ((5, 2, 64), offsets([])), ((5, 2, 64), offsets([0, 0]))):
        q = torch.randn(shape_k[0], 4, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        k = torch.randn(shape_k, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        o = xma.attention_packed(q, k, k, cu)
        dq, dk = torch.autograd.grad(o, (q, k), torch.ones_like(o))
        assert o.shape == q.shape and (o == 0).all() and (dq == 0).all() and (dk == 0).all()
    torch.cuda.synchronize()


def test_offsets_outside_the_stream_touch_nothing():
    """Not a valid cu_seqlens: the values are meaningless, nothing faults and the neighbours of the operands keep."""
    T, H, D = 300, 2, 64
    q, k, v, do = make([T], H, H, D, torch.bfloat16)
    guard = torch.full((T + 512, H, D), 7.0, device="cuda", dtype=torch.bfloat16)
    for values in ([0, 10 ** 6], [-50, 100, 300], [200, 100, 300], [0, 300, 0, 300, 0, 300]):
        run(q, k, v, do, torch.tensor(values, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert_status_clean(q.device)
    assert (guard == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [8, 24, 64, 72, 80, 128])
def test_what_rounding_took_is_kept(dtype, dim):
    """The byte kept for every output element is its rounding, to the two mantissa bits of e5m2 (an eighth) and
    float32: out plus it is that much nearer to the float32 result than half a step of out."""
    from xma import _native as N
    from xma.ops import attention_packed_forward_cuda

    lengths = [300, 1, 31, 160]
    q, k, v, do = make(lengths, 4, 2, dim, dtype, behind=9)
    total, batch = q.size(0), len(lengths)
    out = torch.empty_like(q)
    lse = torch.empty(4, N.attention_stat_rows(total, batch), device="cuda")
    row = -(-dim // 16) * 16
    rest = torch.full((total, 4, row), 0x7F, dtype=torch.uint8, device="cuda")  # NaNs until they are written
    workspace = torch.empty(N.attention_workspace_bytes(total, batch), dtype=torch.uint8, device="cuda")
    scale = 2.0 ** (0 if dim == 8 else -3)
    attention_packed_forward_cuda(q, k, v, offsets(lengths), scale, out, lse, rest, workspace)
    kept = rest[..., :dim].view(torch.float8_e5m2).double() / (4096 if dtype == torch.bfloat16 else 32768)
    owned = slice(0, sum(lengths))
    assert kept[owned].isfinite().all()
    taken = kept[owned].abs()
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # fp16 below 2^-14 steps by 2^-24, whatever the value
    step = (2 * half_step(dtype) * out[owned].double().abs()).clamp_min(tiny)
    assert (taken <= step * 1.13 / 2).all()  # never more than half a step (at a power of two, of the lower one)
    assert (taken > 0.1 * step / 2).double().mean() > 0.5  # and spread over it
    # A row with one key: p = 2^(s c - m) with m the rounded product s c, the exponent the exact one minus m, so p and
    # with it the sum l are off 1 by 2^-24 |m| ln 2 and two steps of ex2; the output is v p / l with p rounded to 1.
    # |m| <= 60 here, so what is taken is below 64 * 2^-24 |v|, far under the step of the type.
    one = lengths[0]
    value = v[one].repeat_interleave(2, 0)
    assert torch.equal(out[one], value) and (kept[one].abs() <= 64 * F32 * value.double().abs()).all()


@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (6, 2, 128), (5, 5, 40), (16, 1, 80)])
def test_factor_of_small_gradients(heads, kv_heads, dim):
    """fp16: the factor that ds is rounded with comes from the largest |do| and |v| of the sequences' rows, exactly."""
    from xma import _native as N
    from xma.ops import attention_packed_backward_cuda, attention_packed_forward_cuda

    lengths = [127, 3, 300]
    q, k, v, do = make(lengths, heads, kv_heads, dim, torch.float16, behind=20)
    v[-20:], do[-20:] = 1e4, 1e4
    total = q.size(0)
    new = lambda t: torch.empty_like(t)
    stats = lambda: torch.empty(heads, N.attention_stat_rows(total, 3), device="cuda")
    out, lse, delta = new(q), stats(), stats()
    rest = torch.empty(total, heads, -(-dim // 16) * 16, dtype=torch.uint8, device="cuda")
    workspace = torch.full((N.attention_workspace_bytes(total, 3),), 0x3C, dtype=torch.uint8, device="cuda")
    attention_packed_forward_cuda(q, k, v, offsets(lengths), 0.1, out, lse, rest, workspace)
    attention_packed_backward_cuda(q, k, v, offsets(lengths), 0.1, out, rest, do, lse, delta, new(q), new(k), new(v), workspace)
    most = workspace[8:16].view(torch.float32)
    assert most.tolist() == [do[:-20].abs().max().item(), v[:-20].abs().max().item()]


@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (128, torch.bfloat16), (48, torch.bfloat16), (80, torch.float16)])
def test_many_work_items(dim, dtype):
    """More work items than SMs, of one and of two query tiles in every order: each CTA goes through several."""
    lengths = [(37 * n * n + 11 * n) % 700 + 1 for n in range(48)]
    check(lengths, 12, 3, dim, dtype, behind=5)


@pytest.mark.parametrize("int_type", [torch.int32, torch.int64])
def test_offsets_out_of_order_are_no_work(int_type):
    """Overlapping sequences of 2^32 row blocks together, more than the plan's counters hold: the rows are left as they were
    and later calls are not touched."""
    from xma import _native as N
    from xma.ops import attention_packed_backward_cuda, attention_packed_forward_cuda

    total, batch = 1 << 22, (1 << 18) + 1
    cu = torch.zeros(batch + 1, dtype=int_type, device="cuda")
    cu[1::2] = total
    q, k, v, do = make([total], 1, 1, 8, torch.bfloat16)
    workspace = torch.empty(N.attention_workspace_bytes(total, batch), dtype=torch.uint8, device="cuda")
    out, dq, dk, dv = (torch.full_like(q, 7.0) for _ in range(4))
    lse, delta = (torch.empty(1, N.attention_stat_rows(total, batch), device="cuda") for _ in range(2))
    rest = torch.zeros(total, 1, 16, dtype=torch.uint8, device="cuda")
    attention_packed_forward_cuda(q, k, v, cu, 0.3, out, lse, rest, workspace)
    attention_packed_backward_cuda(q, k, v, cu, 0.3, out, rest, do, lse, delta, dq, dk, dv, workspace)
    torch.cuda.synchronize()
    assert_status_clean(q.device)
    assert all((t == 7.0).all() for t in (out, dq, dk, dv))
    check([130, 1, 300], 2, 1, 64, torch.bfloat16)


def test_most_heads():
    check([130], 4096, 1, 8, torch.bfloat16)


def test_one_input_learns():
    """Gradients that nobody asked for are not handed out, and the others do not change; one tensor may be all three inputs."""
    lengths = [200, 3, 140]
    q, k, v, do = make(lengths, 4, 4, 64, torch.bfloat16)
    cu = offsets(lengths)
    want = run(q, k, v, do, cu)
    for i, name in enumerate(("dq", "dk", "dv")):
        leaves = [t.detach().requires_grad_(i == j) for j, t in enumerate((q, k, v))]
        xma.attention_packed(*leaves, cu).backward(do)
        assert [t.grad is not None for t in leaves] == [i == j for j in range(3)]
        assert torch.equal(leaves[i].grad, want[name])
    one = q.detach().requires_grad_()
    xma.attention_packed(one, one, one, cu).backward(do)
    parts = run(q, q, q, do, cu)
    total = sum(parts[n].double() for n in ("dq", "dk", "dv"))
    magnitude = sum(parts[n].double().abs() for n in ("dq", "dk", "dv"))
    assert ((one.grad.double() - total).abs() <= 2 * half_step(torch.bfloat16) * magnitude * (1 + 2 ** -7)).all()  # two additions in bf16


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 96])
def test_one_key_has_no_gradient(dtype, dim):
    """A softmax over one key is 1 whatever the score: the first rows' dq, and dk of sequences of one token, are zeros."""
    lengths = [1, 1, 0, 1, 300, 1, 128, 2]
    got = check(lengths, 4, 2, dim, dtype, behind=3)
    at = 0
    for n in lengths:
        if n:
            assert (got["dq"][at] == 0).all()
        if n == 1:
            assert (got["dk"][at] == 0).all()
        at += n


def reference_fp16(q, k, v, do, lengths, scale=None):
    """`reference` with what fp16 adds where numbers fall under its smallest normal one, steps there being 2^-24: half a
    step for every p of a row, which carries 2^9 (in units of its row's largest p) on its way to o and 2^14 on its way to
    dv, and for every ds, which carries the power of two that puts 2 dim max|do| max|v| between 2^14 and 2^15. What o is
    off by is in delta = o . do too, and with it in every ds of the row, times p. Largest finite number: 65504; from 65520
    on the nearest one is infinity."""
    ref = reference(q, k, v, do, lengths, scale=scale)
    H, D = q.shape[1:]
    G, scale = H // k.size(1), scale or 1 / math.sqrt(D)
    e_ds = 2 * D * do.double().abs().max() * v.double().abs().max() * 2.0 ** -14 * 2.0 ** -25
    more = 1 + 2.0 ** -10  # products of two errors, the results' own rounding
    at = 0
    for L in lengths:
        r = slice(at, at + L)
        at += L
        for h in range(H):
            qq, kk, vv, dd = (t.double() for t in (q[r, h], k[r, h // G], v[r, h // G], do[r, h]))
            seen = torch.ones(L, L, dtype=torch.float64, device=q.device).tril()
            p = torch.softmax((qq @ kk.t() * scale).masked_fill(seen == 0, -math.inf), -1)
            e_o = 2.0 ** -34 * (seen @ vv.abs())
            e = seen * e_ds + p * (e_o * dd.abs()).sum(-1, keepdim=True)
            for name, head, term in (("o", h, e_o), ("dv", h // G, 2.0 ** -39 * (seen.t() @ dd.abs())),
                                     ("dq", h, scale * (e @ kk.abs())), ("dk", h // G, scale * (e.t() @ qq.abs()))):
                ref[name][1][r, head] += term * more
    for name, (want, bound) in ref.items():
        over = want.abs() - bound >= 65520
        want[over], bound[over] = want[over].sign() * math.inf, 0.0
    return ref


def assert_within_fp16(name, got, want, bound):
    """assert_within for values of which some are too large for fp16."""
    over = want.isinf()
    assert torch.equal(got[over].double(), want[over]), name
    assert_within(name, got.masked_fill(over, 0), want.masked_fill(over, 0), bound)


def outweighed(gap):
    """One key beside which each of the others weighs exp(-gap), with values and upstream gradients of one sign."""
    L, D = 4000, 64
    q, k, v, do = make([L], 1, 1, D, torch.float16)
    q.zero_(), k.zero_()
    q[..., 0], k[0, :, 0] = 8.0, gap
    v[0], v[1:] = 0.0, v[1:].abs() * 8
    return q, k, v, (do.abs() * 100 + 8).to(torch.float16), [L]


def sharp(q_scale):
    lengths = [1200, 1, 340]
    q, k, v, do = make(lengths, 4, 2, 64, torch.float16, q_scale=q_scale)
    return q, k, v, (do * 400).to(torch.float16), lengths


def growing(top):
    """Scores that rise along the keys, by as much as leaves the accumulator alone from tile to tile and by more."""
    q, k, v, do = make([900], 2, 2, 64, torch.float16)
    q[..., 0], k[..., 0] = 8.0, torch.linspace(0, top, 900, device="cuda")[:, None].to(torch.float16)
    return q, k, v, do, [900]


SMALL_WEIGHTS = ([(outweighed, gap) for gap in (12.0, 18.0, 22.0)] + [(sharp, s) for s in (0.0, 1e-3, 3.0, 20.0)]
                 + [(growing, top) for top in (2.0, 6.0, 11.0, 20.0, 60.0)])


@pytest.mark.parametrize("make_inputs,value", SMALL_WEIGHTS)
def test_small_weights_fp16(make_inputs, value):
    """Keys too small for fp16 beside their row's largest, each alone; thousands of them are not."""
    q, k, v, do, lengths = make_inputs(value)
    ref = reference_fp16(q, k, v, do, lengths)
    with torch.no_grad():
        assert_within("o", xma.attention_packed(q, k, v, offsets(lengths)), *ref["o"])
    assert_status_clean(q.device)


@pytest.mark.parametrize("make_inputs,value", SMALL_WEIGHTS)
def test_gradients_of_small_weights_fp16(make_inputs, value):
    """The same backward: dv of keys that each row hardly looks at is a sum over all the rows."""
    q, k, v, do, lengths = make_inputs(value)
    got, ref = run(q, k, v, do, offsets(lengths)), reference_fp16(q, k, v, do, lengths)
    for name in ("dq", "dk", "dv"):
        assert_within_fp16(name, got[name], *ref[name])
    assert_status_clean(q.device)


@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
def test_non_finite_values_leave_the_factor_alone(what):
    """A sequence whose upstream gradient or values are not finite takes no bit from its neighbours' small gradients."""
    lengths = [100, 60, 300]
    q, k, v, do = make(lengths, 4, 2, 64, torch.float16)
    do = (do * 2.0 ** -8).to(torch.float16)
    do[100:160], v[100:160] = 0.0, 0.0
    clean = run(q, k, v, do, offsets(lengths))
    do[107, 1, 5], v[111, 0, 9], do[120, 2, 8] = what, what, what
    got = run(q, k, v, do, offsets(lengths))
    for name in got:
        assert torch.equal(got[name][:100], clean[name][:100]) and torch.equal(got[name][160:], clean[name][160:])


@pytest.mark.parametrize("dim", [64, 128])
def test_largest_values_fp16(dim):
    """Means of fp16's largest number are that number, whatever rounding does to the weights; an infinity stays one. Beside
    the first key of weight 1 (scores of 0) all others weigh exp(-scale), just above the middle of two steps of fp16."""
    lengths = [700, 33]
    q, k, v, do = make(lengths, 4, 2, dim, torch.float16)
    q.zero_(), k.zero_()
    q[..., 0], k[..., 0] = 1.0, -1.0
    k[0, :, 0], k[700, :, 0] = 0.0, 0.0
    v[..., ::3], v[..., 1::3] = 65504.0, -65504.0
    scale = -math.log(0.5 * (1 + 0.51 * 2.0 ** -10))
    cu = offsets(lengths)
    want, bound = reference(q, k, v, do, lengths, scale=scale)["o"]
    with torch.no_grad():
        o = xma.attention_packed(q, k, v, cu, softmax_scale=scale)
    assert_within("o", o, want, bound)
    got = run(q, k, v, (do * 2.0 ** -10).to(torch.float16), cu, scale)
    assert torch.equal(got["o"], o) and all(t.isfinite().all() for t in got.values())
    v[3, :, 0] = math.inf
    with torch.no_grad():
        assert xma.attention_packed(q, k, v, cu, softmax_scale=scale)[3:700, :, 0].isposinf().all()


@pytest.mark.parametrize("fills", [0, 1, 2, 3, 4, 5, 6, 7, 64])
def test_copies_in_flight_are_waited_for(fills):
    """What a load warp does before its CTA ends, also when another role gave up: the copies that nobody reads any more have
    landed, at every turn of their ring; a copy that never started does not hold it beyond the limit (1 ms)."""
    from xma import _native as N

    size = 8192
    src = torch.randint(0, 256, (max(fills, 1) * size,), dtype=torch.uint8, device="cuda")
    dst = torch.zeros(3, size, dtype=torch.uint8, device="cuda")
    result = torch.full((2,), -1, dtype=torch.int32, device="cuda")
    N.check(N.lib().xma_selftest_settle(src.data_ptr(), fills, dst.data_ptr(), result.data_ptr(), 1_000_000,
                                        torch.cuda.current_stream().cuda_stream), "xma_selftest_settle")
    assert result.tolist() == [1, 0]
    for stage in range(3):
        turns = [j for j in range(fills) if j % 3 == stage]
        want = src[turns[-1] * size: (turns[-1] + 1) * size] if turns else torch.zeros_like(dst[0])
        assert torch.equal(dst[stage], want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_bad_offsets_write_nothing_else(dtype):
    """Outputs, statistics, lists: whatever the offsets hold, what lies around them keeps its bytes."""
    from xma import _native as N
    from xma.ops import attention_packed_backward_cuda, attention_packed_forward_cuda

    T, H, K, D, edge = 300, 4, 2, 40, 4096
    q, k, v, do = make([T], H, K, D, dtype)
    for int_type in (torch.int32, torch.int64):
        for values in ([0, 300], [0, 10 ** 6], [-50, 100, 300], [200, 100, 300], [0, 300, 0, 300, 0, 300], [-7, -7], [400, 500],
                       [0, 0, 0, 129, 129, 300], [301, 300, 0], [-2 ** 31, 2 ** 31 - 1]):
            cu = torch.tensor(values, dtype=int_type, device="cuda")
            B = len(values) - 1
            buffers = []

            def inside(shape, to):
                size = math.prod(shape) * torch.empty(0, dtype=to).element_size()
                raw = torch.full((size + 2 * edge,), 0x5A, dtype=torch.uint8, device="cuda")
                buffers.append((raw, size))
                return raw[edge: edge + size].view(to).view(shape)

            rows = N.attention_stat_rows(T, B)
            workspace = lambda: inside((N.attention_workspace_bytes(T, B),), torch.uint8)
            out, dq, dk, dv = (inside(tuple(t.shape), dtype) for t in (q, q, k, v))
            lse, delta, rest = inside((H, rows), torch.float32), inside((H, rows), torch.float32), inside((T, H, 48), torch.uint8)
            attention_packed_forward_cuda(q, k, v, cu, 0.2, out, lse, rest, workspace())
            attention_packed_backward_cuda(q, k, v, cu, 0.2, out, rest, do, lse, delta, dq, dk, dv, workspace())
            assert_status_clean(q.device)
            for raw, size in buffers:
                assert (raw[:edge] == 0x5A).all() and (raw[edge + size:] == 0x5A).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [24, 64, 128])
def test_short_sequences_keep_what_rounding_takes_from_weights(dtype, dim):
    """Sequences of up to 128 tokens: o is off by its own rounding and by float32's, not by that of the probabilities, which
    go into the product as two numbers: the first cut off (2u), the second rounded (u of that) and at least a step of 2^-24
    in fp16, where a row's largest is 2^9."""
    lengths = [128, 1, 2, 7, 300, 96, 127]
    q, k, v, do = make(lengths, 4, 2, dim, dtype)
    with torch.no_grad():
        o = xma.attention_packed(q, k, v, offsets(lengths))
    u, at, scale = half_step(dtype), 0, 1 / math.sqrt(dim)
    for L in lengths:
        r = slice(at, at + L)
        at += L
        for h in range(4 if L <= 128 else 0):
            qq, kk, vv = (t.double() for t in (q[r, h], k[r, h // 2], v[r, h // 2]))
            seen = torch.ones(L, L, dtype=torch.float64, device="cuda").tril()
            p = torch.softmax((qq @ kk.t() * scale).masked_fill(seen == 0, -math.inf), -1)
            es = (dim + 8) * F32 * (qq.abs() @ kk.abs().t()) * scale * seen  # as in `reference`
            ep = es + es.max(-1, keepdim=True).values + 2.0 ** -16 + 80 * F32
            want = p @ vv
            bound = u * want.abs() * (1 + 2 ** -7) + (p * (ep + 2 * u * u)) @ vv.abs() + 2.0 ** -33 * (seen @ vv.abs()) + 64 * F32 * (p @ vv.abs())
            assert_within("o", o[r, h], want, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("what", [math.inf, -math.inf])
def test_infinite_values_make_infinities(dtype, what):
    """Rows that see an infinite value with a weight above zero get that infinity, in the first tile and behind it."""
    lengths = [60, 400]
    q, k, v, do = make(lengths, 4, 2, 64, dtype, q_scale=0.5)
    clean = xma.attention_packed(q, k, v, offsets(lengths))
    v[5, 0, 3], v[70, 1, 9], v[300, 0, 0] = what, what, what
    o = xma.attention_packed(q, k, v, offsets(lengths))
    assert (o[5:60, :2, 3] == what).all() and (o[70:, 2:, 9] == what).all() and (o[300:, :2, 0] == what).all()
    other = torch.ones_like(o, dtype=torch.bool)
    other[:60, :2, 3], other[60:, 2:, 9], other[60:, :2, 0] = False, False, False
    assert torch.equal(o[other], clean[other])
