"""rmsnorm and fused_residual_add_rmsnorm on the GPU against their formulas in 64 bits.

Bounds: an output of type t is off by half a step of t, plus float32 rounding. A row sum of H terms is added up by
at most 16 (per thread) + 5 + 32 (warps) steps in registers, or ceil(H / 256) + 13 in the two-kernel form; every
other value takes fewer than 24 operations. So the float32 part is below (H / 256 + 80) * 2^-24 of the magnitude
(the same expression with absolute values). Sums over rows add rows / 148 + 64 steps. A kernel that keeps its row's
stream in float32 differs from the reference, which starts from the exact one, by that rounding alone."""

import pytest
import torch

import xma
from block_reference import F32, assert_within, half_step, norm_reference
from gpu_helpers import assert_status_clean

pytestmark = pytest.mark.gpu

EPS = 1e-5
GATES = ("none", "channel", "token", "full")


def make(rows, hidden, dtype, stream_dtype, gate, post, param_dtype=None, seed=0, weight=True, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    param_dtype = param_dtype or dtype
    n = lambda *shape, to=dtype, shift=0.0: (torch.randn(*shape, device=device, generator=g) + shift).to(to).requires_grad_()
    t = {"x": n(rows, hidden), "weight": n(hidden, to=param_dtype, shift=1.0) if weight else None}
    if stream_dtype is not None:
        t["residual"] = n(rows, hidden, to=stream_dtype)
        t["post_weight"] = n(hidden, to=param_dtype, shift=0.5) if post else None
        shape = {"none": None, "channel": (hidden,), "token": (rows, 1), "full": (rows, hidden)}[gate]
        t["gate"] = None if shape is None else n(*shape, to=param_dtype if gate == "channel" else dtype)
    t["dy"] = n(rows, hidden).detach()
    t["dd"] = None if stream_dtype is None else n(rows, hidden, to=stream_dtype).detach()
    return t


def run(t, m, eps=EPS):
    if "residual" not in t:
        return {"y": xma.rmsnorm(t["x"], t["weight"], eps)}
    y, s = xma.fused_residual_add_rmsnorm(t["x"], t["residual"], t["weight"], eps, m, post_weight=t["post_weight"], gate=t["gate"])
    return {"y": y, "stream": s}


def check(t, m, use=("y", "stream"), eps=EPS):
    out = run(t, m, eps)
    rows, hidden = t["x"].shape
    leaves = {k: v for k, v in t.items() if k not in ("dy", "dd") and v is not None}
    dy = t["dy"] if "y" in use else None
    dd = t["dd"] if "stream" in use else None
    pairs = [(out[k], d) for k, d in (("y", dy), ("stream", dd)) if k in out and d is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [d for _, d in pairs], allow_unused=True)
    ref = norm_reference(t["x"], t.get("residual"), t["weight"], t.get("post_weight"), t.get("gate"), eps, m, dy, dd,
                         None if t.get("post_weight") is not None or t.get("gate") is not None else out.get("stream"))
    got = {**out, **{"d_" + k: v for k, v in zip(leaves, grads)}}
    for name, value in got.items():
        if value is None:
            assert name == "d_weight" and "y" not in use  # no path to the weight
            continue
        want, magnitude = ref[name]
        steps = hidden / 256 + 80 + (rows / 148 + 64 if want.dim() == 1 and name.startswith("d_") else 0)
        assert value.dtype == (leaves[name[2:]] if name.startswith("d_") else out[name]).dtype
        tiny = torch.finfo(value.dtype).smallest_normal * torch.finfo(value.dtype).eps  # subnormals step evenly
        assert_within(name, value.reshape(want.shape), want, half_step(value.dtype) * want.abs() * (1 + 2 ** -7) + steps * F32 * magnitude + tiny)
    assert_status_clean(t["x"].device)
    return got


SHAPES = [(1, 1), (3, 7), (5, 8), (2, 64), (130, 96), (7, 256), (33, 1000), (9, 1001), (450, 512), (4, 4096), (301, 2048),
          (149, 8), (5, 7168), (3, 8192), (2, 8200), (2, 8201), (2, 16392), (2, 20001)]
TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
         (torch.float16, torch.float32), (torch.float32, torch.float32)]


@pytest.mark.parametrize("rows,hidden", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rmsnorm(rows, hidden, dtype):
    check(make(rows, hidden, dtype, None, "none", False), 1.0)


@pytest.mark.parametrize("rows,hidden", SHAPES)
@pytest.mark.parametrize("types", range(len(TYPES)))
def test_fused(rows, hidden, types):
    """Every gate, with and without the post norm, at every shape and pair of types."""
    dtype, stream = TYPES[types]
    for i, gate in enumerate(GATES):
        for post in (False, True):
            m = (1.0, 0.22, -1.5, 1.0)[(i + types) % 4]
            check(make(rows, hidden, dtype, stream, gate, post, seed=i), m)


@pytest.mark.parametrize("hidden", [64, 1001, 2048])
@pytest.mark.parametrize("gate", GATES)
def test_float32_parameters(hidden, gate):
    check(make(37, hidden, torch.bfloat16, torch.bfloat16, gate, True, param_dtype=torch.float32), 0.5)


@pytest.mark.parametrize("use", [("y",), ("stream",)])
@pytest.mark.parametrize("hidden", [520, 77])
def test_one_output_used(use, hidden):
    for gate in GATES:
        check(make(19, hidden, torch.float16, torch.float16, gate, gate != "none"), 1.0, use)


def test_without_weight():
    check(make(21, 640, torch.bfloat16, torch.bfloat16, "none", False, weight=False), 1.0)
    check(make(21, 641, torch.bfloat16, None, "none", False, weight=False), 1.0)


@pytest.mark.parametrize("hidden", [256, 250])
def test_unaligned_and_strided_inputs(hidden):
    """Rows that start anywhere, columns of a wider buffer, a transposed view: same values as contiguous copies."""
    g = torch.Generator(device="cuda").manual_seed(3)
    flat = torch.randn(40 * hidden + 3, device="cuda", generator=g).to(torch.bfloat16)
    wide = torch.randn(40, 3 * hidden, device="cuda", generator=g).to(torch.bfloat16)
    w = torch.randn(2 * hidden + 1, device="cuda", generator=g).to(torch.bfloat16)
    views = [flat[3:].view(40, hidden), wide[:, hidden + 1: 2 * hidden + 1], torch.randn(hidden, 40, device="cuda", generator=g).to(torch.bfloat16).t()]
    for x in views:
        for weight in (w[:hidden], w[1: hidden + 1], w[::2][:hidden]):
            y, s = xma.fused_residual_add_rmsnorm(x, views[0], weight, EPS, gate=weight, post_weight=weight)
            y2, s2 = xma.fused_residual_add_rmsnorm(x.clone(memory_format=torch.contiguous_format), views[0].clone(), weight.clone(), EPS, gate=weight.clone(), post_weight=weight.clone())
            # an unaligned row takes another order of the sums: one float32 rounding apart at most, so one step of bf16
            assert ((y - y2).abs() <= 2 * half_step(torch.bfloat16) * y2.abs() + 1e-30).all()
            assert ((s - s2).abs() <= 2 * half_step(torch.bfloat16) * s2.abs() + 1e-5).all()


@pytest.mark.parametrize("shape", [(0, 16), (2, 0, 32)])
def test_no_rows(shape):
    x = torch.zeros(*shape, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(shape[-1], device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y, s = xma.fused_residual_add_rmsnorm(x, x.detach(), w, EPS, gate=w)
    dx, dw = torch.autograd.grad([y, s], [x, w], [y.detach(), s.detach()])
    assert y.shape == x.shape and dx.shape == x.shape and (dw == 0).all()


def test_rows_of_zeros_and_large_values():
    x = torch.zeros(6, 384, device="cuda")
    x[1] = 1e18  # its square is far above float16 and bf16 steps, within float32
    x[2] = 1e-20
    x[3, 5] = 3e4
    t = {"x": x.requires_grad_(), "weight": torch.ones(384, device="cuda", requires_grad=True), "dy": torch.ones(6, 384, device="cuda"), "dd": None}
    check(t, 1.0)


def test_non_finite_rows_stay_alone():
    x = torch.randn(9, 512, device="cuda", dtype=torch.bfloat16)
    clean = xma.rmsnorm(x, None, EPS)
    x[4, 7] = float("nan")
    x[6, 0] = float("inf")
    y = xma.rmsnorm(x, None, EPS)
    others = [0, 1, 2, 3, 5, 7, 8]
    assert torch.equal(y[others], clean[others]) and y[4].isnan().all() and y[6, 0].isnan()


def test_equals_its_parts():
    """The fused call is the composition of its parts, to the rounding of the stream between them."""
    t = make(50, 1024, torch.float32, torch.float32, "channel", True)
    y, s = xma.fused_residual_add_rmsnorm(t["x"], t["residual"], t["weight"], EPS, 0.3, post_weight=t["post_weight"], gate=t["gate"])
    s2 = t["residual"] + 0.3 * t["gate"] * xma.rmsnorm(t["x"], t["post_weight"], EPS)
    y2 = xma.rmsnorm(s2, t["weight"], EPS)
    assert torch.allclose(s, s2, rtol=0, atol=8 * F32 * 16) and torch.allclose(y, y2, rtol=0, atol=16 * F32 * 64)


def test_gradient_against_differences():
    """Directional derivatives in float32: a central difference of step h is off by O(h^2) and 2^-24 |f| / h."""
    t = make(6, 96, torch.float32, torch.float32, "full", True)
    leaves = {k: v for k, v in t.items() if k not in ("dy", "dd")}

    def loss(values):
        y, s = xma.fused_residual_add_rmsnorm(values["x"], values["residual"], values["weight"], EPS, 0.7,
                                              post_weight=values["post_weight"], gate=values["gate"])
        return (y * t["dy"]).double().sum() + (s * t["dd"]).double().sum()

    grads = torch.autograd.grad(loss(leaves), list(leaves.values()))
    for (name, v), d in zip(leaves.items(), grads):
        direction = torch.randn_like(v)
        h = 2.0 ** -8
        up = loss({**leaves, name: (v + h * direction).detach()}).item()
        down = loss({**leaves, name: (v - h * direction).detach()}).item()
        want = (d.double() * direction).sum().item()
        # h^2 / 6 of a third derivative of order one per element, and 2 * 6 * 96 values rounded at 2^-24 of order four
        assert abs((up - down) / (2 * h) - want) <= 0.02 * (d.double() * direction).abs().sum().item() / 10 + 0.05, name


def test_same_results_every_time_and_on_a_side_stream():
    t = make(777, 2048, torch.bfloat16, torch.bfloat16, "channel", True)
    first = check(t, 0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(t, 0.5)
        leaves = {k: v for k, v in t.items() if k not in ("dy", "dd") and v is not None}
        grads = torch.autograd.grad(list(again.values()), list(leaves.values()), [t["dy"], t["dd"]])
    torch.cuda.current_stream().wait_stream(side)
    for k, v in again.items():
        assert torch.equal(v, first[k])
    for k, v in zip(leaves, grads):
        assert torch.equal(v, first["d_" + k])


def test_frozen_parameters_get_no_gradient():
    t = make(11, 128, torch.bfloat16, torch.bfloat16, "channel", True)
    for k in ("weight", "post_weight", "gate"):
        t[k] = t[k].detach()
    y, s = run(t, 0.5).values()
    dx, dr = torch.autograd.grad([y, s], [t["x"], t["residual"]], [t["dy"], t["dd"]])
    full = check(make(11, 128, torch.bfloat16, torch.bfloat16, "channel", True), 0.5)
    assert torch.equal(dx, full["d_x"]) and torch.equal(dr, full["d_residual"])
    with torch.no_grad():
        assert not run(t, 0.5)["y"].requires_grad


def test_captured_step():
    """Forward and backward in a CUDA graph, replayed on new inputs."""
    t = make(65, 1024, torch.bfloat16, torch.bfloat16, "token", True)
    leaves = [v for k, v in t.items() if k not in ("dy", "dd") and v is not None]
    step = lambda: [*(o := list(run(t, 0.5).values())), *torch.autograd.grad(o, leaves, [t["dy"], t["dd"]])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    new = make(65, 1024, torch.bfloat16, torch.bfloat16, "token", True, seed=9)
    with torch.no_grad():
        for k, v in t.items():
            if v is not None:
                v.copy_(new[k])
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, step()):
        assert torch.equal(a, b)


def test_compiled():
    t = make(33, 512, torch.bfloat16, torch.bfloat16, "channel", True)

    def f(x, residual, weight, post_weight, gate):
        return xma.fused_residual_add_rmsnorm(x, residual, weight, EPS, 0.5, post_weight=post_weight, gate=gate)

    leaves = [t[k] for k in ("x", "residual", "weight", "post_weight", "gate")]
    want = f(*leaves)
    got = torch.compile(f, fullgraph=True)(*leaves)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for a, b in zip(torch.autograd.grad(got, leaves, [t["dy"], t["dd"]]), torch.autograd.grad(want, leaves, [t["dy"], t["dd"]])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,hidden", [(2000, 4096), (1400, 6000), (9000, 320), (30000, 64), (1500, 8192), (891, 4104)])
def test_many_rows(rows, hidden):
    """Enough rows for every CTA to go several times round its ring, forward and backward."""
    for types in TYPES:
        check(make(rows, hidden, *types, "channel", True), 0.5)
        check(make(rows, hidden, *types, "full", False), 1.0)
        check(make(rows, hidden, types[0], None, "none", False), 1.0)
    check(make(rows, hidden, torch.bfloat16, torch.bfloat16, "token", True, param_dtype=torch.float32), 0.5)
    check(make(rows, hidden, torch.bfloat16, torch.float32, "none", False), 1.0)


@pytest.mark.parametrize("post", [False, True])
def test_stream_and_branch_are_one_tensor(post):
    """x as its own residual gets the sum of both gradients; gradients of two tensors share no memory."""
    t = make(37, 264, torch.bfloat16, torch.bfloat16, "none", post)
    t["residual"] = t["x"].detach().clone().requires_grad_()
    torch.autograd.backward(list(run(t, None).values()), [t["dy"], t["dd"]])
    dx, dr = t["x"].grad, t["residual"].grad
    assert dx.data_ptr() != dr.data_ptr()
    one = t["x"].detach().requires_grad_()
    y, s = xma.fused_residual_add_rmsnorm(one, one, t["weight"], EPS, post_weight=t["post_weight"])
    got, = torch.autograd.grad([y, s], [one], [t["dy"], t["dd"]])
    assert torch.equal(got, dx + dr)


@pytest.mark.parametrize("rows,hidden", [(5000, 4096), (1500, 6144), (3000, 520), (500, 1001)])
def test_non_finite_rows_stay_alone_in_large_batches(rows, hidden):
    """A row of NaNs or infinities changes no other row, whatever kernel the size picks."""
    t = make(rows, hidden, torch.bfloat16, torch.bfloat16, "token", True)
    pick = [0, 1, rows // 2, rows - 1]
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[pick] = False

    def rows_of(t):
        out = run(t, 0.5)
        return {**out, **dict(zip(("dx", "dr", "dg"), torch.autograd.grad(list(out.values()), [t["x"], t["residual"], t["gate"]], [t["dy"], t["dd"]])))}

    want = rows_of(t)
    with torch.no_grad():
        for i, (name, value) in zip(pick, (("x", float("nan")), ("residual", float("inf")), ("dy", float("nan")), ("gate", float("inf")))):
            t[name][i] = value
    got = rows_of(t)
    for name in want:
        assert torch.equal(got[name][keep], want[name][keep])
    assert got["y"][0].isnan().all() and got["dx"][rows // 2].isnan().all()


@pytest.mark.parametrize("rows,hidden", [(9601, 777), (2401, 4095), (18945, 515), (9473, 1002)])
@pytest.mark.parametrize("types", range(len(TYPES)))
def test_many_rows_of_no_whole_vectors(rows, hidden, types):
    """Rows that start anywhere in a 16-byte piece, the tensors' last bytes outside a whole one."""
    dtype, stream_dtype = TYPES[types]
    assert hidden % 8 and rows * hidden % 8
    check(make(rows, hidden, dtype, stream_dtype, GATES[types % 4], types % 2 == 0), 0.3)
    check(make(rows, hidden, dtype, None, None, False), 1.0)


SMALL = [1.0, 1e-9, 1e-12, 1e-17, 1e-20, 1e-23, 1e-27]
SMALL_SHAPES = [(8, 64), (9, 4096), (7, 1001), (2000, 4096), (4800, 1001), (1400, 6144), (7, 16384), (7, 20001)]


def small_rows(rows, hidden, dtype, stream_dtype, gate, post, names):
    """Rows of which each is scaled by another of SMALL, in the tensors `names`."""
    t = make(rows, hidden, dtype, stream_dtype, gate, post)
    scale = torch.tensor(SMALL, device="cuda")[torch.arange(rows, device="cuda") % len(SMALL)][:, None]
    with torch.no_grad():
        for n in names:
            t[n].mul_(scale)
    return t


SMALL_CALLS = [(torch.float32, None, "none", False, ("x",)), (torch.bfloat16, None, "none", False, ("x",)),
               (torch.float32, torch.float32, "none", True, ("x",)), (torch.bfloat16, torch.bfloat16, "none", False, ("x", "residual")),
               (torch.bfloat16, torch.float32, "channel", True, ("x", "residual")), (torch.float32, torch.float32, "token", True, ("x", "residual")),
               (torch.bfloat16, torch.bfloat16, "full", False, ("x", "residual")), (torch.float32, torch.float32, "full", True, ("x", "residual"))]


@pytest.mark.parametrize("eps", [0.0, 1e-30])
@pytest.mark.parametrize("rows,hidden", SMALL_SHAPES)
def test_small_rows_and_a_small_eps(rows, hidden, eps):
    """Root mean squares whose square is no float32 number, beside ordinary rows."""
    for dtype, stream_dtype, gate, post, names in SMALL_CALLS:
        t = small_rows(rows, hidden, dtype, stream_dtype, gate, post, names)
        with torch.no_grad():
            got = run(t, 0.5, eps)
        ref = norm_reference(t["x"], t.get("residual"), t["weight"], t.get("post_weight"), t.get("gate"), eps, 0.5)
        for name, value in got.items():
            want, magnitude = ref[name]
            tiny = torch.finfo(value.dtype).smallest_normal * torch.finfo(value.dtype).eps
            assert_within(name, value, want, half_step(value.dtype) * want.abs() * (1 + 2 ** -7) + (hidden / 256 + 80) * F32 * magnitude + tiny)
    assert_status_clean(t["x"].device)


def test_rows_of_zeros_without_eps():
    """0 / 0, as the formula says; the rows beside them are what they are alone."""
    for hidden in (64, 4096, 20001):
        x = torch.randn(2500 if hidden == 4096 else 9, hidden, device="cuda")
        clean = xma.rmsnorm(x, None, 0.0)
        x[3], x[5] = 0.0, 1e-25
        y = xma.rmsnorm(x, None, 0.0)
        assert y[3].isnan().all() and (y[5] - 1.0).abs().max() <= 8 * F32
        keep = torch.ones(len(x), dtype=torch.bool, device="cuda")
        keep[[3, 5]] = False
        assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("eps", [0.0, 1e-30])
@pytest.mark.parametrize("rows,hidden", SMALL_SHAPES)
def test_gradients_of_small_rows(rows, hidden, eps):
    """Where the square of a root mean square, or of its reciprocal, is no float32 number, the gradients are."""
    for dtype, stream_dtype, gate, post, names in SMALL_CALLS:
        check(small_rows(rows, hidden, dtype, stream_dtype, gate, post, names), 0.5, eps=eps)


@pytest.mark.parametrize("dtype,stream", TYPES)
@pytest.mark.parametrize("rows,hidden", [(900, 1024), (40, 1001), (3000, 4096)])
def test_residual_add_against_its_definition(rows, hidden, dtype, stream):
    """The backward pass of a plain residual add reads the stream as it was rounded (h, half a step of its type, of each
    element); against the gradients of the exact one that is h sum |dy s rs| in the weight's, and in the rows' once h in
    the stream itself and once in its mean with a."""
    t = make(rows, hidden, dtype, stream, "none", False)
    with torch.no_grad():
        t["residual"].mul_(torch.exp(torch.randn(hidden, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))))
    leaves = [t["x"], t["residual"], t["weight"]]
    grads = torch.autograd.grad(list(run(t, 0.5).values()), leaves, [t["dy"], t["dd"]])
    ref = norm_reference(t["x"], t["residual"], t["weight"], None, None, EPS, 0.5, t["dy"], t["dd"])
    s, dy, w = ref["stream"][0], t["dy"].double(), t["weight"].detach().double()
    rs = torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + EPS)
    h = half_step(stream)
    row = h * (2 + h) * rs.pow(3) * s.abs() * (w * dy * s).abs().mean(-1, keepdim=True)
    extra = {"d_weight": h * (dy * s * rs).abs().sum(0), "d_residual": row, "d_x": 0.5 * row}
    for name, value in zip(("d_x", "d_residual", "d_weight"), grads):
        want, magnitude = ref[name]
        steps = hidden / 256 + 80 + (rows / 148 + 64 if name == "d_weight" else 0)
        u = half_step(value.dtype)
        assert_within(name, value, want, u * want.abs() * (1 + 2 ** -7) + (1 + u) * extra[name] + steps * F32 * magnitude + torch.finfo(value.dtype).tiny)
    assert_status_clean(t["x"].device)


@pytest.mark.parametrize("eps", [0.0, 1e-30])
@pytest.mark.parametrize("rows,hidden", SMALL_SHAPES)
def test_token_gates_of_small_rows(rows, hidden, eps):
    """A token's gate without a post norm: its gradient is a sum over products of a small row with itself."""
    for dtype, stream_dtype in ((torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)):
        check(small_rows(rows, hidden, dtype, stream_dtype, "token", False, ("x", "residual")), 0.5, eps=eps)
        check(small_rows(rows, hidden, dtype, stream_dtype, "token", False, ("x",)), -1.5, eps=eps)
