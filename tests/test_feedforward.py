"""The gated feed-forward block: the CUDA path against 64-bit evaluations, its refusals, its PyTorch form.

Bounds.  ``u`` is the unit roundoff of x's dtype (2^-8 for BF16, 2^-11 for
FP16).  With weights already in x's dtype the path rounds h once (``u |h|``)
and y once, accumulates in FP32 (``K 2^-23`` of the sum of magnitudes, K the
contraction length) and evaluates the activation to a few FP32 ulps (2^-18 of
h).  So ``|y - y64| <= |w_out| (u + 2^-18 + K 2^-23) |h| + u |y|`` element by
element.  The backward reads g and u rounded: with |act''| <= 1,
``E_g = |dh u| (|g| + |act'|) u + u |dg|`` and ``E_u = |dh| |act'| |g| u + u
|du|`` bound its errors in dg and du, which the two products that follow sum in
magnitude.  A factor 1.1 and a floor cover second-order terms and FP16
subnormals.
"""

from __future__ import annotations

import pytest
import torch

from lsso_b200.ball.feedforward import GatedFeedForward, gated_feed_forward, gated_feed_forward_reference

ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _inputs(t, d, h, dtype, weight_dtype, bias, seed=0, device="cuda"):
    gen = torch.Generator().manual_seed(seed + 7 * t + 3 * d + h)
    normal = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, dy = normal(t, d).to(device, dtype), normal(t, d).to(device, dtype)
    w_in = (normal(2 * h, d) / d ** 0.5).to(device, weight_dtype)
    w_out = (normal(d, h) / h ** 0.5).to(device, weight_dtype)
    b_in = (0.3 * normal(2 * h)).to(device, weight_dtype) if bias else None
    b_out = (0.3 * normal(d)).to(device, weight_dtype) if bias else None
    return x, w_in, w_out, b_in, b_out, dy


def _exact(x, w_in, w_out, b_in, b_out, dy, activation):
    """64-bit values and error bounds: {name: (value, bound)} for y and every gradient."""
    kind = x.dtype
    u = ROUNDOFF[kind]
    wide = lambda t: t.detach().to(kind).double()  # noqa: E731  (weights enter in x's dtype)
    xd, wi, wo, dyd = wide(x), wide(w_in), wide(w_out), dy.double()
    hidden = wo.shape[1]
    d = wo.shape[0]
    t = x.shape[0]
    gu = xd @ wi.T + (0 if b_in is None else b_in.double())
    acc_in = (d * 2.0 ** -23) * (xd.abs() @ wi.abs().T + (0 if b_in is None else b_in.double().abs()))
    g, up = gu[:, :hidden], gu[:, hidden:]
    if activation == "silu":
        p = torch.sigmoid(g)
        act, slope = g * p, p * (1 + g * (1 - p))
    else:
        p = 0.5 * torch.erfc(-g * 0.5 ** 0.5)
        act, slope = g * p, p + g * torch.exp(-0.5 * g * g) / (2 * torch.pi) ** 0.5
    h = act * up
    e_h = h.abs() * (u + 2.0 ** -18) + 1.2 * up.abs() * acc_in[:, :hidden] + act.abs() * acc_in[:, hidden:]
    e_h = e_h + 2.0 ** -20 * up.abs()
    y = h @ wo.T + (0 if b_out is None else b_out.double())
    e_y = e_h @ wo.abs().T + hidden * 2.0 ** -23 * (h.abs() @ wo.abs().T) + u * y.abs()
    dh = dyd @ wo
    e_dh = d * 2.0 ** -23 * (dyd.abs() @ wo.abs())
    dg, du = dh * up * slope, dh * act
    e_g = (dh * up).abs() * (g.abs() + slope.abs()) * u + u * dg.abs() + e_dh * (up * slope).abs()
    e_g = e_g + (2.0 ** -18 + 1.2 * acc_in[:, :hidden]) * (dh * up).abs() + acc_in[:, hidden:] * dh.abs()
    e_u = dh.abs() * slope.abs() * g.abs() * u + u * du.abs() + e_dh * act.abs() + 2.0 ** -18 * dh.abs()
    e_u = e_u + 1.2 * acc_in[:, :hidden] * dh.abs()
    dgu, e_gu = torch.cat((dg, du), 1), torch.cat((e_g, e_u), 1)
    uw = ROUNDOFF[w_in.dtype]
    out = {"y": (y, e_y)}
    dx = dgu @ wi
    out["x"] = (dx, e_gu @ wi.abs() + 2 * hidden * 2.0 ** -23 * (dgu.abs() @ wi.abs()) + u * dx.abs())
    dw = dgu.T @ xd
    out["w_in"] = (dw, e_gu.T @ xd.abs() + t * 2.0 ** -23 * (dgu.abs().T @ xd.abs()) + uw * dw.abs())
    dw = dyd.T @ h
    out["w_out"] = (dw, dyd.abs().T @ e_h + t * 2.0 ** -23 * (dyd.abs().T @ h.abs()) + uw * dw.abs())
    if b_in is not None:
        s = dgu.sum(0)
        out["b_in"] = (s, e_gu.sum(0) + t * 2.0 ** -23 * dgu.abs().sum(0) + uw * s.abs())
        s = dyd.sum(0)
        out["b_out"] = (s, t * 2.0 ** -23 * dyd.abs().sum(0) + uw * s.abs())
    return out


def _within(name, actual, expected, bound, kind):
    floor = 2.0 ** -24 * 4 if kind == torch.float16 else 1e-30
    off = (actual.double() - expected).abs() - 1.1 * bound - floor
    assert torch.isfinite(actual).all(), name
    assert off.max().item() <= 0, (name, off.max().item(), bound.mean().item())


SHAPES = [
    (1, 8, 8), (1, 64, 176), (3, 128, 344), (16, 256, 688), (17, 256, 688), (97, 512, 1368), (128, 64, 64),
    (129, 72, 136), (300, 192, 520), (1000, 256, 1024), (4097, 128, 344), (33, 1000, 24), (257, 40, 1992),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize(("dtype", "activation", "bias"), [
    (torch.bfloat16, "silu", False), (torch.float16, "gelu", True), (torch.float16, "silu", True),
    (torch.bfloat16, "gelu", False)])
def test_training_step_matches_64_bits(shape, dtype, activation, bias) -> None:
    from tests.gpu_util import require_native

    require_native()
    x, w_in, w_out, b_in, b_out, dy = _inputs(*shape, dtype, dtype, bias)
    leaves = {n: v.requires_grad_() for n, v in
              (("x", x), ("w_in", w_in), ("w_out", w_out), ("b_in", b_in), ("b_out", b_out)) if v is not None}
    y = gated_feed_forward(x, w_in, w_out, b_in, b_out, activation=activation)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    exact = _exact(x, w_in, w_out, b_in, b_out, dy, activation)
    _within("y", y.detach(), *exact["y"], dtype)
    for name, grad in grads.items():
        assert grad.dtype == leaves[name].dtype and grad.shape == leaves[name].shape
        _within(name, grad, *exact[name], dtype)
    with torch.no_grad():
        again = gated_feed_forward(x, w_in, w_out, b_in, b_out, activation=activation)
    _within("inference", again, *exact["y"], dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 15, 16, 17, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fp32_weights_are_rounded_to_x_dtype_and_get_fp32_gradients(rows, dtype) -> None:
    from tests.gpu_util import require_native

    require_native()
    x, w_in, w_out, b_in, b_out, dy = _inputs(rows, 136, 264, dtype, torch.float32, True)
    with torch.no_grad():  # few rows: FP32 weights streamed
        served = gated_feed_forward(x, w_in, w_out, b_in, b_out)
    exact = _exact(x, w_in, w_out, b_in, b_out, dy, "silu")
    _within("served", served, *exact["y"], dtype)
    leaves = [v.requires_grad_() for v in (x, w_in, w_out, b_in, b_out)]
    y = gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    _within("y", y.detach(), *exact["y"], dtype)
    for name, grad in zip(("x", "w_in", "w_out", "b_in", "b_out"), grads):
        assert grad.dtype == (dtype if name == "x" else torch.float32)
        _within(name, grad, *exact[name], dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_gradients_match_differences(activation) -> None:
    """Directional differences of the 64-bit operator along random directions of every input."""
    from tests.gpu_util import require_native

    require_native()
    x, w_in, w_out, b_in, b_out, dy = _inputs(70, 64, 96, torch.float16, torch.float16, True)
    leaves = [v.requires_grad_() for v in (x, w_in, w_out, b_in, b_out)]
    grads = torch.autograd.grad(gated_feed_forward(*leaves, activation=activation), leaves, dy)
    base = [v.detach().double() for v in leaves]
    gen = torch.Generator().manual_seed(5)
    for i, grad in enumerate(grads):
        step = torch.randn(base[i].shape, generator=gen).cuda().double()
        sides = []
        for sign in (1, -1):
            moved = list(base)
            moved[i] = base[i] + sign * 1e-5 * step
            sides.append((gated_feed_forward_reference(*moved, activation=activation) * dy.double()).sum().item())
        slope = (sides[0] - sides[1]) / 2e-5
        # sums of n independent FP16 roundings: 2^-11 relative each, so well within 1% of the norm's scale
        scale = float((grad.double().norm() * step.norm()).item())
        assert abs(float((grad.double() * step).sum()) - slope) <= 2.0 ** -9 * scale


@pytest.mark.gpu
def test_extreme_activations_stay_finite_and_nan_rows_stay_apart() -> None:
    from tests.gpu_util import require_native

    require_native()
    x, w_in, w_out, _, _, dy = _inputs(260, 64, 128, torch.bfloat16, torch.bfloat16, False)
    x[::2] *= 60  # pre-activations of a few hundred: SiLU and its slope saturate on both sides
    for activation in ("silu", "gelu"):
        leaves = [v.clone().requires_grad_() for v in (x, w_in, w_out)]
        y = gated_feed_forward(*leaves, activation=activation)
        grads = torch.autograd.grad(y, leaves, dy)
        assert all(torch.isfinite(v).all() for v in (y, *grads))
    clean = gated_feed_forward(x, w_in, w_out)
    x[37] = float("nan")
    x[38, 3] = float("inf")
    y = gated_feed_forward(x, w_in, w_out)
    keep = torch.ones(260, dtype=torch.bool, device="cuda")
    keep[37:39] = False
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[37]).all()


@pytest.mark.gpu
def test_layouts_streams_and_repeats() -> None:
    from tests.gpu_util import require_native

    require_native()
    x, w_in, w_out, b_in, b_out, _ = _inputs(4 * 60, 96, 200, torch.bfloat16, torch.bfloat16, True)
    want = gated_feed_forward(x, w_in, w_out, b_in, b_out)
    assert torch.equal(gated_feed_forward(x.view(4, 60, 96), w_in, w_out, b_in, b_out), want.view(4, 60, 96))
    wide = torch.zeros(240, 200, dtype=x.dtype, device="cuda")
    wide[:, 3:99] = x
    assert torch.equal(gated_feed_forward(wide[:, 3:99], w_in, w_out, b_in, b_out), want)  # strided rows
    shifted = torch.empty(240 * 96 + 1, dtype=x.dtype, device="cuda")[1:].view(240, 96)
    shifted.copy_(x)
    assert torch.equal(gated_feed_forward(shifted, w_in, w_out, b_in, b_out), want)  # off the 16-byte boundary
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = gated_feed_forward(x, w_in, w_out, b_in, b_out)
    side.synchronize()
    assert torch.equal(other, want)
    leaves = [v.clone().requires_grad_() for v in (x, w_in, w_out)]
    first = torch.autograd.grad(gated_feed_forward(*leaves).float().square().sum(), leaves)
    second = torch.autograd.grad(gated_feed_forward(*leaves).float().square().sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    # only some gradients wanted
    partial = torch.autograd.grad(gated_feed_forward(leaves[0], w_in, w_out).float().square().sum(), leaves[0])[0]
    assert torch.equal(partial, first[0])
    only = w_out.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(gated_feed_forward(x, w_in, only).float().square().sum(), only)[0], first[2])


@pytest.mark.gpu
@pytest.mark.parametrize(("dim", "hidden", "rows"), [(33, 50, 70), (20, 64, 3), (64, 30, 300)])
def test_widths_that_are_not_multiples_of_eight(dim, hidden, rows) -> None:
    from tests.gpu_util import require_native

    require_native()
    x, w_in, w_out, b_in, b_out, dy = _inputs(rows, dim, hidden, torch.bfloat16, torch.float32, True)
    leaves = [v.requires_grad_() for v in (x, w_in, w_out, b_in, b_out)]
    y = gated_feed_forward(*leaves, activation="gelu")
    grads = torch.autograd.grad(y, leaves, dy)
    exact = _exact(x, w_in, w_out, b_in, b_out, dy, "gelu")
    _within("y", y.detach(), *exact["y"], x.dtype)
    for name, grad in zip(("x", "w_in", "w_out", "b_in", "b_out"), grads):
        _within(name, grad, *exact[name], x.dtype)


@pytest.mark.gpu
def test_no_rows() -> None:
    from tests.gpu_util import require_native

    require_native()
    x, w_in, w_out, _, _, _ = _inputs(1, 64, 64, torch.bfloat16, torch.float32, False)
    leaves = [x[:0].requires_grad_(), w_in.requires_grad_(), w_out.requires_grad_()]
    y = gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y.sum(), leaves)
    assert y.shape == (0, 64) and y.dtype == torch.bfloat16
    assert all(torch.count_nonzero(g) == 0 for g in grads)


@pytest.mark.gpu
def test_refusals() -> None:
    from tests.gpu_util import require_native

    require_native()
    x, w_in, w_out, b_in, b_out, _ = _inputs(4, 64, 64, torch.bfloat16, torch.bfloat16, True)
    with pytest.raises(TypeError, match="bfloat16 or torch.float16"):
        gated_feed_forward(x.float(), w_in, w_out)
    with pytest.raises(TypeError, match="w_in and w_out"):
        gated_feed_forward(x, w_in, w_out.float())
    with pytest.raises(TypeError, match="w_in and w_out"):
        gated_feed_forward(x, w_in.half(), w_out.half())
    with pytest.raises(TypeError, match="b_in and b_out"):
        gated_feed_forward(x, w_in, w_out, b_in, b_out.float())
    with pytest.raises(RuntimeError, match="contiguous w_in"):
        gated_feed_forward(x, w_in.T.contiguous().T, w_out)
    with pytest.raises(RuntimeError, match="w_in must be on"):
        gated_feed_forward(x, w_in.cpu(), w_out)
    from lsso_b200.ball import _native

    lib = _native.library()
    assert lib.lib.lsso_ffn_backward_workspace_size(4, 12, 64) == 0 and "multiples of 8" in lib.last_error()
    args = (x.data_ptr(), 0, 4, 64, 64, w_in.data_ptr(), w_out.data_ptr())
    assert lib.lib.lsso_ffn_forward(*args, 1, None, None, 2, 0, None, x.data_ptr(), x.data_ptr(), None) == 1
    assert "x's type" in lib.last_error()
    assert lib.lib.lsso_ffn_forward(*args, 0, None, None, 2, 7, None, x.data_ptr(), x.data_ptr(), None) == 1
    assert "activation" in lib.last_error()


def test_cpu_refusals_and_reference() -> None:
    x, w_in, w_out, b_in, b_out, _ = _inputs(5, 12, 20, torch.float64, torch.float64, True, device="cpu")
    with pytest.raises(ValueError, match="activation"):
        gated_feed_forward(x, w_in, w_out, activation="tanh")
    with pytest.raises(ValueError, match="CUDA"):
        gated_feed_forward(x, w_in, w_out)
    with pytest.raises(ValueError, match="w_in must have shape"):
        gated_feed_forward(x, w_in[:-1], w_out)
    with pytest.raises(ValueError, match="w_out must have shape"):
        gated_feed_forward(x, w_in, w_out.T)
    with pytest.raises(ValueError, match="x must have shape"):
        gated_feed_forward(x[:, :-1], w_in, w_out)
    with pytest.raises(ValueError, match="b_in must have shape"):
        gated_feed_forward(x, w_in, w_out, b_in[:-1], b_out)
    g, u = (x @ w_in.T + b_in).chunk(2, dim=-1)
    want = (g / (1 + torch.exp(-g)) * u) @ w_out.T + b_out
    torch.testing.assert_close(gated_feed_forward_reference(x, w_in, w_out, b_in, b_out), want)
    leaves = [v.requires_grad_() for v in (x, w_in, w_out, b_in, b_out)]
    for activation in ("silu", "gelu"):
        torch.autograd.gradcheck(
            lambda *v: gated_feed_forward_reference(*v, activation=activation), leaves)  # noqa: B023
    layer = GatedFeedForward(12, 20, bias=True).double()
    assert layer(x).shape == x.shape and layer.w_in.weight.shape == (40, 12)
    with pytest.raises(ValueError, match="implementation"):
        layer(x, implementation="fast")


@pytest.mark.gpu
def test_waits_that_run_out_leave_a_usable_library() -> None:
    """With a one-nanosecond limit the tensor-core kernels take their abort path (nothing hangs or
    faults), the status says so, and the next calls give the bits of the calls before."""
    from lsso_b200.ball import _native, cuda
    from tests.gpu_util import require_native

    require_native()
    cuda.device_status(reset=True)
    for rows in (100, 3000):  # single CTAs and pairs
        x, w_in, w_out, b_in, b_out, dy = _inputs(rows, 256, 688, torch.bfloat16, torch.bfloat16, True)
        leaves = [v.requires_grad_() for v in (x, w_in, w_out, b_in, b_out)]

        def step():
            y = gated_feed_forward(*leaves)  # noqa: B023
            return (y.detach(), *torch.autograd.grad(y, leaves, dy))  # noqa: B023

        want = step()
        torch.cuda.synchronize()
        _native.set_wait_limit_ns(1)
        try:
            step()
            torch.cuda.synchronize()
        finally:
            _native.set_wait_limit_ns(0)
        assert cuda.device_status(reset=True) == 1
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
        assert cuda.device_status(reset=True) == 0


# few rows without gradients: products of few tiles, their contraction split over two, four and eight CTAs
FEW = [(17, 256, 688), (24, 64, 1024), (31, 1024, 64), (97, 512, 1368), (128, 1000, 4096), (129, 512, 520),
       (250, 200, 2000), (400, 136, 344), (512, 1024, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", FEW)
@pytest.mark.parametrize(("dtype", "activation", "bias"), [
    (torch.bfloat16, "silu", True), (torch.float16, "gelu", False), (torch.float16, "silu", True),
    (torch.bfloat16, "gelu", True)])
def test_few_rows_without_gradients(shape, dtype, activation, bias) -> None:
    from tests.gpu_util import require_native

    require_native()
    x, w_in, w_out, b_in, b_out, dy = _inputs(*shape, dtype, dtype, bias)
    want = _exact(x, w_in, w_out, b_in, b_out, dy, activation)["y"]
    with torch.no_grad():
        y = gated_feed_forward(x, w_in, w_out, b_in, b_out, activation=activation)
        _within("y", y, *want, dtype)
        assert torch.equal(y, gated_feed_forward(x, w_in, w_out, b_in, b_out, activation=activation))
        # a row's result depends on its own values alone, whatever the rows beside it hold
        x[0], x[-1] = float("inf"), float("nan")
        other = gated_feed_forward(x, w_in, w_out, b_in, b_out, activation=activation)
    assert torch.equal(y[1:-1], other[1:-1]) and not torch.isfinite(other[[0, -1]]).any()


@pytest.mark.gpu
def test_split_waits_that_run_out_leave_a_usable_library() -> None:
    """The same for the products whose contraction is split over a cluster."""
    from lsso_b200.ball import _native, cuda
    from tests.gpu_util import require_native

    require_native()
    cuda.device_status(reset=True)
    for shape in ((20, 128, 512), (100, 512, 1368), (128, 1024, 4096)):
        args = _inputs(*shape, torch.bfloat16, torch.bfloat16, True)[:5]
        with torch.no_grad():
            want = gated_feed_forward(*args)
            torch.cuda.synchronize()
            _native.set_wait_limit_ns(1)
            try:
                gated_feed_forward(*args)
                torch.cuda.synchronize()
            finally:
                _native.set_wait_limit_ns(0)
            assert cuda.device_status(reset=True) == 1
            assert torch.equal(gated_feed_forward(*args), want)
            assert cuda.device_status(reset=True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 64, 4096), (64, 1024, 4096), (250, 200, 2000), (520, 264, 1096), (1000, 512, 1368)])
@pytest.mark.parametrize(("dtype", "activation"), [(torch.bfloat16, "silu"), (torch.float16, "gelu")])
def test_few_rows_with_gradients(shape, dtype, activation) -> None:
    """Training passes of few tiles, all gradients together, twice, and each alone."""
    from tests.gpu_util import require_native

    require_native()
    x, w_in, w_out, b_in, b_out, dy = _inputs(*shape, dtype, dtype, True)
    want = _exact(x, w_in, w_out, b_in, b_out, dy, activation)
    leaves = {n: v.requires_grad_() for n, v in
              dict(x=x, w_in=w_in, w_out=w_out, b_in=b_in, b_out=b_out).items()}
    y = gated_feed_forward(*leaves.values(), activation=activation)
    _within("y", y.detach(), *want["y"], dtype)
    grads = torch.autograd.grad(y, list(leaves.values()), dy, retain_graph=True)
    for name, grad in zip(leaves, grads):
        _within(name, grad, *want[name], dtype)
    again = torch.autograd.grad(y, list(leaves.values()), dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    for name, leaf in leaves.items():
        _within(name, torch.autograd.grad(y, leaf, dy, retain_graph=True)[0], *want[name], dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 1024, 1368), (6, 512, 1368), (16, 264, 2048)])
def test_few_rows_with_fp32_weights(shape) -> None:
    """Streamed or copied, FP32 weights are rounded to x's dtype first."""
    from tests.gpu_util import require_native

    require_native()
    x, w_in, w_out, b_in, b_out, dy = _inputs(*shape, torch.bfloat16, torch.float32, True)
    with torch.no_grad():
        y = gated_feed_forward(x, w_in, w_out, b_in, b_out)
    _within("y", y, *_exact(x, w_in, w_out, b_in, b_out, dy, "silu")["y"], torch.bfloat16)
