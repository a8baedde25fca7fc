"""The gated feed-forward block at the ends of its value range and with operand types that differ.

``u`` is the unit roundoff of a result's dtype, as in ``test_feedforward.py``.
"""

from __future__ import annotations

import pytest
import torch

from lsso_b200.ball.feedforward import gated_feed_forward
from tests.test_feedforward import ROUNDOFF, _exact, _inputs, _within


# ---------------------------------------------------------------------------- biases of another type than the weights
@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 64, 72), (300, 72, 136), (4200, 64, 136)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("weights", ["x", "fp32"])
def test_bias_gradients_keep_the_dtype_of_the_biases(shape, dtype, weights) -> None:
    """FP32 biases beside 16-bit weights, 16-bit biases beside FP32 weights.  A column sum of dy is exact to
    ``t 2^-23`` of its magnitudes and rounds once to the bias' dtype."""
    from tests.gpu_util import require_native

    require_native()
    weight_dtype, bias_dtype = (dtype, torch.float32) if weights == "x" else (torch.float32, dtype)
    x, w_in, w_out, b_in, b_out, dy = _inputs(*shape, dtype, weight_dtype, True)
    b_in, b_out = b_in.to(bias_dtype), b_out.to(bias_dtype)
    leaves = dict(x=x, w_in=w_in, w_out=w_out, b_in=b_in, b_out=b_out)
    y = gated_feed_forward(*(v.requires_grad_() for v in leaves.values()))
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy, retain_graph=True)))
    exact = _exact(x, w_in, w_out, b_in, b_out, dy, "silu")
    for name in leaves:
        value, bound = exact[name]
        if name in ("b_in", "b_out"):
            bound = bound + (ROUNDOFF[bias_dtype] - ROUNDOFF[weight_dtype]) * value.abs()
        assert grads[name].dtype == leaves[name].dtype
        _within(name, grads[name], value, bound, dtype)
    for name in ("b_in", "b_out"):  # alone: no weight gradient beside it
        alone = torch.autograd.grad(y, leaves[name], dy, retain_graph=True)[0]
        assert torch.equal(alone, grads[name])


@pytest.mark.gpu
def test_fp32_bias_gradients_pass_the_fp16_range() -> None:
    """70000 tokens of gradient 1: the sum is above 65504, and whole numbers below 2^24 add exactly."""
    from tests.gpu_util import require_native

    require_native()
    tokens = 70000
    x = torch.randn(tokens, 16, device="cuda").half()
    w_in, w_out = torch.randn(32, 16, device="cuda").half() / 4, torch.randn(16, 16, device="cuda").half() / 4
    b_in, b_out = torch.zeros(32, device="cuda", requires_grad=True), torch.zeros(16, device="cuda", requires_grad=True)
    y = gated_feed_forward(x, w_in, w_out, b_in, b_out)
    db_in, db_out = torch.autograd.grad(y, (b_in, b_out), torch.ones_like(y))
    assert db_out.dtype == torch.float32 and torch.equal(db_out, torch.full_like(db_out, tokens))
    assert torch.isfinite(db_in).all()


def test_an_unknown_type_of_bias_gradients_is_refused() -> None:
    """Before any pointer is looked at."""
    from lsso_b200 import build
    from lsso_b200.ball import _native

    lib = _native.open_library(build.build())
    args = [16] * 6 + [0, 4, 64, 64, 0, 2, 9] + [16] * 5 + [16, 0, None]
    assert lib.lib.lsso_ffn_backward_mixed(*args) == 1
    assert lib.last_error() == "lsso_ffn_backward_mixed: unknown type"


# ---------------------------------------------------------------------------- large pre-activations
def _probe(values, tokens, dtype, up=None):
    """Operands whose pre-activations are g = ``values`` and u = ``up`` (or 1) exactly, with y[:, 0] = act(g) u and, for
    dy = (1, 0, ..), dx[:, 0] = u act'(g) and dx[:, 1] = act(g) (times w_in's factor, which keeps operands in range).
    The feature beside it has an ordinary pre-activation x[:, 2], and y[:, 1] is its product."""
    hidden, dim = 512, 8
    g = torch.tensor(values, dtype=torch.float64).repeat(-(-tokens // len(values)))[:tokens].cuda()
    u = torch.ones_like(g) if up is None else torch.tensor(up, dtype=torch.float64).repeat(-(-tokens // len(up)))[:tokens].cuda()
    factor = 2.0 ** 8 if up is not None else 1.0
    x = torch.zeros(tokens, dim, dtype=torch.float64, device="cuda")
    x[:, 0], x[:, 1] = g / factor, u / factor
    x[:, 2] = torch.randn(tokens, generator=torch.Generator().manual_seed(tokens)).to(dtype).cuda()
    w_in = torch.zeros(2 * hidden, dim, device="cuda")
    w_in[0, 0], w_in[1, 2] = factor, 1.0
    w_in[hidden:, 1] = factor
    w_out = torch.zeros(dim, hidden, device="cuda")
    w_out[0, 0] = w_out[1, 1] = 1.0
    dy = torch.zeros(tokens, dim, device="cuda", dtype=dtype)
    dy[:, 0] = 1.0
    assert torch.equal(x.to(dtype).double(), x)
    return g, x.to(dtype), w_in.to(dtype), w_out.to(dtype), dy


# exact in BF16 (eight significant bits), up to 1e18 on both sides; FP16 takes those it can hold
SATURATED = [0.0, 0.5, -0.5, 12.0, -12.0, 30.0, -30.0, 39.0, -39.0, 40.25, -40.25, 41.0, -41.0, 50.0, -50.0, 88.0, -88.0,
             200.0, -200.0, 1000.0, -1000.0, 30080.0, -30080.0, 60160.0, -60160.0]
BEYOND = [2.0 ** 20, -2.0 ** 20, 2.0 ** 40, -2.0 ** 40, 2.0 ** 60, -2.0 ** 60, 2.0 ** 100, -2.0 ** 100]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 40, 4224])  # streamed weights, cluster-split tiles, persistent pairs
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_activation_and_slope_far_from_zero(tokens, dtype, activation) -> None:
    """Against 64 bits.  The exponential's argument rounds to 2^-24 of up to 60, so a value is good to 2^-17 of the sum
    of its terms' magnitudes; SiLU below -40 is smaller than 2^-52; GELU's erf polynomial is good to 1.5e-7 where
    e^(-g^2/2) is not smaller still."""
    from tests.gpu_util import require_native

    require_native()
    values = SATURATED + (BEYOND if dtype == torch.bfloat16 else [])

    def act_and_slope(g):
        """Values and error floors of act(g) and act'(g)."""
        if activation == "silu":
            p, q = torch.sigmoid(g), torch.sigmoid(-g)
            error = 2.0 ** -17 * p * (1 + g.abs() * q) + 2.0 ** -52
            return g * p, p * (1 + g * q), 2.0 ** -17 * g.abs() * p + 2.0 ** -52, error
        p, tail = 0.5 * torch.erfc(-g * 0.5 ** 0.5), torch.exp(-0.5 * g * g)
        error = tail.clamp(max=1.5e-7) + 2.0 ** -22 * p
        slope = p + g * tail / (2 * torch.pi) ** 0.5
        return g * p, slope, g.abs() * error, error + 2.0 ** -17 * g.abs() * tail

    for start in range(0, len(values), tokens):
        g, x, w_in, w_out, dy = _probe(values[start:] + values[:start], tokens, dtype)
        act, slope, act_floor, slope_floor = act_and_slope(g)
        beside, _, beside_floor, _ = act_and_slope(x[:, 2].double())

        def check(name, actual, expected, floor):
            tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
            expected = torch.where(expected.abs() < 2.0 ** -126, 0.0, expected)  # FP32 has no such value
            off = (actual.double() - expected).abs() - (2.1 * ROUNDOFF[dtype] * expected.abs() + floor + tiny)
            worst = off.argmax()
            assert off.max() <= 0, (name, g[worst].item(), actual[worst].item(), expected[worst].item())  # noqa: B023

        with torch.no_grad():
            y = gated_feed_forward(x, w_in, w_out, activation=activation)
        check("inference", y[:, 0], act, act_floor)
        check("inference beside", y[:, 1], beside, beside_floor)
        x.requires_grad_()
        y = gated_feed_forward(x, w_in, w_out, activation=activation)
        check("y", y.detach()[:, 0], act, act_floor)
        check("beside", y.detach()[:, 1], beside, beside_floor)
        dx = torch.autograd.grad(y, x, dy)[0]
        check("slope", dx[:, 0], slope, slope_floor)
        check("du", dx[:, 1], act, act_floor)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [40, 4224])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_fp16_preactivations_beyond_its_range_keep_finite_gradients(tokens, activation) -> None:
    """Accumulators of 90112 do not fit the FP16 values that the backward reads; they are held as the largest FP16
    value, which changes neither a closed gate nor an open gate's slope."""
    from tests.gpu_util import require_native

    require_native()
    big = 90112.0  # 352 * 2^8
    _, x, w_in, w_out, dy = _probe([-big, -64.0, big, 1.0], tokens, torch.float16, [1.0, big, 0.25, 1.0])
    x[:, 2] = 0  # the feature beside it: act(0) = 0, so that every exact product is in range
    x.requires_grad_()
    w_in, w_out = w_in.float().requires_grad_(), w_out.float()  # FP32: the exact weight gradients are beyond FP16
    y = gated_feed_forward(x, w_in, w_out, activation=activation)
    dx, dw_in = torch.autograd.grad(y, (x, w_in), dy / 256)  # 1 / 256 takes w_in's factor back
    assert torch.isfinite(y).all() and torch.isfinite(dx).all() and torch.isfinite(dw_in).all()
    assert torch.count_nonzero(y[:2, 0]) == 0 and dx[:2, :2].abs().max() <= 2.0 ** -24
    assert abs(y[2, 0].item() - 0.25 * big) <= 2.0 ** -11 * 0.25 * big
    assert abs(dx[2, 0].item() - 0.25) <= 2.0 ** -10 * 0.25
    assert abs(dx[2, 1].item() - 65504.0) <= 2.0 ** -10 * 65504.0


# ---------------------------------------------------------------------------- one row tile, many columns
@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(100, 64, 16640), (24, 32832, 16)])
@pytest.mark.parametrize(("dtype", "activation", "bias"), [(torch.bfloat16, "silu", True), (torch.float16, "gelu", False)])
def test_one_row_tile_of_many_columns(shape, dtype, activation, bias) -> None:
    """More than 512 column tiles over up to 128 rows: the persistent kernel without a partner CTA."""
    from tests.gpu_util import require_native

    require_native()
    x, w_in, w_out, b_in, b_out, dy = _inputs(*shape, dtype, dtype, bias)
    leaves = {n: v.requires_grad_() for n, v in
              dict(x=x, w_in=w_in, w_out=w_out, b_in=b_in, b_out=b_out).items() if v is not None}
    y = gated_feed_forward(x, w_in, w_out, b_in, b_out, activation=activation)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    exact = _exact(x, w_in, w_out, b_in, b_out, dy, activation)
    _within("y", y.detach(), *exact["y"], dtype)
    for name, grad in grads.items():
        _within(name, grad, *exact[name], dtype)
