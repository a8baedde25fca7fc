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
