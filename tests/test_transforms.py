"""Transforms that the token shell's operators do not take part in are refused, on any device, before any work."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from lsso_b200.ball.dropout import dropout_add, dropout_state
from lsso_b200.ball.embedding import token_embedding
from lsso_b200.ball.feedforward import gated_feed_forward

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _calls(device):
    """{operator: (function of its differentiable inputs, those inputs)}"""
    if device == "cuda":
        from tests.gpu_util import require_native

        require_native()
    make = lambda *s: torch.randn(*s, device=device)  # noqa: E731
    state, ids = dropout_state(1, device=device), torch.tensor([[0, 2, 1]], device=device)
    return {
        "gated_feed_forward": (gated_feed_forward,
                               [make(3, 8).bfloat16(), make(32, 8), make(8, 16), make(32), make(8)]),
        "token_embedding": (lambda weight: token_embedding(ids, weight), [make(4, 8)]),
        "dropout_add": (lambda branch, residual: dropout_add(branch, residual, p=0.5, state=state),
                        [make(1, 3, 8), make(1, 3, 8)]),
    }


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("needs_grad", [False, True])
@pytest.mark.parametrize("name", ["gated_feed_forward", "token_embedding", "dropout_add"])
def test_forward_mode_is_refused(name, needs_grad, device) -> None:
    call, inputs = _calls(device)[name]
    for i in range(len(inputs)):
        with forward_ad.dual_level():
            values = [v.clone().requires_grad_(needs_grad) for v in inputs]
            values[i] = forward_ad.make_dual(values[i], torch.ones_like(values[i]))
            with pytest.raises(NotImplementedError, match=f"{name} .*forward-mode"):
                call(*values)
    if device == "cuda":  # inputs without a tangent run beside a dual level
        with forward_ad.dual_level():
            assert torch.isfinite(call(*inputs)).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", ["gated_feed_forward", "token_embedding", "dropout_add"])
def test_vmap_and_function_transforms_are_refused(name, device) -> None:
    call, inputs = _calls(device)[name]
    with pytest.raises(NotImplementedError, match=f"{name} .*torch.func"):
        torch.vmap(call)(*[v.expand(2, *v.shape) for v in inputs])
    with pytest.raises(NotImplementedError, match=f"{name} .*torch.func"):
        torch.func.grad(lambda *v: call(*v).float().sum())(*inputs)
    with pytest.raises(NotImplementedError, match=f"{name} "):
        torch.func.jvp(call, tuple(inputs), tuple(torch.ones_like(v) for v in inputs))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", ["gated_feed_forward", "token_embedding", "dropout_add"])
def test_tracing_is_refused(name, device) -> None:
    call, inputs = _calls(device)[name]
    with pytest.raises(NotImplementedError, match=f"{name} .*traced"):
        torch.jit.trace(call, tuple(inputs), check_trace=False)
    from torch.fx.experimental.proxy_tensor import make_fx

    with pytest.raises(NotImplementedError, match=f"{name} .*traced"):
        make_fx(lambda *v: call(*v))(*inputs)
