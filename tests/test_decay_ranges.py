"""Decay attention where factors of very different sizes meet: steep decays, growing states, large scales.

Every row is held to three roundings of its magnitude (the definition with absolute values): a pair of tokens meets
through one rounded score, or through a rounded key weight and a rounded state (2 u), and the output is rounded once.
"""

from __future__ import annotations

import pytest
import torch

from lsso_b200.ball.decay import decay_attention
from tests.test_decay import U, exact, inputs

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def native() -> None:
    from tests.gpu_util import require_native

    require_native()


def rows_are_within_three_roundings(q, k, v, dy, l, scale, state=None, mask=None, floor=0.0) -> None:
    """y, dq, dk and dv; ``floor``: what a row's own smallest steps come to."""
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    y = decay_attention(*leaves, l, scale=scale, state=state, valid_mask=mask)
    grads = torch.autograd.grad(y, leaves, dy)
    sides = []
    for size in (lambda t: t, torch.abs):
        wide = [size(t.double()).requires_grad_() for t in (q, k, v)]
        w, _ = exact(*wide, l, abs(scale), None if state is None else size(state), mask)
        sides.append((w, *torch.autograd.grad(w, wide, size(dy.double()))))
    for name, got, want, magnitude in zip(("y", "dq", "dk", "dv"), (y, *grads), *sides):
        error = (got.double() - want).norm(dim=-1)
        within = want.abs().amax(-1) <= 0.99 * torch.finfo(q.dtype).max  # the others are infinite in the type
        assert torch.isfinite(got)[within].all(), name
        assert (error <= 3 * U[q.dtype] * magnitude.norm(dim=-1) + floor)[within].all(), name


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("decay", [-1.0, -1.8, -2.1, -2.2, -2.25, -2.5])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tiny_values_under_steep_decays(dtype, decay, given) -> None:
    """Chunks of zero, tiny and ordinary values under decays whose powers over 32 tokens come near the end of FP32: in
    FP16 the power of two that brings tiny scores into range meets those powers."""
    q, k, v, l, state, _ = inputs(4, 640, 4, 64, 64, dtype, decays=[decay] * 4, state=given, seed=21)
    g = torch.Generator(device="cuda").manual_seed(22)
    kinds = torch.tensor([0.0, 2.0 ** -18, 2.0 ** -9, 1.0], device="cuda")

    def sized(t):
        kind = torch.randint(0, 4, (t.shape[0], 5, t.shape[2], 1), device="cuda", generator=g)
        return (t * kinds[kind].repeat_interleave(128, 1)).to(dtype)

    q, k, v, dy = (sized(t) for t in (q, k, v, torch.randn(v.shape, device="cuda", generator=g)))
    # FP16: a row of 64 results' own smallest steps.  BF16: parts of the sums below 2^-126 vanish, each times 64 features
    # and 128 tokens of values below 2^3, over a row of 64.
    floor = 2.0 ** -25 * 8 if dtype == torch.float16 else 2.0 ** (-126 + 6 + 6 + 7 + 3)
    rows_are_within_three_roundings(q, k, v, dy, l, 0.125, state, floor=floor)


@pytest.mark.parametrize("scale", [2.0 ** 40, 2.0 ** 80])
@pytest.mark.parametrize("decay", [-1.5, -2.1, -2.2, -3.0])
def test_large_scales_under_steep_decays(decay, scale) -> None:
    q, k, v, l, state, mask = inputs(2, 300, 2, 32, 32, torch.bfloat16, decays=[decay], state=True, mask="holes", seed=23)
    dy = torch.randn(v.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(24)).bfloat16()
    rows_are_within_three_roundings(q, k, v, dy, l, scale, state, mask)


@pytest.mark.parametrize("decay", [-0.01, -0.3, -0.34])
@pytest.mark.parametrize("scale", [2.0 ** 19, 2.0 ** 80, 2.0 ** 100])
def test_large_scales_of_weighted_rows(decay, scale) -> None:
    """Heads that weigh their rows once, whose first rows' factor is up to 2^64 times the scale."""
    q, k, v, l, state, mask = inputs(2, 300, 2, 32, 32, torch.bfloat16, decays=[decay], state=True, mask="holes", seed=25)
    dy = torch.randn(v.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(26)).bfloat16()
    rows_are_within_three_roundings(q, k, v, dy, l, scale, state, mask)


@pytest.mark.parametrize("dtype", DTYPES)
def test_states_that_grow_out_of_the_type(dtype) -> None:
    """Growth by up to e^2.2 per token: rows are right until the definition leaves the type, whichever way they are weighed."""
    q, k, v, l, _, _ = inputs(1, 128, 4, 32, 32, dtype, decays=[0.5, 1.0, 2.1, 2.2], seed=29)
    with torch.no_grad():
        y = decay_attention(q[:, :8], 2.0 ** -9 * k[:, :8], v[:, :8], l, scale=2.0 ** -9)
        want, _ = exact(q[:, :8], 2.0 ** -9 * k[:, :8], v[:, :8], l, 2.0 ** -9)
        size, _ = exact(q[:, :8].abs(), 2.0 ** -9 * k[:, :8].abs(), v[:, :8].abs(), l, 2.0 ** -9)
        error = (y.double() - want).norm(dim=-1)
        floor = 2.0 ** -25 * 32 ** 0.5 if dtype == torch.float16 else 0.0  # a row of 32 results' own smallest steps
        assert (error <= 3 * U[dtype] * size.norm(dim=-1) + floor).all()
        assert decay_attention(q, k, v, l).shape == v.shape  # whatever it holds then


@pytest.mark.parametrize(("growth", "length"), [(1e-4, 5000), (0.01, 400), (0.05, 150), (0.075, 150), (0.2, 64)])
@pytest.mark.parametrize(("given", "masked"), [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_states_that_grow(dtype, growth, length, given, masked) -> None:
    """A positive log decay: weights above one, for sequences whose outputs stay within FP16 (but a few rows of the last
    case, whose definition gives up to 6.8e6)."""
    q, k, v, l, state, mask = inputs(1, length, 2, 32, 64, dtype, decays=[growth], state=given, mask="holes" if masked else "none", seed=27)
    g = torch.Generator(device="cuda").manual_seed(28)
    dy = (2.0 ** -8 * torch.randn(v.shape, device="cuda", generator=g)).to(dtype)
    floor = 2.0 ** -25 * 8 if dtype == torch.float16 else 0.0  # a row of 64 results' own smallest steps
    rows_are_within_three_roundings(q, k, 2.0 ** -5 * v, dy, l, 0.25, state, mask, floor=floor)
