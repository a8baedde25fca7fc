"""Decay attention over sequences that are cut into segments and keep no state: the training forward of a long document.

Their segments' states are formed without the parts that a returned state needs, by kernels of their own.  Tolerances
are those of ``test_decay.py``: a pair of tokens in different segments meets through a key weight and a state that are
rounded to the type each.
"""

from __future__ import annotations

import pytest
import torch

from lsso_b200.ball import decay
from lsso_b200.ball.decay import decay_attention, decay_attention_reference
from tests.test_decay import U, check, exact, inputs

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def native() -> None:
    from tests.gpu_util import require_native

    require_native()


def _is_cut(q, v, backward) -> bool:
    return decay._workspace(q.device, (*q.shape, v.shape[-1]), backward)[1] > 16


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", ["none", "holes"])
@pytest.mark.parametrize(("key", "value", "heads", "length"), [(32, 24, 1, 5000), (64, 64, 2, 4097), (72, 40, 1, 4096), (40, 72, 1, 4003), (128, 128, 2, 4608)])
def test_outputs_and_gradients_without_a_state(key, value, heads, length, mask, dtype) -> None:
    q, k, v, l, _, valid = inputs(1, length, heads, key, value, dtype, mask=mask, seed=11)
    assert _is_cut(q, v, False) and _is_cut(q, v, True)
    scale = key ** -0.5
    dy = torch.randn(v.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(12)).to(dtype)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    y = decay_attention(*leaves, l, valid_mask=valid)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(decay_attention(q, k, v, l, valid_mask=valid), y)
    sides = []
    for size in (lambda t: t, torch.abs):
        wide = [size(t.double()).requires_grad_() for t in (q, k, v)]
        w, _ = exact(*wide, l, scale, mask=valid)
        sides.append((w, *torch.autograd.grad(w, wide, size(dy.double()))))
    # FP16 weights below 2^-14: 2^-25 for each of a chunk's 128 tokens, times the other two factors
    top = max(t.abs().max().item() for t in (q, k, v, dy)) ** 2
    extra = 2.0 ** -25 * (128 * max(key, value) * top + 1) if dtype == torch.float16 else 0.0
    for got, want, magnitude in zip((y, *grads), *sides):
        check(got, want, magnitude, dtype, extra)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_long_document(dtype) -> None:
    """65536 tokens against the chunks of the reference in 64 bits, for windows of 2 to 2^11 tokens."""
    q, k, v, l, _, _ = inputs(1, 65536, 8, 64, 64, dtype, seed=13)
    assert _is_cut(q, v, False)
    y = decay_attention(q, k, v, l)
    for head in range(8):
        of_head = [t[:, :, head:head + 1].double() for t in (q, k, v)]
        want = decay_attention_reference(*of_head, l[head:head + 1])
        magnitude = decay_attention_reference(*[t.abs() for t in of_head], l[head:head + 1])
        top = max(t.abs().max().item() for t in of_head) ** 2
        check(y[:, :, head:head + 1], want, magnitude, dtype, 2.0 ** -25 * (128 * 64 * top + 1) if dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_segments_are_the_same_every_time(dtype) -> None:
    """Calls of many segments give the same bits again, whole and masked chunks alike, and so do their gradients."""
    for mask in ("none", "prefix"):
        q, k, v, l, _, valid = inputs(2, 20011, 4, 64, 64, dtype, mask=mask, seed=14)
        assert _is_cut(q, v, False) and _is_cut(q, v, True)
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        dy = torch.randn_like(v)
        want = None
        for _ in range(20):
            y = decay_attention(*leaves, l, valid_mask=valid)
            got = (y.detach(), *torch.autograd.grad(y, leaves, dy))
            want = got if want is None else want
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_same_outputs_with_and_without_the_last_state(dtype) -> None:
    """Asking for the last state changes which kernel forms the segments' states, and with it the outputs by no more than
    the rounding of a key weight."""
    q, k, v, l, _, valid = inputs(1, 9000, 2, 64, 64, dtype, mask="holes", seed=15)
    y = decay_attention(q, k, v, l, valid_mask=valid)
    other, _ = decay_attention(q, k, v, l, valid_mask=valid, return_state=True)
    assert (y.double() - other.double()).norm() <= 2 * U[dtype] * other.double().norm()
