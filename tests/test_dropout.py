"""Dropout with the residual sum: the generator's published vectors, the kernel against it, refusals.

The kept elements must equal the generator's exactly.  Values: the product and
the sum round once each in FP32 (or once together), and the result rounds once
to its dtype: ``2^-23 (|branch scale| + |y|) + u |y|``.
"""

from __future__ import annotations

import pytest
import torch

from lsso_b200.ball.dropout import dropout_add, dropout_add_reference, dropout_state, keep_mask, random_words

ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def test_generator_gives_the_published_vectors() -> None:
    """Known answers of Philox4x32-10 that Salmon et al. publish with the algorithm."""
    words = random_words(4, state=dropout_state(0))
    assert [f"{w:08x}" for w in words.tolist()] == ["6627e8d5", "e169c58d", "bc57ac4c", "9b00dbd8"]


def test_words_are_a_function_of_element_site_step_and_seed() -> None:
    base = random_words(4096, state=dropout_state(5, step=2), site=1)
    assert torch.equal(base[:1001], random_words(1001, state=dropout_state(5, step=2), site=1))
    for state, site in ((dropout_state(6, step=2), 1), (dropout_state(5, step=3), 1), (dropout_state(5, step=2), 2),
                        (dropout_state(5 + 2 ** 32, step=2), 1)):
        other = random_words(4096, state=state, site=site)
        assert (other == base).double().mean() < 0.01
    # mean and neighbours of 2^20 keeps at p = 0.3: within 5 standard deviations
    keep = keep_mask((1024, 1024), p=0.3, state=dropout_state(77)).double()
    assert abs(keep.mean().item() - 0.7) < 5 * (0.21 / 2 ** 20) ** 0.5
    pairs = ((keep[:, :-1] - 0.7) * (keep[:, 1:] - 0.7)).mean().item()
    assert abs(pairs) < 5 * 0.21 / 2 ** 10


TYPES = [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16),
         (torch.float16, torch.float16), (torch.float32, torch.float32)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (7, 8), (65, 192), (2, 33, 250), (130, 1001), (4, 512, 256), (40000, 3)])
@pytest.mark.parametrize(("branch_dtype", "out_dtype"), TYPES)
@pytest.mark.parametrize(("masked", "with_residual"), [(False, True), (True, True), (True, False), (False, False)])
def test_step_matches_the_generator(shape, branch_dtype, out_dtype, masked, with_residual) -> None:
    from tests.gpu_util import require_native

    require_native()
    if not with_residual:
        out_dtype = branch_dtype
    gen = torch.Generator(device="cuda").manual_seed(sum(shape))
    branch = torch.randn(shape, device="cuda", generator=gen).to(branch_dtype).requires_grad_()
    residual = torch.randn(shape, device="cuda", generator=gen).to(out_dtype).requires_grad_() if with_residual else None
    dy = torch.randn(shape, device="cuda", generator=gen).to(out_dtype)
    mask = torch.rand(shape[:-1], device="cuda", generator=gen) > 0.3 if masked else None
    state = dropout_state(2 ** 40 + 12345, step=2 ** 33 + 9, device="cuda")
    p, site = 0.25, 2 ** 32 - 1
    y = dropout_add(branch, residual, p=p, state=state, site=site, valid_mask=mask)
    with torch.no_grad():
        assert torch.equal(dropout_add(branch, residual, p=p, state=state, site=site, valid_mask=mask), y)
    want_state = state.clone()
    state += 7  # the backward uses the state that the forward read
    leaves = [branch] + ([residual] if with_residual else [])
    grads = torch.autograd.grad(y, leaves, dy)
    keep = keep_mask(shape, p=p, state=want_state, site=site)
    live = torch.ones(shape, dtype=torch.bool, device="cuda") if mask is None else mask[..., None].expand(shape)
    scaled = torch.where(keep & live, branch.detach().double() / (1 - p), 0.0)
    exact = torch.where(live, scaled + (residual.detach().double() if with_residual else 0.0), 0.0)
    bound = 2.0 ** -23 * (scaled.abs() + exact.abs()) + ROUNDOFF[out_dtype] * exact.abs()
    floor = 2.0 ** -24 if torch.float16 in (branch_dtype, out_dtype) else 0.0
    assert y.dtype == out_dtype and ((y.detach().double() - exact).abs() <= 1.01 * bound + floor).all()
    exact = torch.where(keep & live, dy.double() / (1 - p), 0.0)
    bound = (2.0 ** -23 + ROUNDOFF[branch_dtype]) * exact.abs()
    assert grads[0].dtype == branch_dtype and ((grads[0].double() - exact).abs() <= 1.01 * bound + floor).all()
    if with_residual:
        assert torch.equal(grads[1], torch.where(live, dy, torch.zeros_like(dy)))


@pytest.mark.gpu
def test_rates_of_zero_and_one_and_non_finite_values() -> None:
    from tests.gpu_util import require_native

    require_native()
    state = dropout_state(1, device="cuda")
    branch = torch.randn(33, 40, device="cuda", dtype=torch.bfloat16)
    residual = torch.randn(33, 40, device="cuda")
    assert torch.equal(dropout_add(branch, residual, p=0.0, state=state), residual + branch.float())
    assert torch.equal(dropout_add(branch, residual, p=1.0, state=state), residual)
    assert torch.count_nonzero(dropout_add(branch, p=1.0, state=state)) == 0
    # dropped and masked elements contribute exactly zero, whatever they hold
    keep = keep_mask(branch.shape, p=0.5, state=state)
    mask = torch.arange(33, device="cuda") < 30
    bad = torch.where(keep, branch, float("nan"))
    bad[30:] = float("inf")
    worse = residual.clone()
    worse[30:] = float("nan")
    y = dropout_add(bad, worse, p=0.5, state=state, valid_mask=mask)
    assert torch.equal(y, dropout_add(branch, residual, p=0.5, state=state, valid_mask=mask))
    empty = dropout_add(branch, residual, p=0.5, state=state, valid_mask=torch.zeros_like(mask))
    assert torch.count_nonzero(empty) == 0


@pytest.mark.gpu
def test_layouts_streams_and_graphs() -> None:
    from tests.gpu_util import require_native

    require_native()
    state = dropout_state(3, device="cuda")
    base = torch.randn(64, 48, device="cuda", dtype=torch.float16)
    residual = torch.randn(64, 48, device="cuda")
    want = dropout_add(base, residual, p=0.4, state=state)
    shifted = torch.empty(64 * 48 + 1, dtype=torch.float16, device="cuda")[1:].view(64, 48)
    shifted.copy_(base)
    assert torch.equal(dropout_add(shifted, residual, p=0.4, state=state), want)  # off the 16-byte boundary
    wide = torch.zeros(64, 100, dtype=torch.float16, device="cuda")
    wide[:, :48] = base
    assert torch.equal(dropout_add(wide[:, :48], residual.T.contiguous().T, p=0.4, state=state), want)  # strided
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = dropout_add(base, residual, p=0.4, state=state)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = dropout_add(base, residual, p=0.4, state=state)
            state[1] += 1
    assert torch.equal(other, want)
    for step in range(3):  # each replay uses the step that the replay before left
        graph.replay()
        torch.cuda.synchronize()
        at = dropout_state(3, step=step, device="cuda")
        assert torch.equal(captured, dropout_add(base, residual, p=0.4, state=at))
    assert state.tolist() == [3, 3]


@pytest.mark.gpu
def test_gpu_refusals() -> None:
    from tests.gpu_util import require_native

    require_native()
    state = dropout_state(3, device="cuda")
    x = torch.randn(4, 8, device="cuda", dtype=torch.float16)
    with pytest.raises(TypeError, match="supports"):
        dropout_add(x.double(), p=0.1, state=state)
    with pytest.raises(TypeError, match="residual must use"):
        dropout_add(x, x.bfloat16(), p=0.1, state=state)
    with pytest.raises(RuntimeError, match="state must be on"):
        dropout_add(x, p=0.1, state=state.cpu())
    from lsso_b200.ball import _native

    lib = _native.library()
    args = (x.data_ptr(), 1, None, 1, None, 4, 8)
    assert lib.lib.lsso_dropout_forward(*args, 1.5, state.data_ptr(), 0, None, x.data_ptr(), None) == 1
    assert "[0, 1]" in lib.last_error()
    assert lib.lib.lsso_dropout_forward(*args, 0.5, None, 0, None, x.data_ptr(), None) == 1
    empty = dropout_add(x[:0], p=0.1, state=state)
    assert empty.shape == (0, 8)


def test_cpu_refusals_and_reference() -> None:
    state = dropout_state(3)
    x = torch.randn(4, 6, 8, dtype=torch.float64)
    for p in (-0.1, 1.1):
        with pytest.raises(ValueError, match="p must be"):
            dropout_add(x, p=p, state=state)
    with pytest.raises(ValueError, match="site"):
        dropout_add(x, p=0.1, state=state, site=-1)
    with pytest.raises(ValueError, match="state"):
        dropout_add(x, p=0.1, state=state[:1])
    with pytest.raises(ValueError, match="residual"):
        dropout_add(x, x[:1], p=0.1, state=state)
    with pytest.raises(ValueError, match="valid_mask"):
        dropout_add(x, p=0.1, state=state, valid_mask=torch.ones(4, dtype=torch.bool))
    with pytest.raises(TypeError, match="valid_mask"):
        dropout_add(x, p=0.1, state=state, valid_mask=torch.ones(4, 6))
    with pytest.raises(ValueError, match="CUDA"):
        dropout_add(x, p=0.1, state=state)
    mask = torch.rand(4, 6) > 0.5
    y = dropout_add_reference(x, x, p=0.5, state=state, site=4, valid_mask=mask)
    keep = keep_mask(x.shape, p=0.5, state=state, site=4)
    torch.testing.assert_close(y, torch.where(mask[..., None], x + torch.where(keep, 2 * x, 0.0), 0.0))
    assert torch.equal(dropout_add_reference(x, x, p=1.0, state=state), x)
