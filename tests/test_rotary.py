"""Rotary positions against the definition in 64 bits, gradients, layouts, positions, refusals.

A turned feature is two products and a sum in FP32 of factors that are within 2^-23 of the cosine and sine (their
rounding, and that of the angle's fraction of a turn, pi 2^-24): ``2^-21 (|a| + |b|) magnitude``, and the result's own
rounding ``u |y|``.
"""

from __future__ import annotations

import math

import pytest
import torch

from lsso_b200.ball.rotary import rotary, rotary_frequencies, rotary_reference

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def exact(x, frequencies, positions, interleaved, magnitude, sign=1.0):
    """(turned, |a| + |b| of every feature's pair) with complex numbers in 64 bits."""
    f = frequencies.numel()
    x = x.detach().double()
    positions = torch.arange(x.shape[1], device=x.device) if positions is None else positions
    turn = torch.polar(torch.full((), magnitude, dtype=torch.float64, device=x.device), sign * positions.double()[..., None] * frequencies.double())
    first = torch.arange(f, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else f)
    z = torch.complex(x[..., first], x[..., second]) * turn[..., None, :]
    y, size = x.clone(), torch.zeros_like(x)
    y[..., first], y[..., second] = z.real, z.imag
    size[..., first] = size[..., second] = x[..., first].abs() + x[..., second].abs()
    return y, size * magnitude


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pairs", [1, 3, 8])
def test_reference_follows_the_definition(interleaved, pairs) -> None:
    x = torch.randn(2, 7, 3, 16, dtype=torch.float64, requires_grad=True)
    f = rotary_frequencies(2 * pairs)[0]
    positions = torch.randint(0, 10 ** 6, (2, 7))
    y = rotary_reference(x, f, positions, interleaved=interleaved, magnitude=1.25)
    assert torch.allclose(y, exact(x, f, positions, interleaved, 1.25)[0], rtol=1e-9, atol=1e-9)
    dy = torch.randn_like(y)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert torch.allclose(dx, exact(dy, f, positions, interleaved, 1.25, -1.0)[0], rtol=1e-9, atol=1e-9)
    torch.autograd.gradcheck(lambda t: rotary_reference(t, f, positions, interleaved=interleaved, magnitude=1.25), x)


def test_scores_depend_on_distance_alone() -> None:
    q, k = torch.randn(2, 1, 1, 1, 32, dtype=torch.float64)
    f = rotary_frequencies(32)[0]
    score = lambda i, j: (rotary_reference(q, f, torch.tensor([i])) * rotary_reference(k, f, torch.tensor([j]))).sum()  # noqa: E731
    assert torch.allclose(score(5, 3), score(1005, 1003), rtol=1e-9)


def test_frequencies_and_their_scalings() -> None:
    plain, one = rotary_frequencies(8, base=100.0)
    assert torch.allclose(plain, torch.tensor([1, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64)) and one == 1.0
    assert torch.allclose(rotary_frequencies(8, base=100.0, scaling="linear", factor=4.0)[0], plain / 4)
    wider = rotary_frequencies(8, base=100.0, scaling="base", factor=4.0)[0]
    assert wider[0] == 1 and torch.allclose(wider[-1], plain[-1] / 4)
    blend, magnitude = rotary_frequencies(64, scaling="blend", factor=8.0, original_length=4096)
    plain = rotary_frequencies(64)[0]
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(blend[turns > 32], plain[turns > 32]) and torch.allclose(blend[turns < 1], plain[turns < 1] / 8)
    assert (blend[:-1] > blend[1:]).all() and magnitude == 1 + 0.1 * math.log(8)
    for wrong in (dict(features=7), dict(features=0), dict(features=True), dict(features=8, scaling="x"),
                  dict(features=8, factor=0.5), dict(features=8, base=0.0), dict(features=8, scaling="blend", factor=2.0, fast_turns=1.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**wrong)


def test_refusals() -> None:
    x, f = torch.randn(2, 3, 1, 8), rotary_frequencies(8)[0]
    with pytest.raises(ValueError, match="requires CUDA"):
        rotary(x, f)
    with pytest.raises(ValueError, match="x must have shape"):
        rotary(x[0], f)
    with pytest.raises(ValueError, match="1 to 4 pairs"):
        rotary(x, rotary_frequencies(10)[0])
    with pytest.raises(TypeError, match="frequencies must use"):
        rotary(x, f.half())
    with pytest.raises(ValueError, match="gradients for frequencies"):
        rotary(x, f.clone().requires_grad_())
    with pytest.raises(ValueError, match="positions must have shape"):
        rotary(x, f, torch.arange(4))
    with pytest.raises(TypeError, match="positions must use"):
        rotary(x, f, torch.arange(3).half())
    with pytest.raises(ValueError, match="gradients for positions"):
        rotary(x, f, torch.arange(3.0).requires_grad_())


SHAPES = [(1, 1, 1, 2, 1), (2, 5, 3, 8, 4), (1, 300, 1, 64, 32), (3, 33, 16, 32, 16), (2, 17, 5, 80, 24), (2, 9, 2, 128, 64),
          (1, 7, 3, 18, 5), (4, 1, 12, 64, 32), (2, 3, 1, 6, 3), (1, 2, 2, 4096, 2048), (5, 129, 7, 40, 20), (1, 2, 3, 12, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_turns_and_gradients(shape, interleaved, dtype) -> None:
    from tests.gpu_util import require_native

    require_native()
    batch, length, heads, dim, pairs = shape
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    x = torch.randn(batch, length, heads, dim, device="cuda", generator=g).to(dtype).requires_grad_()
    dy = torch.randn(batch, length, heads, dim, device="cuda", generator=g).to(dtype)
    f = rotary_frequencies(2 * pairs, device="cuda")[0]
    far = torch.randint(0, 2 ** 22, (batch, length), device="cuda", generator=g)
    kinds = [None, far, far[0].int(), far.float(), far[0].double() / 3, -far]
    for i, positions in enumerate(kinds):
        freq, magnitude = (f.float(), 1.0) if i == 1 else (f, 1.2)
        y = rotary(x, freq, positions, interleaved=interleaved, magnitude=magnitude)
        (dx,) = torch.autograd.grad(y, x, dy)
        for got, source, sign in ((y, x, 1.0), (dx, dy, -1.0)):
            want, size = exact(source, freq, positions, interleaved, magnitude, sign)
            bound = 2.0 ** -21 * size + 1.01 * U[dtype] * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
            assert got.dtype == dtype and got.is_contiguous() and ((got.double() - want).abs() <= bound).all()
            assert torch.equal(got[..., 2 * pairs:], source[..., 2 * pairs:])


@pytest.mark.gpu
def test_views_streams_copies_and_capture() -> None:
    from tests.gpu_util import require_native

    require_native()
    packed = torch.randn(3, 40, 5 * 48 + 24, device="cuda").bfloat16()
    f = rotary_frequencies(32, device="cuda")[0]
    view = packed[..., 24:].unflatten(-1, (5, 48))
    want = rotary(view.contiguous(), f)
    assert torch.equal(rotary(view, f), want)
    assert torch.equal(rotary(view.transpose(1, 2).contiguous().transpose(1, 2), f), want)
    odd = torch.empty(view.numel() + 1, device="cuda", dtype=view.dtype)[1:].view(view.shape).copy_(view)
    assert torch.equal(rotary(odd, f), want)
    assert torch.equal(rotary(view[:1].expand(3, -1, -1, -1), f), want[:1].expand(3, -1, -1, -1))
    kept = torch.full((1, 1, 1, 8), float("nan"), device="cuda")
    assert torch.isnan(rotary(kept, f[:2])).all()
    assert rotary(view[:, :0], f).shape == (3, 0, 5, 48) and rotary(view[:, :, :0], f).shape == (3, 40, 0, 48)
    positions = torch.arange(40, device="cuda")
    x = view.contiguous()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        rotary(x, f, positions)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = rotary(x, f, positions)
    positions += 1000
    graph.replay()
    assert torch.equal(y, rotary(x, f, positions)) and not torch.equal(y, want)


@pytest.mark.gpu
def test_refusals_on_the_gpu() -> None:
    from tests.gpu_util import require_native

    require_native()
    f = rotary_frequencies(8, device="cuda")[0]
    x = torch.randn(1, 2, 1, 9, device="cuda")
    with pytest.raises(ValueError, match="even head width"):
        rotary(x, f)
    with pytest.raises(TypeError, match="supports"):
        rotary(x[..., :8].double(), f)
    with pytest.raises(RuntimeError, match="must be on"):
        rotary(x[..., :8], f.cpu())
    with pytest.raises(RuntimeError, match="supported launch range"):
        rotary(torch.zeros(1, 1, 1, 4100, device="cuda"), rotary_frequencies(4098, device="cuda")[0])
    with pytest.raises(NotImplementedError, match="torch.func"):
        torch.func.grad(lambda t: rotary(t, f).sum())(x[..., :8].contiguous())
