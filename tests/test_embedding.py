"""Token embedding and its gradient: exact forward, gradient against 64 bits, refusals.

The forward is one FP32 product rounded once: equal, bit for bit, to the same
product in PyTorch.  A row's gradient is a sum of n FP32-rounded additions:
off by at most ``n 2^-24`` of the sum of magnitudes, times the scale, plus one
rounding of the product (2^-23) and one to the weight's dtype.
"""

from __future__ import annotations

import pytest
import torch

from lsso_b200.ball.embedding import TokenEmbedding, token_embedding, token_embedding_reference

ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _check_step(ids, weight, dy, scale, mask, padding, dtype):
    weight = weight.detach().requires_grad_()
    y = token_embedding(ids, weight, scale=scale, valid_mask=mask, padding_idx=padding, dtype=dtype)
    grad, = torch.autograd.grad(y, weight, dy)
    want = (weight.detach().float()[ids.long().clamp(0, weight.shape[0] - 1)] * scale)
    live = torch.ones_like(ids, dtype=torch.bool) if mask is None else mask
    live = live & (ids >= 0) & (ids < weight.shape[0])
    want = torch.where(live[..., None], want, torch.zeros_like(want)).to(dtype)
    assert y.dtype == dtype and torch.equal(y.detach(), want)
    counted = live if padding is None else live & (ids != padding)
    rows = dy[counted].double()
    at = ids[counted].long()
    zero = torch.zeros(weight.shape, dtype=torch.float64, device="cuda")
    exact = zero.index_add(0, at, rows) * scale
    size = zero.index_add(0, at, rows.abs()) * abs(scale)
    n = torch.bincount(at, minlength=weight.shape[0]).double()[:, None]
    bound = (n * 2.0 ** -24 + 2.0 ** -23) * size + ROUNDOFF[weight.dtype] * exact.abs()
    if weight.dtype == torch.float16:
        bound = bound + 2.0 ** -24
    assert grad.dtype == weight.dtype
    assert ((grad.double() - exact).abs() <= 1.01 * bound).all()
    assert torch.count_nonzero(grad[n.squeeze(1) == 0]) == 0
    y = token_embedding(ids, weight, scale=scale, valid_mask=mask, padding_idx=padding, dtype=dtype)
    assert torch.equal(torch.autograd.grad(y, weight, dy)[0], grad)  # the same bits again


@pytest.mark.gpu
@pytest.mark.parametrize(("tokens", "vocab", "dim"), [
    (1, 1, 1), (1, 50021, 64), (2, 2, 8), (31, 5, 12), (32, 1, 96), (33, 7, 100), (64, 3, 256), (65, 1000, 36),
    (2047, 300, 33), (2048, 511, 128), (2049, 512, 130), (5000, 8, 128), (4096, 100003, 24), (20000, 1, 40),
    (70001, 70000, 16), (1500000, 17, 8),
])
@pytest.mark.parametrize(("weight_dtype", "dtype"), [
    (torch.float32, torch.bfloat16), (torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
    (torch.float16, torch.float32)])
def test_step_matches_64_bits(tokens, vocab, dim, weight_dtype, dtype) -> None:
    from tests.gpu_util import require_native

    require_native()
    gen = torch.Generator(device="cuda").manual_seed(tokens + vocab + dim)
    ids = torch.randint(0, vocab, (tokens,), device="cuda", generator=gen)
    weight = torch.randn(vocab, dim, device="cuda", generator=gen).to(weight_dtype)
    dy = torch.randn(tokens, dim, device="cuda", generator=gen).to(dtype)
    _check_step(ids, weight, dy, 1.0, None, None, dtype)
    mask = torch.rand(tokens, device="cuda", generator=gen) > 0.4
    _check_step(ids, weight, dy, dim ** 0.5, mask, vocab // 2, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("pattern", ["one", "two", "runs", "last", "none", "edge"])
def test_rows_that_cross_or_fill_chunks(pattern) -> None:
    from tests.gpu_util import require_native

    require_native()
    gen = torch.Generator(device="cuda").manual_seed(3)
    tokens, vocab, dim = 4097, 600, 72
    ids = torch.randint(0, vocab, (tokens,), device="cuda", generator=gen)
    mask = None
    if pattern == "one":
        ids.fill_(599)
    elif pattern == "two":
        ids = torch.where(torch.arange(tokens, device="cuda") % 2 == 0, 0, 511)
    elif pattern == "runs":
        ids = torch.arange(tokens, device="cuda") // 32 % vocab  # every row fills one chunk exactly
    elif pattern == "last":
        ids[:] = 5
        ids[-1] = 599
    elif pattern == "none":
        mask = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    else:
        mask = torch.arange(tokens, device="cuda") < 64  # chunks end where the tokens without a gradient begin
        ids = torch.where(mask, 1, 2)
    weight = torch.randn(vocab, dim, device="cuda", generator=gen)
    dy = torch.randn(tokens, dim, device="cuda", generator=gen)
    _check_step(ids, weight, dy, 0.5, mask, None, torch.float32)


@pytest.mark.gpu
def test_masked_tokens_are_not_looked_at() -> None:
    """Masked ids may lie outside the table, and masked upstream rows may hold anything."""
    from lsso_b200.ball import cuda
    from tests.gpu_util import require_native

    require_native()
    cuda.device_status(reset=True)
    ids = torch.tensor([[3, 1, -7], [10 ** 12, 2, 2]], device="cuda")
    mask = torch.tensor([[True, True, False], [False, True, True]], device="cuda")
    weight = torch.randn(4, 16, device="cuda", requires_grad=True)
    dy = torch.randn(2, 3, 16, device="cuda")
    dy[~mask] = float("nan")
    y = token_embedding(ids, weight, valid_mask=mask, scale=2.0)
    grad, = torch.autograd.grad(y, weight, dy)
    assert torch.count_nonzero(y[~mask]) == 0 and torch.equal(y[mask], 2 * weight.detach()[ids[mask]])
    torch.testing.assert_close(grad[2], 2 * (dy[1, 1] + dy[1, 2]))
    assert torch.equal(grad[3], 2 * dy[0, 0]) and torch.count_nonzero(grad[0]) == 0
    assert cuda.device_status(reset=True) == 0


@pytest.mark.gpu
def test_an_id_outside_the_table_is_reported() -> None:
    from lsso_b200.ball import cuda
    from tests.gpu_util import require_native

    require_native()
    cuda.device_status(reset=True)
    for bad in (4, -1, 2 ** 40):
        ids = torch.tensor([0, bad, 3], device="cuda")
        weight = torch.randn(4, 16, device="cuda", requires_grad=True)
        y = token_embedding(ids, weight)
        assert torch.count_nonzero(y[1]) == 0 and torch.equal(y[2], weight[3])
        with pytest.raises(RuntimeError, match="outside the embedding's vocabulary"):
            cuda.check_device_status()
        grad, = torch.autograd.grad(y.sum(), weight)
        assert torch.equal(grad[0], torch.ones(16, device="cuda")) and torch.count_nonzero(grad[1:3]) == 0
        assert cuda.device_status(reset=True) == 3


@pytest.mark.gpu
def test_layouts_and_types_of_ids() -> None:
    from tests.gpu_util import require_native

    require_native()
    gen = torch.Generator(device="cuda").manual_seed(9)
    ids = torch.randint(0, 300, (40, 50), device="cuda", generator=gen)
    weight = torch.randn(300, 64, device="cuda", generator=gen)
    want = weight[ids]
    assert torch.equal(token_embedding(ids.int(), weight), want)
    assert torch.equal(token_embedding(ids.T, weight), want.transpose(0, 1))  # strided ids
    off = torch.empty(300 * 64 + 1, device="cuda")[1:].view(300, 64)
    off.copy_(weight)
    assert torch.equal(token_embedding(ids, off), want)  # table off the 16-byte boundary
    leaf = weight.clone().requires_grad_()
    dy = torch.randn(40, 50, 65, device="cuda", generator=gen)[..., 1:]  # strided upstream gradient
    grads = [torch.autograd.grad(token_embedding(i, leaf), leaf, dy)[0] for i in (ids, ids.int())]
    assert torch.equal(*grads)
    torch.testing.assert_close(grads[0], torch.zeros_like(weight).index_add_(0, ids.flatten(), dy.reshape(-1, 64)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = torch.autograd.grad(token_embedding(ids, leaf), leaf, dy)[0]
    side.synchronize()
    assert torch.equal(other, grads[0])


@pytest.mark.gpu
def test_no_tokens_and_refusals() -> None:
    from tests.gpu_util import require_native

    require_native()
    weight = torch.randn(10, 16, device="cuda", requires_grad=True)
    y = token_embedding(torch.empty(0, 5, dtype=torch.int64, device="cuda"), weight)
    assert y.shape == (0, 5, 16)
    assert torch.count_nonzero(torch.autograd.grad(y.sum(), weight)[0]) == 0
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError, match="supports"):
        token_embedding(ids, weight.double())
    with pytest.raises(TypeError, match="the output uses"):
        token_embedding(ids, weight, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="contiguous weight"):
        token_embedding(ids, weight[:, ::2])
    with pytest.raises(RuntimeError, match="ids must be on"):
        token_embedding(ids.cpu(), weight)
    from lsso_b200.ball import _native

    lib = _native.library()
    assert lib.lib.lsso_embedding_backward_workspace_size(0, 4, 4) == 0 and "positive" in lib.last_error()
    size = lib.lib.lsso_embedding_backward_workspace_size(3, 10, 16)
    out = torch.empty(10, 16, device="cuda")
    args = (ids.data_ptr(), 1, None, 3, out.data_ptr(), 2, 10, 16)
    assert lib.lib.lsso_embedding_backward(*args, 10, 1.0, out.data_ptr(), 2, out.data_ptr(), size, None) == 1
    assert "padding" in lib.last_error()
    assert lib.lib.lsso_embedding_backward(*args, -1, 1.0, out.data_ptr(), 2, out.data_ptr(), size - 1, None) == 4


def test_cpu_refusals_and_reference() -> None:
    weight = torch.randn(10, 16, dtype=torch.float64)
    ids = torch.tensor([[1, 2], [9, 3]])
    with pytest.raises(TypeError, match="int64 or torch.int32"):
        token_embedding(ids.float(), weight)
    with pytest.raises(ValueError, match="CUDA"):
        token_embedding(ids, weight)
    with pytest.raises(ValueError, match="padding_idx"):
        token_embedding(ids, weight, padding_idx=10)
    with pytest.raises(ValueError, match="valid_mask"):
        token_embedding(ids, weight, valid_mask=torch.ones(2, dtype=torch.bool))
    with pytest.raises(TypeError, match="valid_mask"):
        token_embedding(ids, weight, valid_mask=torch.ones(2, 2))
    with pytest.raises(ValueError, match="weight must have shape"):
        token_embedding(ids, weight[0])
    mask = torch.tensor([[True, False], [True, True]])
    layer = TokenEmbedding(10, 16, scale=4.0, padding_idx=9)
    y = layer(ids, mask, dtype=torch.bfloat16)
    assert y.dtype == torch.bfloat16 and torch.count_nonzero(y[0, 1]) == 0
    torch.testing.assert_close(y[0, 0], (layer.weight[1] * 4).to(torch.bfloat16))
    y.float().sum().backward()
    assert torch.count_nonzero(layer.weight.grad[9]) == 0 and torch.count_nonzero(layer.weight.grad[2]) == 0
    assert torch.equal(token_embedding_reference(ids, weight), weight[ids])
