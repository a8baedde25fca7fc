"""Decay attention and its single-token step against the definition in 64 bits, gradients, states, masks, refusals.

Tolerances, with u half a step of the type (BF16 2^-8, FP16 2^-11) and M the same output with every input replaced by
its absolute value.  A pair of tokens meets through a score rounded to the type (u), or through a key weight and a
state rounded to it (2 u), so that an output is off by at most ``2 u M`` and its own rounding ``u |y|``; FP32 sums of up
to 128 + 128 terms, chunks and exponentials add ``2^-15 M``.  FP16 key weights below 2^-14 are off by 2^-25 each.  For
random signs the four roundings are independent, ``u / sqrt 3`` each at most, so the relative L2 error stays below
``4^(1/2) / 3^(1/2) u < 1.2 u``; 2 u is asked.  States are FP32 sums: ``2^-15 M`` and 2^-18 in L2.
"""

from __future__ import annotations

import math

import pytest
import torch

from lsso_b200.ball.decay import (decay_attention, decay_attention_reference, decay_attention_step,
                                  decay_attention_step_reference)

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def exact(q, k, v, log_decay, scale, state=None, mask=None):
    """(y, last state) by all pairs of tokens, differentiable, in 64 bits."""
    q, k, v = q.double(), k.double(), v.double()
    batch, length, heads, _ = q.shape
    if mask is None:
        mask = torch.ones(batch, length, dtype=torch.bool, device=q.device)
    rank = mask.double().cumsum(-1)
    live = mask[..., None, None]
    q, k, v = (torch.where(live, t, 0.0) for t in (q, k, v))
    rate = log_decay.double().clamp_min(-1e4)[None, :, None]
    apart = (rank[:, None, :, None] - rank[:, None, None, :]).clamp_min(0)
    pairs = torch.ones(length, length, dtype=torch.bool, device=q.device).tril() & mask[:, None, None, :]
    weight = torch.where(pairs, torch.exp(rate[..., None] * apart), 0.0)
    y = torch.einsum("bhij,bjhv->bihv", torch.einsum("bihk,bjhk->bhij", q, k) * weight, v)
    count = rank[:, None, -1:]
    last = torch.einsum("bjhk,bhj,bjhv->bhkv", k, torch.exp(rate * (count - rank[:, None])), v)
    if state is not None:
        state = state.double()
        y = y + torch.einsum("bihk,bhi,bhkv->bihv", q, torch.exp(rate * rank[:, None]), state)
        last = last + state * torch.exp(rate * count)[..., None]
    return torch.where(live, y * scale, 0.0), last


def inputs(batch, length, heads, key, value, dtype, *, mask="none", state=False, decays="spread", seed=0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    new = lambda *shape: torch.randn(*shape, device=device, generator=g)  # noqa: E731
    q, k = new(batch, length, heads, key).to(dtype), new(batch, length, heads, key).to(dtype)
    v = new(batch, length, heads, value).to(dtype)
    if decays == "spread":  # windows of 2 to 2^11 tokens
        log_decay = torch.log1p(-2.0 ** -(1 + 10 * torch.arange(heads, device=device) / max(1, heads - 1)))
    else:
        log_decay = torch.tensor(decays, device=device)[torch.arange(heads, device=device) % len(decays)]
    s0 = 3 * new(batch, heads, key, value) if state else None
    valid = None
    if mask == "prefix":
        lengths = torch.randint(0, length + 1, (batch, 1), device=device, generator=g)
        lengths[0] = 0
        valid = torch.arange(length, device=device) < lengths
    elif mask == "holes":
        valid = torch.rand(batch, length, device=device, generator=g) < 0.6
    elif mask == "suffix":
        valid = torch.arange(length, device=device) >= torch.randint(0, length, (batch, 1), device=device, generator=g)
    return q, k, v, log_decay, s0, valid


# ---------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("length", [0, 1, 63, 64, 65, 200])
@pytest.mark.parametrize(("mask", "state"), [("none", False), ("holes", True), ("prefix", True)])
def test_reference_follows_the_definition(length, mask, state) -> None:
    q, k, v, l, s0, valid = inputs(3, length, 2, 6, 5, torch.float64, mask=mask, state=state, decays=[-0.02, -math.inf], device="cpu") \
        if length else inputs(3, 0, 2, 6, 5, torch.float64, state=state, device="cpu")
    leaves = [t.double().requires_grad_() for t in (q, k, v)] + ([s0.double().requires_grad_()] if state else [])
    given = leaves[3] if state else None
    y, last = decay_attention_reference(*leaves[:3], l, state=given, valid_mask=valid, return_state=True, scale=0.3)
    if not length:
        assert y.shape == (3, 0, 2, 5) and torch.equal(last, torch.zeros_like(last) if given is None else given)
        return
    want, want_last = exact(*leaves[:3], l, 0.3, given, valid)
    assert torch.allclose(y, want, rtol=1e-10, atol=1e-10) and torch.allclose(last, want_last, rtol=1e-10, atol=1e-10)
    up = torch.randn_like(want), torch.randn_like(want_last)
    for a, b in zip(torch.autograd.grad((y, last), leaves, up), torch.autograd.grad((want, want_last), leaves, up)):
        assert torch.allclose(a, b, rtol=1e-9, atol=1e-9)


def test_reference_gradients_against_differences() -> None:
    q, k, v, l, s0, valid = inputs(2, 5, 2, 3, 4, torch.float64, mask="holes", state=True, decays=[-0.3, -0.05], device="cpu")
    leaves = [t.double().requires_grad_() for t in (q, k, v, l, s0)]
    torch.autograd.gradcheck(lambda q, k, v, l, s: decay_attention_reference(q, k, v, l, state=s, valid_mask=valid, return_state=True), leaves)


def test_recurrence_of_single_steps_is_the_sequence() -> None:
    q, k, v, l, s0, valid = inputs(3, 9, 2, 4, 6, torch.float64, mask="holes", state=True, device="cpu")
    s0 = s0.double()
    y, last = decay_attention_reference(q, k, v, l, state=s0, valid_mask=valid, return_state=True)
    s = s0.clone()
    for t in range(9):
        row = decay_attention_step_reference(q[:, t], k[:, t], v[:, t], l, s, valid_mask=valid[:, t])
        assert torch.allclose(row, y[:, t], rtol=1e-12, atol=1e-12)
    assert torch.allclose(s, last, rtol=1e-12, atol=1e-12)


def test_refusals() -> None:
    q, k, v, l, s0, _ = inputs(2, 3, 2, 8, 16, torch.bfloat16, state=True, device="cpu")
    run = decay_attention
    with pytest.raises(ValueError, match="requires CUDA"):
        run(q, k, v, l)
    with pytest.raises(ValueError, match="q must have shape"):
        run(q[0], k, v, l)
    with pytest.raises(ValueError, match="k must have q's shape"):
        run(q, k[:, :2], v, l)
    with pytest.raises(ValueError, match="v must have shape"):
        run(q, k, v[:, :, :1], l)
    with pytest.raises(TypeError, match="one dtype"):
        run(q, k, v.half(), l)
    with pytest.raises(ValueError, match="log_decay must have shape"):
        run(q, k, v, l[:1])
    with pytest.raises(TypeError, match="floating-point"):
        run(q, k, v, l.long())
    with pytest.raises(ValueError, match="state must have shape"):
        run(q, k, v, l, state=s0[:1])
    with pytest.raises(ValueError, match="valid_mask must have shape"):
        run(q, k, v, l, valid_mask=torch.ones(2, 4, dtype=torch.bool))
    with pytest.raises(TypeError, match="torch.bool"):
        run(q, k, v, l, valid_mask=torch.ones(2, 3))
    with pytest.raises(ValueError, match="requires CUDA"):
        decay_attention_step(q[:, 0], k[:, 0], v[:, 0], l, s0)
    with pytest.raises(ValueError, match="q must have shape"):
        decay_attention_step(q, k, v, l, s0)


# ---------------------------------------------------------------------------- GPU
def check(got, want, magnitude, dtype, extra=0.0) -> None:
    """``got`` within the bound above of ``want``; ``magnitude`` is M."""
    got, want = got.detach().double(), want.detach()
    assert got.shape == want.shape and torch.isfinite(got).all()
    if dtype == torch.float32:
        bound, most = 2.0 ** -15 * magnitude, 2.0 ** -18
    else:
        u = U[dtype]
        bound, most = 1.02 * ((2 * u + 2.0 ** -15) * magnitude + u * want.abs()) + extra, 2 * u
    error = (got - want).abs()
    assert (error <= bound + 1e-30).all(), f"largest error over its bound {(error / (bound + 1e-30)).max().item():.3g}"
    if want.numel() > 256 and want.norm() > 0:
        assert error.norm() <= most * want.norm(), f"L2 {(error.norm() / want.norm()).item():.3g}, asked {most:.3g}"


def compare(q, k, v, l, s0, valid, *, scale=None, seed=9) -> None:
    """Outputs and gradients, from and to states where there is one."""
    dtype, key = q.dtype, q.shape[-1]
    scale = key ** -0.5 if scale is None else scale
    g = torch.Generator(device=q.device).manual_seed(seed)
    dy = torch.randn(v.shape, device=q.device, generator=g).to(dtype)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)] + ([s0.clone().requires_grad_()] if s0 is not None else [])
    given = leaves[3] if s0 is not None else None
    carried = s0 is not None
    with torch.no_grad():
        plain = decay_attention(*leaves[:3], l, scale=scale, state=given, valid_mask=valid, return_state=True)
    y, last = decay_attention(*leaves[:3], l, scale=scale, state=given, valid_mask=valid, return_state=True)
    assert torch.equal(y, plain[0]) and torch.equal(last, plain[1])
    dlast = torch.randn(last.shape, device=q.device, generator=g)
    grads = torch.autograd.grad((y, last) if carried else (y,), leaves, (dy, dlast) if carried else (dy,))
    wide = [t.detach().double().requires_grad_() for t in leaves]
    sides = []
    for sign in (False, True):
        x = [t.detach().abs().requires_grad_() if sign else t for t in wide]
        w, wl = exact(*x[:3], l, abs(scale) if sign else scale, x[3] if carried else None, valid)
        up = [t.double().abs() if sign else t.double() for t in ((dy, dlast) if carried else (dy,))]
        sides.append((w, wl, torch.autograd.grad((w, wl) if carried else (w,), x, up)))
    (w, wl, wg), (m, ml, mg) = sides
    # FP16 weights below 2^-14: 2^-25 for each of a chunk's 128 tokens, times the other two factors
    extra = 0.0
    if dtype == torch.float16:
        top = max(t.detach().abs().max().item() for t in (q, k, v, dy)) ** 2
        extra = 2.0 ** -25 * 128 * max(key, v.shape[-1]) * top * max(scale, 1.0) + 2.0 ** -25
    check(y, w, m, dtype, extra)
    check(last, wl, ml, torch.float32)
    for a, b, c in zip(grads[:3], wg, mg):
        check(a, b, c, dtype, extra)
        assert a.dtype == dtype
    if carried:
        check(grads[3], wg[3], mg[3], torch.float32)
    if valid is not None:
        for t in (y, *grads[:3]):
            assert not t[~valid].any()


WIDTHS = [(8, 8), (16, 24), (32, 32), (64, 64), (40, 72), (72, 40), (128, 128), (128, 16), (8, 128), (96, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize(("key", "value"), WIDTHS)
@pytest.mark.parametrize("length", [1, 127, 130, 300])
def test_sequences_of_every_width(key, value, length, dtype) -> None:
    from tests.gpu_util import require_native

    require_native()
    compare(*inputs(2, length, 3, key, value, dtype, seed=length + key))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("length", [1, 2, 33, 128, 129, 257, 1000])
@pytest.mark.parametrize("mask", ["none", "prefix", "holes", "suffix"])
@pytest.mark.parametrize("state", [False, True])
def test_masks_and_states(length, mask, state, dtype) -> None:
    from tests.gpu_util import require_native

    require_native()
    compare(*inputs(3, length, 2, 32, 48, dtype, mask=mask, state=state, seed=length))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize(("key", "value"), [(64, 64), (128, 128), (72, 40), (24, 104)])
def test_states_of_every_kernel_width(key, value, dtype) -> None:
    from tests.gpu_util import require_native

    require_native()
    compare(*inputs(2, 391, 3, key, value, dtype, mask="holes", state=True, seed=3))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decays_from_none_to_all(dtype) -> None:
    """No decay at all, the smallest, strong ones whose powers leave FP32, and a token that sees itself alone."""
    from tests.gpu_util import require_native

    require_native()
    decays = [0.0, -1e-6, -0.7, -3.0, -30.0, -200.0, -2e4, -math.inf]
    for mask in ("none", "holes"):
        compare(*inputs(2, 290, 8, 32, 32, dtype, state=True, mask=mask, decays=decays, seed=1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize(("batch", "heads", "length"), [(1, 1, 5000), (1, 3, 3001), (2, 2, 2304)])
@pytest.mark.parametrize(("mask", "state"), [("none", False), ("holes", True)])
def test_long_sequences_of_few_heads(batch, heads, length, mask, state, dtype) -> None:
    from tests.gpu_util import require_native

    require_native()
    compare(*inputs(batch, length, heads, 32, 24, dtype, mask=mask, state=state, seed=5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize(("size", "up"), [(1.0, 2.0 ** -12), (2.0 ** -9, 1.0), (64.0, 64.0)])
def test_small_and_large_values(size, up, dtype) -> None:
    """Scores and states far from one keep their precision, in FP16 beyond its range too (outputs stay within it)."""
    from tests.gpu_util import require_native

    require_native()
    q, k, v, l, _, _ = inputs(2, 300, 3, 64, 64, dtype, seed=2)
    q, k, v = q * size, k * size, v / size
    dy = (torch.randn(v.shape, device="cuda") * up / size).to(dtype)
    scale = 2.0 ** -6 / size / size
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    y = decay_attention(*leaves, l, scale=scale)
    grads = torch.autograd.grad(y, leaves, dy)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    want, _ = exact(*wide, l, scale)
    for a, b in zip((y, *grads), (want, *torch.autograd.grad(want, wide, dy.double()))):
        if b.abs().max() > 0.9 * torch.finfo(dtype).max:  # beyond the type: dq of the second case is dy v k 2^12, 2^9 2^9 2^-9 2^12
            continue
        # values below 2^-14 have FP16's smallest step of 2^-24
        allowed = 2 * U[dtype] * b.norm() + (2.0 ** -25 * b.numel() ** 0.5 if dtype == torch.float16 else 0.0)
        assert (a.double() - b).norm() <= allowed


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("filler", [float("nan"), float("inf"), -float("inf")])
def test_masked_tokens_may_hold_anything(filler, dtype) -> None:
    from tests.gpu_util import require_native

    require_native()
    q, k, v, l, s0, valid = inputs(3, 333, 2, 40, 64, dtype, mask="holes", state=True)
    dy = torch.randn(v.shape, device="cuda").to(dtype)
    results = []
    for fill in (0.0, filler):
        leaves = [torch.where(valid[..., None, None], t, fill).to(dtype).requires_grad_() for t in (q, k, v)] + [s0.clone().requires_grad_()]
        y, last = decay_attention(*leaves[:3], l, state=leaves[3], valid_mask=valid, return_state=True)
        up = torch.where(valid[..., None, None], dy, fill).to(dtype)
        results.append((y, last, *torch.autograd.grad((y, last), leaves, (up, torch.ones_like(last)))))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_views_of_a_packed_projection_are_read_in_place() -> None:
    from tests.gpu_util import require_native

    require_native()
    b, n, h, dk, dv = 2, 261, 3, 40, 72
    packed = torch.randn(b, n, h * (2 * dk + dv), device="cuda").bfloat16().requires_grad_()
    q, k, v = packed.split((h * dk, h * dk, h * dv), dim=-1)
    views = [t.unflatten(-1, (h, -1)) for t in (q, k, v)]
    l = torch.tensor([-0.1, -0.01, -0.001], device="cuda")
    copies = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in views]
    dy = torch.randn(b, n, h, dv, device="cuda").bfloat16()
    y, want = decay_attention(*views, l), decay_attention(*copies, l)
    assert torch.equal(y, want)
    (grad,) = torch.autograd.grad(y, packed, dy)
    grads = torch.autograd.grad(want, copies, dy)
    assert torch.equal(grad, torch.cat([t.flatten(2) for t in grads], dim=-1))
    # heads before tokens, an odd offset, a broadcast sample: read in place or copied, the values are the same
    moved = [t.detach().transpose(1, 2).contiguous().transpose(1, 2) for t in copies]
    odd = [torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)[1:].view(t.shape).copy_(t.detach()) for t in copies]
    wide = [t.detach()[:1].expand(b, -1, -1, -1) for t in copies]
    assert torch.equal(decay_attention(*moved, l), want) and torch.equal(decay_attention(*odd, l), want)
    assert torch.equal(decay_attention(*wide, l), want[:1].expand(b, -1, -1, -1))
    # an upstream gradient that is broadcast, and one of the last state alone
    y, last = decay_attention(*copies, l, return_state=True)
    a = torch.autograd.grad(y.sum(), copies, retain_graph=True)
    assert all(torch.equal(s, t) for s, t in zip(a, torch.autograd.grad(y, copies, torch.ones_like(y), retain_graph=True)))
    dq, dk_, dv_ = torch.autograd.grad(last, copies, torch.ones_like(last))
    assert not dq.any() and dk_.any() and dv_.any()


@pytest.mark.gpu
def test_other_streams_empty_inputs_and_two_calls_at_once() -> None:
    from tests.gpu_util import require_native

    require_native()
    q, k, v, l, s0, valid = inputs(1, 2500, 2, 64, 64, torch.bfloat16, mask="holes", state=True)
    want = decay_attention(q, k, v, l, state=s0, valid_mask=valid, return_state=True)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(decay_attention(q, k, v, l, state=s0, valid_mask=valid, return_state=True))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for pair in got for a, b in zip(pair, want))
    y, last = decay_attention(q[:, :0], k[:, :0], v[:, :0], l, state=s0, return_state=True)
    assert y.shape == (1, 0, 2, 64) and torch.equal(last, s0) and last.data_ptr() != s0.data_ptr()
    y, last = decay_attention(q[:0], k[:0], v[:0], l, return_state=True)
    assert y.shape == (0, 2500, 2, 64) and last.shape == (0, 2, 64, 64)
    leaf = q[:, :0].clone().requires_grad_()
    s = s0.clone().requires_grad_()
    y, last = decay_attention(leaf, k[:, :0], v[:, :0], l, state=s, return_state=True)
    assert torch.equal(torch.autograd.grad(last, s, s0)[0], s0)


@pytest.mark.gpu
@pytest.mark.parametrize(("batch", "length", "heads"), [(2, 300, 4), (1, 3000, 2)])
def test_captured_calls_replay(batch, length, heads) -> None:
    from tests.gpu_util import require_native

    require_native()
    q, k, v, l, s0, valid = inputs(batch, length, heads, 32, 64, torch.float16, mask="holes", state=True)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, s0)]
    dy, dlast = torch.randn_like(v), torch.randn_like(s0)

    def step():
        y, last = decay_attention(*leaves[:3], l, state=leaves[3], valid_mask=valid, return_state=True)
        return (y, last, *torch.autograd.grad((y, last), leaves, (dy, dlast)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (1, 2):
        fresh = inputs(batch, length, heads, 32, 64, torch.float16, mask="holes", state=True, seed=seed)
        with torch.no_grad():
            for leaf, t in zip(leaves, (*fresh[:3], fresh[4])):
                leaf.copy_(t)
            valid.copy_(fresh[5])
        graph.replay()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize(("batch", "heads", "key", "value"), [(1, 1, 8, 8), (1, 8, 32, 32), (5, 3, 40, 72), (3, 2, 128, 128), (2, 2, 24, 120), (4, 2, 128, 8)])
@pytest.mark.parametrize("masked", [False, True])
def test_single_step(batch, heads, key, value, masked, dtype) -> None:
    """The state within three FP32 roundings; y within those of its sum of ``key`` products and its own."""
    from tests.gpu_util import require_native

    require_native()
    q, k, v, l, s0, _ = inputs(batch, 1, heads, key, value, dtype, state=True, seed=key)
    q, k, v = q[:, 0], k[:, 0], v[:, 0]
    valid = torch.arange(batch, device="cuda") % 2 == 1 if masked else None
    wide = s0.double().clone()
    want = decay_attention_step_reference(q, k, v, l, wide, valid_mask=valid)
    y64 = torch.einsum("bhk,bhkv->bhv", q.double(), wide) * key ** -0.5
    size = torch.einsum("bhk,bhkv->bhv", q.double().abs(), wide.abs()) * key ** -0.5
    apart, s = torch.full_like(s0, 7.0), s0.clone()
    y = decay_attention_step(q, k, v, l, s, valid_mask=valid, new_state=apart)
    assert torch.equal(s, s0)
    assert torch.equal(decay_attention_step(q, k, v, l, s, valid_mask=valid), y) and torch.equal(s, apart)
    kv = (k.double()[..., None] * v.double()[..., None, :]).abs()
    assert ((s.double() - wide).abs() <= 2.0 ** -21 * (s0.double().abs() + kv)).all()
    live = torch.ones(batch, dtype=torch.bool, device="cuda") if valid is None else valid
    error = (y.double() - y64).abs()[live]
    assert (error <= ((key + 8) * 2.0 ** -23 * size + U[dtype] * y64.abs())[live] + (2.0 ** -25 if dtype == torch.float16 else 0)).all()
    assert y.dtype == dtype and want.shape == y.shape and not y[~live].any() and torch.equal(s[~live], s0[~live])


@pytest.mark.gpu
def test_prompt_then_single_steps() -> None:
    """A prompt and steps after it give what the whole sequence gives."""
    from tests.gpu_util import require_native

    require_native()
    q, k, v, l, _, _ = inputs(3, 150, 4, 32, 40, torch.bfloat16, seed=4)
    whole, end = decay_attention(q, k, v, l, return_state=True)
    _, s = decay_attention(q[:, :140], k[:, :140], v[:, :140], l, return_state=True)
    rows = [decay_attention_step(q[:, t], k[:, t], v[:, t], l, s) for t in range(140, 150)]
    assert (s - end).norm() <= 2.0 ** -17 * end.norm()
    rows, want = torch.stack(rows, dim=1).double(), exact(q, k, v, l, 32 ** -0.5)[0][:, 140:]
    assert (rows - want).norm() <= 1.0 * U[torch.bfloat16] * want.norm()
    assert (whole[:, 140:].double() - want).norm() <= 2 * U[torch.bfloat16] * want.norm()


@pytest.mark.gpu
def test_refusals_on_the_gpu() -> None:
    from tests.gpu_util import require_native

    require_native()
    q, k, v, l, s0, _ = inputs(2, 3, 2, 16, 8, torch.bfloat16, state=True)
    with pytest.raises(TypeError, match="supports"):
        decay_attention(q.float(), k.float(), v.float(), l)
    with pytest.raises(ValueError, match="multiples of 8"):
        decay_attention(q[..., :12], k[..., :12], v, l)
    with pytest.raises(ValueError, match="multiples of 8"):
        wide = torch.zeros(2, 3, 2, 136, device="cuda", dtype=torch.bfloat16)
        decay_attention(q, k, wide, l)
    with pytest.raises(TypeError, match="log_decay"):
        decay_attention(q, k, v, l.double())
    with pytest.raises(ValueError, match="gradient of log_decay"):
        decay_attention(q, k, v, l.clone().requires_grad_())
    with pytest.raises(TypeError, match="state must use"):
        decay_attention(q, k, v, l, state=s0.bfloat16())
    with pytest.raises(RuntimeError, match="must be on"):
        decay_attention(q, k, v, l.cpu())
    rows = q[:, 0], k[:, 0], v[:, 0]
    with pytest.raises(RuntimeError, match="contiguous state"):
        decay_attention_step(*rows, l, s0.transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(ValueError, match="new_state must be"):
        decay_attention_step(*rows, l, s0, new_state=s0[:1])
    with pytest.raises(ValueError, match="no gradient"):
        decay_attention_step(rows[0].clone().requires_grad_(), *rows[1:], l, s0)
    with pytest.raises(RuntimeError, match="overlaps"):
        pool = torch.zeros(3, 2, 16, 8, device="cuda")
        decay_attention_step(*rows, l, pool[:2], new_state=pool[1:])
    with pytest.raises(RuntimeError):  # a second derivative
        leaf = q.clone().requires_grad_()
        (grad,) = torch.autograd.grad(decay_attention(leaf, k, v, l).sum(), leaf, create_graph=True)
        torch.autograd.grad(grad.sum(), leaf)
    with pytest.raises(NotImplementedError, match="torch.func"):
        torch.func.grad(lambda t: decay_attention(t, k, v, l).float().sum())(q)
