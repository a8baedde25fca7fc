"""Decay attention at its edges: offsets beyond 32 bits, long sequences in parts, padding, unaligned gradients, states
changed under a graph, concurrent captured calls, a thread's first call, and waits that run out."""

from __future__ import annotations

import threading

import pytest
import torch

from lsso_b200.ball.decay import decay_attention, decay_attention_step
from tests.test_decay import U, check, compare, exact, inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def native() -> None:
    from tests.gpu_util import require_native

    require_native()


def test_offsets_beyond_32_bits() -> None:
    """Samples 2^31 elements apart (4 GB), and tokens 2^22 elements apart."""
    b, n, h, d = 2, 200, 2, 32
    far = torch.empty(2 ** 31 + 2 ** 20, device="cuda", dtype=torch.bfloat16)
    apart = torch.empty(n * 2 ** 23, device="cuda", dtype=torch.bfloat16)
    for store, strides in ((far, (2 ** 31, 64, 32, 1)), (apart, (2 ** 22, 2 ** 23, 32, 1))):
        q, k, v, l, _, _ = inputs(b, n, h, d, d, torch.bfloat16)
        views = []
        for i, t in enumerate((q, k, v)):
            view = store.as_strided((b, n, h, d), strides, i * n * 64 if strides[1] == 64 else i * 64)
            view.copy_(t)
            views.append(view.requires_grad_(False))
        want = decay_attention(q, k, v, l)
        assert torch.equal(decay_attention(*views, l), want)
        if strides[1] == 64:  # gradients of far views
            leaves = [t.clone().requires_grad_() for t in (q, k, v)]
            grads = torch.autograd.grad(decay_attention(*leaves, l), leaves, want)
            far_leaves = [t.detach().requires_grad_() for t in views]
            assert all(torch.equal(a, c) for a, c in zip(grads, torch.autograd.grad(decay_attention(*far_leaves, l), far_leaves, want)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_sequences_equal_their_parts(dtype) -> None:
    """70 001 tokens in one call, and in calls of odd lengths from state to state: within the roundings of both."""
    q, k, v, l, s0, valid = inputs(1, 70001, 2, 32, 40, dtype, mask="holes", state=True, seed=8)
    y, last = decay_attention(q, k, v, l, state=s0, valid_mask=valid, return_state=True)
    at, s, parts = 0, s0, []
    for n in (1, 127, 4097, 30000, 20011, 15765):
        piece = [t[:, at:at + n] for t in (q, k, v)]
        part, s = decay_attention(*piece, l, state=s, valid_mask=valid[:, at:at + n], return_state=True)
        parts.append(part)
        at += n
    assert at == 70001
    assert (s - last).norm() <= 2.0 ** -17 * last.norm()
    parts = torch.cat(parts, dim=1).double()
    assert (parts - y.double()).norm() <= 4 * U[dtype] * y.double().norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tokens_of_very_different_sizes(dtype) -> None:
    """Tokens whose values differ by up to 2^8 keep each its own precision: every row within 3 u of its magnitude (the
    definition with absolute values), for decays that leave all but nothing of a chunk's first token at its last."""
    q, k, v, l, _, _ = inputs(2, 400, 6, 64, 64, dtype, decays=[-0.001, -0.03, -0.07, -0.08, -0.13, -0.5])
    g = torch.Generator(device="cuda").manual_seed(3)
    sized = lambda t: (t * 2.0 ** -torch.randint(0, 9, (*t.shape[:2], 1, 1), device="cuda", generator=g)).to(dtype)  # noqa: E731
    leaves = [sized(t).requires_grad_() for t in (q, k, v)]
    dy = sized(torch.randn(v.shape, device="cuda", generator=g))
    y = decay_attention(*leaves, l)
    grads = torch.autograd.grad(y, leaves, dy)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    want, _ = exact(*wide, l, 0.125)
    wants = (want, *torch.autograd.grad(want, wide, dy.double()))
    sizes = [t.detach().abs().requires_grad_() for t in wide]
    size, _ = exact(*sizes, l, 0.125)
    sizes = (size, *torch.autograd.grad(size, sizes, dy.double().abs()))
    for a, b, m in zip((y, *grads), wants, sizes):
        error = (a.double() - b).norm(dim=-1)
        floor = 2.0 ** -25 * 8 if dtype == torch.float16 else 0.0  # a row of 64 results' own smallest steps
        assert (error <= 3 * U[dtype] * m.detach().norm(dim=-1) + floor).all()


@pytest.mark.parametrize("large", ["first", "last"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_tokens_that_nothing_is_left_of(dtype, masked, large) -> None:
    """Strong decays leave nothing of one half of a chunk at its end (in time, and against it), but its tokens' own
    scores remain, here 2^18 times those of the other half: each row within 3 u of its magnitude, as above."""
    q, k, v, l, _, _ = inputs(2, 300, 5, 64, 64, dtype, decays=[-2.0, -4.0, -20.0, -60.0, -100.0])
    g = torch.Generator(device="cuda").manual_seed(4)
    half = torch.arange(300, device="cuda") % 128 < 64
    size = torch.where(half == (large == "first"), 2.0, 2.0 ** -8)[None, :, None, None]
    mask = torch.rand(2, 300, device="cuda", generator=g) < 0.8 if masked else None
    leaves = [(t * size).to(dtype).requires_grad_() for t in (q, k, v)]
    dy = (torch.randn(v.shape, device="cuda", generator=g) * size).to(dtype)
    y = decay_attention(*leaves, l, valid_mask=mask)
    grads = torch.autograd.grad(y, leaves, dy)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    want, _ = exact(*wide, l, 0.125, mask=mask)
    wants = (want, *torch.autograd.grad(want, wide, dy.double()))
    sizes = [t.detach().abs().requires_grad_() for t in wide]
    size, _ = exact(*sizes, l, 0.125, mask=mask)
    sizes = (size, *torch.autograd.grad(size, sizes, dy.double().abs()))
    for a, b, m in zip((y, *grads), wants, sizes):
        error = (a.double() - b).norm(dim=-1)
        floor = 2.0 ** -25 * 8 if dtype == torch.float16 else 0.0  # a row of 64 results' own smallest steps
        assert (error <= 3 * U[dtype] * m.detach().norm(dim=-1) + floor).all()


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("decay", [-0.01, -0.5, -30.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_chunks_of_zeros_and_of_tiny_values(dtype, decay, given) -> None:
    """Every chunk's q, k, v and dy are zero, tiny or ordinary, each for itself: rows within 3 u of their magnitude."""
    q, k, v, l, state, _ = inputs(4, 640, 4, 64, 64, dtype, decays=[decay] * 4, state=given)
    g = torch.Generator(device="cuda").manual_seed(5)
    kinds = torch.tensor([0.0, 2.0 ** -18, 2.0 ** -3, 1.0], device="cuda")

    def sized(t):
        kind = torch.randint(0, 4, (t.shape[0], 5, t.shape[2], 1), device="cuda", generator=g)
        return (t * kinds[kind].repeat_interleave(128, 1)).to(dtype)

    leaves = [sized(t).requires_grad_() for t in (q, k, v)]
    dy = sized(torch.randn(v.shape, device="cuda", generator=g))
    y = decay_attention(*leaves, l, state=state)
    grads = torch.autograd.grad(y, leaves, dy)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    want, _ = exact(*wide, l, 0.125, state)
    wants = (want, *torch.autograd.grad(want, wide, dy.double()))
    sizes = [t.detach().abs().requires_grad_() for t in wide]
    size, _ = exact(*sizes, l, 0.125, None if state is None else state.abs())
    sizes = (size, *torch.autograd.grad(size, sizes, dy.double().abs()))
    for a, b, m in zip((y, *grads), wants, sizes):
        error = (a.double() - b).norm(dim=-1)
        # FP16: a row of 64 results' own smallest steps.  BF16: parts of the sums below 2^-126 (results here reach down to
        # 1e-160) vanish, and the rows' factors, e^(128 |l|) where they are applied after the sums (l = -0.01 here), bring
        # back at most 2^2, with room 2^32: 2^-94, times two values below 2^3, 64 features and
        # 128 tokens, over a row of 64.
        floor = 2.0 ** -25 * 8 if dtype == torch.float16 else 2.0 ** (-94 + 6 + 6 + 7 + 3)
        assert (error <= 3 * U[dtype] * m.detach().norm(dim=-1) + floor).all()


@pytest.mark.parametrize("small", ["q", "k", "v", "dy", "state"])
def test_one_tensor_of_small_values(small) -> None:
    """BF16 values of 1e-12 (a loss's mean over many tokens) under decays of windows down to two tokens."""
    tiny = 2.0 ** -40
    q, k, v, l, state, _ = inputs(2, 300, 6, 64, 64, torch.bfloat16, decays=[-0.03, -0.17, -0.18, -0.3, -0.5, -0.52], state=True)
    g = torch.Generator(device="cuda").manual_seed(6)
    size = lambda name: tiny if small == name else 1.0  # noqa: E731
    leaves = [(t * size(n)).requires_grad_() for n, t in zip("qkv", (q, k, v))]
    state = state * (tiny if small in ("k", "v", "state") else 1.0)
    dy = (torch.randn(v.shape, device="cuda", generator=g) * size("dy")).to(v.dtype)
    y = decay_attention(*leaves, l, state=state)
    grads = torch.autograd.grad(y, leaves, dy)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    want, _ = exact(*wide, l, 0.125, state)
    wants = (want, *torch.autograd.grad(want, wide, dy.double()))
    sizes = [t.detach().abs().requires_grad_() for t in wide]
    magnitude, _ = exact(*sizes, l, 0.125, state.abs())
    magnitudes = (magnitude, *torch.autograd.grad(magnitude, sizes, dy.double().abs()))
    for a, b, m in zip((y, *grads), wants, magnitudes):
        error = (a.double() - b).norm(dim=-1)
        assert (error <= 3 * U[torch.bfloat16] * m.detach().norm(dim=-1) + 2.0 ** -72).all()


@pytest.mark.parametrize("where", ["first", "last"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_small_scores_of_tokens_far_from_their_chunks_end(dtype, where) -> None:
    """The first (or last) 16 tokens of a chunk have queries and keys of 2^-8, the others of one; values are ordinary."""
    q, k, v, l, _, _ = inputs(2, 128, 4, 64, 64, dtype, decays=[-0.02, -0.05, -0.07, -0.076])
    g = torch.Generator(device="cuda").manual_seed(7)
    t = torch.arange(128, device="cuda")
    small = torch.where(t < 16 if where == "first" else t >= 112, 2.0 ** -8, 1.0)[None, :, None, None]
    leaves = [(a * b).to(dtype).requires_grad_() for a, b in ((q, small), (k, small), (v, 1.0))]
    dy = torch.randn(v.shape, device="cuda", generator=g).to(dtype)
    y = decay_attention(*leaves, l)
    grads = torch.autograd.grad(y, leaves, dy)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    want, _ = exact(*wide, l, 0.125)
    wants = (want, *torch.autograd.grad(want, wide, dy.double()))
    sizes = [t.detach().abs().requires_grad_() for t in wide]
    size, _ = exact(*sizes, l, 0.125)
    sizes = (size, *torch.autograd.grad(size, sizes, dy.double().abs()))
    for a, b, m in zip((y, *grads), wants, sizes):
        error = (a.double() - b).norm(dim=-1)
        floor = 2.0 ** -25 * 8 if dtype == torch.float16 else 0.0  # a row of 64 results' own smallest steps
        assert (error <= 3 * U[dtype] * m.detach().norm(dim=-1) + floor).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_padding_at_both_ends(dtype) -> None:
    """Whole chunks of masked tokens before, behind and between valid ones, a single valid token, none."""
    q, k, v, l, s0, _ = inputs(5, 1500, 2, 64, 32, dtype, state=True, seed=6)
    valid = torch.zeros(5, 1500, dtype=torch.bool, device="cuda")
    valid[0, 700:900] = True
    valid[1, 3] = True
    valid[1, 1400:] = True
    valid[2, 1499] = True
    valid[3, :130] = True
    compare(q, k, v, l, s0, valid)
    compare(q, k, v, l, None, valid)


def test_growing_states_and_extreme_scales() -> None:
    """The formula holds for a decay above one, and for scales that are tiny, zero or negative."""
    for rate, scale in ((0.01, None), (0.4, None), (-0.1, 1e-9), (-0.1, -2.0)):
        compare(*inputs(2, 200, 2, 32, 32, torch.bfloat16, state=True, decays=[rate]), scale=scale)
    q, k, v, l, s0, _ = inputs(2, 200, 2, 32, 32, torch.bfloat16, state=True)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, s0)]
    y, last = decay_attention(*leaves[:3], l, state=leaves[3], scale=0.0, return_state=True)
    assert not y.any() and torch.isfinite(last).all()
    grads = torch.autograd.grad((y, last), leaves, (torch.ones_like(y), torch.ones_like(last)))
    want = torch.autograd.grad(exact(*[t.double() for t in leaves[:3]], l, 0.0, leaves[3].double())[1], leaves[1:], torch.ones_like(last).double())
    assert not grads[0].any()
    for a, b, dtype in zip(grads[1:], want, (torch.bfloat16, torch.bfloat16, torch.float32)):
        check(a, b.double(), b.double().abs() + 64 * 8.0, dtype)


def test_gradients_of_the_last_state_may_be_any_view() -> None:
    q, k, v, l, s0, _ = inputs(2, 150, 2, 16, 24, torch.bfloat16, state=True)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, s0)]
    up = torch.randn(2, 2, 16, 24, device="cuda")
    odd = torch.empty(up.numel() + 1, device="cuda")[1:].view(up.shape).copy_(up)
    turned = up.transpose(2, 3).contiguous().transpose(2, 3)
    _, last = decay_attention(*leaves[:3], l, state=leaves[3], return_state=True)
    want = torch.autograd.grad(last, leaves, up, retain_graph=True)
    for view in (odd, turned):
        got = torch.autograd.grad(last, leaves, view, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    shared = torch.autograd.grad(last, leaves, torch.ones(1, device="cuda").expand(up.shape))
    assert all(torch.isfinite(t).all() for t in shared)


def test_a_state_stepped_under_a_graph_is_noticed() -> None:
    q, k, v, l, s0, _ = inputs(1, 10, 2, 16, 16, torch.bfloat16, state=True)
    leaf = q.clone().requires_grad_()
    y = decay_attention(leaf, k, v, l, state=s0)
    with torch.no_grad():
        decay_attention_step(q[:, 0], k[:, 0], v[:, 0], l, s0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), leaf)
    with torch.inference_mode():
        s = torch.zeros_like(s0)
        assert decay_attention_step(q[:, 0], k[:, 0], v[:, 0], l, s).shape == (1, 2, 16)
        decay_attention_step(q[:, 0], k[:, 0], v[:, 0], l, s0)


def test_two_captured_calls_run_at_once() -> None:
    """Two graphs of cut sequences replayed on two streams: neither touches the other's workspace."""
    sides = []
    for seed in (1, 2):
        args = inputs(1, 6000, 2, 64, 64, torch.bfloat16, mask="holes", state=True, seed=seed)
        q, k, v, l, s0, valid = args
        leaves = [t.clone().requires_grad_() for t in (q, k, v, s0)]
        dy = torch.randn_like(v)

        def call(leaves=leaves, l=l, valid=valid, dy=dy):
            y, last = decay_attention(*leaves[:3], l, state=leaves[3], valid_mask=valid, return_state=True)
            return (y, last, *torch.autograd.grad((y, last), leaves, (dy, torch.ones_like(last))))

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            want = [t.clone() for t in call()]
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs = call()
        sides.append((stream, graph, outs, want))
    for _ in range(5):
        for stream, graph, _, _ in sides:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, outs, want in sides:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_first_cuda_call_of_a_thread() -> None:
    q, k, v, l, s0, _ = inputs(2, 100, 2, 32, 32, torch.bfloat16, state=True)
    want = decay_attention(q, k, v, l)
    seen = []

    def call() -> None:
        try:
            seen.append(decay_attention(q, k, v, l))
        except RuntimeError as error:
            seen.append(error)

    torch.cuda.synchronize()
    thread = threading.Thread(target=call)
    thread.start()
    thread.join()
    assert isinstance(seen[0], torch.Tensor), seen[0]
    torch.cuda.synchronize()
    assert torch.equal(seen[0], want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize(("key", "value", "batch", "length"), [(32, 32, 2, 400), (128, 128, 2, 400), (72, 40, 2, 300), (40, 72, 2, 300), (64, 64, 1, 5000)])
def test_waits_that_run_out_end_the_call(key, value, batch, length, dtype) -> None:
    """With a limit of 1 ns waits that would have completed give up: the call ends, the status says so, and the next
    calls are those of before (states carried, so that every product runs; masked, so that every barrier does)."""
    from lsso_b200.ball import _native, cuda

    q, k, v, l, s0, valid = inputs(batch, length, 2, key, value, dtype, mask="holes", state=True, decays=[-0.01, -5.0])
    leaves = [t.clone().requires_grad_() for t in (q, k, v, s0)]
    dy = torch.randn_like(v)

    def call():
        y, last = decay_attention(*leaves[:3], l, state=leaves[3], valid_mask=valid, return_state=True)
        grads = torch.autograd.grad((y, last), leaves, (dy, torch.ones_like(last)))
        torch.cuda.synchronize()
        return (y, last, *grads)

    want = call()
    cuda.check_device_status()
    _native.set_wait_limit_ns(1)
    try:
        call()
        assert cuda.device_status(reset=False) in (0, 1)  # 0: no wait was late
        cuda.device_status(reset=True)
    finally:
        _native.set_wait_limit_ns(0)
    assert all(torch.equal(a, b) for a, b in zip(call(), want))
    cuda.check_device_status()
