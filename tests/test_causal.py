"""The causal mixer and the shell with it: composition, causality, continued sequences, the CUDA path, a captured step.

The CUDA path is compared with the FP32 reference path by relative L2, at 1e-2
per layer (BF16 operands and activations, as for the LSSO layers) or 1.25x the
error of the reference path's own BF16 run.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from lsso import LSSOConfig
from lsso_b200.ball.causal import CausalMixer
from lsso_b200.ball.decay import decay_attention_reference
from lsso_b200.ball.rotary import rotary_reference
from lsso_b200.ball.shell import SequenceShell

OPTIONS = dict(depth=2, vocab=11, gated="silu", hidden=40, embedding_scale=4.0, mixer="causal", mixer_options=dict(windows=(4.0, 64.0)))


def _batch(device="cpu", batch=3, length=13):
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 11, (batch, length), generator=gen).to(device)
    mask = torch.ones(batch, length, dtype=torch.bool, device=device)
    mask[1, length * 2 // 3:] = False
    mask[2] = False
    return ids, mask


def test_mixer_is_the_composition_of_its_operators() -> None:
    torch.manual_seed(0)
    mixer = CausalMixer(LSSOConfig(24, 3, 4, bias=True), windows=(2.0, 32.0), rotary=dict(base=100.0)).double()
    assert mixer.log_decay.dtype == torch.float32 and mixer.frequencies.dtype == torch.float64
    assert torch.allclose(mixer.log_decay.exp(), torch.tensor([0.5, 0.875, 1 - 1 / 32]))
    x = torch.randn(2, 9, 24, dtype=torch.float64)
    projected = x @ mixer.w_qkv.weight.T + mixer.w_qkv.bias
    q, k, v = projected[..., :12].unflatten(-1, (3, 4)), projected[..., 12:24].unflatten(-1, (3, 4)), projected[..., 24:].unflatten(-1, (3, 8))
    f = mixer.frequencies
    y = decay_attention_reference(rotary_reference(q, f), rotary_reference(k, f), v, mixer.log_decay)
    y = y * (y.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    want = y.flatten(2) @ mixer.w_o.weight.T + mixer.w_o.bias
    torch.testing.assert_close(mixer(x), want)


def test_tokens_see_the_past_alone_and_masked_ones_are_absent() -> None:
    torch.manual_seed(0)
    mixer = CausalMixer(LSSOConfig(16, 2, 4)).double()
    x = torch.randn(1, 12, 16, dtype=torch.float64)
    changed = x.clone()
    changed[:, 7:] = torch.randn(1, 5, 16, dtype=torch.float64)
    torch.testing.assert_close(mixer(x)[:, :7], mixer(changed)[:, :7])
    mask = torch.rand(1, 12) < 0.6
    y = mixer(x, mask)
    torch.testing.assert_close(y[mask], mixer(x[mask][None])[0])
    assert not y[~mask].any()


@pytest.mark.parametrize("parts", [(13,), (1,) * 13, (5, 1, 1, 6), (12, 1)])
def test_shell_continues_a_sequence(parts) -> None:
    torch.manual_seed(0)
    shell = SequenceShell(LSSOConfig(32, 2, 16), **OPTIONS).double().eval()
    ids, mask = _batch()
    want = shell(ids, mask)
    state, got, at = shell.new_state(3), [], 0
    with torch.no_grad():
        for n in parts:
            got.append(shell(ids[:, at:at + n], mask[:, at:at + n], state=state))
            at += n
    torch.testing.assert_close(torch.cat(got, dim=1), want)
    assert state[0].position.tolist() == mask.sum(-1).tolist()


def test_training_step_and_names() -> None:
    torch.manual_seed(0)
    shell = SequenceShell(LSSOConfig(32, 2, 16), dropout=0.1, **OPTIONS)
    ids, mask = _batch()
    shell(ids, mask).square().mean().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in shell.parameters())
    assert "blocks.0.mixer.log_decay" in shell.state_dict() and "blocks.0.mixer.frequencies" not in shell.state_dict()
    other = SequenceShell(LSSOConfig(32, 2, 16), dropout=0.1, **(OPTIONS | dict(mixer_options=None)))
    other.load_state_dict(shell.state_dict())
    assert torch.equal(other.blocks[1].mixer.log_decay, shell.blocks[1].mixer.log_decay)


def test_refusals() -> None:
    shell = SequenceShell(LSSOConfig(32, 2, 16), dropout=0.1, **OPTIONS)
    ids, mask = _batch()
    state = shell.new_state(3)
    with pytest.raises(RuntimeError, match="for evaluation"):
        shell(ids, mask, state=state)
    shell.eval()
    with pytest.raises(RuntimeError, match="no_grad"):
        shell(ids, mask, state=state)
    with torch.no_grad():
        with pytest.raises(ValueError, match="the state must hold"):
            shell(ids[:2], mask[:2], state=state)
        with pytest.raises(ValueError, match="each of the 2 blocks"):
            shell(ids, mask, state=state[:1])
        mixer = shell.blocks[0].mixer
        x = torch.randn(3, 4, 32)
        with pytest.raises(ValueError, match="position_ids cannot"):
            mixer(x, position_ids=torch.arange(4), state=state[0])
        with pytest.raises(TypeError, match="CUDA tensors"):
            mixer(x, implementation="cuda")
        with pytest.raises(ValueError, match="x must have shape"):
            mixer(x[..., :8])
    with pytest.raises(RuntimeError, match="only a shell with mixer='causal'"):
        SequenceShell(LSSOConfig(32, 2, 16)).new_state(1)
    with pytest.raises(ValueError, match="mixer must be"):
        SequenceShell(LSSOConfig(32, 2, 16), mixer="other")
    with pytest.raises(ValueError, match="mixer_options"):
        SequenceShell(LSSOConfig(32, 2, 16), mixer_options=dict(windows=(2, 3)))
    with pytest.raises(ValueError, match="windows"):
        CausalMixer(LSSOConfig(32, 2, 16), windows=(0.5, 3.0))


@pytest.mark.gpu
@pytest.mark.parametrize(("dim", "heads", "rank"), [(128, 4, 32), (256, 8, 32), (192, 3, 48)])
def test_cuda_shell_matches_the_reference_path_in_bf16(dim, heads, rank) -> None:
    from tests.gpu_util import relative_l2, require_native

    require_native()
    torch.manual_seed(0)
    shell = SequenceShell(LSSOConfig(dim, heads, rank), **(OPTIONS | dict(depth=4, hidden=344))).cuda()
    ids, mask = _batch("cuda", 3, 300)

    def run(implementation, amp):
        for p in shell.parameters():
            p.grad = None
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=amp):
            y = shell(ids, mask, implementation=implementation)
        y.float().square().mean().backward()
        return y.detach().float(), [p.grad.detach().clone() for p in shell.parameters()]

    y_cuda, g_cuda = run("cuda", True)
    y_ref, g_ref = run("reference", False)
    y_bf16, g_bf16 = run("reference", True)
    assert not y_cuda[1, 200:].any() and not y_cuda[2].any()
    assert relative_l2(y_cuda, y_ref) <= max(1e-2, 1.25 * relative_l2(y_bf16, y_ref))
    for (name, _), a, b, c in zip(shell.named_parameters(), g_cuda, g_ref, g_bf16):
        ge, ge_ref = relative_l2(a, b), relative_l2(c, b)
        assert ge <= max(1e-2, 1.25 * ge_ref), (name, ge, ge_ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_cuda_shell_answers_token_by_token(dtype) -> None:
    """Prompt and steps on the CUDA path, the steps replayed from one captured graph, against whole sequences."""
    from tests.gpu_util import relative_l2, require_native

    require_native()
    torch.manual_seed(0)
    shell = SequenceShell(LSSOConfig(128, 4, 32), **(OPTIONS | dict(depth=3))).cuda().eval()
    ids, mask = _batch("cuda", 3, 160)
    mask[2, :150] = True  # this one starts, and ends before the others
    prompt = 140
    with torch.no_grad():
        want = shell(ids, mask)
        with torch.autocast("cuda", dtype=dtype):
            whole = shell(ids, mask, implementation="cuda")
            state = shell.new_state(3)
            head = shell(ids[:, :prompt], mask[:, :prompt], implementation="cuda", state=state)
            with torch.autocast("cuda", dtype=torch.bfloat16):
                ref_bf16 = shell(ids, mask)
            assert relative_l2(head, want[:, :prompt]) <= max(1e-2, 1.25 * relative_l2(ref_bf16[:, :prompt], want[:, :prompt]))
            token, live = ids[:, prompt:prompt + 1].clone(), mask[:, prompt:prompt + 1].clone()
            saved = [(s.memory.clone(), s.position.clone()) for s in state]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                shell(token, live, implementation="cuda", state=state)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                row = shell(token, live, implementation="cuda", state=state)
            for s, (memory, position) in zip(state, saved):
                s.memory.copy_(memory)
                s.position.copy_(position)
            rows = []
            for t in range(prompt, 160):
                token.copy_(ids[:, t:t + 1])
                live.copy_(mask[:, t:t + 1])
                graph.replay()
                rows.append(row.clone())
    got = torch.cat(rows, dim=1)
    assert not got[~mask[:, prompt:]].any()
    assert relative_l2(got, want[:, prompt:]) <= max(1e-2, 1.25 * relative_l2(ref_bf16[:, prompt:], want[:, prompt:]))
    assert state[2].position.tolist() == mask.sum(-1).tolist()


@pytest.mark.gpu
def test_training_step_replays_as_a_graph() -> None:
    from tests.gpu_util import require_native

    require_native()
    torch.manual_seed(0)
    shell = SequenceShell(LSSOConfig(64, 2, 32), dropout=0.2, **OPTIONS).cuda()
    ids, mask = _batch("cuda", 3, 200)
    params = list(shell.parameters())

    def step():
        with torch.autocast("cuda", dtype=torch.float16):
            y = shell(ids, mask, implementation="cuda")
        return y, torch.autograd.grad(y.float().square().sum(), params)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y, grads = step()
    with torch.no_grad():
        shell.dropout_state[1] = 5
    graph.replay()
    torch.cuda.synchronize()
    with torch.no_grad():
        shell.dropout_state[1] = 5
    y_eager, grads_eager = step()
    assert torch.equal(y, y_eager) and all(torch.equal(a, b) for a, b in zip(grads, grads_eager))
