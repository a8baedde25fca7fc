"""The sequence shell with the package's operators around the mixer: gated feed-forward, dropout, scaled embedding."""

from __future__ import annotations

import pytest
import torch

from lsso import LSSOConfig
from lsso_b200.ball.dropout import dropout_state, keep_mask
from lsso_b200.ball.shell import SequenceShell

OPTIONS = dict(depth=2, vocab=11, gated="silu", hidden=40, dropout=0.25, dropout_seed=9, embedding_scale=4.0)


def _batch(device="cpu", batch=2, length=13):
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 11, (batch, length), generator=gen).to(device)
    mask = torch.ones(batch, length, dtype=torch.bool, device=device)
    mask[1, length * 2 // 3:] = False
    return ids, mask


def test_reference_shell_is_the_composition_of_its_operators() -> None:
    torch.manual_seed(0)
    shell = SequenceShell(LSSOConfig(32, 2, 16, bias=True), **OPTIONS).double()
    ids, mask = _batch()
    state = shell.dropout_state.clone()
    out = shell(ids, mask)
    zero = torch.zeros(1, dtype=torch.float64)
    x = torch.where(mask[:, :, None], 4.0 * shell.embedding.weight[ids], zero)
    for i, block in enumerate(shell.blocks):
        for j, branch in enumerate((lambda v: block.mixer(block.norm1(v), valid_mask=mask),  # noqa: B023
                                    lambda v: _gated(block.mlp, block.norm2(v)))):  # noqa: B023
            keep = keep_mask(x.shape, p=0.25, state=state, site=2 * i + j)
            x = torch.where(mask[:, :, None], x + torch.where(keep, branch(x) / 0.75, zero), zero)
    torch.testing.assert_close(out, x)
    assert torch.count_nonzero(out[1, 8:]) == 0
    assert shell.dropout_state.tolist() == [9, 1]  # one training forward
    assert not torch.equal(shell(ids, mask), out)  # another step: other elements dropped


def _gated(mlp, x):
    g, u = (x @ mlp.w_in.weight.T + mlp.w_in.bias).chunk(2, dim=-1)
    return (g * torch.sigmoid(g) * u) @ mlp.w_out.weight.T + mlp.w_out.bias


def test_evaluation_drops_nothing_and_keeps_the_step() -> None:
    torch.manual_seed(0)
    shell = SequenceShell(LSSOConfig(32, 2, 16), **OPTIONS).double().eval()
    ids, mask = _batch()
    assert torch.equal(shell(ids, mask), shell(ids, mask))
    assert shell.dropout_state.tolist() == [9, 0]


def test_default_shell_has_the_same_parameters_as_before() -> None:
    plain = SequenceShell(LSSOConfig(32, 2, 16), depth=1, vocab=8, mlp_ratio=2.0)
    names = {n for n, _ in plain.named_parameters()}
    assert {"embedding.weight", "blocks.0.mlp.0.weight", "blocks.0.mlp.2.weight"} <= names
    assert "dropout_state" not in plain.state_dict()
    gated = SequenceShell(LSSOConfig(32, 2, 16), **OPTIONS)
    assert "dropout_state" in gated.state_dict() and "embedding.weight" in gated.state_dict()


@pytest.mark.gpu
def test_cuda_shell_matches_the_reference_path_in_bf16() -> None:
    """As the plain shell's test: each tensor within the per-layer BF16 budget
    (1e-2) or 1.25x the error of the reference path's own BF16 run of it."""
    from tests.gpu_util import relative_l2, require_native

    require_native()
    torch.manual_seed(0)
    shell = SequenceShell(LSSOConfig(128, 4, 48), **(OPTIONS | dict(depth=4, hidden=344))).cuda()
    ids, mask = _batch("cuda", 2, 300)

    def run(implementation, amp):
        for p in shell.parameters():
            p.grad = None
        with torch.no_grad():
            shell.dropout_state.copy_(dropout_state(9))  # the same dropped elements in every run
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=amp):
            y = shell(ids, mask, implementation=implementation)
        y.float().square().mean().backward()
        return y.detach().float(), [p.grad.detach().clone() for p in shell.parameters()]

    y_cuda, g_cuda = run("cuda", True)
    y_ref, g_ref = run("reference", False)
    y_bf16, g_bf16 = run("reference", True)
    assert torch.count_nonzero(y_cuda[1, 200:]) == 0
    assert relative_l2(y_cuda, y_ref) <= max(1e-2, 1.25 * relative_l2(y_bf16, y_ref))
    for (name, _), a, b, c in zip(shell.named_parameters(), g_cuda, g_ref, g_bf16):
        ge, ge_ref = relative_l2(a, b), relative_l2(c, b)
        assert ge <= max(1e-2, 1.25 * ge_ref), (name, ge, ge_ref)


@pytest.mark.gpu
def test_training_step_replays_as_a_graph() -> None:
    """A captured step follows the dropout state from replay to replay and equals the eager step bit for bit."""
    from tests.gpu_util import require_native

    require_native()
    torch.manual_seed(0)
    shell = SequenceShell(LSSOConfig(64, 2, 32), **OPTIONS).cuda()
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
        shell.dropout_state.copy_(dropout_state(9))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert shell.dropout_state.tolist() == [9, 2]
    with torch.no_grad():
        shell.dropout_state.copy_(dropout_state(9, step=1))
    y_eager, grads_eager = step()
    torch.cuda.synchronize()
    assert torch.equal(y, y_eager)
    assert all(torch.equal(a, b) for a, b in zip(grads, grads_eager))
