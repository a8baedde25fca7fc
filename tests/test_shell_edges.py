"""The sequence shell's construction checks, and its blocks recomputed in the backward."""

from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from lsso import LSSOConfig
from lsso_b200.ball.feedforward import GatedFeedForward
from lsso_b200.ball.shell import SequenceShell, ShellBlock

CONFIG = LSSOConfig(32, 2, 16)


def test_a_gated_block_needs_features() -> None:
    for options in (dict(gated="silu"), dict(gated="silu", hidden=0), dict(gated="gelu", hidden=-8),
                    dict(gated="silu", mlp_ratio=0.01)):
        with pytest.raises(ValueError, match="hidden"):
            SequenceShell(CONFIG, **options)
        with pytest.raises(ValueError, match="hidden"):
            ShellBlock(CONFIG, **options)
    with pytest.raises(ValueError, match="hidden"):
        GatedFeedForward(32, 0)
    assert SequenceShell(CONFIG, gated="silu", mlp_ratio=2.0).blocks[0].mlp.w_out.in_features == 64
    assert SequenceShell(CONFIG, gated="silu", hidden=40).blocks[0].mlp.w_out.in_features == 40


def test_hidden_without_a_feed_forward_is_refused() -> None:
    with pytest.raises(ValueError, match="hidden"):
        SequenceShell(CONFIG, hidden=40)
    assert SequenceShell(CONFIG, hidden=40, mlp_ratio=1.0).blocks[0].mlp[0].out_features == 40
    assert SequenceShell(CONFIG).blocks[0].mlp is None


def _gradients(shell, ids, mask, implementation, reentrant, **autocast):
    """Gradients of one training step, its blocks recomputed in the backward unless ``reentrant`` is None."""
    forwards = [block.forward for block in shell.blocks]
    if reentrant is not None:
        for block in shell.blocks:
            block.forward = (lambda f: lambda *args: checkpoint(f, *args, use_reentrant=reentrant))(block.forward)
    for p in shell.parameters():
        p.grad = None
    try:
        with torch.autocast(**autocast):
            y = shell(ids, mask, implementation=implementation)
        y.float().square().sum().backward()
        return [p.grad.clone() for p in shell.parameters()]
    finally:
        for block, forward in zip(shell.blocks, forwards):
            block.forward = forward


def _shell():
    torch.manual_seed(0)
    shell = SequenceShell(LSSOConfig(64, 2, 32), depth=2, vocab=11, gated="silu", hidden=40, dropout=0.25, dropout_seed=9,
                          embedding_scale=4.0)
    ids = torch.randint(0, 11, (2, 13))
    mask = torch.ones(2, 13, dtype=torch.bool)
    mask[1, 8:] = False
    return shell, ids, mask


@pytest.mark.parametrize("reentrant", [False, True])
def test_blocks_with_dropout_can_be_recomputed(reentrant) -> None:
    """A block recomputed in the backward drops the elements that its forward dropped, although the shell's step has
    moved on meanwhile."""
    shell, ids, mask = _shell()
    shell.double()
    start = shell.dropout_state.clone()
    want = _gradients(shell, ids, mask, "reference", None, device_type="cpu", enabled=False)
    assert shell.dropout_state.tolist() == [9, 1]
    shell.dropout_state.copy_(start)
    got = _gradients(shell, ids, mask, "reference", reentrant, device_type="cpu", enabled=False)
    assert shell.dropout_state.tolist() == [9, 1]
    for (name, _), a, b in zip(shell.named_parameters(), got, want):
        torch.testing.assert_close(a, b, msg=name)


@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [False, True])
def test_cuda_blocks_with_dropout_can_be_recomputed(reentrant) -> None:
    from tests.gpu_util import require_native

    require_native()
    shell, ids, mask = _shell()
    shell, ids, mask = shell.cuda(), ids.cuda(), mask.cuda()
    start = shell.dropout_state.clone()
    want = _gradients(shell, ids, mask, "cuda", None, device_type="cuda", dtype=torch.bfloat16)
    shell.dropout_state.copy_(start)
    got = _gradients(shell, ids, mask, "cuda", reentrant, device_type="cuda", dtype=torch.bfloat16)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
