"""The sequence shell's construction checks."""

from __future__ import annotations

import pytest

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
