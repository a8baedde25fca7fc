"""The causal mixer as a module: made without memory, moved and loaded, and the configurations that it refuses."""

from __future__ import annotations

import pytest
import torch

from lsso import LSSOConfig
from lsso_b200.ball.causal import CausalMixer
from lsso_b200.ball.shell import SequenceShell

CONFIG = LSSOConfig(32, 2, 16)
OPTIONS = dict(windows=(4.0, 64.0), rotary=dict(base=500.0, scaling="blend", factor=4.0))


@pytest.mark.parametrize("assign", [False, True])
def test_made_on_the_meta_device(assign) -> None:
    """``to_empty`` and a loaded checkpoint, or a checkpoint that is assigned, give the mixer that was saved."""
    torch.manual_seed(0)
    ready = CausalMixer(CONFIG, **OPTIONS)
    with torch.device("meta"):
        mixer = CausalMixer(CONFIG, **OPTIONS)
    assert mixer.log_decay.is_meta and mixer.frequencies.is_meta
    if not assign:
        mixer = mixer.to_empty(device="cpu")
        assert torch.equal(mixer.log_decay, ready.log_decay)
    mixer.load_state_dict(ready.state_dict(), assign=assign)
    assert torch.equal(mixer.log_decay, ready.log_decay) and torch.equal(mixer.frequencies, ready.frequencies)
    assert mixer.log_decay.dtype == torch.float32 and mixer.frequencies.dtype == torch.float64
    x = torch.randn(2, 9, 32)
    assert torch.equal(mixer(x), ready(x))


def test_a_shell_made_on_the_meta_device() -> None:
    options = dict(depth=2, vocab=11, gated="silu", hidden=40, embedding_scale=4.0, mixer="causal", mixer_options=OPTIONS)
    torch.manual_seed(0)
    ready = SequenceShell(CONFIG, **options)
    with torch.device("meta"):
        shell = SequenceShell(CONFIG, **options)
    shell = shell.to_empty(device="cpu")
    shell.load_state_dict(ready.state_dict())
    ids = torch.randint(0, 11, (2, 7))
    assert torch.equal(shell(ids), ready(ids))


def test_casts_and_moves_leave_the_constants() -> None:
    mixer = CausalMixer(CONFIG, **OPTIONS)
    decay, frequencies = mixer.log_decay.clone(), mixer.frequencies.clone()
    for change in (lambda m: m.half(), lambda m: m.double(), lambda m: m.to(torch.bfloat16), lambda m: m.to_empty(device="cpu")):
        mixer = change(mixer)
        assert torch.equal(mixer.log_decay, decay) and torch.equal(mixer.frequencies, frequencies)
        assert mixer.log_decay.dtype == torch.float32 and mixer.frequencies.dtype == torch.float64
    assert mixer.to("meta").log_decay.is_meta


@pytest.mark.parametrize("change", [dict(core_mode="static"), dict(core_mode="zero"), dict(rank_rotary=False)])
def test_ablations_of_the_other_mixer_are_refused(change) -> None:
    config = LSSOConfig(32, 2, 16, **change)
    SequenceShell(config, depth=1)
    with pytest.raises(ValueError, match="core_mode must be 'dynamic' and rank_rotary True"):
        CausalMixer(config)
    with pytest.raises(ValueError, match="core_mode must be 'dynamic' and rank_rotary True"):
        SequenceShell(config, depth=1, mixer="causal")


@pytest.mark.parametrize(("dim", "heads", "rank", "label"), [(32, 2, 12, "rank"), (48, 4, 16, "dim // num_heads"), (32, 2, 136, "rank"), (272, 2, 16, "dim // num_heads")])
def test_widths_that_the_kernels_lack_are_refused_before_any_work(dim, heads, rank, label, monkeypatch) -> None:
    from lsso_b200.ball import projection

    monkeypatch.setattr(projection, "layer_images", lambda *_: pytest.fail("work was done"))
    mixer = CausalMixer(LSSOConfig(dim, heads, rank))
    assert mixer(torch.randn(1, 3, dim)).shape == (1, 3, dim)
    with pytest.raises(ValueError, match=f"{label} of multiples of 8"):
        mixer(torch.randn(1, 3, dim), implementation="cuda")


@pytest.mark.gpu
def test_states_that_the_kernels_lack_are_refused_before_any_work(monkeypatch) -> None:
    from lsso_b200.ball import projection
    from tests.gpu_util import require_native

    require_native()
    mixer = CausalMixer(CONFIG).cuda()
    x = torch.randn(2, 3, 32, device="cuda").bfloat16()
    good = mixer.new_state(2)
    with torch.no_grad():
        mixer(x, state=good, implementation="cuda")
        monkeypatch.setattr(projection, "layer_images", lambda *_: pytest.fail("work was done"))
        for memory in (good.memory.double(), good.memory.cpu(), good.memory.bfloat16()):
            kept = memory.clone()
            with pytest.raises(TypeError, match="state of torch.float32"):
                mixer(x, state=good._replace(memory=memory), implementation="cuda")
            assert torch.equal(memory, kept)
