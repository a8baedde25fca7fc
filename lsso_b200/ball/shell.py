"""End-to-end drivers of the mixer: a sequence-model shell and vision position IDs.

``SequenceShell`` stacks pre-LayerNorm residual blocks around ``LSSO`` the way
the reference's experiment encoder does (experiments/train_transformers.py:
479-556, ``SequenceBlock``): ``x + mixer(norm1(x))`` with the normalised
activations cast to the autocast dtype before the mixer, padded tokens zeroed
after each residual, and an optional ``x + mlp(norm2(x))`` (``mlp_ratio=0``
leaves it out, as BASELINE config 4 does).  Tokens enter through an
``Embedding`` initialised N(0, 0.02).

Three options replace the PyTorch layers around the mixer by the package's
operators, on either implementation: ``gated`` (a gated feed-forward block,
``feedforward.py``, in the MLP's place), ``dropout`` (dropout with the residual
sum and the padding mask in one pass, ``dropout.py``, on both branches of every
block) and ``embedding_scale`` (a scaled embedding with the mask applied and a
deterministic gradient, ``embedding.py``).

``mixer="causal"`` puts the causal mixer (``causal.py``: decay attention with
rotary positions) in LSSO's place.  Such a shell can continue a sequence:
``new_state`` and the ``state`` argument run prompts and then single tokens.

``vision_position_ids`` is the timm adapter's position rule
(integrations/timm.py:143-156): position 0 for the class token and centered
one-dimensional coordinates for the patches.
"""

from __future__ import annotations

import torch
from torch import nn

from .causal import CausalMixer, CausalState
from .config import LSSOConfig
from .dropout import dropout_add, dropout_add_reference, dropout_state
from .embedding import TokenEmbedding
from .feedforward import GatedFeedForward
from .model import LSSO


def vision_position_ids(length: int, device: torch.device | None = None) -> torch.Tensor:
    """FP32 [length]: 0 for the class token, then p - (length - 2)/2 for patch p."""
    if length <= 0:
        return torch.empty(0, device=device, dtype=torch.float32)
    patches = torch.arange(length - 1, device=device, dtype=torch.float32)
    patches -= 0.5 * (length - 2)
    return torch.cat((torch.zeros(1, device=device, dtype=torch.float32), patches))


class ShellBlock(nn.Module):
    """Pre-norm residual block: x + LSSO(norm(x)), padded tokens zero (optional MLP).

    ``gated`` ("silu" or "gelu"): a gated feed-forward block of ``hidden``
    features (default ``round(dim * mlp_ratio)``) in the MLP's place.  One of
    ``hidden`` and ``mlp_ratio`` has to give it features; ``hidden`` alone,
    with neither ``gated`` nor ``mlp_ratio``, is refused.
    ``dropout``: the rate on both branches in training mode; the block's
    branches use the generator sites ``site`` and ``site + 1``.
    ``mixer``: "lsso", or "causal" for a :class:`CausalMixer` with
    ``mixer_options``.
    """

    def __init__(self, config: LSSOConfig, *, mlp_ratio: float = 0.0, gated: str | None = None,
                 hidden: int | None = None, dropout: float = 0.0, site: int = 0, mixer: str = "lsso",
                 mixer_options: dict | None = None) -> None:
        super().__init__()
        if mixer not in ("lsso", "causal"):
            raise ValueError(f"mixer must be 'lsso' or 'causal', got {mixer!r}")
        if mixer == "lsso" and mixer_options:
            raise ValueError("mixer_options are the causal mixer's: set mixer='causal'")
        self.norm1 = nn.LayerNorm(config.dim)
        self.mixer = LSSO(config) if mixer == "lsso" else CausalMixer(config, **(mixer_options or {}))
        self.mlp = None
        self.dropout, self.site = float(dropout), site
        if hidden is not None and hidden < 1:
            raise ValueError(f"hidden must be positive, got {hidden}")
        if hidden is not None and gated is None and mlp_ratio <= 0:
            raise ValueError(f"hidden={hidden} needs a feed-forward block: set gated or mlp_ratio")
        hidden = int(round(config.dim * mlp_ratio)) if hidden is None else hidden
        if gated is not None:
            if hidden < 1:
                raise ValueError(f"a gated block needs features: set hidden or mlp_ratio (mlp_ratio={mlp_ratio})")
            self.norm2 = nn.LayerNorm(config.dim)
            self.mlp = GatedFeedForward(config.dim, hidden, activation=gated, bias=config.bias)
        elif mlp_ratio > 0:
            self.norm2 = nn.LayerNorm(config.dim)
            self.mlp = nn.Sequential(nn.Linear(config.dim, hidden, bias=config.bias), nn.GELU(),
                                     nn.Linear(hidden, config.dim, bias=config.bias))

    def _residual(self, x, branch, valid_mask, implementation, state, site):
        """x + branch (with dropout in training), padded tokens zero."""
        if self.training and self.dropout > 0:
            if state is None:
                raise ValueError("a block with dropout needs the generator state in training mode")
            add = dropout_add if implementation == "cuda" else dropout_add_reference
            return add(branch, x, p=self.dropout, state=state, site=site, valid_mask=valid_mask)
        x = x + branch
        if valid_mask is not None:
            x = torch.where(valid_mask[:, :, None], x, torch.zeros_like(x))
        return x

    def forward(self, x: torch.Tensor, valid_mask: torch.Tensor | None, implementation: str,
                state: torch.Tensor | None = None, memory: CausalState | None = None) -> torch.Tensor:
        """``state``: the dropout generator's; ``memory``: the causal mixer's."""
        normalized = self.norm1(x)
        if normalized.device.type == "cuda" and torch.is_autocast_enabled():
            amp = torch.get_autocast_dtype("cuda")
            if implementation == "cuda" and amp not in (torch.float16, torch.bfloat16):
                raise TypeError("the CUDA LSSO sequence path supports FP16 or BF16 AMP")
            normalized = normalized.to(dtype=amp)
        options = {} if memory is None else {"state": memory}
        branch = self.mixer(normalized, valid_mask=valid_mask, implementation=implementation, **options)
        x = self._residual(x, branch, valid_mask, implementation, state, self.site)
        if self.mlp is not None:
            if isinstance(self.mlp, GatedFeedForward):
                branch = self.mlp(self.norm2(x).to(dtype=normalized.dtype), implementation=implementation)
            else:
                branch = self.mlp(self.norm2(x))
            x = self._residual(x, branch, valid_mask, implementation, state, self.site + 1)
        return x


class SequenceShell(nn.Module):
    """Token embedding plus ``depth`` pre-norm LSSO blocks (dim 128, 4 heads,
    rank 48, depth 4, vocabulary 8, no MLP).

    ``gated``, ``hidden``, ``dropout``: as in :class:`ShellBlock`, for every
    block.  ``embedding_scale``: a :class:`TokenEmbedding` with this scale (the
    parameter keeps the name ``embedding.weight``).  With dropout, the buffer
    ``dropout_state`` holds ``[dropout_seed, step]`` and a training forward
    advances the step, in a captured graph as well.  Data-parallel ranks need a
    ``dropout_seed`` each, which DistributedDataParallel keeps only with
    ``broadcast_buffers=False`` and which a loaded checkpoint overwrites.  The
    blocks get a copy of the state, so they may be recomputed in the backward
    (activation checkpointing, block by block); recomputing the whole shell
    would advance the step again.  ``mixer``, ``mixer_options``: as in
    :class:`ShellBlock`, for every block.
    """

    def __init__(self, config: LSSOConfig, *, depth: int = 4, vocab: int = 8, mlp_ratio: float = 0.0,
                 gated: str | None = None, hidden: int | None = None, dropout: float = 0.0, dropout_seed: int = 0,
                 embedding_scale: float | None = None, mixer: str = "lsso", mixer_options: dict | None = None) -> None:
        super().__init__()
        if embedding_scale is None:
            self.embedding = nn.Embedding(vocab, config.dim)
            nn.init.normal_(self.embedding.weight, mean=0.0, std=0.02)
        else:
            self.embedding = TokenEmbedding(vocab, config.dim, scale=embedding_scale)
        self.blocks = nn.ModuleList(
            ShellBlock(config, mlp_ratio=mlp_ratio, gated=gated, hidden=hidden, dropout=dropout, site=2 * i, mixer=mixer,
                       mixer_options=mixer_options)
            for i in range(depth))
        if dropout > 0:
            self.register_buffer("dropout_state", dropout_state(dropout_seed))
        else:
            self.dropout_state = None

    def new_state(self, batch: int) -> list[CausalState]:
        """The state of ``batch`` sequences before their first token (``mixer="causal"``), one entry per block."""
        if not all(isinstance(block.mixer, CausalMixer) for block in self.blocks):
            raise RuntimeError("only a shell with mixer='causal' has a state")
        return [block.mixer.new_state(batch) for block in self.blocks]

    def forward(self, token_ids: torch.Tensor, valid_mask: torch.Tensor | None = None, *,
                implementation: str = "reference", state: list[CausalState] | None = None) -> torch.Tensor:
        """Hidden states ``[batch, length, dim]``.

        ``state`` (from :meth:`new_state`, under ``torch.no_grad()``, in
        evaluation mode): the tokens continue the sequences it stands for, and
        it moves on behind them, in a captured graph as well.
        """
        if state is not None:
            if not all(isinstance(block.mixer, CausalMixer) for block in self.blocks):
                raise RuntimeError("only a shell with mixer='causal' has a state")
            if len(state) != len(self.blocks):
                raise ValueError(f"the state must have an entry for each of the {len(self.blocks)} blocks, got {len(state)}")
            if self.training and self.dropout_state is not None:
                raise RuntimeError("a state is for evaluation: call eval() first")
        if isinstance(self.embedding, TokenEmbedding):
            x = self.embedding(token_ids, valid_mask, implementation=implementation)
        else:
            x = self.embedding(token_ids)
            if valid_mask is not None:
                x = torch.where(valid_mask[:, :, None], x, torch.zeros_like(x))
        generator = self.dropout_state
        if self.training and generator is not None:
            generator = generator.clone()
            self.dropout_state[1] += 1
        for i, block in enumerate(self.blocks):
            x = block(x, valid_mask, implementation, generator, None if state is None else state[i])
        return x


__all__ = ["SequenceShell", "ShellBlock", "vision_position_ids"]
