"""Causal token mixer with a state: linear attention with a decay per head over rotary queries and keys.

``CausalMixer`` stands where ``LSSO`` stands in a block and takes the same
configuration: per head ``rank`` query and key features and ``head_dim`` value
features from one packed projection, rotary positions on queries and keys, the
decay attention of ``decay.py``, an RMS norm of every head's output and an
output projection.  Unlike ``LSSO`` a token sees itself and the tokens before
it alone, so a sequence can be continued: a ``CausalState`` holds the heads'
memories and the number of tokens seen, prompts run in chunks and single
tokens by one step each.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn.functional as F
from torch import nn

from .config import CoreMode, LSSOConfig
from .decay import decay_attention, decay_attention_reference, decay_attention_step
from .rotary import rotary, rotary_frequencies, rotary_reference

_EPSILON = 1e-6


class CausalState(NamedTuple):
    """What a batch of sequences has left behind; updated in place."""

    memory: torch.Tensor    # [batch, heads, rank, head_dim], FP32 (FP64 under the FP64 reference)
    position: torch.Tensor  # [batch] int64: valid tokens so far


class CausalMixer(nn.Module):
    """Decay attention as a token mixer (``config.rank`` key features, ``config.head_dim`` value features per head).

    ``windows``: the first and the last head's decay window in tokens, the
    heads between spaced evenly over its logarithm (``decay = 1 - 1 /
    window``, a constant of the model).  ``rotary``: arguments of
    ``rotary_frequencies`` (base, scaling, ...) beside the width.  The
    configuration's ablations (``core_mode``, ``rank_rotary``) are LSSO's and
    refused here.  The CUDA path projects to BF16 whatever the input's type.
    """

    def __init__(self, config: LSSOConfig, *, windows: tuple[float, float] = (8.0, 512.0), rotary: dict | None = None) -> None:
        super().__init__()
        if config.core_mode is not CoreMode.DYNAMIC or not config.rank_rotary:
            raise ValueError("CausalMixer has no compact core and always rotates queries and keys: core_mode must be 'dynamic' and "
                             f"rank_rotary True, got {config.core_mode.value!r} and {config.rank_rotary}")
        if config.rank % 2:
            raise ValueError(f"rotary positions require an even rank, got rank={config.rank}")
        if not all(w >= 1 for w in windows) or len(windows) != 2:
            raise ValueError(f"windows must be two lengths of at least one token, got {windows}")
        self.config = config
        heads = config.num_heads
        self.widths = (2 * heads * config.rank, heads * config.head_dim)
        self.w_qkv = nn.Linear(config.dim, sum(self.widths), bias=config.bias)
        self.w_o = nn.Linear(config.dim, config.dim, bias=config.bias)
        self._windows, self._rotary = tuple(windows), dict(rotary or {})
        _, self.magnitude = rotary_frequencies(config.rank, **self._rotary)
        for name, value in self._constants().items():
            self.register_buffer(name, value, persistent=name == "log_decay")

    def _constants(self) -> dict[str, torch.Tensor]:
        heads, windows = self.config.num_heads, self._windows
        spread = torch.arange(heads, dtype=torch.float64) / max(1, heads - 1)
        window = windows[0] * (windows[1] / windows[0]) ** spread
        frequencies, _ = rotary_frequencies(self.config.rank, **self._rotary)
        return {"log_decay": torch.log1p(-1 / window).float(), "frequencies": frequencies}

    def _constant(self, name: str, device: torch.device) -> torch.Tensor:
        with torch.device("cpu"):
            return self._constants()[name].to(device=device)

    def _apply(self, fn, recurse=True):
        # module-wide dtype changes leave the constants in their precision, and what to_empty() gives a module that was
        # made on the meta device is filled in
        constants = {name: getattr(self, name) for name in ("log_decay", "frequencies")}
        super()._apply(fn, recurse)
        for name, value in constants.items():
            device = getattr(self, name).device
            empty = value.is_meta and device.type != "meta"
            setattr(self, name, self._constant(name, device) if empty else value.to(device=device))
        return self

    def _load_from_state_dict(self, *args, **kwargs) -> None:
        super()._load_from_state_dict(*args, **kwargs)
        if self.frequencies.is_meta and not self.log_decay.is_meta:  # assigned to a module on the meta device
            self.frequencies = self._constant("frequencies", self.log_decay.device)

    def new_state(self, batch: int) -> CausalState:
        """The state before any token."""
        c, like = self.config, self.w_o.weight
        kind = torch.float64 if like.dtype == torch.float64 else torch.float32
        return CausalState(torch.zeros(batch, c.num_heads, c.rank, c.head_dim, dtype=kind, device=like.device),
                           torch.zeros(batch, dtype=torch.int64, device=like.device))

    def _check(self, x, valid_mask, position_ids, state, implementation) -> None:
        c = self.config
        if implementation not in ("reference", "cuda"):
            raise ValueError(f"implementation must be 'reference' or 'cuda', got {implementation!r}")
        if x.ndim != 3 or x.shape[-1] != c.dim:
            raise ValueError(f"x must have shape [B, N, {c.dim}], got {tuple(x.shape)}")
        if valid_mask is not None:
            if valid_mask.shape != x.shape[:2]:
                raise ValueError(f"valid_mask must have shape {tuple(x.shape[:2])}, got {tuple(valid_mask.shape)}")
            if valid_mask.dtype != torch.bool:
                raise TypeError(f"valid_mask must have dtype torch.bool, got {valid_mask.dtype}")
        if position_ids is not None and state is not None:
            raise ValueError("position_ids cannot be given with a state, which counts the tokens itself")
        if state is not None:
            shape = (x.shape[0], c.num_heads, c.rank, c.head_dim)
            if tuple(state.memory.shape) != shape or tuple(state.position.shape) != shape[:1]:
                raise ValueError(f"the state must hold memories {shape} and positions {shape[:1]}, got "
                                 f"{tuple(state.memory.shape)} and {tuple(state.position.shape)}")
            if torch.is_grad_enabled():
                raise RuntimeError("a state is updated in place: run with it under torch.no_grad()")
        if implementation == "cuda":
            for label, width in (("rank", c.rank), ("dim // num_heads", c.head_dim)):
                if width % 8 or not 8 <= width <= 128:
                    raise ValueError(f"implementation='cuda' supports {label} of multiples of 8 from 8 to 128, got {width}")
            if x.dtype not in (torch.float16, torch.bfloat16) or not x.is_cuda:
                raise TypeError(f"implementation='cuda' supports CUDA tensors of torch.float16 or torch.bfloat16, got {x.dtype} on {x.device}")
            for name, parameter in self.named_parameters():
                if parameter.dtype != torch.float32 or parameter.device != x.device:
                    raise TypeError(f"implementation='cuda' requires {name} to use torch.float32 on {x.device}")
            if state is not None and (state.memory.dtype != torch.float32 or state.memory.device != x.device):
                raise TypeError(f"implementation='cuda' requires a state of torch.float32 on {x.device}, got "
                                f"{state.memory.dtype} on {state.memory.device}")

    def _positions(self, x, valid_mask, position_ids, state):
        """Rotary positions: of valid tokens in order (where nothing else is given, None for 0, 1, ..)."""
        if position_ids is not None:
            return position_ids
        if valid_mask is None:
            if state is None:
                return None
            return state.position[:, None] + torch.arange(x.shape[1], device=x.device)
        order = (valid_mask.cumsum(-1) - 1).clamp_min(0)
        return order if state is None else state.position[:, None] + order

    def forward(self, x: torch.Tensor, valid_mask: torch.Tensor | None = None, position_ids: torch.Tensor | None = None, *,
                state: CausalState | None = None, implementation: str = "reference") -> torch.Tensor:
        """``[B, N, dim]`` to the same; masked tokens are as though absent and give zeros.

        ``position_ids`` ``[N]`` or ``[B, N]`` replace the count of valid
        tokens.  ``state`` (from :meth:`new_state`, under ``torch.no_grad()``)
        precedes the first token and is updated in place.
        """
        self._check(x, valid_mask, position_ids, state, implementation)
        positions = self._positions(x, valid_mask, position_ids, state)
        run = self._forward_cuda if implementation == "cuda" else self._forward_reference
        y = run(x, valid_mask, positions, state)
        if state is not None:
            state.position.add_(x.shape[1] if valid_mask is None else valid_mask.sum(-1))
        return y

    def _split(self, projected, turn, positions):
        """Rotated queries and keys, and values, of a packed projection."""
        heads = self.config.num_heads
        both, values = projected.split(self.widths, dim=-1)
        both = turn(both.unflatten(-1, (2 * heads, -1)), self.frequencies, positions, magnitude=self.magnitude)
        q, k = both.split(heads, dim=2)
        return q, k, values.unflatten(-1, (heads, -1))

    def _forward_cuda(self, x, valid_mask, positions, state):
        from . import projection

        wants_backward = torch.is_grad_enabled() and (x.requires_grad or self.w_qkv.weight.requires_grad or self.w_o.weight.requires_grad)
        images = projection.layer_images(self.w_qkv.weight, self.w_o.weight, wants_backward)
        projected = projection.input_projection(x, self.w_qkv.weight, self.w_qkv.bias, valid_mask, images)
        q, k, v = self._split(projected, rotary, positions)
        if state is None:
            y = decay_attention(q, k, v, self.log_decay, valid_mask=valid_mask)
        elif x.shape[1] == 1:
            live = None if valid_mask is None else valid_mask[:, 0]
            y = decay_attention_step(q[:, 0], k[:, 0], v[:, 0], self.log_decay, state.memory, valid_mask=live)[:, None]
        else:
            y, last = decay_attention(q, k, v, self.log_decay, state=state.memory, valid_mask=valid_mask, return_state=True)
            state.memory.copy_(last)
        y = F.rms_norm(y, y.shape[-1:], eps=_EPSILON).flatten(2)
        return projection.output_projection(y, self.w_o.weight, self.w_o.bias, x.dtype, valid_mask, images)

    def _forward_reference(self, x, valid_mask, positions, state):
        if valid_mask is not None:
            x = torch.where(valid_mask[..., None], x, torch.zeros((), dtype=x.dtype, device=x.device))
        projected = self.w_qkv(x)
        with torch.autocast(device_type=x.device.type, enabled=False):
            q, k, v = self._split(projected, rotary_reference, positions)
            y = decay_attention_reference(q, k, v, self.log_decay, valid_mask=valid_mask, return_state=state is not None,
                                          state=None if state is None else state.memory)
            if state is not None:
                y, last = y
                state.memory.copy_(last)
            y = F.rms_norm(y, y.shape[-1:], eps=_EPSILON).flatten(2)
        y = self.w_o(y).to(x.dtype)
        return y if valid_mask is None else torch.where(valid_mask[..., None], y, torch.zeros((), dtype=y.dtype, device=y.device))

    def extra_repr(self) -> str:
        c = self.config
        return f"dim={c.dim}, num_heads={c.num_heads}, rank={c.rank}"


__all__ = ["CausalMixer", "CausalState"]
