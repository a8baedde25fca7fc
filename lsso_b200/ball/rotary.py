"""Rotary positions: queries and keys turned by their position, feature pair by feature pair.

``rotary(x, frequencies, positions)`` turns pair i of the first ``2 f``
features of every head, ``f = len(frequencies)``, by the angle ``position *
frequencies[i]`` and multiplies it by ``magnitude``; the other features are
copied.  Pairs are features ``(i, i + f)`` or, ``interleaved``, ``(2 i, 2 i +
1)``.  Angles are formed in 64 bits, so far positions keep their precision.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _native

_POSITION_TYPES = {torch.int64: 0, torch.int32: 1, torch.float32: 2, torch.float64: 3}
_strides: dict[tuple, ctypes.Array] = {}  # as the library takes them


def rotary_frequencies(features: int, *, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_length: int = 4096, fast_turns: float = 32.0, slow_turns: float = 1.0,
                       device: torch.device | str | None = None) -> tuple[torch.Tensor, float]:
    """``(frequencies, magnitude)`` for :func:`rotary` over ``features`` (even) features, FP64.

    ``base ** (-2 i / features)``, for contexts ``factor`` times as long as
    the model was trained for by ``scaling``: ``"linear"`` divides every
    frequency by the factor; ``"base"`` raises the base so that the slowest
    pair is divided by it and the fastest stays; ``"blend"`` divides the pairs
    that turn fewer than ``slow_turns`` times within ``original_length``, keeps
    those that turn more than ``fast_turns`` times, blends between, and raises
    the magnitude by ``0.1 ln(factor)``.
    """
    if isinstance(features, bool) or not isinstance(features, int) or features < 2 or features % 2:
        raise ValueError(f"features must be a positive even integer, got {features!r}")
    if scaling not in (None, "linear", "base", "blend"):
        raise ValueError(f"scaling must be None, 'linear', 'base' or 'blend', got {scaling!r}")
    if factor < 1 or base <= 0:
        raise ValueError(f"factor must be at least 1 and base positive, got {factor} and {base}")
    half = features // 2
    i = torch.arange(half, dtype=torch.float64) / half
    if scaling == "base":
        base = base * factor ** (half / max(1, half - 1))
    frequencies, magnitude = base ** -i, 1.0
    if scaling == "linear":
        frequencies = frequencies / factor
    elif scaling == "blend":
        if not fast_turns > slow_turns:
            raise ValueError(f"fast_turns must exceed slow_turns, got {fast_turns} and {slow_turns}")
        turns = original_length * frequencies / (2 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        frequencies = frequencies * keep + frequencies / factor * (1 - keep)
        magnitude = 1 + 0.1 * math.log(factor)
    return frequencies.to(device=device), magnitude


def _check(x, frequencies, positions) -> None:
    if x.ndim != 4:
        raise ValueError(f"x must have shape [batch, length, heads, dim], got {tuple(x.shape)}")
    if frequencies.ndim != 1 or not 1 <= frequencies.numel() <= x.shape[-1] // 2:
        raise ValueError(f"frequencies must hold 1 to {x.shape[-1] // 2} pairs, got shape {tuple(frequencies.shape)}")
    if frequencies.dtype not in (torch.float64, torch.float32):
        raise TypeError(f"frequencies must use torch.float64 or torch.float32, got {frequencies.dtype}")
    if frequencies.requires_grad:
        raise ValueError("rotary does not support gradients for frequencies")
    if positions is not None:
        if positions.dtype not in _POSITION_TYPES:
            raise TypeError(f"positions must use int64, int32, float32 or float64, got {positions.dtype}")
        if tuple(positions.shape) not in ((x.shape[1],), tuple(x.shape[:2])):
            raise ValueError(f"positions must have shape [{x.shape[1]}] or {tuple(x.shape[:2])}, got {tuple(positions.shape)}")
        if positions.requires_grad:
            raise ValueError("rotary does not support gradients for positions")
    for name, value in (("frequencies", frequencies), ("positions", positions)):
        if value is not None and value.device != x.device:
            raise RuntimeError(f"{name} must be on {x.device}, got {value.device}")


def _usual(x, frequencies, positions) -> bool:
    """Whether all of _check holds, in one expression (a microsecond less than asking one by one)."""
    shape, device = x.shape, x.device
    return (len(shape) == 4 and frequencies.dtype is torch.float64 and frequencies.ndim == 1
            and 1 <= frequencies.shape[0] <= shape[3] // 2 and frequencies.device == device and not frequencies.requires_grad
            and (positions is None or (positions.dtype is torch.int64 and positions.shape == shape[:2]
                                       and positions.device == device)))


def rotary_reference(x, frequencies, positions=None, *, interleaved=False, magnitude=1.0) -> torch.Tensor:
    """The same operator in PyTorch (any device, autograd by PyTorch)."""
    _check(x, frequencies, positions)
    f = frequencies.numel()
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    positions = torch.arange(x.shape[1], device=x.device) if positions is None else positions
    angle = (positions.double()[..., None] * frequencies.double())[..., None, :]
    cos, sin = (torch.cos(angle) * magnitude).to(wide), (torch.sin(angle) * magnitude).to(wide)
    part = x[..., : 2 * f].to(wide)
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else part.split(f, dim=-1)
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)
    return torch.cat((turned.to(x.dtype), x[..., 2 * f:]), dim=-1)


def _turn(x, frequencies, positions, interleaved, magnitude, backward):
    batch, length, heads, dim = x.shape
    y = x.new_empty((batch, length, heads, dim))
    if not y.numel():
        return y
    s = x.stride()
    if s[3] != 1 or (s[0] | s[1] | s[2]) % 2 or s[0] < 0 or s[1] < 0 or s[2] < 0 or x.data_ptr() % (2 * x.element_size()):
        x = x.clone(memory_format=torch.contiguous_format)
        s = x.stride()
    strides = _strides.get(s)
    if strides is None:
        if len(_strides) >= 4096:
            _strides.clear()
        strides = _strides[s] = (ctypes.c_int64 * 3)(*s[:3])
    _native.run("lsso_rotary", x.device, x.data_ptr(), strides, _native.ELEMENT_TYPES[x.dtype], batch, length,
                heads, dim, frequencies.numel(), frequencies.data_ptr(), int(frequencies.dtype is torch.float64),
                _native._ptr(positions), 0 if positions is None else _POSITION_TYPES[positions.dtype],
                int(positions is not None and positions.ndim == 2), int(interleaved), int(backward), magnitude,
                y.data_ptr())
    return y


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, frequencies, positions, interleaved, magnitude):
        ctx.save_for_backward(frequencies, positions)
        ctx.layout = interleaved, magnitude
        return _turn(x, frequencies, positions, interleaved, magnitude, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        frequencies, positions = ctx.saved_tensors
        return _turn(dy, frequencies, positions, *ctx.layout, True), None, None, None, None


def rotary(x: torch.Tensor, frequencies: torch.Tensor, positions: torch.Tensor | None = None, *,
           interleaved: bool = False, magnitude: float = 1.0) -> torch.Tensor:
    """``x`` ``[batch, length, heads, dim]`` turned by its positions, as a new contiguous tensor.

    ``x`` is BF16, FP16 or FP32 with an even ``dim``; queries and keys that
    are adjacent heads of one projection go in one call, strided views are
    read in place.  ``frequencies`` (FP64 or FP32) holds one angle per
    position for each turned pair, as :func:`rotary_frequencies` gives them;
    ``positions`` is ``[length]`` or ``[batch, length]``, int64, int32, FP32
    or FP64 (default 0, 1, ..).
    """
    _native.refuse_transforms("rotary", x, frequencies, positions)
    if not _usual(x, frequencies, positions):
        _check(x, frequencies, positions)
    if not x.is_cuda:
        raise ValueError("rotary requires CUDA tensors; use rotary_reference elsewhere")
    if x.dtype not in _native.ELEMENT_TYPES:
        raise TypeError(f"rotary supports torch.bfloat16, torch.float16 and torch.float32, got {x.dtype}")
    if x.shape[-1] % 2:
        raise ValueError(f"rotary requires an even head width, got {x.shape[-1]}")
    frequencies = frequencies.contiguous()
    positions = None if positions is None else positions.contiguous()
    if torch.is_grad_enabled() and x.requires_grad:
        return _Rotary.apply(x, frequencies, positions, bool(interleaved), float(magnitude))
    return _turn(x, frequencies, positions, bool(interleaved), float(magnitude), False)


__all__ = ["rotary", "rotary_frequencies", "rotary_reference"]
