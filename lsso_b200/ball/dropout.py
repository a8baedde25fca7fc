"""Dropout with the residual sum, from a counter-based generator.

``dropout_add(branch, residual, p=..., state=..., site=...)`` is
``residual + branch * keep / (1 - p)`` in one kernel.  ``keep`` is never
stored: element ``4 j + i`` (flat index) is kept when word ``i`` of
Philox4x32-10 (Salmon et al., SC 2011) at counter ``(j mod 2^32, j div 2^32,
site, step mod 2^32)`` and key ``seed`` is at least ``round(p 2^32)``, so the
backward computes it again.  ``state`` is an int64 CUDA tensor ``[seed,
step]``: advance ``state[1]`` once per training step (in a captured graph,
too) and give every dropout of a step its own ``site``.  Where activations are
recomputed in the backward, pass a copy of the state that stays as it is until
then.  The index is that of the tensor at hand: ranks that each hold a part of
the batch or of the sequence need a seed each, or they drop the same elements
of their parts.
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _native

_M32 = 0xFFFFFFFF


def dropout_state(seed: int, *, step: int = 0, device: torch.device | str | None = None) -> torch.Tensor:
    """The generator state ``[seed, step]`` as :func:`dropout_add` takes it."""
    return torch.tensor([seed, step], dtype=torch.int64, device=device)


def random_words(count: int, *, state: torch.Tensor, site: int = 0) -> torch.Tensor:
    """The 32-bit words (as int64) of flat indices ``0 .. count - 1`` (PyTorch; any device)."""
    j = torch.arange((count + 3) // 4, device=state.device)
    seed, step = state[0], state[1]
    c = [j & _M32, j >> 32, torch.full_like(j, site), (step & _M32).expand_as(j)]
    k0, k1 = seed & _M32, (seed >> 32) & _M32
    for _ in range(10):
        # 64-bit products wrap modulo 2^64, so both 32-bit halves are exact
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & _M32) ^ c[1] ^ k0, b & _M32, ((a >> 32) & _M32) ^ c[3] ^ k1, a & _M32]
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return torch.stack(c, dim=1).reshape(-1)[:count]


def keep_mask(shape, *, p: float, state: torch.Tensor, site: int = 0) -> torch.Tensor:
    """The elements that :func:`dropout_add` keeps, as a bool tensor (PyTorch; any device)."""
    words = random_words(math.prod(shape), state=state, site=site)
    return (words >= round(p * 2 ** 32)).reshape(shape)


def dropout_add_reference(branch, residual=None, *, p, state, site=0, valid_mask=None) -> torch.Tensor:
    """The same operator in PyTorch (any device, first-order autograd by PyTorch)."""
    _check(branch, residual, p, state, site, valid_mask)
    out_dtype = branch.dtype if residual is None else residual.dtype
    wide = torch.float64 if torch.float64 in (branch.dtype, out_dtype) else torch.float32
    keep = keep_mask(branch.shape, p=p, state=state, site=site)
    scale = 0.0 if p == 1 else 1 / (1 - p)
    y = torch.where(keep, branch.to(wide) * scale, torch.zeros((), dtype=wide, device=branch.device))
    if residual is not None:
        y = y + residual.to(wide)
    if valid_mask is not None:
        y = torch.where(valid_mask[..., None], y, torch.zeros((), dtype=wide, device=branch.device))
    return y.to(out_dtype)


def _check(branch, residual, p, state, site, valid_mask) -> None:
    if branch.ndim < 1:
        raise ValueError("branch must have at least one dimension")
    if not 0 <= p <= 1:
        raise ValueError(f"p must be in [0, 1], got {p}")
    if isinstance(site, bool) or not isinstance(site, int) or not 0 <= site <= _M32:
        raise ValueError(f"site must be an integer in [0, 2^32), got {site!r}")
    if state.dtype != torch.int64 or tuple(state.shape) != (2,):
        raise ValueError(f"state must be an int64 tensor [seed, step], got {state.dtype} {tuple(state.shape)}")
    if residual is not None and residual.shape != branch.shape:
        raise ValueError(f"residual must have branch's shape {tuple(branch.shape)}, got {tuple(residual.shape)}")
    if valid_mask is not None:
        if valid_mask.shape != branch.shape[:-1]:
            raise ValueError(f"valid_mask must have shape {tuple(branch.shape[:-1])}, got {tuple(valid_mask.shape)}")
        if valid_mask.dtype != torch.bool:
            raise TypeError(f"valid_mask must have dtype torch.bool, got {valid_mask.dtype}")
    for name, value in (("residual", residual), ("state", state), ("valid_mask", valid_mask)):
        if value is not None and value.device != branch.device:
            raise RuntimeError(f"{name} must be on {branch.device}, got {value.device}")


def _forward(branch, residual, p, state, site, mask, used):
    y = torch.empty_like(branch if residual is None else residual)
    if y.numel():
        types = _native.ELEMENT_TYPES
        width = branch.shape[-1]
        _native.run("lsso_dropout_forward", branch.device, branch.data_ptr(), types[branch.dtype],
                    _native._ptr(residual), types[y.dtype], _native._ptr(mask), branch.numel() // width, width, p,
                    state.data_ptr(), site, _native._ptr(used), y.data_ptr())
    return y


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, branch, residual, p, state, site, mask):
        # the state may move on before the backward runs: the kernel keeps a copy of what it read
        used = torch.empty(2, dtype=torch.int64, device=branch.device)
        y = _forward(branch, residual, p, state, site, mask, used)
        ctx.save_for_backward(used, mask)
        ctx.p, ctx.site, ctx.branch_dtype = p, site, branch.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        used, mask = ctx.saved_tensors
        needs_branch, needs_residual = ctx.needs_input_grad[:2]
        dbranch = dresidual = None
        dy = dy.contiguous()
        if needs_residual:
            dresidual = dy if mask is None else torch.empty_like(dy)
        if needs_branch:
            dbranch = torch.empty_like(dy, dtype=ctx.branch_dtype)
        if dy.numel() and (needs_branch or (needs_residual and mask is not None)):
            types = _native.ELEMENT_TYPES
            width = dy.shape[-1]
            _native.run("lsso_dropout_backward", dy.device, dy.data_ptr(), types[dy.dtype], types[ctx.branch_dtype],
                        _native._ptr(mask), dy.numel() // width, width, ctx.p, used.data_ptr(), ctx.site,
                        _native._ptr(dbranch), _native._ptr(None if mask is None else dresidual))
        return dbranch, dresidual, None, None, None, None


def dropout_add(branch: torch.Tensor, residual: torch.Tensor | None = None, *, p: float, state: torch.Tensor,
                site: int = 0, valid_mask: torch.Tensor | None = None) -> torch.Tensor:
    """``residual + branch * keep / (1 - p)``, zero where ``valid_mask`` is unset.

    ``branch`` ``[.., width]`` is BF16, FP16 or FP32; ``residual`` (optional)
    has its shape and its dtype or FP32, and decides the output's dtype;
    ``valid_mask`` is bool over the leading dimensions.  Non-contiguous inputs
    are copied.  A dropped element contributes exactly zero, whatever it holds.
    """
    _native.refuse_transforms("dropout_add", branch, residual, state, valid_mask)
    _check(branch, residual, p, state, site, valid_mask)
    if not branch.is_cuda:
        raise ValueError("dropout_add requires CUDA tensors; use dropout_add_reference elsewhere")
    if branch.dtype not in _native.ELEMENT_TYPES:
        raise TypeError(f"dropout_add supports torch.bfloat16, torch.float16 and torch.float32, got {branch.dtype}")
    if residual is not None and residual.dtype not in (branch.dtype, torch.float32):
        raise TypeError(f"residual must use {branch.dtype} or torch.float32, got {residual.dtype}")
    branch = branch.contiguous()
    residual = None if residual is None else residual.contiguous()
    state = state.contiguous()
    mask = None if valid_mask is None else valid_mask.contiguous()
    if torch.is_grad_enabled() and (branch.requires_grad or (residual is not None and residual.requires_grad)):
        return _DropoutAdd.apply(branch, residual, float(p), state, site, mask)
    return _forward(branch, residual, float(p), state, site, mask, None)


__all__ = ["dropout_add", "dropout_add_reference", "dropout_state", "keep_mask", "random_words"]
