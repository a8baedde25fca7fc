"""Token embedding with scaling, and its gradient by sorted tokens.

``token_embedding(ids, weight, scale=..., valid_mask=...)`` is
``scale * weight[ids]`` with masked tokens zero, in the wanted output dtype.
The backward sorts the tokens by id and sums each row's upstream gradients in
FP32, in an order that depends on the ids alone: deterministic, no atomics.
"""

from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _native


def _check(ids, weight, valid_mask, padding_idx) -> None:
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"ids must use torch.int64 or torch.int32, got {ids.dtype}")
    if weight.ndim != 2 or 0 in weight.shape:
        raise ValueError(f"weight must have shape [vocab, dim], got {tuple(weight.shape)}")
    if valid_mask is not None:
        if valid_mask.shape != ids.shape:
            raise ValueError(f"valid_mask must have shape {tuple(ids.shape)}, got {tuple(valid_mask.shape)}")
        if valid_mask.dtype != torch.bool:
            raise TypeError(f"valid_mask must have dtype torch.bool, got {valid_mask.dtype}")
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f"padding_idx must be a row of the table (0..{weight.shape[0] - 1}), got {padding_idx}")
    for name, value in (("ids", ids), ("valid_mask", valid_mask)):
        if value is not None and value.device != weight.device:
            raise RuntimeError(f"{name} must be on {weight.device}, got {value.device}")


def token_embedding_reference(ids, weight, *, scale=1.0, valid_mask=None, padding_idx=None, dtype=None):
    """The same operator in PyTorch (any device)."""
    _check(ids, weight, valid_mask, padding_idx)
    safe = ids if valid_mask is None else torch.where(valid_mask, ids, torch.zeros_like(ids))
    y = nn.functional.embedding(safe, weight, padding_idx).to(torch.promote_types(weight.dtype, torch.float32)) * scale
    if valid_mask is not None:
        y = torch.where(valid_mask[..., None], y, torch.zeros_like(y))
    return y.to(weight.dtype if dtype is None else dtype)


def _forward(ids, weight, scale, mask, dtype):
    types = _native.ELEMENT_TYPES
    vocab, dim = weight.shape
    y = weight.new_empty((*ids.shape, dim), dtype=dtype)
    if y.numel():
        _native.run("lsso_embedding_forward", weight.device, ids.data_ptr(), int(ids.dtype == torch.int64),
                    _native._ptr(mask), ids.numel(), weight.data_ptr(), types[weight.dtype], vocab, dim, scale,
                    y.data_ptr(), types[dtype])
    return y


class _TokenEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, mask, padding_idx, dtype):
        ctx.save_for_backward(ids, mask)
        ctx.weight_meta = (weight.shape, weight.dtype)
        ctx.scale, ctx.padding = scale, -1 if padding_idx is None else padding_idx
        return _forward(ids, weight, scale, mask, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        ids, mask = ctx.saved_tensors
        (vocab, dim), dtype = ctx.weight_meta
        device = dy.device
        types = _native.ELEMENT_TYPES
        if not ids.numel():
            return None, dy.new_zeros((vocab, dim), dtype=dtype), None, None, None, None
        dy = dy.contiguous()
        grad = dy.new_empty((vocab, dim), dtype=dtype)
        scratch = _native.workspace("lsso_embedding_backward_workspace_size", device, ids.numel(), vocab, dim)
        _native.run("lsso_embedding_backward", device, ids.data_ptr(), int(ids.dtype == torch.int64),
                    _native._ptr(mask), ids.numel(), dy.data_ptr(), types[dy.dtype], vocab, dim, ctx.padding,
                    ctx.scale, grad.data_ptr(), types[dtype], scratch.data_ptr(), scratch.numel())
        return None, grad, None, None, None, None


def token_embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0,
                    valid_mask: torch.Tensor | None = None, padding_idx: int | None = None,
                    dtype: torch.dtype | None = None) -> torch.Tensor:
    """``scale * weight[ids]`` as ``[*ids.shape, dim]`` in ``dtype`` (default: the weight's).

    ``weight`` ``[vocab, dim]`` and ``dtype`` are FP32, BF16 or FP16; ``ids``
    int64 or int32.  Tokens whose ``valid_mask`` is unset give zero rows, take
    no part in the gradient, and their ids are not looked at; the row
    ``padding_idx`` has a zero gradient.  An id outside the table gives a zero
    row and sets the device status (``cuda.check_device_status()`` raises).
    """
    _native.refuse_transforms("token_embedding", weight, ids, valid_mask)
    _check(ids, weight, valid_mask, padding_idx)
    if not weight.is_cuda:
        raise ValueError("token_embedding requires CUDA tensors; use token_embedding_reference elsewhere")
    dtype = weight.dtype if dtype is None else dtype
    for name, value in (("weight", weight.dtype), ("the output", dtype)):
        if value not in _native.ELEMENT_TYPES:
            raise TypeError(f"token_embedding supports torch.float32, torch.bfloat16 and torch.float16, {name} uses {value}")
    if not weight.is_contiguous():
        raise RuntimeError("token_embedding requires a contiguous weight")
    ids = ids.contiguous()
    mask = None if valid_mask is None else valid_mask.contiguous()
    if torch.is_grad_enabled() and weight.requires_grad:
        return _TokenEmbedding.apply(ids, weight, float(scale), mask, padding_idx, dtype)
    return _forward(ids, weight, float(scale), mask, dtype)


class TokenEmbedding(nn.Module):
    """Embedding table ``weight [vocab, dim]`` (FP32, N(0, 0.02)) with an output scale."""

    def __init__(self, vocab: int, dim: int, *, scale: float = 1.0, padding_idx: int | None = None) -> None:
        super().__init__()
        self.weight = nn.Parameter(torch.empty(vocab, dim))
        self.scale, self.padding_idx = float(scale), padding_idx
        nn.init.normal_(self.weight, mean=0.0, std=0.02)

    def forward(self, ids: torch.Tensor, valid_mask: torch.Tensor | None = None, *,
                dtype: torch.dtype | None = None, implementation: str = "reference") -> torch.Tensor:
        if implementation not in ("reference", "cuda"):
            raise ValueError(f"implementation must be 'reference' or 'cuda', got {implementation!r}")
        run = token_embedding if implementation == "cuda" else token_embedding_reference
        return run(ids, self.weight, scale=self.scale, valid_mask=valid_mask, padding_idx=self.padding_idx, dtype=dtype)


__all__ = ["TokenEmbedding", "token_embedding", "token_embedding_reference"]
