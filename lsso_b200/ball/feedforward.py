"""Gated feed-forward block of the token shell.

``gated_feed_forward(x, w_in, w_out)`` is ``(act(g) * u) w_out^T`` with
``[g | u] = x w_in^T``: ``w_in`` ``[2 hidden, dim]`` holds the gate rows, then
the up rows.  Both projections, the activation and the product are one tcgen05
kernel; a training forward keeps ``[g | u]`` (in FP16 at most +-65504) and the
product.  Operands have x's dtype (BF16 or FP16), products accumulate in FP32.  FP32 weights are rounded
to x's dtype in the call and get FP32 gradients; weights that already have x's
dtype (a served model's, laid out once) are used in place.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import nn
from torch.autograd.function import once_differentiable

from . import _native

_ACTIVATIONS = {"silu": 0, "gelu": 1}


def _check(x, w_in, w_out, b_in, b_out, activation) -> None:
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if w_in.ndim != 2 or w_in.shape[0] % 2 or 0 in w_in.shape:
        raise ValueError(f"w_in must have shape [2 * hidden, dim], got {tuple(w_in.shape)}")
    hidden, dim = w_in.shape[0] // 2, w_in.shape[1]
    if tuple(w_out.shape) != (dim, hidden):
        raise ValueError(f"w_out must have shape {(dim, hidden)}, got {tuple(w_out.shape)}")
    if x.ndim < 1 or x.shape[-1] != dim:
        raise ValueError(f"x must have shape [.., {dim}], got {tuple(x.shape)}")
    for name, value, shape in (("b_in", b_in, (2 * hidden,)), ("b_out", b_out, (dim,))):
        if value is not None and tuple(value.shape) != shape:
            raise ValueError(f"{name} must have shape {shape}, got {tuple(value.shape)}")
    for name, value in (("w_in", w_in), ("w_out", w_out), ("b_in", b_in), ("b_out", b_out)):
        if value is not None and value.device != x.device:
            raise RuntimeError(f"{name} must be on {x.device}, got {value.device}")


def gated_feed_forward_reference(x, w_in, w_out, b_in=None, b_out=None, *, activation="silu") -> torch.Tensor:
    """The same operator in PyTorch (any device), in FP32 or FP64, rounded once."""
    _check(x, w_in, w_out, b_in, b_out, activation)
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    cast = lambda t: None if t is None else t.to(wide)  # noqa: E731
    with torch.autocast(device_type=x.device.type, enabled=False):
        g, u = F.linear(x.to(wide), cast(w_in), cast(b_in)).chunk(2, dim=-1)
        h = (F.silu(g) if activation == "silu" else F.gelu(g)) * u
        return F.linear(h, cast(w_out), cast(b_out)).to(x.dtype)


def _forward(x, w_in, w_out, b_in, b_out, activation, keep):
    """(y, kept, h) for x [T, D]; kept (g and u, for the backward) is None unless ``keep``."""
    types = _native.ELEMENT_TYPES
    t, d = x.shape
    hidden = w_out.shape[1]
    bias = b_in if b_in is not None else b_out
    h = x.new_empty((t, hidden))
    kept = x.new_empty((t, 2, hidden)) if keep else None
    y = torch.empty_like(x)
    _native.run("lsso_ffn_forward", x.device, x.data_ptr(), types[x.dtype], t, d, hidden, w_in.data_ptr(),
                w_out.data_ptr(), types[w_in.dtype], _native._ptr(b_in), _native._ptr(b_out),
                2 if bias is None else types[bias.dtype], activation, _native._ptr(kept), h.data_ptr(), y.data_ptr())
    return y, kept, h


def _cast(w_in, w_out, dtype):
    """Both weights in ``dtype`` (one launch when they are FP32)."""
    if w_in.dtype == dtype:
        return w_in, w_out
    a, b = torch.empty_like(w_in, dtype=dtype), torch.empty_like(w_out, dtype=dtype)
    _native.run("lsso_ffn_cast", w_in.device, w_in.data_ptr(), a.data_ptr(), w_in.numel(), w_out.data_ptr(),
                b.data_ptr(), w_out.numel(), _native.ELEMENT_TYPES[dtype])
    return a, b


class _GatedFeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out, b_in, b_out, activation):
        a, b = _cast(w_in, w_out, x.dtype)
        y, kept, h = _forward(x, a, b, b_in, b_out, activation, True)
        ctx.save_for_backward(x, kept, h, a, b)
        ctx.activation, ctx.weight_dtype = activation, w_in.dtype
        ctx.bias_dtype = next((v.dtype for v in (b_in, b_out) if v is not None), w_in.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, kept, h, w_in, w_out = ctx.saved_tensors
        types = _native.ELEMENT_TYPES
        needs = ctx.needs_input_grad
        device, kind, bias_kind = x.device, ctx.weight_dtype, ctx.bias_dtype
        (t, d), hidden = x.shape, h.shape[1]
        dy = _aligned(dy.contiguous())
        dx = torch.empty_like(x) if needs[0] else None
        dw_in = torch.empty_like(w_in, dtype=kind) if needs[1] else None
        dw_out = torch.empty_like(w_out, dtype=kind) if needs[2] else None
        db_in = x.new_empty((2 * hidden,), dtype=bias_kind) if needs[3] else None
        db_out = x.new_empty((d,), dtype=bias_kind) if needs[4] else None
        scratch = _native.workspace("lsso_ffn_backward_workspace_size", device, t, d, hidden)
        _native.run("lsso_ffn_backward_mixed", device, dy.data_ptr(), x.data_ptr(), kept.data_ptr(), h.data_ptr(),
                    w_in.data_ptr(), w_out.data_ptr(), types[x.dtype], t, d, hidden, ctx.activation, types[kind],
                    types[bias_kind], _native._ptr(dx), _native._ptr(dw_in), _native._ptr(dw_out),
                    _native._ptr(db_in), _native._ptr(db_out), scratch.data_ptr(), scratch.numel())
        return dx, dw_in, dw_out, db_in, db_out, None


def gated_feed_forward(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, b_in: torch.Tensor | None = None,
                       b_out: torch.Tensor | None = None, *, activation: str = "silu") -> torch.Tensor:
    """``(act(g) * u) w_out^T + b_out`` with ``[g | u] = x w_in^T + b_in``, in x's dtype.

    ``x`` ``[.., dim]`` is BF16 or FP16; both weights are FP32 or have x's
    dtype, contiguous; the biases have one of these dtypes, the same for both.
    ``activation`` is ``"silu"`` or ``"gelu"`` (by erf).  Widths that are not
    multiples of 8 are padded with zeros (copies of x and the weights).
    Without gradients, one row (or a few of a small block) streams the weights,
    FP32 ones rounded as they are read; otherwise the tensor-core path runs.
    """
    _native.refuse_transforms("gated_feed_forward", x, w_in, w_out, b_in, b_out)
    _check(x, w_in, w_out, b_in, b_out, activation)
    if not x.is_cuda:
        raise ValueError("gated_feed_forward requires CUDA tensors; use gated_feed_forward_reference elsewhere")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"gated_feed_forward supports x with dtype torch.bfloat16 or torch.float16, got {x.dtype}")
    if w_in.dtype != w_out.dtype or w_in.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"w_in and w_out must both use {x.dtype} or torch.float32, got {w_in.dtype} and {w_out.dtype}")
    biases = [b.dtype for b in (b_in, b_out) if b is not None]
    if any(b not in (x.dtype, torch.float32) for b in biases) or len(set(biases)) > 1:
        raise TypeError(f"b_in and b_out must both use {x.dtype} or torch.float32, got {biases}")
    for name, value in (("w_in", w_in), ("w_out", w_out), ("b_in", b_in), ("b_out", b_out)):
        if value is not None and not value.is_contiguous():
            raise RuntimeError(f"gated_feed_forward requires contiguous {name}")
    hidden, dim = w_out.shape[1], x.shape[-1]
    shape = x.shape
    rows = x.numel() // dim
    if rows == 0:
        # no rows: no work; gradients (zeros) through PyTorch
        return gated_feed_forward_reference(x, w_in, w_out, b_in, b_out, activation=activation)
    extra_d, extra_h = -dim % 8, -hidden % 8
    if extra_d or extra_h:
        x = F.pad(x, (0, extra_d))
        w_in = F.pad(w_in.view(2, hidden, dim), (0, extra_d, 0, extra_h)).reshape(-1, dim + extra_d)
        w_out = F.pad(w_out, (0, extra_h, 0, extra_d))
        b_in = None if b_in is None else F.pad(b_in.view(2, hidden), (0, extra_h)).reshape(-1)
        b_out = None if b_out is None else F.pad(b_out, (0, extra_d))
    if x.ndim != 2 or not x.is_contiguous():
        x = x.reshape(rows, dim + extra_d).contiguous()
    x, w_in, w_out = _aligned(x), _aligned(w_in), _aligned(w_out)
    act = _ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (x.requires_grad or w_in.requires_grad or w_out.requires_grad
                                    or any(b is not None and b.requires_grad for b in (b_in, b_out))):
        y = _GatedFeedForward.apply(x, w_in, w_out, b_in, b_out, act)
    else:
        if w_in.dtype != x.dtype and not _native.library().lib.lsso_ffn_streams_weights(rows, dim + extra_d,
                                                                                         hidden + extra_h):
            w_in, w_out = _cast(w_in, w_out, x.dtype)
        y = _forward(x, w_in, w_out, b_in, b_out, act, False)[0]
    if extra_d:
        y = y[:, :dim]
    return y if y.shape == shape else y.reshape(shape)


def _aligned(value: torch.Tensor) -> torch.Tensor:
    """The tensor, or a copy where its first element is not on a 16-byte boundary."""
    return value if value.data_ptr() % 16 == 0 else value.clone()


class GatedFeedForward(nn.Module):
    """``w_out (act(w_gate x) * w_up x)`` with FP32 parameters: ``w_in`` packs the gate and up rows."""

    def __init__(self, dim: int, hidden: int, *, activation: str = "silu", bias: bool = False) -> None:
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
        if dim < 1 or hidden < 1:
            raise ValueError(f"dim and hidden must be positive, got {dim} and {hidden}")
        self.activation = activation
        self.w_in = nn.Linear(dim, 2 * hidden, bias=bias)
        self.w_out = nn.Linear(hidden, dim, bias=bias)

    def forward(self, x: torch.Tensor, *, implementation: str = "reference") -> torch.Tensor:
        if implementation not in ("reference", "cuda"):
            raise ValueError(f"implementation must be 'reference' or 'cuda', got {implementation!r}")
        run = gated_feed_forward if implementation == "cuda" else gated_feed_forward_reference
        return run(x, self.w_in.weight, self.w_out.weight, self.w_in.bias, self.w_out.bias, activation=self.activation)


__all__ = ["GatedFeedForward", "gated_feed_forward", "gated_feed_forward_reference"]
