"""Linear attention with a decay per head: chunks for prompts and training, one step per token for serving.

Per sample and head, over the valid tokens in order (a masked token is as
though it were not there; its output is zero)::

    S_t = exp(log_decay) S_{t-1} + k_t v_t^T        y_t = scale * S_t^T q_t

``decay_attention`` runs whole sequences (and their gradients) in chunks on the
tensor cores, from a given state and to the last one when asked;
``decay_attention_step`` runs one token per sample on the state.  States are
FP32 ``[batch, heads, key, value]``.  The decay is a constant of the model:
its gradient is not computed (``decay_attention_reference`` has it).
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _native

_CHUNK = 64


def _check(q, k, v, log_decay, state, valid_mask, lead: int) -> None:
    """``lead``: leading dimensions of the tokens (2 = [batch, length], 1 = [batch])."""
    shape = ("batch", "length")[:lead]
    if q.ndim != lead + 2:
        raise ValueError(f"q must have shape [{', '.join(shape)}, heads, key], got {tuple(q.shape)}")
    if k.shape != q.shape:
        raise ValueError(f"k must have q's shape {tuple(q.shape)}, got {tuple(k.shape)}")
    if v.ndim != q.ndim or v.shape[:-1] != q.shape[:-1]:
        raise ValueError(f"v must have shape {tuple(q.shape[:-1])} + (value,), got {tuple(v.shape)}")
    batch, heads, key, value = q.shape[0], q.shape[-2], q.shape[-1], v.shape[-1]
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k and v must have one dtype, got {q.dtype}, {k.dtype} and {v.dtype}")
    if tuple(log_decay.shape) != (heads,):
        raise ValueError(f"log_decay must have shape {(heads,)}, got {tuple(log_decay.shape)}")
    if not log_decay.is_floating_point():
        raise TypeError(f"log_decay must be a floating-point tensor, got {log_decay.dtype}")
    if state is not None:
        if tuple(state.shape) != (batch, heads, key, value):
            raise ValueError(f"state must have shape {(batch, heads, key, value)}, got {tuple(state.shape)}")
    if valid_mask is not None:
        if valid_mask.shape != q.shape[:lead]:
            raise ValueError(f"valid_mask must have shape {tuple(q.shape[:lead])}, got {tuple(valid_mask.shape)}")
        if valid_mask.dtype != torch.bool:
            raise TypeError(f"valid_mask must have dtype torch.bool, got {valid_mask.dtype}")
    for name, value_ in (("k", k), ("v", v), ("log_decay", log_decay), ("state", state), ("valid_mask", valid_mask)):
        if value_ is not None and value_.device != q.device:
            raise RuntimeError(f"{name} must be on {q.device}, got {value_.device}")


def _check_cuda(name, q, k, v, log_decay, dtypes) -> None:
    if not q.is_cuda:
        raise ValueError(f"{name} requires CUDA tensors; use {name}_reference elsewhere")
    if q.dtype not in dtypes:
        raise TypeError(f"{name} supports {', '.join(str(d) for d in dtypes)}, got {q.dtype}")
    if log_decay.dtype != torch.float32:
        raise TypeError(f"log_decay must use torch.float32, got {log_decay.dtype}")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} does not compute the gradient of log_decay; detach it or use {name}_reference")
    for label, width in (("key", q.shape[-1]), ("value", v.shape[-1])):
        if width % 8 or not 8 <= width <= 128:
            raise ValueError(f"{name} supports {label} widths that are multiples of 8 from 8 to 128, got {width}")


_HALVES = frozenset((torch.bfloat16, torch.float16))


def _usual(q, k, v, log_decay, state, valid_mask, lead: int) -> bool:
    """Whether all of _check and _check_cuda but the types holds, in one expression (2 us less than asking one by one)."""
    shape, values, kind, device = q.shape, v.shape, q.dtype, q.device
    if len(shape) != lead + 2 or len(values) != lead + 2 or k.shape != shape or not q.is_cuda:
        return False
    batch, heads, key, value = shape[0], shape[-2], shape[-1], values[-1]
    return (values[:-1] == shape[:-1] and k.dtype is kind and v.dtype is kind and log_decay.dtype is torch.float32
            and log_decay.shape == (heads,) and 8 <= key <= 128 and 8 <= value <= 128 and not (key | value) % 8
            and k.device == device and v.device == device and log_decay.device == device
            and (state is None or (state.shape == (batch, heads, key, value) and state.device == device))
            and (valid_mask is None or (valid_mask.shape == shape[:lead] and valid_mask.dtype is torch.bool
                                        and valid_mask.device == device)))


def decay_attention_reference(q, k, v, log_decay, *, scale=None, state=None, valid_mask=None, return_state=False):
    """The same operator in PyTorch (any device; first-order autograd by PyTorch, the decay's gradient included)."""
    _check(q, k, v, log_decay, state, valid_mask, 2)
    batch, length, heads, key = q.shape
    value = v.shape[-1]
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    scale = key ** -0.5 if scale is None else scale
    mask = torch.ones(batch, length, dtype=torch.bool, device=q.device) if valid_mask is None else valid_mask
    pad = -length % _CHUNK

    def chunks(t):  # [B, H, chunks, 64, d], masked rows zero
        t = torch.where(mask[..., None, None], t.to(wide), torch.zeros((), dtype=wide, device=t.device))
        return torch.nn.functional.pad(t.transpose(1, 2), (0, 0, 0, pad)).unflatten(2, (-1, _CHUNK))

    live = torch.nn.functional.pad(mask, (0, pad)).unflatten(1, (-1, _CHUNK))[:, None]
    rank = live.to(wide).cumsum(-1)  # [B, 1, chunks, 64], counts the token itself
    rate = log_decay.to(wide).clamp_min(-1e4)[None, :, None, None]
    x, y, z = chunks(q) * scale, chunks(k), chunks(v)
    apart = rank[..., :, None] - rank[..., None, :]
    lower = torch.ones(_CHUNK, _CHUNK, dtype=torch.bool, device=q.device).tril() & live[..., None, :]
    weight = torch.where(lower, torch.exp(rate[..., None] * apart.clamp_min(0)), torch.zeros((), dtype=wide, device=q.device))
    out = (x @ y.mT * weight) @ z
    count = rank[..., -1:]
    added = (y * torch.exp(rate * (count - rank))[..., None]).mT @ z
    whole = torch.exp(rate * count)[..., None]
    into = torch.exp(rate * rank)[..., None]
    s = q.new_zeros((batch, heads, key, value), dtype=wide) if state is None else state.to(wide)
    before = []
    for c in range(added.shape[2]):
        before.append(s)
        s = s * whole[:, :, c] + added[:, :, c]
    if before:
        out = out + (x @ torch.stack(before, dim=2)) * into
    out = out.flatten(2, 3)[:, :, :length].transpose(1, 2)
    out = torch.where(mask[..., None, None], out, torch.zeros((), dtype=wide, device=q.device)).to(q.dtype)
    return (out, s.to(torch.promote_types(wide, torch.float32))) if return_state else out


def decay_attention_step_reference(q, k, v, log_decay, state, *, scale=None, valid_mask=None, new_state=None):
    """The same step in PyTorch (any device, no autograd): writes ``new_state`` (default: ``state``), returns y."""
    _check(q, k, v, log_decay, state, valid_mask, 1)
    with torch.no_grad():
        wide = state.dtype
        scale = q.shape[-1] ** -0.5 if scale is None else scale
        after = state * torch.exp(log_decay.to(wide))[:, None, None] + k.to(wide)[..., None] * v.to(wide)[..., None, :]
        y = (q.to(wide)[..., None] * after).sum(-2) * scale
        if valid_mask is not None:
            after = torch.where(valid_mask[:, None, None, None], after, state)
            y = torch.where(valid_mask[:, None, None], y, torch.zeros((), dtype=wide, device=y.device))
        (state if new_state is None else new_state).copy_(after)
        return y.to(q.dtype)


# ---------------------------------------------------------------------------- the native calls
_arrays: dict[tuple, ctypes.Array] = {}
_sizes: dict[tuple, int] = {}


def _array(strides: tuple) -> ctypes.Array:
    """Strides as the library takes them (made once per set of strides: 0.6 us each)."""
    found = _arrays.get(strides)
    if found is None:
        if len(_arrays) >= 4096:
            _arrays.clear()
        found = _arrays[strides] = (ctypes.c_int64 * len(strides))(*strides)
    return found


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, ctypes.Array]:
    """``t`` (copied if a tensor map cannot describe it) and its strides."""
    strides = t.stride()
    sb, sn, sh, sd = strides
    if sd == 1 and not (sb | sn | sh) % 8 and sb > 0 and sn > 0 and sh > 0 and not t.data_ptr() % 16:
        return t, _array(strides[:3])
    b, n, h, d = t.shape
    for _ in range(2):
        sb, sn, sh, sd = t.stride()
        # the stride of an axis of one is never used: any allowed value
        sh = d if h == 1 else sh
        sn = h * d if n == 1 else sn
        sb = n * h * d if b == 1 else sb
        if sd == 1 and min(sb, sn, sh) > 0 and not (sb | sn | sh) % 8 and not t.data_ptr() % 16:
            return t, _array((sb, sn, sh))
        t = t.clone(memory_format=torch.contiguous_format)
    raise RuntimeError("a fresh tensor was not aligned to 16 bytes")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _workspace(device: torch.device, sizes: tuple, backward: bool) -> tuple[int | None, int, torch.Tensor | None]:
    """Pointer, bytes and owner of a call's scratch (none where the sequences are not cut)."""
    key = (device.index, *sizes, backward)
    size = _sizes.get(key)
    if size is None:
        lib = _native.library()
        with torch.cuda.device(device):
            size = lib.lib.lsso_decay_workspace_size(*sizes, int(backward))
        if size == 0:
            lib.check(1)
        if len(_sizes) >= 4096:
            _sizes.clear()
        _sizes[key] = size
    if size <= 16:
        return None, 0, None
    scratch = torch.empty((size,), dtype=torch.uint8, device=device)
    return scratch.data_ptr(), size, scratch


def _forward(q, k, v, log_decay, scale, state, mask, return_state):
    batch, length, heads, key = q.shape
    value = v.shape[3]
    y = q.new_empty((batch, length, heads, value))
    last = None
    if return_state:
        last = torch.empty((batch, heads, key, value), dtype=torch.float32, device=q.device)
    if not y.numel():
        if last is not None:
            last.zero_() if state is None else last.copy_(state)
        return y, last
    (q, qs), (k, ks), (v, vs), (_, ys) = _rows(q), _rows(k), _rows(v), _rows(y)
    sizes = (batch, length, heads, key, value)
    device = q.device
    scratch, scratch_bytes, _owner = _workspace(device, sizes, False)
    _native.run("lsso_decay_forward", device, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
                _native.ELEMENT_TYPES[q.dtype], log_decay.data_ptr(), _native._ptr(mask), *sizes, scale,
                _native._ptr(state), _native._ptr(last), y.data_ptr(), ys, scratch, scratch_bytes)
    return y, last


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, scale, state, mask, return_state):
        ctx.set_materialize_grads(False)
        y, last = _forward(q, k, v, log_decay, scale, state, mask, return_state)
        ctx.save_for_backward(q, k, v, log_decay, state, mask)
        ctx.scale = scale
        return (y, last) if return_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast=None):
        q, k, v, log_decay, state, mask = ctx.saved_tensors
        batch, length, heads, key = q.shape
        value = v.shape[-1]
        needs_state = state is not None and ctx.needs_input_grad[5]
        dstate = torch.empty_like(state) if needs_state else None
        new = lambda like: like.new_empty(like.shape)  # noqa: E731
        dq, dk, dv = new(q), new(k), new(v)
        if not v.numel():
            if needs_state:
                dstate.zero_() if dlast is None else dstate.copy_(dlast)
            return dq, dk, dv, None, None, dstate, None, None
        if dy is None:
            dy = torch.zeros_like(v, memory_format=torch.contiguous_format)
        dlast = None if dlast is None else _aligned(dlast)
        (q, qs), (k, ks), (v, vs), (dy, ys) = _rows(q), _rows(k), _rows(v), _rows(dy)
        (dq, dqs), (dk, dks), (dv, dvs) = _rows(dq), _rows(dk), _rows(dv)
        sizes = (batch, length, heads, key, value)
        scratch, scratch_bytes, _owner = _workspace(q.device, sizes, True)
        _native.run("lsso_decay_backward", q.device, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, dy.data_ptr(),
                    ys, _native.ELEMENT_TYPES[q.dtype], log_decay.data_ptr(), _native._ptr(mask), *sizes, ctx.scale,
                    _native._ptr(state), _native._ptr(dlast), dq.data_ptr(), dqs, dk.data_ptr(), dks, dv.data_ptr(), dvs,
                    _native._ptr(dstate), scratch, scratch_bytes)
        return dq, dk, dv, None, None, dstate, None, None


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *,
                    scale: float | None = None, state: torch.Tensor | None = None,
                    valid_mask: torch.Tensor | None = None, return_state: bool = False):
    """Causal linear attention over ``[batch, length, heads, ..]``: y, or ``(y, last state)``.

    ``q``, ``k`` ``[batch, length, heads, key]`` and ``v`` ``[.., value]`` are
    BF16 or FP16 with widths that are multiples of 8 from 8 to 128;
    ``log_decay`` ``[heads]`` FP32, at most zero in use (``-inf``: a token sees
    itself alone; above zero the state grows, as far as the types reach; FP16
    heads below -0.076 take the slower of two paths); ``scale`` defaults to
    ``key ** -0.5``; ``state`` FP32 ``[batch, heads, key, value]`` precedes the first token (default zero);
    ``valid_mask`` is bool ``[batch, length]``.  What masked tokens hold does
    not matter; a valid token that is not finite may spoil the outputs of its
    128-token chunk before it, too.  Views whose strides are multiples of 8
    elements (slices of a packed projection) are read in place, others copied.
    Gradients: q, k, v and state.
    """
    _native.refuse_transforms("decay_attention", q, k, v, log_decay, state, valid_mask)
    if not _usual(q, k, v, log_decay, state, valid_mask, 2):
        _check(q, k, v, log_decay, state, valid_mask, 2)
        _check_cuda("decay_attention", q, k, v, log_decay, (torch.bfloat16, torch.float16))
    elif q.dtype not in _HALVES or (log_decay.requires_grad and torch.is_grad_enabled()):
        _check_cuda("decay_attention", q, k, v, log_decay, (torch.bfloat16, torch.float16))
    if state is not None and state.dtype != torch.float32:
        raise TypeError(f"state must use torch.float32, got {state.dtype}")
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    log_decay = log_decay.contiguous()
    state = None if state is None else _aligned(state)
    mask = None if valid_mask is None else valid_mask.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (state is not None and state.requires_grad)):
        return _DecayAttention.apply(q, k, v, log_decay, scale, state, mask, return_state)
    y, last = _forward(q, k, v, log_decay, scale, state, mask, return_state)
    return (y, last) if return_state else y


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                         state: torch.Tensor, *, scale: float | None = None, valid_mask: torch.Tensor | None = None,
                         new_state: torch.Tensor | None = None) -> torch.Tensor:
    """One token per sample: updates ``state`` in place, returns y ``[batch, heads, value]``.

    ``q``, ``k`` ``[batch, heads, key]`` and ``v`` ``[batch, heads, value]``
    are BF16, FP16 or FP32; ``state`` is FP32 ``[batch, heads, key, value]``,
    contiguous.  ``new_state`` (optional, like ``state`` and apart from it)
    receives the new state and ``state`` stays as it is.  Samples whose
    ``valid_mask`` ``[batch]`` is unset keep their state and give zero rows.
    Not differentiable: train with :func:`decay_attention`.
    """
    _native.refuse_transforms("decay_attention_step", q, k, v, log_decay, state, valid_mask)
    kind, device = q.dtype, q.device
    if not _usual(q, k, v, log_decay, state, valid_mask, 1) or kind not in _native.ELEMENT_TYPES or log_decay.requires_grad:
        _check(q, k, v, log_decay, state, valid_mask, 1)
        _check_cuda("decay_attention_step", q, k, v, log_decay, (torch.bfloat16, torch.float16, torch.float32))
    target = state if new_state is None else new_state
    for name, value in (("state", state),) if new_state is None else (("state", state), ("new_state", new_state)):
        if value.dtype is not torch.float32 or value.shape != state.shape or value.device != device:
            raise ValueError(f"{name} must be FP32 {tuple(state.shape)} on {device}, got {value.dtype} "
                             f"{tuple(value.shape)} on {value.device}")
        if not value.is_contiguous():
            raise RuntimeError(f"decay_attention_step requires a contiguous {name}")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad
                                    or target.requires_grad):
        raise ValueError("decay_attention_step has no gradient; call it under torch.no_grad() or use decay_attention")
    batch, heads, key = q.shape
    value = v.shape[2]
    y = q.new_empty((batch, heads, value))
    if not y.numel():
        return y
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    if qs[2] != 1 or ks[2] != 1 or vs[2] != 1:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        qs, ks, vs = q.stride(), k.stride(), v.stride()
    if not log_decay.is_contiguous():
        log_decay = log_decay.contiguous()
    if valid_mask is not None and not valid_mask.is_contiguous():
        valid_mask = valid_mask.contiguous()
    at = state.data_ptr()
    _native.run("lsso_decay_step", device, q.data_ptr(), _array(qs[:2]), k.data_ptr(), _array(ks[:2]), v.data_ptr(),
                _array(vs[:2]), _native.ELEMENT_TYPES[kind], log_decay.data_ptr(), _native._ptr(valid_mask), batch, heads,
                key, value, key ** -0.5 if scale is None else scale, at, at if new_state is None else new_state.data_ptr(),
                y.data_ptr())
    if not target.is_inference():
        increment_version(target)  # a graph that kept it for its backward says so
    return y


__all__ = ["decay_attention", "decay_attention_reference", "decay_attention_step", "decay_attention_step_reference"]
