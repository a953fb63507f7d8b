"""Norms before and after a block, fused with the block's gate, the residual scale and the residual add, and with the FP8
quantisation that the next block's projections start from."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from . import _host

_KINDS = {"rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER}
_plans: dict = {}
_fast = None          # the native host path, False without one


class _Plan:
    __slots__ = ("desc", "addr", "index", "rows", "hidden", "y", "scale", "device")


def _vector(v: Optional[torch.Tensor], name: str, h: int, x: torch.Tensor) -> Optional[torch.Tensor]:
    if v is None:
        return None
    assert v.shape == (h,) and v.device == x.device, f"{name} must be [H] on x's device"
    assert v.dtype in (x.dtype, torch.float32), f"{name} must have x's type or float32"
    return v.contiguous()


def _gate(gate: Optional[torch.Tensor], x: torch.Tensor, h: int):
    """(mode, tensor, row stride)"""
    if gate is None:
        return _lib.GATE_NONE, None, 0
    assert gate.device == x.device, "gate must be on x's device"
    assert gate.dtype in (x.dtype, torch.float32), "gate must have x's type or float32"
    if gate.shape == (h,):
        return _lib.GATE_CHANNEL, gate.contiguous(), 0
    if gate.shape == x.shape and h > 1:
        g = _host.as_rows(gate, h)
        return _lib.GATE_FULL, g, _host.row_stride(g, h)
    if gate.shape == x.shape[:-1] + (1,):
        g = gate.reshape(-1)
        if g.numel() > 1 and g.stride(0) < 1:
            g = g.contiguous()
        return _lib.GATE_TOKEN, g, g.stride(0) if g.numel() > 1 else 1
    raise ValueError("gate must be [H] (per channel), [..., 1] (per token) or [..., H]")


def _distinct(t: torch.Tensor) -> bool:
    """No two elements of ``t`` share memory (each stride, in order of size, passes over all that lies below it)."""
    reach = 0
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda d: d[1]):
        if stride <= reach:
            return False
        reach += (size - 1) * stride
    return True


def _make_plan(x, post, pre, w_post, b_post, w_pre, b_pre, residual, gate, residual_scale, eps, kind, weight_offset, quantize,
               inplace, flags):
    """Checks one call; returns its plan and the tensors whose addresses the kernel gets."""
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor: this package has no CPU path")
    if kind not in _KINDS:
        raise ValueError(f"Unsupported norm: {kind}")
    assert x.dtype in _host.DTYPES, "x must be bfloat16, float16 or float32"
    assert x.dim() >= 1 and x.shape[-1] > 0, "x must be [..., H]"
    assert eps >= 0, "eps must not be negative"
    h = x.shape[-1]
    if h > _lib.NORM_MAX_H:
        raise ValueError(f"rows of more than {_lib.NORM_MAX_H} elements are not supported")
    _host.rows_of(x, h, _lib.NORM_MAX_ROWS)
    if residual is not None:
        assert residual.shape == x.shape and residual.device == x.device, "residual must have x's shape and device"
        assert residual.dtype in (x.dtype, torch.float32), "residual must have x's type or float32"
    w_post, b_post = _vector(w_post, "weight", h, x), _vector(b_post, "bias", h, x)
    w_pre, b_pre = _vector(w_pre, "weight", h, x), _vector(b_pre, "bias", h, x)
    mode, gate, ldg = _gate(gate, x, h)
    x2 = _host.as_rows(x, h)
    r2 = None if residual is None else _host.as_rows(residual, h)
    if inplace:
        assert residual is not None, "inplace needs a residual"
        assert x.numel() == 0 or (r2.data_ptr() == residual.data_ptr() and _distinct(residual)), \
            "inplace needs a residual with contiguous rows that do not overlap"
    p = _Plan()
    m = x2.shape[0]
    rdt = x.dtype if residual is None else residual.dtype
    p.index, p.device, p.rows = x.device.index, x.device, m
    shape = tuple(x.shape)
    strides = _host.strides_of(shape)
    p.hidden = (shape, strides, rdt)
    if not post and residual is None and gate is None and residual_scale == 1.0:
        p.hidden = None             # the rows themselves
    p.y = p.scale = None
    if pre:
        p.y = (shape, strides, _host.FP8 if quantize else x.dtype)
        if quantize:
            groups = shape[:-1] + (-(-h // 128),)
            p.scale = (groups, _host.strides_of(groups), torch.float32)
    dt = lambda t: 0 if t is None else _host.DTYPES[t.dtype]                       # noqa: E731
    p.desc, p.addr = _host.struct(
        _lib.Norm, m, h, _KINDS[kind], _host.DTYPES[x.dtype], _host.DTYPES[rdt], post, pre, mode, dt(gate), dt(w_post), dt(b_post),
        dt(w_pre), dt(b_pre), flags, eps, residual_scale, weight_offset, _host.row_stride(x2, h), _host.row_stride(r2, h), ldg,
        _host.row_stride(r2, h) if inplace else h)
    return p, (x2, r2, gate, w_post, b_post, w_pre, b_pre)


def _block_norm(x, post, pre, w_post, b_post, w_pre, b_pre, residual, gate, residual_scale, eps, kind, weight_offset, quantize,
                inplace):
    global _fast
    if _fast is None and torch.cuda.is_available():
        _fast = _host.fast()
    if _fast and kind in _KINDS:
        r = _fast.norm(post, pre, kind == "layer", quantize, inplace, residual_scale, eps, weight_offset, x, residual, gate, w_post, b_post,
                       w_pre, b_pre)
        if r is not None:
            if type(r) is int:
                _lib.check(r, "block_norm")
            return r
    residual_scale, eps, weight_offset = float(residual_scale), float(eps), float(weight_offset)
    flags = _host.env_flags(1) if _lib.env_set() else 0
    tensors = (x, residual, gate, w_post, b_post, w_pre, b_pre)
    key = (post, pre, kind, residual_scale, eps, weight_offset, quantize, inplace, flags,
           (x.shape, x.dtype, x.device, x.is_contiguous()),
           None if residual is None else (residual.shape, residual.dtype, residual.device, residual.is_contiguous()),
           None if gate is None else (gate.shape, gate.dtype, gate.device, gate.is_contiguous()),
           None if w_post is None else (w_post.shape, w_post.dtype, w_post.device, w_post.is_contiguous()),
           None if b_post is None else (b_post.shape, b_post.dtype, b_post.device, b_post.is_contiguous()),
           None if w_pre is None else (w_pre.shape, w_pre.dtype, w_pre.device, w_pre.is_contiguous()),
           None if b_pre is None else (b_pre.shape, b_pre.dtype, b_pre.device, b_pre.is_contiguous()))
    p = _plans.get(key)
    if p is None:
        p, tensors = _make_plan(x, post, pre, w_post, b_post, w_pre, b_pre, residual, gate, residual_scale, eps, kind,
                                weight_offset, quantize, inplace, flags)
        if all(k is None or k[3] for k in key[9:]):
            _host.keep(_plans, key, p)      # (every tensor contiguous: what the call gets is what the kernel gets)
    empty, device = _host.empty, p.device
    if inplace:
        hidden = residual
    elif p.hidden is None:
        hidden = None
    else:
        shape, strides, dtype = p.hidden
        hidden = empty(shape, strides, dtype=dtype, device=device)
    y = scale = None
    if pre:
        shape, strides, dtype = p.y
        y = empty(shape, strides, dtype=dtype, device=device)
        if quantize:
            shape, strides, dtype = p.scale
            scale = empty(shape, strides, dtype=dtype, device=device)
    if p.rows:
        x2, residual, gate, w_post, b_post, w_pre, b_pre = tensors
        args = (p.addr, x2.data_ptr(), None if residual is None else residual.data_ptr(), None if gate is None else gate.data_ptr(),
                None if w_post is None else w_post.data_ptr(), None if b_post is None else b_post.data_ptr(),
                None if w_pre is None else w_pre.data_ptr(), None if b_pre is None else b_pre.data_ptr(),
                None if hidden is None else hidden.data_ptr(), y.data_ptr() if pre else None, scale.data_ptr() if quantize else None, _host.raw_stream(p.index))
        if _host.current_device() == p.index:
            rc = _lib.lib().b200moe_block_norm(*args)
        else:
            with torch.cuda.device(device):
                rc = _lib.lib().b200moe_block_norm(*args)
        if rc != _lib.OK:
            _lib.check(rc, "block_norm")
    return (y, scale) if quantize else y, x if hidden is None else hidden


def norm_before_block(
    x: torch.Tensor,
    weight: Optional[torch.Tensor],
    *,
    bias: Optional[torch.Tensor] = None,
    residual: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    residual_scale: float = 1.0,
    eps: float = 1e-6,
    kind: str = "rms",
    weight_offset: float = 0.0,
    quantize: bool = False,
    inplace: bool = False,
):
    """The last block's output ``x [..., H]`` joins the residual stream, which is normalised for the next block::

        hidden = residual + residual_scale * gate * x           (no residual: residual_scale * gate * x)
        y      = norm(hidden) * (weight_offset + weight) + bias

    ``kind``: "rms" or "layer".  Returns ``(y, hidden)``; with ``quantize`` ``y`` is the pair ``(q float8_e4m3fn, scale
    fp32 [..., ceil(H/128)])`` that ``fp8_block_linear`` and ``fused_experts`` take.  ``weight_offset=1`` is the convention of
    the reference's Gemma norms (src/flaggems_sglang/ops/gemma_rms_norm.py:18-117).

    ``gate``: ``[H]`` per channel, ``[..., 1]`` per token or ``[..., H]``.  ``residual`` has x's type or float32, and ``hidden`` has
    the residual's; ``inplace`` writes ``hidden`` over ``residual`` (x and residual are then the same rows or share none, and
    neither gate nor vectors share memory with residual).  Without residual, gate and scale ``hidden`` is ``x`` itself.  All
    arithmetic is fp32; ``y`` is taken from ``hidden`` before that is rounded; a layer norm's rows may have a mean that is large against their
    deviation.  Vectors and gate have x's type or float32; ``weight=None`` is a norm without weights.  H up to 16384, rows up to 2^30;
    a 1-D gate of H elements is per channel whatever the number of rows.  A NaN or an infinity concerns its own row only
    (quantised: a group's scale is that of its numbers, its values are what the formula gives).  Forward only: no gradient is recorded."""
    return _block_norm(x, False, True, None, None, weight, bias, residual, gate, residual_scale, eps, kind, weight_offset,
                       bool(quantize), bool(inplace))


def norm_after_block(
    x: torch.Tensor,
    weight: Optional[torch.Tensor],
    *,
    bias: Optional[torch.Tensor] = None,
    residual: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    residual_scale: float = 1.0,
    eps: float = 1e-6,
    kind: str = "rms",
    weight_offset: float = 0.0,
    next_norm: bool = False,
    next_weight: Optional[torch.Tensor] = None,
    next_bias: Optional[torch.Tensor] = None,
    quantize: bool = False,
    inplace: bool = False,
):
    """A block's output is normalised before it joins the residual stream::

        hidden = residual + residual_scale * gate * (norm(x) * (weight_offset + weight) + bias)

    Returns ``hidden``; with ``next_weight`` (or ``next_norm=True`` for a norm without weights) also the next block's input, as
    ``(norm(hidden) * (weight_offset + next_weight) + next_bias, hidden)`` in one pass over the rows.  The other arguments are those
    of ``norm_before_block``; ``quantize`` concerns the next block's input."""
    following = bool(next_norm) or next_weight is not None
    assert following or (next_bias is None and not quantize), "next_bias and quantize need next_weight or next_norm=True"
    y, hidden = _block_norm(x, True, following, weight, bias, next_weight, next_bias, residual, gate, residual_scale, eps, kind,
                            weight_offset, bool(quantize), bool(inplace))
    return (y, hidden) if following else hidden
