"""Gated activation between two products, optionally quantised for the second one."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from . import _host
from .fused_moe import _ACTS

_plans: dict = {}
_fast = None          # the native host path, False without one


def _make_plan(x, activation, quantize):
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor: this package has no CPU path")
    act = _ACTS.get(activation)
    if act is None:
        raise ValueError(f"Unsupported activation: {activation}")
    assert x.dtype in _host.DTYPES, "x must be bfloat16, float16 or float32"
    assert x.dim() >= 1 and x.shape[-1] > 0 and x.shape[-1] % 2 == 0, "x must be [..., 2I]"
    i = _host.counted(x.shape[-1] // 2, _lib.ACT_MAX_I)
    _host.rows_of(x, 2 * i, _lib.MAX_ROWS)
    x2 = _host.as_rows(x, 2 * i)
    lead = tuple(x.shape[:-1])
    y, groups = lead + (i,), lead + (-(-i // 128),)
    plan = (act, i, x2.shape[0], _host.row_stride(x2, 2 * i), _host.DTYPES[x.dtype], x.device, x.device.index,
            y, _host.strides_of(y), _host.FP8 if quantize else x.dtype, groups, _host.strides_of(groups))
    return plan, x2


def gated_activation(
    x: torch.Tensor,
    activation: str = "silu",
    *,
    swiglu_alpha: float = 1.0,
    swiglu_limit: Optional[float] = None,
    quantize: bool = False,
):
    """``act(gate) * linear`` of rows ``x [..., 2I]`` that hold the gate half, then the linear half.

    ``activation``: "silu", "gelu" (the normal distribution's, not a tanh) or "swiglu_oai" (gate clamped from above and linear to
    ``[-limit, limit]`` where ``swiglu_limit`` is given and not zero, then ``g * sigmoid(alpha * g) * (linear + 1)``), as in ``fused_experts``.
    fp32 arithmetic, one rounding: to x's type, or with ``quantize`` to ``(q float8_e4m3fn [..., I], scale fp32 [..., ceil(I/128)])``.  Before
    it the result is within 2^-19 of itself, for 16-bit rows a further 2^-24 |alpha g| (GELU: 2^-24 g^2).  Rows to 2^31 - 256, I to
    65535 * 4096.  Forward only."""
    global _fast
    if _fast is None and torch.cuda.is_available():
        _fast = _host.fast()
    if _fast and activation in _ACTS:
        r = _fast.activation(_ACTS[activation], swiglu_alpha, swiglu_limit or 0.0, bool(quantize), x)
        if r is not None:
            if type(r) is int:
                _lib.check(r, "gated_activation")
            return r
    key = (x.shape, x.dtype, x.device, x.is_contiguous(), activation, bool(quantize))
    plan = _plans.get(key)
    if plan is None:
        plan, x = _make_plan(x, activation, quantize)
        if key[3]:
            _host.keep(_plans, key, plan)
    act, i, m, ldx, dtype, device, index, shape, strides, out, groups, group_strides = plan
    y = _host.empty(shape, strides, dtype=out, device=device)
    scale = _host.empty(groups, group_strides, dtype=torch.float32, device=device) if quantize else None
    if m:
        args = (x.data_ptr(), ldx, dtype, m, i, act, swiglu_alpha, swiglu_limit or 0.0, y.data_ptr(),
                scale.data_ptr() if quantize else None, _host.env_flags(1) if _lib.env_set() else 0, _host.raw_stream(index))
        if _host.current_device() == index:
            rc = _lib.lib().b200moe_gated_activation(*args)
        else:
            with torch.cuda.device(index):
                rc = _lib.lib().b200moe_gated_activation(*args)
        if rc != _lib.OK:
            _lib.check(rc, "gated_activation")
    return (y, scale) if quantize else y
