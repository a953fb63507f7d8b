"""Linear layer with block-quantised FP8 weights: the projections that stand around the experts of such a model (shared
expert, dense layers, attention), on the weights' own 128 x 128 block scales."""
from __future__ import annotations

import os
from typing import Optional

import torch

from .. import _lib
from . import _host
from .fused_moe import _deferred_status_check, _status_word, check_status

_plans: dict = {}
_fast = None          # the native host path, False without one


class _Plan:
    __slots__ = ("desc", "addr", "index", "device", "rows", "out", "work")


def _aligned_rows(x: torch.Tensor, k: int) -> torch.Tensor:
    """``x`` as [rows, k] with contiguous rows that start on 16 bytes; copied where they do not."""
    x = x if x.dim() == 2 else x.reshape(-1, k)
    if (x.stride(1) != 1 and k != 1) or (x.shape[0] > 1 and (x.stride(0) < k or x.stride(0) * x.element_size() % 16)) or \
            x.data_ptr() % 16:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x)
    return x


def _make_plan(x, weight, weight_scale, bias, x_scale, out_dtype, tile, split, flags):
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor: this package has no CPU path")
    assert weight.dim() == 2 and weight.dtype == _host.FP8, "weight must be [N, K] float8_e4m3fn"
    n, k = weight.shape
    dev = x.device
    assert x.dim() >= 1 and x.shape[-1] == k, "x and weight differ in K"
    assert n > 0 and k > 0 and k % 16 == 0, "K must be a multiple of 16"
    _host.counted(n, _lib.MAX_ROWS)
    _host.rows_of(x, _host.counted(k, _lib.LINEAR_MAX_K), _lib.MAX_ROWS)
    g = -(-k // 128)
    assert weight.device == dev and weight_scale.device == dev, "x, weight and weight_scale must be on one device"
    assert weight_scale.shape == (-(-n // 128), g), "weight_scale must be [ceil(N/128), ceil(K/128)]"
    assert weight.stride(1) == 1 and (n == 1 or (weight.stride(0) >= k and weight.stride(0) % 16 == 0)), \
        "weight rows must be contiguous and start on 16 bytes"
    if x.dtype == _host.FP8:
        assert x_scale is not None, "float8_e4m3fn x needs x_scale"
        assert x_scale.shape == x.shape[:-1] + (g,) and x_scale.device == dev, "x_scale must be [..., ceil(K/128)] on x's device"
        odt, xdt = out_dtype or torch.bfloat16, _lib.X_E4M3
    else:
        assert x_scale is None, "x_scale goes with float8_e4m3fn x"
        assert x.dtype in (torch.bfloat16, torch.float16), "x must be bfloat16, float16 or float8_e4m3fn"
        odt, xdt = out_dtype or x.dtype, _host.DTYPES[x.dtype]
    if odt not in _host.DTYPES:
        raise ValueError(f"Unsupported output type: {odt}")
    if bias is not None:
        assert bias.shape == (n,) and bias.device == dev, "bias must be [N] on x's device"
        assert bias.dtype in _host.DTYPES, "bias must be bfloat16, float16 or float32"
    x2 = _aligned_rows(x, k)
    p = _Plan()
    m = x2.shape[0]
    shape = tuple(x.shape[:-1]) + (n,)
    p.index, p.device, p.rows, p.out = dev.index, dev, m, (shape, _host.strides_of(shape), odt)
    p.desc, p.addr = _host.struct(_lib.Linear, m, n, k, xdt, _host.DTYPES[odt], 0 if bias is None else _host.DTYPES[bias.dtype], flags,
                                  tile, split, 0, _host.row_stride(x2, k), weight.stride(0) if n > 1 else k)
    with torch.cuda.device(dev):        # (the library asks the current device what it holds)
        p.work = _lib.lib().b200moe_fp8_linear_workspace_bytes(p.addr)
    return p, x2


def fp8_block_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    *,
    x_scale: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
    tile: int = 0,
    split: int = 0,
) -> torch.Tensor:
    """``x [..., K] @ weight[N, K].T + bias`` with ``float8_e4m3fn`` weights and one fp32 scale per 128 x 128 block.

    ``weight_scale``: ``[ceil(N/128), ceil(K/128)]`` (``quant.quantize_fp8_block`` makes both for stacked weights).  ``x`` is
    bfloat16 or float16 and is quantised per 1 x 128 group within the call, with the bits that ``per_token_group_quant_fp8``
    gives; or it is ``float8_e4m3fn`` already, with its scales ``x_scale [..., ceil(K/128)]``, as ``norm_before_block`` and
    ``gated_activation`` return them with ``quantize=True``.  The sums are fp32 and rounded once, to ``out_dtype`` (default:
    the type of a 16-bit ``x``, else bfloat16; float32 is possible).  ``bias``: ``[N]``.

    K is a multiple of 16 up to 65536, N and the rows up to 2^31 - 256, no rows are an empty result.  ``weight`` may have strided rows that start on
    16 bytes; rows of ``x`` that do not are copied.  A NaN or an infinity makes its own row of the result NaN and no other.
    Forward only: no gradient is recorded.  ``tile`` / ``split`` pick the kernel by hand (tuning aid)."""
    global _fast
    if _fast is None and torch.cuda.is_available():
        _fast = _host.fast()
    if _fast and out_dtype is None and tile == 0 and split == 0 and x.is_cuda:
        status = _status_word(x.device)
        r = _fast.linear(x, weight, weight_scale, bias, x_scale, status)
        if r is not None:
            if type(r) is int:
                _lib.check(r, "fp8_block_linear")
            _deferred_status_check(x.device, status)
            return r
    env = _lib.env_set()
    flags = _host.env_flags(env)
    key = (x.shape, x.dtype, x.device, x.is_contiguous(), weight.shape, weight.dtype, weight.device, weight.stride(),
           weight_scale.shape, weight_scale.device, out_dtype, tile, split, flags,
           None if bias is None else (bias.shape, bias.dtype, bias.device),
           None if x_scale is None else (x_scale.shape, x_scale.device))
    p = _plans.get(key)
    if p is None:
        p, x = _make_plan(x, weight, weight_scale, bias, x_scale, out_dtype, tile, split, flags)
        if key[3]:
            _host.keep(_plans, key, p)      # (contiguous rows, copied or not, have one stride)
    elif x.data_ptr() & 15:
        x = _aligned_rows(x, weight.shape[1])
    assert weight.data_ptr() & 15 == 0, "weight rows must be contiguous and start on 16 bytes"
    if weight_scale.dtype is not torch.float32 or not weight_scale.is_contiguous():
        weight_scale = weight_scale.to(torch.float32).contiguous()
    if x_scale is not None and (x_scale.dtype is not torch.float32 or not x_scale.is_contiguous()):
        x_scale = x_scale.to(torch.float32).contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    shape, strides, dtype = p.out
    index, device = p.index, p.device
    out = _host.empty(shape, strides, dtype=dtype, device=device)
    if not p.rows:
        return out
    # (the workspace is torch's: kept for this stream by its allocator, or for the graph under capture, so that no two share it)
    work = _host.empty((p.work,), (1,), dtype=torch.uint8, device=device) if p.work else None
    status = _status_word(device)
    args = (p.addr, x.data_ptr(), None if x_scale is None else x_scale.data_ptr(), weight.data_ptr(), weight_scale.data_ptr(),
            None if bias is None else bias.data_ptr(), None if work is None else work.data_ptr(), p.work, out.data_ptr(),
            status.data_ptr(), _host.raw_stream(index))
    if _host.current_device() == index:
        rc = _lib.lib().b200moe_fp8_linear(*args)
    else:
        with torch.cuda.device(index):
            rc = _lib.lib().b200moe_fp8_linear(*args)
    if rc != _lib.OK:
        _lib.check(rc, "fp8_block_linear")
    if not env or os.environ.get("B200MOE_DEFERRED_STATUS", "1") != "0":
        _deferred_status_check(device, status)
    if env and os.environ.get("B200MOE_CHECK_STATUS", "0") == "1":
        check_status(device)
    return out
