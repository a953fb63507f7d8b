"""What the operators around the experts share on the host.  A decode call is one launch of a few microseconds.  Contiguous
tensors on the current device go through the native path (``fast``), 4 to 6 us a call.  The others are checked in Python, where a
call whose tensors look like an earlier one's (shapes, types, devices, layout; never addresses) finds its checks and the
description of the problem in a plan, 9 to 12 us."""
from __future__ import annotations

import ctypes as C
import os
from typing import Optional

import torch

from .. import _lib
from .fused_moe import _current_device, _raw_stream

DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}
FP8 = torch.float8_e4m3fn
MAX_PLANS = 512

empty = torch.empty_strided         # (1.4 us; torch.empty with the same arguments 2.4)
raw_stream = _raw_stream
current_device = _current_device


def fast():
    """The native host path of contiguous calls (csrc/fastcall.cpp), or False where it was not built for this torch and this
    library: the calls then take the Python path to the same kernels."""
    lib = _lib.lib()
    try:
        from .. import _fastcall
    except ImportError:
        return False
    if not torch.__version__.startswith(_fastcall.torch_version) or _fastcall.version != _lib.VERSION:
        return False
    entries = (lib.b200moe_block_norm, lib.b200moe_gated_activation, lib.b200moe_fp8_linear, lib.b200moe_fp8_linear_workspace_bytes,
               lib.b200moe_env_set)
    _fastcall.init(*(C.cast(f, C.c_void_p).value for f in entries))
    return _fastcall


def env_flags(env: int) -> int:
    """B200MOE_FLAG_* from the environment; ``env``: whether it holds any of this library's variables."""
    return _lib.FLAG_NO_PDL if env and os.environ.get("B200MOE_NO_PDL", "0") == "1" else 0


def keep(plans: dict, key, plan):
    if len(plans) >= MAX_PLANS:
        plans.clear()
    plans[key] = plan


def strides_of(shape) -> tuple:
    out, step = [], 1
    for n in reversed(shape):
        out.append(step)
        step *= max(n, 1)
    return tuple(reversed(out))


def counted(m: int, most: int) -> int:
    """``m`` rows (or elements of a row): a description holds 32 bits, which a larger number would not fit into."""
    if m > most:
        raise ValueError(f"sizes of more than {most} are not supported")
    return m


def rows_of(t: torch.Tensor, h: int, most: int) -> int:
    return counted(t.numel() // h, most)


def as_rows(t: torch.Tensor, h: int) -> torch.Tensor:
    """[rows, h] with contiguous rows: a view where the strides allow it, else a copy."""
    t = t if t.dim() == 2 else t.reshape(-1, h)
    if (t.stride(1) != 1 and h != 1) or (t.shape[0] > 1 and t.stride(0) < h):
        t = t.contiguous()
    return t


def row_stride(t: Optional[torch.Tensor], h: int) -> int:
    return h if t is None or t.shape[0] <= 1 else t.stride(0)


def struct(cls, *values):
    """(the structure, its address)"""
    s = cls(C.sizeof(cls), *values)
    return s, C.addressof(s)
