"""CPU: sizes near and beyond 32 bits are refused at the C ABI, before anything is launched, and the two sides agree on the limits."""
import ctypes as C
import re
from pathlib import Path

HEADER = Path(__file__).resolve().parent.parent / "include" / "b200moe.h"


def test_limits_are_the_headers():
    from flaggems_sglang_b200 import _lib
    text = HEADER.read_text()
    for name in ("MAX_ROWS", "NORM_MAX_ROWS", "ACT_MAX_I", "LINEAR_MAX_K", "NORM_MAX_H"):
        value = re.search(rf"#define B200MOE_{name} (\([^)]*\)|\S+)", text).group(1)
        assert eval(value) == getattr(_lib, name), name


def test_linear(built_lib):
    from flaggems_sglang_b200 import _lib

    def run(**kw):
        v = dict(struct_bytes=C.sizeof(_lib.Linear), M=1, N=128, K=128, x_dtype=_lib.X_E4M3, ldx=128, ldw=128)
        v.update(kw)
        return built_lib.b200moe_fp8_linear(C.byref(_lib.Linear(**v)), 256, 256, 256, 256, None, None, 0, 256, 256, None)

    # (rounding these up to whole tiles passes 2^31)
    for m in (_lib.MAX_ROWS + 1, 2 ** 31 - 100, 2 ** 31 - 1):
        assert run(M=m) == _lib.ERR_TOO_LARGE
        assert run(N=m) == _lib.ERR_TOO_LARGE
        d = _lib.Linear(struct_bytes=C.sizeof(_lib.Linear), M=m, N=128, K=128, ldx=128, ldw=128)
        assert built_lib.b200moe_fp8_linear_workspace_bytes(C.byref(d)) == 0


def test_activation_and_norm(built_lib):
    from flaggems_sglang_b200 import _lib
    f = built_lib.b200moe_gated_activation
    assert f(16, 1 << 40, 0, 1, _lib.ACT_MAX_I + 1, 0, 1.0, 0.0, 16, None, 0, None) == _lib.ERR_TOO_LARGE
    assert f(16, 16, 0, _lib.MAX_ROWS + 1, 8, 0, 1.0, 0.0, 16, None, 0, None) == _lib.ERR_TOO_LARGE
    n = _lib.Norm(struct_bytes=C.sizeof(_lib.Norm), M=_lib.NORM_MAX_ROWS + 1, H=8, dtype=2, residual_dtype=2, pre=1, ldx=8, ldr=8, ldh=8)
    assert built_lib.b200moe_block_norm(C.byref(n), 32, None, None, None, None, None, None, 32, 32, None, None) == _lib.ERR_TOO_LARGE


def test_the_python_layer_counts_before_it_converts():
    """A ctypes field takes the low 32 bits of a larger number without a word: 2^32 + 1 rows became one."""
    import pytest
    import torch
    from flaggems_sglang_b200 import _lib
    from flaggems_sglang_b200.ops import _host
    assert C.c_int32(2 ** 32 + 1).value == 1
    t = torch.zeros(1, 2).expand(2 ** 32 + 1, 2)
    for most in (_lib.MAX_ROWS, _lib.NORM_MAX_ROWS):
        with pytest.raises(ValueError):
            _host.rows_of(t, 2, most)
        assert _host.rows_of(t[:most], 2, most) == most
