"""CPU: what a kernel reads of the kernel before it is no read-only data.

Kernels are launched programmatically: one starts while its predecessor still writes, and waits (griddepcontrol.wait) before it reads.  That
orders ordinary loads.  Read-only loads (ld.global.nc, __ldg, or any load from a `const ... __restrict__` argument of a kernel, for which the
compiler may choose them) are defined only for memory that nothing writes from the kernel's start to its end.  No run can show the
difference reliably, so the sources are looked at."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "flaggems-sglang_b200" / "csrc"


def _code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def _kernel_arguments(text):
    """The argument lists of the file's kernels."""
    out = []
    for m in re.finditer(r"__global__[^;{]*?(\w+_kernel)\s*\(", text):
        depth, i = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        out.append((m.group(1), text[m.end():i - 1]))
    return out


@pytest.mark.parametrize("name", ["linear_fp8.cu", "norm.cu", "activation.cu", "quant.cuh"])
def test_operators_around_the_experts(name):
    text = _code(name)
    assert "__ldg(" not in text and "ld.global.nc" not in text
    for kernel, arguments in _kernel_arguments(text):
        assert not re.search(r"const\s+\w+\s*\*\s*__restrict__", arguments), kernel


@pytest.mark.parametrize("name", ["prep.cu", "router.cu", "ep.cu", "gemm_simt.cu"])
def test_rows_that_enter_the_experts(name):
    """Tokens come from a norm that lets the next kernel start early, router logits from a product that does; lists, sorted rows and pairs from the
    kernels of the call itself."""
    text = _code(name)
    assert "__ldg(" not in text and "ld.global.nc" not in text
    for kernel, arguments in _kernel_arguments(text):
        assert not re.search(r"const\s+\w+\s*\*\s*__restrict__", arguments), kernel


def test_the_kernels_are_found():
    assert {k for k, _ in _kernel_arguments(_code("linear_fp8.cu"))} >= {"linear_quant_kernel", "fp8_linear_decode_kernel", "fp8_linear_token_kernel"}
    assert {k for k, _ in _kernel_arguments(_code("prep.cu"))} >= {"gather_rows_kernel", "gather_routed_kernel", "group_quant_fp8_kernel", "finalize_pairs_kernel"}
