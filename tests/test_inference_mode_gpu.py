"""GPU: calls in and outside of inference mode, in any order, in one process."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

CODE = """
import sys; sys.path[:0] = [%r, %r]
import contextlib, importlib
import torch, flaggems_sglang_b200 as F
from flaggems_sglang_b200.quant import quantize_fp8_block
fm = importlib.import_module("flaggems_sglang_b200.ops.fused_moe")
d = torch.device("cuda:0")
x = torch.randn(40, 512, device=d).to(torch.bfloat16)
w, s = quantize_fp8_block(torch.randn(1, 256, 512, device=d)); w, s = w[0], s[0]
first, then = ((torch.inference_mode, contextlib.nullcontext), (contextlib.nullcontext, torch.inference_mode))[%d]
with first():
    want = F.fp8_block_linear(x, w, s)
with then():
    for _ in range(2 * fm.STATUS_COPY_EVERY + 2):
        y = F.fp8_block_linear(x, w, s)
    assert torch.equal(y, want)
    fm._status_word(d).fill_(103)
    try:
        F.check_status()
        raise SystemExit("not raised")
    except RuntimeError as e:
        assert "code 103" in str(e), e
    F.check_status()
with first():
    fm._status_word(d).fill_(102)
    raised = 0
    for _ in range(2 * fm.STATUS_COPY_EVERY + 2):
        try:
            F.fp8_block_linear(x, w, s)
        except RuntimeError as e:
            assert "code 102" in str(e), e
            raised += 1
        torch.cuda.synchronize()
    assert raised == 1, raised
F.check_status(); print("done")
"""


@pytest.mark.parametrize("order", [0, 1])
def test_the_first_call_in_one_mode_and_the_others_in_the_other(cuda_device, order):
    code = CODE % (str(ROOT), str(ROOT / "flaggems-sglang_b200"), order)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stdout + r.stderr
