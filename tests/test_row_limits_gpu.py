"""GPU: calls on more rows than 32 bits count are refused before anything is copied or launched.  (The rows are one row, repeated: the
tensors hold a few bytes.)"""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [2 ** 31, 2 ** 32 + 1, 2 ** 32 + 4096])
def test_rows(cuda_device, rows):
    import flaggems_sglang_b200 as F
    x = torch.zeros(1, 16, device=cuda_device, dtype=torch.bfloat16).expand(rows, 16)
    w, s = torch.zeros(8, 16, device=cuda_device).to(torch.float8_e4m3fn), torch.ones(1, 1, device=cuda_device)
    before = torch.cuda.memory_allocated()
    for call in (lambda: F.norm_before_block(x, None), lambda: F.norm_after_block(x, None), lambda: F.gated_activation(x),
                 lambda: F.gated_activation(x, quantize=True), lambda: F.fp8_block_linear(x, w, s),
                 lambda: F.fp8_block_linear(x.view(2, rows // 2, 16) if rows % 2 == 0 else x[None], w, s)):
        with pytest.raises(ValueError, match="not supported"):
            call()
    assert torch.cuda.memory_allocated() == before


def test_width(cuda_device):
    import flaggems_sglang_b200 as F
    from flaggems_sglang_b200 import _lib
    x = torch.zeros(1, 1, device=cuda_device).expand(1, 2 ** 33 + 16)
    with pytest.raises(ValueError, match="not supported"):
        F.gated_activation(x)
    w = torch.zeros(1, 16, device=cuda_device).to(torch.float8_e4m3fn).expand(2 ** 32 + 128, 16)
    with pytest.raises((ValueError, AssertionError)):
        F.fp8_block_linear(torch.zeros(1, 16, device=cuda_device).half(), w, torch.ones(1, 1, device=cuda_device).expand(2 ** 25 + 1, 1))
    i = _lib.ACT_MAX_I
    x = torch.full((1, 2 * i), 1.0, device=cuda_device, dtype=torch.bfloat16)          # the widest row
    x[0, :i] = 32.0
    y = F.gated_activation(x)
    assert y.shape == (1, i) and bool((y == 32).all())
