"""GPU: the pair kernels with the reduction split in four, clusters of eight CTAs: picked by hand only, and on the sizes at which shares are
one slice long, unequal, or fewer than asked for."""
import pytest
import torch

from oracle import block_ops as B

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tile", [2, 3])
@pytest.mark.parametrize("split", [3, 4, 7, 8])
@pytest.mark.parametrize("m,n,k", [(1, 128, 640), (70, 130, 1040), (257, 700, 2048), (600, 513, 1168), (300, 300, 512), (520, 260, 384), (130, 260, 128),
                                   (2000, 1500, 1040)])
def test_pairs_split_in_four(cuda_device, tile, split, m, n, k):
    """Tolerance as for the other kernels: half a step of the type and 2^-11 of the terms' magnitude."""
    import flaggems_sglang_b200 as F
    g = torch.Generator(device=cuda_device).manual_seed(m)
    w = (torch.randn(n, k, device=cuda_device, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    ws = torch.rand(-(-n // 128), -(-k // 128), device=cuda_device, generator=g) * 1e-3 + 1e-4
    xq, xs = B.group_quant(torch.randn(m, k, device=cuda_device, generator=g))
    bias = torch.randn(n, device=cuda_device, generator=g)
    want, mag = B.linear(xq, xs, w, ws, bias)
    for dt in (torch.float32, torch.bfloat16):
        out = F.fp8_block_linear(xq, w, ws, bias, x_scale=xs, out_dtype=dt, tile=tile, split=split)
        d = (out.double() - want).abs()
        assert (d <= torch.finfo(dt).eps / 2 * want.abs() + 2.0 ** -11 * mag + 2.0 ** -25).all()
        assert torch.equal(out, F.fp8_block_linear(xq, w, ws, bias, x_scale=xs, out_dtype=dt, tile=tile, split=split))
    F.check_status()
