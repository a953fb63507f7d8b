"""GPU: layer norms of rows whose mean is large against their deviation, in every kernel.

A sum of a row takes at most 32 terms in a thread and ten pairwise steps, its mean a division: 43 roundings, 2^-18.5 of the magnitude.

Equal elements.  The differences from that mean are exact and equal, at most 2^-18.5 of the value, and their own mean is off by 2^-18.5 of
them: 2^-37 of the value is left, 2^-22 of 30000.  The root of eps = 1e-6 makes that at most 2^-12; the variance that is left is below eps.

Small deviations (root mean square 2^-4.75, at most 2^-4) from 32768.  The differences are exact and at most 2^-2.7; their mean is off by
2^-21.2, 2^-16.4 of the deviation, and taken from the squares' mean by 2^-14.2 of the variance, 2^-15.2 of its root; the squares' mean by 2^-18.5 of 6.6
variances, 2^-16.8 of the root.  Of results up to 1.7 that is 2^-13.9 in all.

1000 plus normally distributed values: differences up to 5, their mean off by 2^-16.2, the root by 2^-19.5 of 5: 2^-15.5 on either side."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# a row to a CTA, streamed with and without tests per chunk, the ring of long rows, rows off 16 bytes
SIZES = [(2, 1000), (3, 7168), (40, 4096), (600, 7168), (3000, 1000), (4000, 1528), (900, 8192), (300, 16384), (290, 8200), (5, 16383), (700, 2047)]


def rows(m, h, dev):
    v = torch.tensor([30000.0, 1000.0, -12345.0, 0.1, 333.25, 7.0], device=dev)
    return v[torch.arange(m, device=dev) % len(v)][:, None].expand(m, h).contiguous()


@pytest.mark.parametrize("m,h", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_equal_elements_give_zero(cuda_device, m, h, dtype):
    import flaggems_sglang_b200 as F
    x = rows(m, h, cuda_device).to(dtype)
    zero = torch.zeros_like(x)
    for y in (F.norm_before_block(x, None, residual=zero, kind="layer")[0], F.norm_after_block(x, None, residual=zero, kind="layer"),
              F.norm_after_block(x, None, residual=x, kind="layer", next_norm=True)[0]):
        assert float(y.float().abs().max()) <= 2.0 ** -12
    q, s = F.norm_before_block(x, None, residual=zero, kind="layer", quantize=True)[0]
    assert float((q.float() * s.repeat_interleave(128, 1)[:, :h]).abs().max()) <= 2.0 ** -12


@pytest.mark.parametrize("m,h", SIZES)
def test_small_deviations_from_a_large_mean(cuda_device, m, h):
    """32768 plus multiples of 2^-8 up to 2^-4: all of them floats."""
    import flaggems_sglang_b200 as F
    g = torch.Generator(device=cuda_device).manual_seed(h)
    x = 32768 + torch.randint(-16, 17, (m, h), device=cuda_device, generator=g).float() / 256
    d = x.double() - x.double().mean(1, keepdim=True)
    want = d / (d.square().mean(1, keepdim=True) + 1e-6).sqrt()
    for y in (F.norm_before_block(x, None, residual=torch.zeros_like(x), kind="layer")[0], F.norm_after_block(x, None, kind="layer")):
        assert float((y.double() - want).abs().max()) <= 2.0 ** -13


def test_a_result_does_not_depend_on_the_number_of_rows(cuda_device):
    """One row by itself and among enough others to stream, and both against 64 bits: values that need all of their digits."""
    import flaggems_sglang_b200 as F
    for h in (1000, 4096, 7168):
        x = (1000 + torch.randn(1200, h, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(h)))
        many, one = F.norm_after_block(x, None, kind="layer"), F.norm_after_block(x[:1], None, kind="layer")
        assert float((many[:1] - one).abs().max()) <= 2.0 ** -14
