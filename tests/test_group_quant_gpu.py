"""GPU: the 1 x 128 e4m3 quantisation within the operators around the experts, bit by bit against the definition in torch's fp32:
scale = max(amax, 1e-10) / 448, value = e4m3(v / scale), both IEEE divisions.

Everything here scales by powers of two as long as nothing is subnormal, so all mantissas at a few exponents are all floats.  Rows of
chosen fp32 values come out of the gated activation: at a gate of 32 sigmoid is 1 - 2^-46, which is 1, and the result is 32 times the linear half."""
import pytest
import torch

from oracle import block_ops as B

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def quantised(y):
    """(q, scale) of the fp32 rows y, which are the activation's results exactly."""
    import flaggems_sglang_b200 as F
    x = torch.cat([torch.full_like(y, 32.0), y / torch.full((), 32.0, device=y.device)], -1)
    assert torch.equal(F.gated_activation(x), y)
    return F.gated_activation(x, quantize=True)


def scale_of(amax):
    return amax.clamp_min(1e-10) / torch.full((), 448.0, device=amax.device)      # (a tensor: by a number CUDA torch multiplies with its reciprocal)


@pytest.mark.parametrize("exponent", [-34, -33, 0, 5, 126, 127])
def test_every_scale(cuda_device, exponent):
    """All 2^23 maxima of a binade: the lowest (1e-10 lies in it), one in between, the two highest."""
    step = 1 << 17
    for first in range(0, 1 << 23, step):
        bits = torch.arange(first, first + step, device=cuda_device, dtype=torch.int32) + ((exponent + 127) << 23)
        amax = bits.view(torch.float32)
        y = torch.zeros(step, 128, device=cuda_device)
        y[torch.arange(step, device=cuda_device), torch.arange(step, device=cuda_device) % 128] = amax
        q, s = quantised(y)
        assert torch.equal(s[:, 0], scale_of(amax))
        assert torch.equal(q.float().amax(1), (amax / s[:, 0]).clamp_max(448).to(FP8).float())


def boundaries(dev):
    """The points between neighbouring e4m3 values, the ties: 126 of them, up to 432."""
    v = torch.arange(127, dtype=torch.uint8, device=dev).view(FP8).float()
    return (v[1:] + v[:-1]) / 2


@pytest.mark.parametrize("exponent", [-30, 0, 100])
def test_values_next_to_every_boundary(cuda_device, exponent):
    """fp32 values at, and up to two steps beside, each boundary of e4m3 under scales of random maxima."""
    g = torch.Generator(device=cuda_device).manual_seed(exponent)
    rows = 4000
    mantissa = torch.randint(0, 1 << 23, (rows,), device=cuda_device, generator=g, dtype=torch.int32)
    mantissa[:64] = torch.arange(64, device=cuda_device, dtype=torch.int32) << 17           # maxima that make exact ties
    amax = (mantissa + ((exponent + 127) << 23)).view(torch.float32)
    s = scale_of(amax)[:, None]
    near = boundaries(cuda_device)[None] * s
    for off in range(-2, 3):
        v = (near.view(torch.int32) + off).view(torch.float32)
        v = torch.where(torch.rand(v.shape, device=cuda_device, generator=g) < 0.5, v, -v)
        y = torch.cat([amax[:, None], v, torch.zeros_like(s)], 1)
        q, got = quantised(y)
        assert torch.equal(got, s)
        want = (y / s).clamp(-448, 448).to(FP8)
        bad = q.float() != want.float()
        assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values at {off} steps from a boundary"


@pytest.mark.parametrize("dtype,mantissas,exponents", [(torch.bfloat16, 128, (-20, 0, 30)), (torch.float16, 1024, (3, 15))])
def test_every_16_bit_value_over_every_maximum(cuda_device, dtype, mantissas, exponents):
    """Rows quantised by the linear layer, read back through the unit matrix: every mantissa of the maximum, over it every value down to
    2^-20 of it (beyond, all are zero)."""
    import flaggems_sglang_b200 as F
    unit, one = torch.eye(128, device=cuda_device).to(FP8), torch.ones(1, 1, device=cuda_device)
    m = 1 + torch.arange(mantissas, device=cuda_device, dtype=torch.float64) / mantissas
    for e in exponents:
        values = torch.cat([m * 2.0 ** (e - d) for d in range(21)])
        values = torch.cat([values, values.new_zeros(-values.numel() % 127)]).view(-1, 127)
        values *= 1 - 2 * (torch.arange(127, device=cuda_device) % 2)
        for a in (m * 2.0 ** e).split(128):
            x = torch.cat([a[:, None, None].expand(-1, values.shape[0], 1), values[None].expand(a.numel(), -1, -1)], 2)
            x = torch.where(x.abs() <= a[:, None, None], x, torch.zeros_like(x)).to(dtype).view(-1, 128)
            out = F.fp8_block_linear(x, unit, one, out_dtype=torch.float32)
            q, s = B.group_quant(x)
            assert torch.equal(out, q.float() * s)
            few = F.fp8_block_linear(x[:8], unit, one, out_dtype=torch.float32)          # quantised by the product's own kernel
            assert torch.equal(few, out[:8])
    F.check_status()


def test_an_infinite_scale(cuda_device):
    """Numbers beside an infinity are zero, the infinity itself is NaN: both quotients by an infinite scale."""
    y = torch.randn(3, 256, device=cuda_device)
    y[1, 5] = float("inf")
    q, s = quantised(y)
    assert s[1].tolist()[0] == float("inf") and torch.isfinite(s[0]).all() and torch.isfinite(s[1, 1])
    want = torch.zeros(128, device=cuda_device)
    want[5] = float("nan")
    assert torch.equal(q[1, :128].float().nan_to_num(7.0), want.nan_to_num(7.0))
    assert torch.equal(q[1, 128:].float(), (y[1, 128:] / s[1, 1]).to(FP8).float())
