"""GPU: the gated activation's own error, on fp32 rows, where no rounding to fewer bits covers it.

Derivation.  exp2 is within 2^-22 relative (4 units of 2^-24), its argument's rounding is carried along, so e = exp(-|z|) is within 5 units.
1 + e takes at most half of that and a rounding, its reciprocal after a step of Newton's iteration two units, and z < 0 multiplies with e itself:
5 + 1 there.  Two more products: 5 + 1 + 2.5 + 1 + 2 + 2 = 13.5 units, below 2^-20.  alpha g rounds once more: |z| units.  Results below the least
normal number may be zero: 2^-126 times the linear half."""
import pytest
import torch

from oracle import block_ops as B

pytestmark = pytest.mark.gpu


def rows(dev, lo, hi, n=1 << 18):
    g = torch.Generator(device=dev).manual_seed(int(hi))
    gate = lo + (hi - lo) * torch.rand(n, device=dev, generator=g, dtype=torch.float64)
    return gate.float().view(-1, 1024), torch.randn(n // 1024, 1024, device=dev, generator=g)


def relative(got, want, allowed, floor):
    d = (got.double() - want).abs()
    tol = allowed * want.abs() + floor
    bad = d > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst 2^{float((d[bad] / want[bad].abs()).max().log2()):.1f} of the result"


@pytest.mark.parametrize("lo,hi", [(-1, 1), (-8, 8), (-40, 40), (-86, -40), (-120, 120)])
def test_silu(cuda_device, lo, hi):
    import flaggems_sglang_b200 as F
    g, u = rows(cuda_device, lo, hi)
    x = torch.cat([g, u], 1)
    g, u = g.double(), u.double()
    relative(F.gated_activation(x), g * torch.sigmoid(g) * u, 2.0 ** -20, 2.0 ** -126 * (1 + g.abs()) * u.abs())


@pytest.mark.parametrize("alpha", [1.0, 2.0, -0.5, 1.702])
def test_swiglu(cuda_device, alpha):
    """alpha as the kernel has it, a float; powers of two multiply exactly."""
    import flaggems_sglang_b200 as F
    g, u = rows(cuda_device, -40, 40)
    x = torch.cat([g, u], 1)
    z = g.double() * float(torch.tensor(alpha, dtype=torch.float32))
    want = g.double() * torch.sigmoid(z) * (u.double() + 1)
    exact = abs(alpha) in (0.5, 1.0, 2.0)
    # u + 1 rounds once: half a unit of the larger of the two
    slack = 2.0 ** -24 * (g.double() * torch.sigmoid(z)).abs() * (1 + u.double().abs())
    relative(F.gated_activation(x, "swiglu_oai", swiglu_alpha=alpha), want, 2.0 ** -20 + (0 if exact else 2.0 ** -24 * z.abs()), slack + 2.0 ** -120)


def test_silu_at_the_ends(cuda_device):
    import flaggems_sglang_b200 as F
    inf, nan = float("inf"), float("nan")
    g = torch.tensor([[inf, -inf, nan, 3e38, -3e38, 0.0, -0.0, 200.0, -200.0]], device=cuda_device)
    one = torch.ones_like(g)
    y = F.gated_activation(torch.cat([g, one], 1))[0].tolist()
    assert y[0] == inf and y[1] != y[1] and y[2] != y[2] and y[3] == float(g[0, 3]) and y[4] == 0 and y[5] == 0 and y[6] == 0
    assert y[7] == 200 and y[8] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lo,hi", [(-1, 1), (-4, 4), (-13, -4), (-40, 40)])
def test_gelu(cuda_device, dtype, lo, hi):
    """Units of 2^-24: the fitted polynomial and its roundings 7, the reciprocal 2, which the function turns into at most 2.3 times as many,
    the exponential 5, three products 3: 20, below 2^-19, of the result, in the tail too.  16-bit rows: two roundings of g^2 / 2 more.  Then
    half a step of the type."""
    import flaggems_sglang_b200 as F
    g, u = rows(cuda_device, lo, hi)
    x = torch.cat([g, u], 1).to(dtype)
    g, u = x.double().chunk(2, 1)
    want = g * (0.5 * torch.special.erfc(-g * 0.5 ** 0.5)) * u
    half, least = (0, 2.0 ** -126) if dtype == torch.float32 else (torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)
    relative(F.gated_activation(x, "gelu"), want, 2.0 ** -19 + half + (2.0 ** -24 * g.square() if half else 0), least + 2.0 ** -126 * (g * u).abs())


def test_gelu_at_the_ends(cuda_device):
    import flaggems_sglang_b200 as F
    inf, nan = float("inf"), float("nan")
    g = torch.tensor([[inf, -inf, nan, 3e38, -3e38, 0.0, -0.0, 20.0, -20.0]], device=cuda_device)
    y = F.gated_activation(torch.cat([g, torch.ones_like(g)], 1), "gelu")[0].tolist()
    assert y[0] == inf and y[1] != y[1] and y[2] != y[2] and y[3] == float(g[0, 3]) and y[4] == 0 and y[5] == 0 and y[6] == 0
    assert y[7] == 20 and y[8] == 0
