"""GPU: the FP8 linear layer behind kernels that still write what it reads when it starts (programmatic launches), in buffers that are used
again and again, so that a line kept from the call before would show.  Bit for bit what the same calls give one at a time."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _weights(n, k, dev, seed):
    from flaggems_sglang_b200.quant import quantize_fp8_block
    g = torch.Generator(device=dev).manual_seed(seed)
    q, s = quantize_fp8_block(torch.randn(1, n, k, device=dev, generator=g) * k ** -0.5)
    return q[0], s[0]


@pytest.mark.parametrize("m", [1, 8, 40, 150, 600])
def test_rows_and_scales_of_the_kernel_before(cuda_device, m):
    """Quantising norm and quantising activation in front, other rows every time, outputs in the memory that the ones before have left."""
    import flaggems_sglang_b200 as F
    h, i = 1024, 768
    w13, s13 = _weights(2 * i, h, cuda_device, 1)
    wd, sd = _weights(h, i, cuda_device, 2)
    g = torch.Generator(device=cuda_device).manual_seed(m)
    # (rows of very different size: another row's scales would be far off)
    xs = [(torch.randn(m, h, device=cuda_device, generator=g) * 4.0 ** (n % 5)).to(torch.bfloat16) for n in range(24)]

    def block(x, sync):
        wait = torch.cuda.synchronize if sync else (lambda: None)
        (q, s), hidden = F.norm_before_block(x, None, residual=x, quantize=True)
        wait()
        a = F.fp8_block_linear(q, w13, s13, x_scale=s)
        wait()
        aq, sa = F.gated_activation(a, quantize=True)
        wait()
        y = F.fp8_block_linear(aq, wd, sd, x_scale=sa)
        wait()
        z = F.fp8_block_linear(hidden, w13, s13)
        return y, z

    want = [block(x, True) for x in xs]
    for _ in range(3):
        got = []
        for x in xs:
            y, z = block(x, False)
            got.append((y.clone(), z.clone()))
            del y, z
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    F.check_status()


@pytest.mark.parametrize("m", [3, 48, 300])
def test_weights_written_in_the_stream_ahead(cuda_device, m):
    """The weights and their scales are written in place just before the call."""
    import flaggems_sglang_b200 as F
    n, k = 1152, 2048
    sets = [_weights(n, k, cuda_device, seed) for seed in range(4)]
    x = torch.randn(m, k, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(m)).to(torch.bfloat16)
    want = []
    for w, s in sets:
        torch.cuda.synchronize()
        want.append(F.fp8_block_linear(x, w, s))
    w, s = sets[0][0].clone(), sets[0][1].clone()
    for _ in range(5):
        for (a, b), o in zip(sets, want):
            w.view(torch.uint8).copy_(a.view(torch.uint8))
            s.copy_(b)
            F.gated_activation(x)                     # (a kernel that lets the next one start early)
            assert torch.equal(F.fp8_block_linear(x, w, s), o)
    F.check_status()
