"""GPU: fp16 cross attention where the values, the gradients of the output or the weights lie far from one another."""

import pytest
import torch

import torchsoftdtw_b200 as T  # noqa: F401

pytestmark = pytest.mark.gpu

# The head widths of each kernel: tensor-core ones, warp-level ones.
WIDTHS = [32, 64, 128, 20, 33, 100]


@pytest.mark.parametrize("size", [2.0**-12, 1.0, 2.0**12])
@pytest.mark.parametrize("N", [1, 150])
@pytest.mark.parametrize("d", WIDTHS)
def test_the_remainder_of_the_output(cuda, d, N, size):
    """out and out_lo together are the output to twice the type's bits, here the mean m of two states, small ones too.

    out drops r, |r| <= u |m| or 2^-25 (u = 2^-11 half a step). out_lo rounds 2^11 r by u of it or 2^-25: u |r| or 2^-36 of
    r, at most u^2 |m| + 2^-36 + 2^-36. m itself comes from a sum and a product in 32 bits: 2^-23 |m|."""
    g = torch.Generator().manual_seed(8)
    q = torch.zeros(2, N, 2, d, dtype=torch.float16, device=cuda)
    k = torch.randn(2, 2, 1, d, generator=g).half().cuda()
    v = (torch.randn(2, 2, 1, d, generator=g) * size).half().cuda()
    out, lo, _ = torch.ops.torchsoftdtw_b200.attention(q, k, v, None, None, -1, 1.0)
    mean = v.double().mean(1, keepdim=True)
    off = (out.double() + lo.double() * 2.0**-11 - mean).abs() - ((2.0**-22 + 2.0**-23) * mean.abs() + 2.0**-35)
    worst = off.max().item()
    assert worst <= 0
