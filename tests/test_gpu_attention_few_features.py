"""GPU: dq of few features in 16 bits, of widths that the tensor-core kernels do not take."""

import math

import pytest
import torch

import sequence_plain as plain
import torchsoftdtw_b200 as T

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("d", [9, 12, 20, 31])
def test_dq_of_few_odd_features(cuda, d, dtype):
    """A few large dS carry dq, so that their rounding has to be made good: dq may be off by its own rounding, 0.42 u over
    its elements (u half a step), and by delta's part, 0.2 u at d = 8 to 32. In squares 0.46 u; rounding dS adds 0.5 u, together
    0.68 u. The bound lies between."""
    g = torch.Generator().manual_seed(84)
    q, k, v, dout = [(torch.randn(2, n, h, d, generator=g, dtype=torch.float64) * f).to(dtype).cuda()
                     for n, h, f in ((2000, 2, 1.5), (600, 1, 1.0), (600, 1, 1.0), (2000, 2, 1.0))]
    leaf = q.detach().requires_grad_(True)
    (got,) = torch.autograd.grad(T.cross_attention(leaf, k, v), leaf, dout)
    vals, _ = plain.attention(q, k, v, torch.tensor([2000, 2000]), torch.tensor([600, 600]), -1, 1 / math.sqrt(d), dout)
    off = ((got.double() - vals["dq"]).norm() / vals["dq"].norm()).item() / (torch.finfo(dtype).eps / 2)
    assert off <= 0.55
