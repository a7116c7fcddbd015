"""GPU: one row of a longer series (a decoded token) and the band."""

import ctypes
import math

import pytest
import torch

import sequence_plain as plain
import torchsoftdtw_b200 as T
from torchsoftdtw_b200 import _ext

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("N,M,bw", [(150, 333, 9), (333, 150, 20), (64, 64, 0)])
def test_a_row_on_its_interval(cuda, dtype, N, M, bw):
    """A row alone is a series of length one, whose row spans all states whatever the band; on the states of its
    interval in the longer series it is that series' row, within the two bounds."""
    g = torch.Generator().manual_seed(15)
    q, k, v = [torch.randn(1, n, h, 64, generator=g, dtype=torch.float64).to(dtype).cuda() for n, h in ((N, 4), (M, 2), (M, 2))]
    whole = T.cross_attention(q, k, v, bandwidth=bw)
    _, errs = plain.attention(q, k, v, torch.tensor([N]), torch.tensor([M]), bw, 1 / math.sqrt(64))
    lo, hi = ctypes.c_int64(), ctypes.c_int64()
    for i in (0, 1, N // 2, N - 1):
        row = q[:, i:i + 1]
        assert torch.equal(T.cross_attention(row, k, v, bandwidth=bw), T.cross_attention(row, k, v))
        _ext.capi().sdtw_band_row_range(i, N, M, bw, ctypes.byref(lo), ctypes.byref(hi))
        part = slice(lo.value, hi.value + 1)
        plain.check("row", T.cross_attention(row, k[:, part], v[:, part])[:, 0], whole[:, i].double(), 2 * errs["out"][:, i])
