"""GPU: waits of the tensor-core kernels that run out, where the tile that they are about is the last one of its rows, or is being
cleared behind a length."""

import pytest
import torch

import torchsoftdtw_b200 as T
from torchsoftdtw_b200 import _ext

pytestmark = pytest.mark.gpu

STALLS = [(1, "out"), (2, "dq"), (3, "dk")]


def stalled(which, name, N, M, d, lens=(None, None)):
    """One warp of the first CTA withholds an arrival: the kernel ends, the CTA's rows are NaN, the other sample's right, the
    error is reported, and the next call is right."""
    lib = _ext.capi()
    T.check_errors()
    g = torch.Generator(device="cuda").manual_seed(9)
    t = [torch.randn(2, n, 2, d, generator=g, device="cuda").to(torch.bfloat16) for n in (N, M, M, N)]

    def forward():
        leaves = [x.detach().requires_grad_(True) for x in t[:3]]
        return leaves, T.cross_attention(*leaves, *lens)

    def everything(leaves, out):
        return dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, t[3]))))

    want = everything(*forward())
    torch.cuda.synchronize()
    lib.sdtw_set_wait_timeout(0.2)
    try:
        made = forward() if which > 1 else None
        lib.sdtw_debug_attention_stall(which)
        got = everything(*made) if which > 1 else {"out": forward()[1].detach()}
        torch.cuda.synchronize()
    finally:
        lib.sdtw_debug_attention_stall(0)
        lib.sdtw_set_wait_timeout(2.0)
    broken = bool(got[name][0, 0, 0].isnan().all())
    assert broken
    assert torch.equal(got[name][1], want[name][1])
    with pytest.raises(RuntimeError, match="timed out"):
        T.check_errors()
    again = everything(*forward())
    assert all(torch.equal(again[n], want[n]) for n in want)
    T.check_errors()


@pytest.mark.parametrize("N,M", [(60, 60), (128, 64), (200, 100), (100, 200)])
@pytest.mark.parametrize("which,name", STALLS)
@pytest.mark.parametrize("d", [64, 128])
def test_in_the_last_tiles(cuda, d, which, name, N, M):
    """Few tiles: the warps that are not stalled have theirs when the wait runs out."""
    stalled(which, name, N, M, d)


@pytest.mark.parametrize("length", [60, 100, 600])
@pytest.mark.parametrize("which,name", STALLS)
@pytest.mark.parametrize("d", [64, 128])
def test_beside_a_padded_tile(cuda, d, which, name, length):
    """The stalled sample's last tile is loaded and cleared while the others wait (the short ones), or after."""
    lens = torch.tensor([length, 650], device=cuda), torch.tensor([length, 640], device=cuda)
    stalled(which, name, 700, 650, d, lens)
