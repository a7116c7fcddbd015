"""GPU: fp16 gradients of cross attention where the values, the gradients of the output or the weights lie far from one
another: dq, dk and dv are as exact there as where all are near one.

The bound, on the relative error over a region's elements (root of the sums of squares), u = 2^-11 half a step: rounding a result
costs 0.42 u (uniform within a half step, 0.58 u of a value between 1 and 2, 0.72 of that over mantissas spread evenly in
the logarithm); so does rounding the operand of the last product (P or dS), whose terms add with random signs; delta, from an
output whose weights were rounded, less than that again. In squares 0.73 u, and u is allowed. Operands below fp16's normal
numbers would be off by up to 2^-25 each, whatever their size.
"""

import math

import pytest
import torch

import torchsoftdtw_b200 as T

pytestmark = pytest.mark.gpu

U = 2.0**-11


def tensors(B, N, M, Hq, Hkv, d, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g, dtype=torch.float64).cuda()
            for s in ((B, N, Hq, d), (B, M, Hkv, d), (B, M, Hkv, d), (B, N, Hq, d))]


def both(t, bandwidth=-1):
    """dq, dk, dv of the operator and of its definition in 64 bits, on t rounded to fp16."""
    q, k, v, dout = [x.half() for x in t]
    assert all(x.isfinite().all() for x in (q, k, v, dout))
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    got = torch.autograd.grad(T.cross_attention(*leaves, bandwidth=bandwidth), leaves, dout)
    wide = [x.double().detach().requires_grad_(True) for x in (q, k, v)]
    rep = q.shape[2] // k.shape[2]
    N, M = q.shape[1], k.shape[1]
    s = torch.einsum("bnhd,bmhd->bhnm", wide[0], wide[1].repeat_interleave(rep, 2)) / math.sqrt(q.shape[3])
    if bandwidth >= 0:
        assert N == M > 1
        i = torch.arange(N, device=q.device)
        s = s.masked_fill((i.view(-1, 1) - i.view(1, -1)).abs() > bandwidth, -math.inf)
    out = torch.einsum("bhnm,bmhd->bnhd", s.softmax(-1), wide[2].repeat_interleave(rep, 2))
    want = torch.autograd.grad(out, wide, dout.double())
    return dict(zip(("dq", "dk", "dv"), zip(got, want)))


def check(res, region=slice(None)):
    for name, (got, want) in res.items():
        g, w = got[:, region].double(), want[:, region]
        finite = bool(g.isfinite().all())
        assert finite, name
        # Results below fp16's normal numbers round by 2^-26 in the mean, whatever their size.
        slack = 2.0**-25 * math.sqrt(w.numel())
        off = ((g - w).norm().item() - slack) / (U * w.norm().item())
        assert off <= 1, name


# The head widths of each kernel: tensor-core ones, warp-level ones.
WIDTHS = [32, 64, 128, 20, 33, 100]


@pytest.mark.parametrize("d", WIDTHS)
def test_large_values_and_small_gradients(cuda, d):
    """Values of thousands, and gradients of the output that all point along one of them: products far above a row's |dout|."""
    t = tensors(2, 150, 4, 2, 1, d, 1)
    t[2] *= 8000
    t[3] = 2.0**-12 * t[2][:, :1].sign().expand_as(t[3])
    check(both(t))


@pytest.mark.parametrize("d", WIDTHS)
def test_small_values_and_large_gradients(cuda, d):
    t = tensors(1, 260, 2048, 2, 1, d, 2)
    t[2] *= 2.0**-12
    t[3] *= 2.0**12
    check(both(t))


@pytest.mark.parametrize("exponent", [-16, -18])
@pytest.mark.parametrize("d", WIDTHS)
def test_gradients_that_differ_along_a_band(cuda, d, exponent):
    """The second half of the series has far smaller gradients: its states, which no row of the first half reaches, lose
    nothing by the first half's size."""
    t = tensors(1, 512, 512, 2, 1, d, 3)
    t[0] *= 4
    t[1] *= 0.25
    t[3] *= 2.0**11
    t[3][:, 256:] *= 2.0**exponent
    res = both(t, 16)
    check(res, slice(256 + 40, None))
    check(res, slice(0, 256 - 40))


@pytest.mark.parametrize("d", WIDTHS)
def test_values_that_differ_along_a_band(cuda, d):
    t = tensors(1, 512, 512, 2, 1, d, 4)
    t[2] *= 2.0**4
    t[2][:, 256:] *= 2.0**-14
    t[3][:, 256:] *= 2.0**6
    res = both(t, 16)
    check(res, slice(256 + 40, None))
    check(res, slice(0, 256 - 40))


@pytest.mark.parametrize("d", WIDTHS)
def test_small_weights_and_large_gradients(cuda, d):
    """Half of the states have weights of 2^-28 and less in every row, and gradients of normal size through large dout."""
    t = tensors(1, 200, 128, 2, 1, d, 5)
    t[0] *= 0.5
    t[0][..., 0] = math.sqrt(d)
    t[1][:, 64:, :, 0] -= 15.0  # e^-15 of the others' weights, 2^-6 and less
    t[2] *= 2.0**-8
    t[3] *= 2.0**11
    res = both(t)
    check(res)
    check({"dv": res["dv"]}, slice(64, None))


@pytest.mark.parametrize("d", WIDTHS)
def test_gradients_of_nothing(cuda, d):
    """Rows without a gradient beside others, and values of zero."""
    t = tensors(2, 150, 170, 2, 1, d, 6)
    t[3][:, 64:] = 0
    t[2][1] = 0
    res = both(t)
    assert (res["dq"][0][:, 64:] == 0).all() and (res["dq"][0][1] == 0).all() and (res["dk"][0][1] == 0).all()
    check(res)


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


@pytest.mark.parametrize("d", [64, 33])
def test_replayed_on_gradients_of_another_size(cuda, d):
    """The scale is that of the replay's inputs, not of the capture's: equal bits to an eager call, in any order."""
    sets = []
    for size in (1.0, 2.0**-12, 2.0**10):
        t = [x.half() for x in tensors(2, 150, 170, 4, 2, d, 11)]
        t[3] = (t[3] * size).half()
        leaves = [x.clone().requires_grad_(True) for x in t[:3]]
        sets.append((t, torch.autograd.grad(T.cross_attention(*leaves, bandwidth=20), leaves, t[3])))
    held = [x.clone() for x in sets[0][0]]
    leaves = [x.requires_grad_(True) for x in held[:3]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad(T.cross_attention(*leaves, bandwidth=20), leaves, held[3])
    for which in (1, 0, 2, 1):
        held[3].copy_(sets[which][0][3])
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(grads, sets[which][1]):
            assert torch.equal(got, want)
