"""GPU: cross attention and its gradients against a plain implementation in 64 bits, elementwise within bounds
that follow from the roundings the kernels make (sequence_plain.py), at the sizes, masks, layouts and ways of
calling where they can go wrong."""

import math
import os
import subprocess
import sys

import pytest
import torch

import sequence_plain as plain
import torchsoftdtw_b200 as T
from torchsoftdtw_b200 import _ext

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]

# B, N, M, Hq, Hkv, d, bandwidth
SHAPES = [
    (1, 1, 1, 1, 1, 1, -1),
    (2, 1, 37, 4, 2, 64, -1),
    (3, 5, 7, 2, 1, 33, -1),
    (2, 17, 1, 3, 3, 16, -1),
    (1, 1, 5000, 8, 1, 128, -1),
    (5, 3, 777, 6, 2, 80, -1),
    (2, 40, 600, 4, 4, 64, -1),
    (2, 128, 128, 2, 2, 64, -1),
    (2, 129, 257, 4, 2, 64, -1),
    (1, 200, 130, 2, 2, 128, 8),
    (2, 130, 300, 4, 1, 80, 0),
    (2, 64, 64, 2, 2, 96, 3),
    (2, 300, 200, 2, 1, 40, 32),
    (1, 511, 513, 1, 1, 127, -1),
    (2, 1000, 300, 2, 2, 32, 5),
    (1, 257, 1025, 3, 1, 72, 64),
    (3, 100, 90, 2, 2, 8, 0),
    (1, 40, 5000, 2, 1, 64, -1),
    (2, 30, 4001, 2, 2, 128, 100),
    (1, 600, 700, 1, 1, 128, -1),
    (1, 700, 600, 2, 1, 64, 40),
]


def make(shape, dtype, seed, ragged, train=True):
    B, N, M, Hq, Hkv, d, _ = shape
    g = torch.Generator().manual_seed(seed)
    t = [torch.randn(*s, generator=g, dtype=torch.float64).to(dtype).cuda() * f
         for s, f in (((B, N, Hq, d), 1.5), ((B, M, Hkv, d), 1.0), ((B, M, Hkv, d), 1.0), ((B, N, Hq, d), 1.0))]
    if ragged:
        lx = torch.randint(0, N + 1, (B,), generator=g)
        ly = torch.randint(0, M + 1, (B,), generator=g)
        lx[0], ly[0] = N, M
        if B > 1:
            lx[1], ly[1] = max(1, N // 2), 1
        if B > 2:
            ly[2] = 0
        for b in range(B):  # nothing past the lengths may be used
            t[0][b, lx[b]:] = math.nan
            t[1][b, ly[b]:] = math.nan
            t[2][b, ly[b]:] = math.inf
            t[3][b, lx[b]:] = math.nan
    else:
        lx, ly = torch.full((B,), N), torch.full((B,), M)
    return t, lx, ly


def run(t, lx, ly, bw, scale=None, given=True, grads=True):
    q, k, v, dout = t
    leaves = [x.detach().requires_grad_(grads) for x in (q, k, v)]
    lens = (lx.cuda(), ly.cuda()) if given else (None, None)
    out = T.cross_attention(*leaves, *lens, bandwidth=bw, scale=scale)
    res = {"out": out.detach()}
    if grads:
        res.update(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout)))
    return res


def compare(t, lx, ly, bw, res, scale=None):
    scale = 1 / math.sqrt(t[0].shape[-1]) if scale is None else scale
    vals, errs = plain.attention(*t[:3], lx, ly, bw, scale, t[3] if "dq" in res else None)
    for name, got in res.items():
        plain.check(name, got, vals[name], errs[name])


@pytest.mark.parametrize("ragged", [False, True], ids=["full", "ragged"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_and_gradients(cuda, shape, dtype, ragged):
    t, lx, ly = make(shape, dtype, 7, ragged)
    compare(t, lx, ly, shape[-1], run(t, lx, ly, shape[-1], given=ragged))
    T.check_errors(cuda)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(2, 1, 300, 4, 2, 64, -1), (2, 150, 170, 4, 2, 64, 9)], ids=str)
def test_forward_alone_is_the_same(cuda, shape, dtype):
    t, lx, ly = make(shape, dtype, 3, True)
    a = run(t, lx, ly, shape[-1], grads=False)["out"]
    b = run(t, lx, ly, shape[-1], grads=True)["out"]
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("layout", ["heads first", "fused", "expanded", "odd stride", "reversed features", "offset"])
def test_strides(cuda, dtype, layout):
    B, N, M, H, d, bw = 2, 140, 150, 2, 64, 20
    g = torch.Generator(device="cuda").manual_seed(5)

    def rnd(*s):
        return torch.randn(*s, generator=g, device=cuda).to(dtype)

    if layout == "heads first":
        t = [rnd(B, H, n, d).transpose(1, 2) for n in (N, M, M, N)]
    elif layout == "fused":
        kv = rnd(B, M, 2, H, d)
        t = [rnd(B, N, 3, H, d)[:, :, 1], kv[:, :, 0], kv[:, :, 1], rnd(B, N, H, 2 * d)[..., d:]]
    elif layout == "expanded":
        t = [rnd(B, N, H, d), rnd(1, M, H, d).expand(B, M, H, d), rnd(B, M, 1, d).expand(B, M, H, d),
             rnd(1, 1, 1, d).expand(B, N, H, d)]
    elif layout == "odd stride":
        t = [rnd(B, n, H, d + 3)[..., :d] for n in (N, M, M, N)]
    elif layout == "offset":
        t = [rnd(B * n * H * d + 1)[1:].view(B, n, H, d) for n in (N, M, M, N)]
    else:
        t = [rnd(B, n, d, H).transpose(2, 3) for n in (N, M, M, N)]
    lx, ly = torch.tensor([N, N - 37]), torch.tensor([M - 3, M])
    compare(t, lx, ly, bw, run(t, lx, ly, bw))


def test_many_samples(cuda):
    """More samples and heads than one dimension of a grid may hold."""
    B, N, M, H, d = 20000, 2, 3, 4, 16
    q, k, v = (torch.randn(B, n, H, d, device=cuda, dtype=torch.bfloat16).requires_grad_(True) for n in (N, M, M))
    out = T.cross_attention(q, k, v)
    grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    for b in (0, 9999, B - 1):
        vals, errs = plain.attention(q[b:b + 1].detach(), k[b:b + 1].detach(), v[b:b + 1].detach(), torch.tensor([N]),
                                     torch.tensor([M]), -1, 0.25, torch.ones_like(out[b:b + 1]))
        for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
            plain.check(name, got[b:b + 1].detach(), vals[name], errs[name])


def test_one_tensor_in_all_places(cuda):
    """Self attention: the gradients of the three uses add up."""
    x = torch.randn(2, 150, 2, 64, device=cuda, dtype=torch.bfloat16).requires_grad_(True)
    dout = torch.randn_like(x)
    (dx,) = torch.autograd.grad(T.cross_attention(x, x, x, bandwidth=9), x, dout)
    leaves = [x.detach().clone().requires_grad_(True) for _ in range(3)]
    parts = torch.autograd.grad(T.cross_attention(*leaves, bandwidth=9), leaves, dout)
    # Autograd adds three bf16 numbers in two sums, each off by at most u = 2^-8 of itself (half a step): together
    # u |a + b| + u (|a + b| (1 + u) + |c|) <= 2 u (1 + u) (|a| + |b| + |c|).
    bound = 2 * 2.0**-8 * (1 + 2.0**-8) * sum(p.double().abs() for p in parts)
    assert ((dx.double() - sum(p.double() for p in parts)).abs() <= bound).all()


def test_inference_mode_and_no_grad(cuda):
    t, lx, ly = make((2, 100, 120, 4, 2, 64, 9), torch.bfloat16, 67, True)
    want = run(t, lx, ly, 9, grads=False)["out"]
    leaves = [x.detach().requires_grad_(True) for x in t[:3]]
    for mode in (torch.inference_mode, torch.no_grad):
        with mode():
            out = T.cross_attention(*leaves, lx.cuda(), ly.cuda(), bandwidth=9)
        assert torch.equal(out, want) and not out.requires_grad


def test_refusals(cuda):
    q, k = torch.zeros(2, 3, 4, 8, device=cuda), torch.zeros(2, 5, 2, 8, device=cuda)
    for kw, message in (
        (dict(v=k.cpu()), "same device"),
        (dict(lengths_x=torch.tensor([1, 2])), "lengths_x must be on"),
        (dict(lengths_y=torch.tensor([1.0, 2.0], device=cuda)), "lengths_y must be int32 or int64"),
        (dict(lengths_x=torch.tensor([1, 2, 3], device=cuda)), "lengths_x must have shape"),
        (dict(v=k.half()), "same dtype"),
    ):
        with pytest.raises(RuntimeError, match=message):
            T.cross_attention(q, k, kw.pop("v", k), **kw)
    with pytest.raises(RuntimeError, match="positions must have shape"):
        T.norm_rotate(q, positions=torch.zeros(3, 2, device=cuda))
    with pytest.raises(RuntimeError, match="positions must be float32"):
        T.norm_rotate(q, positions=torch.zeros(2, 3, device=cuda, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="weight must have shape"):
        T.norm_rotate(q, torch.ones(4, device=cuda))
    with pytest.raises(RuntimeError, match="rotary_dim"):
        T.norm_rotate(q, rotary_dim=3)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_one_state_takes_all_weight(cuda, dtype):
    """M = 1, and a band of one state a row: out is that state, to the bit in 16-bit types; dq and dk are sums of
    terms that cancel, within the bounds."""
    for shape in ((2, 150, 1, 2, 1, 64, -1), (2, 400, 20, 2, 2, 64, 0), (1, 1, 1, 8, 2, 128, -1)):
        t, lx, ly = make(shape, dtype, 11, False)
        compare(t, lx, ly, shape[-1], run(t, lx, ly, shape[-1]))
        if shape[2] == 1 and dtype != torch.float32:
            out = run(t, lx, ly, shape[-1])["out"]
            assert torch.equal(out, t[2].repeat_interleave(shape[3] // shape[4], 2).expand_as(out))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N", [1, 130])
def test_scores_far_from_zero(cuda, dtype, N):
    """Weights that underflow, and scores of the whole range of a softmax, stay finite and within the bounds."""
    shape = (1, N, 300, 2, 2, 64, -1)
    t, lx, ly = make(shape, dtype, 13, False)
    t[0] *= 20
    compare(t, lx, ly, -1, run(t, lx, ly, -1))
    t[1][:, 17] = 0
    compare(t, lx, ly, -1, run(t, lx, ly, -1, scale=-0.25), scale=-0.25)


@pytest.mark.parametrize("size", [2.0**-14, 2.0**11])
def test_small_and_large_gradients_in_fp16(cuda, size):
    """fp16 gradients of the output far below and above one: dS stays inside the type wherever dq, dk and dv do."""
    for shape in ((1, 200, 260, 4, 2, 64, -1), (1, 150, 300, 1, 1, 128, 20)):
        t, lx, ly = make(shape, torch.float16, 61, False)
        t[3] *= size
        t[2] *= 4
        res = run(t, lx, ly, shape[-1])
        assert all(x.isfinite().all() for x in res.values())
        compare(t, lx, ly, shape[-1], res)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(3, 1, 70, 4, 2, 64, -1), (3, 200, 70, 4, 2, 64, 4)], ids=str)
def test_bad_lengths_are_reported(cuda, shape, dtype):
    T.check_errors(cuda)
    t, lx, ly = make(shape, dtype, 17, False)
    for a, b in ((shape[1] + 1, 5), (1, -1)):
        lx2, ly2 = lx.clone(), ly.clone()
        lx2[1], ly2[1] = a, b
        res = run(t, lx2, ly2, shape[-1])
        assert res["out"][1].isnan().all() and not res["out"][0].isnan().any() and not res["out"][2].isnan().any()
        for name in ("dq", "dk", "dv"):
            assert (res[name][1] == 0).all() and res[name].isfinite().all()
        with pytest.raises(RuntimeError, match="length"):
            T.check_errors(cuda)


@pytest.mark.parametrize("N", [3, 150])
def test_a_band_wider_than_the_series_is_none(cuda, N):
    t, lx, ly = make((2, N, 170, 2, 2, 64, -1), torch.bfloat16, 73, True)
    want = run(t, lx, ly, -1)
    for bw in (170, 2**40, 2**63 - 1):
        got = run(t, lx, ly, bw)
        assert all(torch.equal(got[n], want[n]) for n in want)


def test_int32_and_mixed_lengths(cuda):
    t, lx, ly = make((3, 40, 50, 2, 2, 32, 6), torch.float32, 19, True)
    want = run(t, lx, ly, 6)
    for a, b in ((torch.int32, torch.int32), (torch.int32, torch.int64)):
        got = run(t, lx.to(a), ly.to(b), 6)
        assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(0, 4, 5, 2, 2, 16, -1), (2, 0, 5, 2, 2, 16, -1), (2, 4, 0, 2, 2, 16, -1)], ids=str)
def test_empty_sides(cuda, shape, dtype):
    t, lx, ly = make(shape, dtype, 23, False)
    res = run(t, lx, ly, -1)
    for name, like in zip(("out", "dq", "dk", "dv"), (t[0], t[0], t[1], t[2])):
        assert res[name].shape == like.shape and (res[name] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(2, 1, 9000, 8, 2, 64, -1), (2, 300, 280, 4, 2, 128, 30)], ids=str)
def test_same_bits_every_time(cuda, shape, dtype):
    t, lx, ly = make(shape, dtype, 29, True)
    a = run(t, lx, ly, shape[-1])
    for _ in range(3):
        b = run(t, lx, ly, shape[-1])
        assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_a_row_alone_is_the_row_among_others(cuda, dtype):
    """One query a call (a decoded token) gives what the whole series gives, within the two bounds."""
    shape = (2, 150, 333, 4, 2, 64, -1)
    t, lx, ly = make(shape, dtype, 31, False)
    whole = run(t, lx, ly, -1, grads=False)["out"]
    _, errs = plain.attention(*t[:3], lx, ly, -1, 0.125)
    for i in (0, 77, 149):
        row = T.cross_attention(t[0][:, i:i + 1], t[1], t[2])
        plain.check("row", row[:, 0], whole[:, i].double(), 2 * errs["out"][:, i])


@pytest.mark.parametrize("shape", [(2, 1, 2000, 4, 2, 64, -1), (2, 200, 220, 4, 2, 64, 12)], ids=str)
def test_streams_and_graphs(cuda, shape):
    """Two calls at once on two streams; then two graphs, captured, replayed on new inputs in turn."""
    sets = [make(shape, torch.bfloat16, s, True) for s in (37, 41)]
    want = [run(*s, shape[-1]) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append([run(*s, shape[-1]) for _ in range(5)][-1])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(g[n], w[n]) for n in w)
    (t, lx, ly), (t2, lx2, ly2) = sets
    graphs = []
    for _ in range(2):
        leaves = [x.detach().clone().requires_grad_(True) for x in t[:3]]
        dout, dlx, dly = t[3].clone(), lx.cuda(), ly.cuda()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = T.cross_attention(*leaves, dlx, dly, bandwidth=shape[-1])
            grads = torch.autograd.grad(out, leaves, dout)
        graphs.append((graph, leaves, dout, dlx, dly, [out.detach(), *grads]))
    for which in (0, 1, 0):
        for n, (graph, leaves, dout, dlx, dly, outs) in enumerate(graphs):
            (tt, a, b), w = sets[(which + n) % 2], want[(which + n) % 2]
            with torch.no_grad():
                for leaf, x in zip(leaves, tt):
                    leaf.copy_(x)
            dout.copy_(tt[3])
            dlx.copy_(a)
            dly.copy_(b)
            graph.replay()
        torch.cuda.synchronize()
        for n, (*_, outs) in enumerate(graphs):
            w = want[(which + n) % 2]
            for got_t, name in zip(outs, ("out", "dq", "dk", "dv")):
                assert torch.equal(got_t, w[name]), name


def test_compile(cuda):
    t, lx, ly = make((2, 50, 60, 4, 2, 64, 9), torch.bfloat16, 43, False)
    w = torch.rand(64, device=cuda)

    def step(q, k, v):
        return T.cross_attention(T.norm_rotate(q, w), T.norm_rotate(k, w), v, bandwidth=9).float().square().sum()

    grads = []
    for f in (step, torch.compile(step)):
        leaves = [x.detach().requires_grad_(True) for x in t[:3]]
        grads.append(torch.autograd.grad(f(*leaves), leaves))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


def test_offsets_past_32_bits(cuda):
    """A cache of 2^31 + elements a tensor: the last states are read from their own place."""
    M, H, d = 1100000, 16, 128
    k = torch.zeros(1, M, H, d, dtype=torch.bfloat16, device=cuda)
    v = torch.zeros(1, M, H, d, dtype=torch.bfloat16, device=cuda)
    assert k.numel() > 2**31
    q = torch.ones(1, 1, H, d, dtype=torch.bfloat16, device=cuda)
    k[0, M - 5] = 8.0  # a score of 8 sqrt(128): all the weight but M e^-90
    v[0, M - 5] = torch.arange(d, device=cuda).to(torch.bfloat16)
    out = T.cross_attention(q, k, v)
    assert torch.equal(out, v[:, M - 5].view(1, 1, H, d))


def test_differences(cuda):
    """fp32 gradients against central differences of the kernel's own outputs along random directions. With step
    h the two results are off by at most 2 e / (2 h) from the outputs' bounds e, and by (4/3) |D(h) - D(h/2)| from
    the curvature (the error of D falls with h^2; its next term is taken up by the factor 2 instead of 4/3)."""
    shape = (2, 9, 11, 4, 2, 16, 3)
    t, lx, ly = make(shape, torch.float32, 47, False)
    lx[1], ly[1] = 6, 8
    res = run(t, lx, ly, 3)
    _, errs = plain.attention(*t[:3], lx, ly, 3, 0.25, t[3])
    h = 2.0**-5
    for which, name in enumerate(("dq", "dk", "dv")):
        direction = torch.randn_like(t[which])

        def loss(step):
            moved = [x + step * direction if n == which else x for n, x in enumerate(t[:3])]
            out = T.cross_attention(*moved, lx.cuda(), ly.cuda(), bandwidth=3)
            return (out.double() * t[3].double()).sum().item()

        D = [(loss(s) - loss(-s)) / (2 * s) for s in (h, h / 2)]
        noise = 1.5 * (errs["out"] * t[3].double().abs()).sum().item() / (h / 2)
        slope = (res[name].double() * direction.double()).sum().item()
        slack = (errs[name] * direction.double().abs()).sum().item()
        assert abs(D[1] - slope) <= 2 * abs(D[0] - D[1]) + noise + slack, name


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_first_gradient_of_a_process(cuda, dtype):
    """The first gradient of a process, whose thread has made no CUDA call before."""
    code = ("import torch, torchsoftdtw_b200 as T; x = torch.randn(1, 200, 2, 64, device='cuda', dtype=torch." + dtype + ")"
            ".requires_grad_(True); g, = torch.autograd.grad(T.cross_attention(x, x, x).float().sum(), x); "
            "y = T.norm_rotate(x); h, = torch.autograd.grad(y.float().sum(), x); "
            "assert bool(g.isfinite().all() and h.isfinite().all())")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_only_the_wanted_gradients(cuda):
    t, lx, ly = make((1, 5, 6, 2, 2, 16, -1), torch.float32, 53, False)
    k = t[1].detach().requires_grad_(True)
    out = T.cross_attention(t[0], k, t[2])
    (dk,) = torch.autograd.grad(out.sum(), k, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(dk.sum(), k)


def test_a_training_step_together(cuda):
    """Queries and keys normed and rotated along the diagonal, attention inside the band, the loss on its result,
    all gradients and their clipping: against the same step in plain 64-bit operations."""
    B, N, M, H, d, bw = 3, 60, 45, 2, 16, 12
    g = torch.Generator().manual_seed(59)
    x, y = torch.randn(B, N, H * d, generator=g).cuda(), torch.randn(B, M, H * d, generator=g).cuda()
    lx, ly = torch.tensor([60, 41, 7]).cuda(), torch.tensor([45, 30, 45]).cuda()
    params = [(torch.randn(H * d, H * d, generator=g) * (H * d) ** -0.5).cuda().requires_grad_(True) for _ in range(3)]
    params += [torch.ones(d, device=cuda, requires_grad=True) for _ in range(2)]
    pos_y = torch.arange(M, device=cuda) * ((lx - 1) / (ly - 1)).view(B, 1)
    loss_fn = T.SoftDTW(gamma=1.0, bandwidth=bw, normalize=True)

    def step(plain_step):
        wq, wk, wv, nq, nk = params
        q, k, v = ((s @ w).view(B, -1, H, d) for s, w in ((x, wq), (y, wk), (y, wv)))
        if plain_step:
            q, k, v = q.double(), k.double(), v.double()
            ones = torch.ones(B, device=cuda)

            def turned(z, n, pos):
                z = z / (z.square().mean(-1, keepdim=True) + 1e-6).sqrt() * n.double()
                a = pos.double().unsqueeze(-1) * 10000.0 ** (-torch.arange(0, d, 2, device=cuda).double() / d)
                c, s = a.cos().unsqueeze(2), a.sin().unsqueeze(2)
                f, e = z.chunk(2, -1)
                return torch.cat((f * c - e * s, f * s + e * c), -1)

            q = turned(q, nq, torch.arange(N, device=cuda) * ones.view(B, 1))
            k = turned(k, nk, pos_y)
            mask = plain.cell_mask(B, N, M, lx, ly, bw).cuda().view(B, 1, N, M)
            s = (torch.einsum("bnhd,bmhd->bhnm", q, k) / math.sqrt(d)).masked_fill(~mask, -1e30)
            p = torch.where(mask, torch.softmax(s, -1), 0.0)
            o = torch.einsum("bhnm,bmhd->bnhd", p, v).reshape(B, N, H * d).float()
        else:
            q = T.norm_rotate(q, nq, lx)
            k = T.norm_rotate(k, nk, ly, pos_y)
            o = T.cross_attention(q, k, v, lx, ly, bandwidth=bw).reshape(B, N, H * d)
        loss = loss_fn(o, y, lx, ly).sum()
        return loss, torch.autograd.grad(loss, params)

    loss, grads = step(False)
    want_loss, want = step(True)
    # The attention's inputs and outputs agree to fp32 roundings (a few 1e-6 of their size); the loss's own fp32
    # gradient contract is 1e-5 of the largest entry, and so is each product's after it.
    torch.testing.assert_close(loss, want_loss, rtol=2e-5, atol=0)
    for a, b in zip(grads, want):
        assert (a - b).abs().max() <= 1e-4 * b.abs().max()
    for p, gr in zip(params, grads):
        p.grad = gr.clone()
    norm = T.clip_grad_norm_(params, 0.5)
    exact = torch.sqrt(sum(b.double().square().sum() for b in grads))
    assert abs(norm.item() - exact.item()) <= 2**-20 * exact.item()
    factor = min(1.0, 0.5 / (exact.item() + 1e-6))
    for p, gr in zip(params, grads):
        torch.testing.assert_close(p.grad, (gr.double() * factor).float(), rtol=2**-20, atol=0)
    T.check_errors(cuda)


@pytest.mark.parametrize("which,name", [(1, "out"), (2, "dq"), (3, "dk")])
@pytest.mark.parametrize("d", [64, 128])
def test_a_wait_that_runs_out_ends_the_kernel(cuda, d, which, name):
    """One warp of the first CTA withholds an arrival: the waits behind it end at their limit, its rows are NaN, the others'
    right, the error is reported, and the next call is right."""
    lib = _ext.capi()
    T.check_errors(cuda)
    t, lx, ly = make((2, 700, 650, 2, 2, d, -1), torch.bfloat16, 71, False)
    want = run(t, lx, ly, -1)
    torch.cuda.synchronize()
    lib.sdtw_set_wait_timeout(0.2)
    try:
        if which > 1:  # the forward as usual
            leaves = [x.detach().requires_grad_(True) for x in t[:3]]
            out = T.cross_attention(*leaves)
        lib.sdtw_debug_attention_stall(which)
        got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, t[3]))) if which > 1 else run(t, lx, ly, -1, grads=False)
        torch.cuda.synchronize()
    finally:
        lib.sdtw_debug_attention_stall(0)
        lib.sdtw_set_wait_timeout(2.0)
    assert got[name][0, 0, 0].isnan().all()  # the first CTA's: sample 0, head 0, first rows
    assert torch.equal(got[name][1], want[name][1]) and torch.equal(got[name][0, :, 1], want[name][0, :, 1])
    with pytest.raises(RuntimeError, match="timed out"):
        T.check_errors(cuda)
    again = run(t, lx, ly, -1)
    assert all(torch.equal(again[n], want[n]) for n in want)
    T.check_errors(cuda)


@pytest.mark.parametrize("B,N,M,Hq,Hkv,d", [(2, 300, 300, 4, 2, 128), (1, 4000, 1000, 2, 1, 16), (2, 300, 2000, 4, 4, 64),
                                            (1, 20, 30000, 4, 4, 128), (2, 1, 4000, 8, 2, 128)])
def test_float32_over_long_sums(cuda, B, N, M, Hq, Hkv, d):
    """Relative error over an output's elements, where roundings of one sign would add up.

    An operand in two parts is off by 2^-24, the dropped product of tails by 2^-24: a product by 2^-22.4, and by a third
    of that as a root mean square over operands. A score adds the same to its weight's exponent (scores have a standard
    deviation of 1.5). A sum of n parts in 32 bits adds half of 2^-24 n^(1/2) at most where roundings have either sign:
    2^-20.6 for n = 940 tiles (30000 states). Five such terms in squares stay below 2^-19.
    """
    t, lx, ly = make((B, N, M, Hq, Hkv, d, -1), torch.float32, 81, False)
    got = run(t, lx, ly, -1, given=False)
    q, k, v, dout = [x.double().detach().requires_grad_() for x in t]
    kk, vv = [x.repeat_interleave(Hq // Hkv, 2) for x in (k, v)]
    p = (torch.einsum("bnhd,bmhd->bhnm", q, kk) * d**-0.5).softmax(-1)
    out = torch.einsum("bhnm,bmhd->bnhd", p, vv)
    want = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), dout)), out=out.detach())
    for name, w in want.items():
        assert ((got[name].double() - w).norm() / w.norm()).item() <= 2**-19, name


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("d", [8, 16, 32])
def test_dq_of_few_features(cuda, d, dtype):
    """With few features a few large dS carry dq: their rounding has to be made good.

    Rounding dq itself costs 0.42 u over its elements (uniform within a half step, 0.58 u of a value between 1 and 2,
    0.72 of that over mantissas spread evenly in the logarithm). delta takes the output's weights, rounded: 0.35 u of a
    part of dq that is a third to a half of it at d = 8 to 32. Together 0.46 u; rounding dS adds 0.5 u, in squares 0.68 u.
    """
    t, lx, ly = make((2, 2000, 600, 2, 1, d, -1), dtype, 83, False)
    got = run(t, lx, ly, -1, given=False)["dq"]
    vals, _ = plain.attention(*t[:3], lx, ly, -1, 1 / math.sqrt(d), t[3])
    want = vals["dq"]
    assert ((got.double() - want).norm() / want.norm()).item() <= 0.55 * torch.finfo(dtype).eps / 2
