"""GPU: the head norm with rotation and its gradients against a plain implementation in 64 bits."""

import math

import pytest
import torch

import sequence_plain as plain
import torchsoftdtw_b200 as T

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]

# B, N, H, d, rotary, interleaved
SHAPES = [
    (1, 1, 1, 1, 0, False),
    (1, 1, 1, 2, 2, True),
    (2, 3, 5, 33, 32, False),
    (2, 3, 5, 33, 18, True),
    (8, 1, 8, 64, 64, False),
    (2, 37, 3, 64, 64, True),
    (2, 50, 4, 128, 128, False),
    (1, 70, 2, 96, 64, True),
    (1, 70, 2, 96, 48, False),
    (3, 11, 7, 80, 20, False),
    (2, 9, 2, 256, 256, False),
    (2, 9, 2, 255, 2, True),
    (1, 5, 33, 16, 16, False),
    (1, 5, 3, 8, 8, True),
    (1, 900, 13, 200, 100, False),
    (4, 130, 1, 40, 0, False),
]


def make(shape, dtype, seed, ragged, positions, weight):
    B, N, H, d, *_ = shape
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, N, H, d, generator=g) * 2).to(dtype).cuda()
    dy = torch.randn(B, N, H, d, generator=g).to(dtype).cuda()
    lengths = torch.full((B,), N)
    if ragged:
        lengths = torch.randint(0, N + 1, (B,), generator=g)
        for b in range(B):
            x[b, lengths[b]:] = math.nan
            dy[b, lengths[b]:] = math.nan
    pos = {"": None, "int": torch.randint(0, 1 << 20, (B, N), generator=g), "int32": torch.randint(-50, 50, (N,), generator=g).int(),
           "real": torch.rand(B, N, generator=g) * 5000}[positions]
    w = None if weight is None else (1 + 0.2 * torch.randn(d, generator=g)).to(dtype if weight == "same" else torch.float32).cuda()
    return x, dy, lengths, None if pos is None else pos.cuda(), w


def run(x, dy, lengths, pos, w, rotary, interleaved, base=10000.0, eps=1e-6):
    x = x.detach().requires_grad_(True)
    leaves = [x] + ([] if w is None else [w.detach().requires_grad_(True)])
    y = T.norm_rotate(x, leaves[1] if w is not None else None, None if lengths is None else lengths.cuda(), pos, rotary,
                      base, interleaved, eps)
    grads = torch.autograd.grad(y, leaves, dy)
    res = {"y": y.detach(), "dx": grads[0]}
    if w is not None:
        res["dweight"] = grads[1]
    return res


def compare(res, x, dy, lengths, pos, w, rotary, interleaved, base=10000.0, eps=1e-6):
    if lengths is None:
        lengths = torch.full((x.shape[0],), x.shape[1])
    vals, errs = plain.norm_rotate(x, w, lengths, pos, rotary, base, interleaved, eps, dy)
    for name, got in res.items():
        plain.check(name, got, vals[name], errs[name])


@pytest.mark.parametrize("ragged,positions,weight", [(False, "", None), (True, "int", "float32"), (True, "real", "same"),
                                                     (False, "int32", "float32")])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_and_gradients(cuda, shape, dtype, ragged, positions, weight):
    args = make(shape, dtype, 3, ragged, positions, weight)
    compare(run(*args, *shape[4:]), *args, *shape[4:])
    T.check_errors(cuda)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("layout", ["heads first", "fused", "odd stride", "expanded", "reversed features", "offset"])
def test_strides(cuda, dtype, layout):
    B, N, H, d = 2, 19, 4, 64

    def rnd(*s):
        return torch.randn(*s, device=cuda).to(dtype)

    torch.manual_seed(5)
    x, dy = {
        "heads first": lambda: [rnd(B, H, N, d).transpose(1, 2) for _ in range(2)],
        "fused": lambda: [rnd(B, N, 3, H, d)[:, :, 1] for _ in range(2)],
        "odd stride": lambda: [rnd(B, N, H, d + 1)[..., :d] for _ in range(2)],
        "expanded": lambda: [rnd(B, N, 1, d).expand(B, N, H, d), rnd(d).expand(B, N, H, d)],
        "reversed features": lambda: [rnd(B, N, d, H).transpose(2, 3) for _ in range(2)],
        "offset": lambda: [rnd(B * N * H * d + 1)[1:].view(B, N, H, d) for _ in range(2)],
    }[layout]()
    w, pos = torch.rand(d, device=cuda), torch.arange(2 * N, device=cuda)[::2].expand(B, N)
    args = (x, dy, None, pos, w)
    compare(run(*args, 64, False), *args, 64, False)


def test_far_positions_keep_their_angles(cuda):
    """Neighbouring positions beyond 2^24 and up to 2^40: a 32-bit angle would be off by whole turns."""
    x = torch.randn(1, 6, 2, 64, device=cuda)
    dy = torch.randn(1, 6, 2, 64, device=cuda)
    pos = torch.tensor([[0, 1, 2**24 + 1, 2**31 + 5, 2**40 + 3, -(2**33) - 1]], device=cuda)
    args = (x, dy, None, pos, None)
    compare(run(*args, 16, True, 1e6), *args, 16, True, 1e6)


def test_zero_rows_and_large_values(cuda):
    for dtype, big in ((torch.float32, 1e15), (torch.bfloat16, 1e15), (torch.float16, 6e4)):
        x = torch.randn(1, 4, 2, 64, device=cuda).to(dtype)
        x[0, 1] = 0
        x[0, 2] = big
        dy = torch.randn(1, 4, 2, 64, device=cuda).to(dtype)
        args = (x, dy, None, None, torch.ones(64, device=cuda))
        res = run(*args, 64, False)
        assert all(t.isfinite().all() for t in res.values())
        compare({"y": res["y"]}, *args, 64, False)


def test_bad_lengths_are_reported(cuda):
    T.check_errors(cuda)
    args = make((3, 5, 2, 64, 64, False), torch.float32, 7, False, "", "same")
    lengths = torch.tensor([5, 6, -1])
    res = run(args[0], args[1], lengths, *args[3:], 64, False)
    assert res["y"][1:].isnan().all() and res["y"][0].isfinite().all()
    assert (res["dx"][1:] == 0).all() and res["dweight"].isfinite().all()
    with pytest.raises(RuntimeError, match="length"):
        T.check_errors(cuda)


def test_empty(cuda):
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        x = torch.zeros(shape, device=cuda, requires_grad=True)
        w = torch.ones(8, device=cuda, requires_grad=True)
        y = T.norm_rotate(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
        assert y.shape == x.shape and dx.shape == x.shape and (dw == 0).all()


def test_same_bits_streams_and_graphs(cuda):
    shape = (4, 300, 6, 128, 128, False)
    sets = [make(shape, torch.bfloat16, s, True, "int", "float32") for s in (11, 13)]
    want = [run(*s, *shape[4:]) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append([run(*s, *shape[4:]) for _ in range(4)][-1])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(a[n], b[n]) for n in b)
    x, dy, lengths, pos, w = [None if t is None else t.clone().cuda() for t in sets[0]]
    x.requires_grad_(True)
    w.requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = T.norm_rotate(x, w, lengths, pos)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
    for s, ref in ((sets[1], want[1]), (sets[0], want[0])):
        with torch.no_grad():
            for t, new in zip((x, dy, lengths, pos, w), s):
                t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref["y"]) and torch.equal(dx, ref["dx"]) and torch.equal(dw, ref["dweight"])


def test_differences(cuda):
    """fp32 gradients against central differences of the kernel's own outputs (see test_gpu_attention.py)."""
    args = make((2, 5, 3, 16, 12, True), torch.float32, 17, False, "real", "same")
    x, dy, lengths, pos, w = args
    res = run(*args, 12, True)
    _, errs = plain.norm_rotate(x, w, lengths, pos, 12, 10000.0, True, 1e-6, dy)
    h = 2.0**-5
    for name, at in (("dx", 0), ("dweight", 1)):
        direction = torch.randn_like((x, w)[at])

        def loss(step):
            xs, ws = (x + step * direction, w) if at == 0 else (x, w + step * direction)
            return (T.norm_rotate(xs, ws, None, pos, 12, 10000.0, True).double() * dy.double()).sum().item()

        D = [(loss(s) - loss(-s)) / (2 * s) for s in (h, h / 2)]
        noise = 1.5 * (errs["y"] * dy.double().abs()).sum().item() / (h / 2)
        slope = (res[name].double() * direction.double()).sum().item()
        slack = (errs[name] * direction.double().abs()).sum().item()
        assert abs(D[1] - slope) <= 2 * abs(D[0] - D[1]) + noise + slack, name
