"""GPU: the global norm and clipping against 64-bit sums. The norm's squares are formed and added in 32 bits only
64 at a time, so it is off by at most 2^-19 of itself in float32 (64 * 2^-24 halved by the root, and its own rounding) and
n 2^-52 where a float64 tensor makes all of it 64-bit; a clipped entry by the norm's error and a half step of its type."""

import math

import pytest
import torch

import torchsoftdtw_b200 as T

pytestmark = pytest.mark.gpu

F32, F16, BF16, F64 = torch.float32, torch.float16, torch.bfloat16, torch.float64


def tensors(spec, seed=0, scale=0.02):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g, dtype=F64) * scale).to(t).cuda() for s, t in spec]


def reference(ts, kind):
    if kind == 2.0:
        return math.sqrt(sum(t.double().square().sum().item() for t in ts))
    return max((t.double().abs().max().item() for t in ts if t.numel()), default=0.0)


def close(ts, out, norm, max_norm, kind):
    wide = any(t.dtype == F64 for t in ts)
    want = reference(ts, kind)
    rel = (1e-10 if wide else 2**-19) if kind == 2.0 else (0.0 if wide else 2**-24)
    assert norm.dtype == (F64 if wide else F32) and norm.dim() == 0
    assert abs(norm.item() - want) <= rel * want
    coef = min(1.0, max_norm / (want + 1e-6))
    for t, o in zip(ts, out):
        assert o.dtype == t.dtype and o.shape == t.shape
        w = t.double() * coef
        step = max(torch.finfo(t.dtype).eps / 2, 0 if t.dtype == F64 else 2**-23)
        assert ((o.double() - w).abs() <= (rel + step + 2**-52) * w.abs() + (2**-25 if t.dtype == F16 else 0)).all()


SPECS = {
    "one": [((1,), F32)],
    "few": [((7,), F32), ((33, 65), BF16), ((), F16), ((0, 4), F32), ((129,), F64)],
    "single type": [((257, 129), F32)] * 5,
    "half": [((1000,), F16), ((3, 5, 7), F16)],
    "chunks": [((32768,), BF16), ((32769,), BF16), ((32767,), F32), ((65536 * 3 + 5,), F16)],
    "many": [((i % 97 + 1,), (F32, BF16, F16)[i % 3]) for i in range(1000)],
    "table": [((i % 5,), F32) for i in range(64)],
    "table + 1": [((17,), F32) for i in range(65)],
    "two tables": [((9,), F32) for i in range(2000)],
}


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("max_norm", [0.01, 1e6, 0.0])
@pytest.mark.parametrize("spec", list(SPECS))
def test_values(cuda, spec, max_norm, kind):
    ts = tensors(SPECS[spec], 1)
    before = [t.clone() for t in ts]
    out, norm = T.clip_grads(ts, max_norm, kind)
    assert all(torch.equal(a, b) for a, b in zip(ts, before))
    close(ts, out, norm, max_norm, kind)
    assert torch.equal(T.global_norm(ts, kind), norm)
    params = [t.clone() for t in ts]
    for p, t in zip(params, before):
        p.grad = t.clone()
    n = T.clip_grad_norm_(params, max_norm, kind)
    assert torch.equal(n, norm)
    assert all(torch.equal(p.grad, o) for p, o in zip(params, out))


def test_large_sum_and_repeatable(cuda):
    ts = tensors([((1 << 22,), F32), ((3000, 3001), BF16), ((5,), F32)], 2)
    out, norm = T.clip_grads(ts, 1.0)
    close(ts, out, norm, 1.0, 2.0)
    for _ in range(3):
        again, n = T.clip_grads(ts, 1.0)
        assert torch.equal(n, norm) and all(torch.equal(a, b) for a, b in zip(again, out))


@pytest.mark.parametrize("value,dtype", [(1e30, F32), (3e38, BF16), (1e-30, F32), (1e-44, F32), (6e4, F16), (1e-300, F64)])
def test_squares_outside_the_type(cuda, value, dtype):
    """Squares that overflow or underflow 32 bits do not spoil the norm."""
    ts = [torch.full((100,), value, dtype=dtype, device=cuda), torch.zeros(50000, dtype=dtype, device=cuda)]
    norm = T.global_norm(ts)
    want = 10 * ts[0][0].double().item()
    if want > torch.finfo(norm.dtype).max:
        assert norm.item() == math.inf
    else:
        assert abs(norm.item() - want) <= 2**-19 * want + 2.0**-149 * (norm.dtype == F32)


def test_nan_and_infinity(cuda):
    for kind in (2.0, math.inf):
        ts = tensors([((50,), F32), ((70000,), BF16)], 3)
        ts[1][65000] = math.nan
        out, norm = T.clip_grads(ts, 1.0, kind)
        assert norm.isnan() and all(o.isnan().all() for o in out)
        ts[1][65000] = -math.inf
        out, norm = T.clip_grads(ts, 1.0, kind)
        assert norm.item() == math.inf
        assert (out[0] == 0).all() and out[1][65000].isnan() and (out[1][:65000] == 0).all()
        p = ts[0].clone()
        p.grad = ts[1].clone()[:50].float()
        q = ts[1].clone()
        q.grad = ts[1].clone()
        keep = [p.grad.clone(), q.grad.clone()]
        with pytest.raises(RuntimeError, match="not finite"):
            T.clip_grad_norm_([p, q], 1.0, kind, error_if_nonfinite=True)
        assert torch.equal(p.grad, keep[0]) and torch.equal(q.grad, keep[1])


def test_layouts(cuda):
    torch.manual_seed(4)
    base = torch.randn(40, 50, device=cuda)
    ts = [base.t(), torch.randn(6, 7, 8, device=cuda).permute(2, 0, 1), torch.randn(30, 20, device=cuda)[:, ::2],
          torch.randn(1001, device=cuda)[1:], torch.randn(5, 1, device=cuda).expand(5, 9)]
    out, norm = T.clip_grads(ts, 0.5)
    close(ts, out, norm, 0.5, 2.0)
    mixed = [torch.empty(50, 40, device=cuda), torch.empty(8, 6, 7, device=cuda), torch.empty(30, 20, device=cuda)[:, ::2],
             torch.empty(1003, device=cuda)[3:], torch.empty(5, 9, device=cuda)]
    res, norm2 = T.clip_grads(ts, 0.5, out=mixed)
    assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(res, out))
    inside = [ts[0].clone(), torch.randn(30, 20, device=cuda)[:, ::2]]
    want = [t.clone() for t in inside]
    res, norm3 = T.clip_grads(inside, 0.5, out=inside)
    close(want, res, norm3, 0.5, 2.0)


def test_shared_memory_is_refused(cuda):
    a = torch.randn(100, device=cuda)
    with pytest.raises(RuntimeError, match="shares memory"):
        T.clip_grads([a, a], 1.0, out=[a, a])
    with pytest.raises(RuntimeError, match="shares memory"):
        T.clip_grads([a[:60]], 1.0, out=[a[40:]])
    with pytest.raises(RuntimeError, match="shares memory"):
        T.clip_grads([a[:50], a[50:]], 1.0, out=[a[50:], torch.empty(50, device=cuda)])
    out, norm = T.clip_grads([a, a], 1.0)  # read twice, counted twice
    close([a, a], out, norm, 1.0, 2.0)
    p = torch.randn(10, device=cuda)
    p.grad = torch.randn(10, device=cuda)
    keep = p.grad.clone()
    n = T.clip_grad_norm_([p, p], 0.1)  # a parameter listed twice has one gradient
    close([keep], [p.grad], n, 0.1, 2.0)


def test_in_place_below_the_bound_writes_nothing(cuda):
    a = tensors([((1000,), F32)], 5)[0]
    keep = a.clone()
    T.clip_grads([a], 1e9, out=[a])
    assert torch.equal(a, keep)


def test_nothing_to_clip(cuda):
    assert T.clip_grads([], 1.0)[1].item() == 0 and T.global_norm([]).item() == 0
    assert T.clip_grad_norm_([torch.zeros(3, device=cuda)], 1.0).item() == 0
    empty = [torch.empty(0, device=cuda)]
    out, norm = T.clip_grads(empty, 1.0)
    assert norm.item() == 0 and out[0].numel() == 0


def test_streams_and_graph(cuda):
    sets = [tensors([((70000,), F32), ((300, 300), BF16)], s) for s in (6, 7)]
    want = [T.clip_grads(s, 0.3) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append([T.clip_grads(s, 0.3) for _ in range(5)][-1])
    torch.cuda.synchronize()
    for (o, n), (wo, wn) in zip(got, want):
        assert torch.equal(n, wn) and all(torch.equal(a, b) for a, b in zip(o, wo))
    bufs = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, norm = T.clip_grads(bufs, 0.3, out=bufs)
    for s, (wo, wn) in zip(sets, want):
        for b, t in zip(bufs, s):
            b.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, wn) and all(torch.equal(a, b) for a, b in zip(bufs, wo))
