"""GPU: clipping of views of one buffer: allowed where no entry that is written is another tensor's, refused otherwise."""

import random

import pytest
import torch

import torchsoftdtw_b200 as T

pytestmark = pytest.mark.gpu


def expected(ts, max_norm):
    """Clipped copies, in 64 bits."""
    norm = torch.stack([t.double().square().sum() for t in ts]).sum().sqrt().item()
    return [t.double() * min(1.0, max_norm / (norm + 1e-6)) for t in ts], norm


def near(got, want):
    """A norm is off by 2^-19 in float32, an entry by that and its rounding."""
    worst = ((got.double() - want).abs() - 2.0**-18 * want.abs()).max().item()
    assert worst <= 0


@pytest.mark.parametrize("cut", [
    lambda a: [a[:, :40], a[:, 40:]],
    lambda a: [a[:, 0::3], a[:, 1::3], a[:, 2::3]],
    lambda a: [a[0::2], a[1::2]],
    lambda a: [a[:16, :50], a[16:, 50:], a[16:, :50], a[:16, 50:]],
    lambda a: [a[:, 40:].t(), a[:, :40].t()],
    lambda a: [a.view(30, 10, 10)[:, :, :4], a.view(30, 10, 10)[:, :, 4:]],
    lambda a: [a.view(-1)[1:], a.view(-1)[:1]],
], ids=["columns", "every third column", "every second row", "quarters", "transposed", "three dimensions", "offset"])
def test_slices_of_one_matrix(cuda, cut):
    a = torch.randn(30, 100, device=cuda)
    want, norm = expected(cut(a), 0.5)
    res, n = T.clip_grads(cut(a), 0.5)
    near(n, torch.tensor(norm, device=cuda))
    for g, w in zip(res, want):
        near(g, w)
    b = a.clone()
    params = [torch.zeros_like(t) for t in cut(b)]
    for p, t in zip(params, cut(b)):
        p.grad = t
    T.clip_grad_norm_(params, 0.5)
    for t, w in zip(cut(b), want):
        near(t, w)
    near(b, expected([a], 0.5)[0][0])


@pytest.mark.parametrize("cut", [
    lambda a: [a[:, :41], a[:, 40:]],
    lambda a: [a[:, 0::3], a[:, 0::2]],
    lambda a: [a[:, :40], a.t()[39:, :]],
    lambda a: [a[3], a[:, 7]],
    lambda a: [a.view(torch.float16)[:, ::2], a[:, 99:]],
], ids=["columns", "third and second columns", "transposed", "row and column", "types"])
def test_slices_that_share_entries(cuda, cut):
    a = torch.randn(30, 100, device=cuda)
    keep = a.clone()
    with pytest.raises(RuntimeError, match="shares memory"):
        T.clip_grads(cut(a), 0.5, out=cut(a))
    assert torch.equal(a, keep)
    T.clip_grads(cut(a), 0.5)  # read alone they may


def test_an_output_with_entries_in_one_place(cuda):
    """Refused before anything is written."""
    a, b = torch.randn(50, device=cuda), torch.randn(5, 1, device=cuda)
    keep = a.clone(), b.clone()
    with pytest.raises(RuntimeError, match="several entries in one place"):
        T.clip_grads([a, b.expand(5, 9)], 0.1, out=[a, b.expand(5, 9)])
    assert torch.equal(a, keep[0]) and torch.equal(b, keep[1])


def test_random_views(cuda):
    """Pairs of strided views are refused exactly where they share an entry."""
    rng = random.Random(10)
    buf = torch.randn(400, device=cuda)
    index = torch.arange(400)
    refused = 0
    for _ in range(600):
        views = []
        while len(views) < 2:
            size = [rng.randint(1, 6) for _ in range(rng.randint(1, 3))]
            stride = [rng.choice([1, 2, 3, 5, 8, 13, 20, 40]) for _ in size]
            at = rng.randint(0, 150)
            if at + sum((s - 1) * d for s, d in zip(size, stride)) >= 400:
                continue
            ids = index.as_strided(size, stride, at).flatten().tolist()
            if len(set(ids)) == len(ids):
                views.append((size, stride, at, set(ids)))
        ts = [buf.as_strided(*v[:3]) for v in views]
        if views[0][3] & views[1][3]:
            refused += 1
            with pytest.raises(RuntimeError, match="shares memory"):
                T.clip_grads(ts, 1.0, out=ts)
        else:
            T.clip_grads(ts, 1.0, out=ts)
    assert 50 < refused < 550  # both kinds are there
