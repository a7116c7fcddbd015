"""GPU: the global norm over the whole range of float64, and clipping by it.

Sums run in 64 bits: a norm of n entries is off by at most n 2^-52 of itself, and by half the smallest subnormal number. A
clipped entry carries that, the factor's two roundings and its own (2^-53 each); a factor below 2^-1022 is a subnormal number,
off by 2^-1075 whatever its size."""

import math
from fractions import Fraction

import pytest
import torch

import torchsoftdtw_b200 as T

pytestmark = pytest.mark.gpu

LEAST = 2.0**-1074


def exact_norm(values):
    """The norm of some floats, correctly to 60 bits or more, as a fraction."""
    total = sum(Fraction(v) ** 2 for v in values)
    if not total:
        return Fraction(0)
    shift = 2 * max(0, 700 - (total.numerator.bit_length() - total.denominator.bit_length()) // 2)
    return Fraction(math.isqrt(total.numerator * 2**shift // total.denominator), 2 ** (shift // 2))


@pytest.mark.parametrize("values", [
    [1e305], [1.7e308], [1e305, 0.5, -3.0], [1e308, -1e308], [4e304] * 100, [2.6e120, 2.5e120, 1e121], [1e200, 1e-200, 1e-320],
    [1e-320], [5e-324], [5e-324] * 4 + [0.0] * 7, [1e-320, -1e-310, 1e-300], [4e-121, 3.8e-121, 1e-130], [1e-150, 1e-170],
], ids=lambda v: f"{v[0]:g} of {len(v)}")
def test_the_whole_range_of_float64(cuda, values):
    ts = [torch.tensor(values, dtype=torch.float64, device=cuda), torch.zeros(20000, dtype=torch.float32, device=cuda)]
    norm = T.global_norm(ts)
    want = exact_norm(values)
    rel = Fraction(len(values) + 2, 2**52)
    assert norm.dtype == torch.float64 and math.isfinite(norm.item())
    assert abs(Fraction(norm.item()) - want) <= rel * want + Fraction(LEAST) / 2
    out, norm2 = T.clip_grads(ts, 1.0)
    assert torch.equal(norm, norm2)
    coef = min(Fraction(1), 1 / (want + Fraction(1e-6)))
    for got, v in zip(out[0].tolist(), values):
        w = coef * Fraction(v)
        slack = abs(Fraction(v)) * Fraction(LEAST) / 2 + Fraction(LEAST) / 2
        assert abs(Fraction(got) - w) <= (rel + Fraction(3, 2**53)) * abs(w) + slack
    assert (out[1] == 0).all()
