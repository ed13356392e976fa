"""Rotary tables hold the nearest 64-bit fraction of each plane's frequency: bounds in whole numbers, without roots or logarithms."""
import math
from fractions import Fraction

import pytest

torch = pytest.importorskip("torch")
from msnhnet_b200 import tokens  # noqa: E402

# pi to 60 digits, from below
PI = Fraction(314159265358979323846264338327950288419716939937510582097494, 10 ** 59)


@pytest.fixture
def ops():
    handle = tokens.TokenOps.__new__(tokens.TokenOps)
    handle.device = torch.device("cpu")
    return handle


def near(turns, dim, i, base, slower=Fraction(1)):
    """Whether turns / 2^64, half a unit (and a hundredth) off at most, is base ** (-2 i / dim) / (2 pi slower): both sides to the power of dim."""
    bound, want = Fraction(51, 100), Fraction(1) / Fraction(base) ** (2 * i)
    least, most = ((Fraction(turns) + d) / 2 ** 64 * 2 * PI * slower for d in (-bound, bound))
    return max(least, 0) ** dim < want < most ** dim


@pytest.mark.parametrize("dim", [2, 8, 64, 128])
@pytest.mark.parametrize("base", [10000.0, 500000.0, 1234.5678, 3.0])
def test_frequencies_are_the_nearest_fractions(ops, dim, base):
    for i, turns in enumerate(ops.rotary_table(dim, base=base).turns.tolist()):
        assert near(turns, dim, i, base), i
    for i, turns in enumerate(ops.rotary_table(dim, base=base, stretch="all", factor=3.7).turns.tolist()):
        assert near(turns, dim, i, base, Fraction(3.7)), i


@pytest.mark.parametrize("dim", [4, 8, 12])
def test_stretched_by_the_base(ops, dim):
    base, factor = 10000.0, 5.5
    for i, turns in enumerate(ops.rotary_table(dim, base=base, stretch="base", factor=factor).turns.tolist()):
        # (base * factor ** (dim / (dim - 2))) ** (-2 i / dim), to the power of dim * (dim - 2)
        want = Fraction(1) / (Fraction(base) ** (dim - 2) * Fraction(factor) ** dim) ** (2 * i)
        least, most = ((Fraction(turns) + d) / 2 ** 64 * 2 * PI for d in (Fraction(-51, 100), Fraction(51, 100)))
        assert max(least, 0) ** (dim * (dim - 2)) < want < most ** (dim * (dim - 2)), i


def test_slow_planes_are_stretched_and_fast_ones_are_not(ops):
    dim, base, factor, trained = 64, 500000.0, 8.0, 8192
    got = ops.rotary_table(dim, base=base, stretch="slow", factor=factor, trained=trained).turns.tolist()
    kinds = set()
    for i, turns in enumerate(got):
        times = trained * base ** (-2 * i / dim) / (2 * math.pi)
        if times > 4.001 or times < 0.999:
            assert near(turns, dim, i, base, Fraction(factor if times < 1 else 1.0)), i
            kinds.add(times < 1)
        else:
            kept = (times - 1) / 3
            one = base ** (-2 * i / dim) / (2 * math.pi)
            assert math.isclose(turns / 2 ** 64, one * (kept + (1 - kept) / factor), rel_tol=1e-13)
            kinds.add(None)
    assert kinds == {True, False, None}


@pytest.mark.parametrize("more,turns", [({"base": math.inf}, 1), ({"factor": math.inf, "stretch": "all"}, 0), ({"factor": math.inf, "stretch": "base"}, 1)])
def test_infinite_bases_and_factors_leave_planes_still(ops, more, turns):
    got = ops.rotary_table(8, **more).turns.tolist()
    assert got[turns:] == [0] * (4 - turns) and (not turns or near(got[0], 8, 0, 2.0))
