"""How small and how far angles of rotary positions may be: the slow planes' sines at the first positions, and positions as far as frequencies carry."""
import decimal
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from msnhnet_b200 import tokens
    handle = tokens.TokenOps(0)
    yield handle
    handle.close()


def signed(turns):
    """Fractions of a turn from -1/2 on, of whole numbers modulo 2^64."""
    return ((turns + 2 ** 63) % 2 ** 64 - 2 ** 63) / 2 ** 64


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("base,more", [(500000.0, {"stretch": "all", "factor": 8.0}), (1e7, {}), (1e30, {})])
def test_rotary_keeps_small_angles(ops, base, more, interleaved):
    dim, at = 128, [1, -1, 2, 3, 17, 1000]
    table = ops.rotary_table(dim, base=base, interleaved=interleaved, **more)
    x = torch.zeros(len(at), 1, dim, device="cuda")
    a, b = (slice(0, dim, 2), slice(1, dim, 2)) if interleaved else (slice(0, dim // 2), slice(dim // 2, dim))
    x[..., a] = 1.0
    y = ops.rotary(x, torch.tensor(at, dtype=torch.int32, device="cuda"), table)
    angle = torch.tensor([[2 * math.pi * signed(p * t) for t in table.turns.tolist()] for p in at], dtype=torch.float64, device="cuda")
    want = torch.sin(angle)
    # what x turns into is the sine. The fraction is rounded to 24 bits: 2^-24 of the angle, and a sine's slope is 1 at most, so it is off by no more than
    # 2^-24 |angle| (which is 2^-24 of the sine itself where angles are small, and more towards half a turn, where the sine is small again); the sine to two
    # units (2^-22 of it), times a magnitude of 1
    off = (y[:, 0, b].double() - want).abs()
    assert bool((off <= 2.0 ** -24 * angle.abs() + 2.0 ** -22 * want.abs()).all()), float((off - 2.0 ** -24 * angle.abs() - 2.0 ** -22 * want.abs()).max())


PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494")


def test_rotary_of_far_positions_goes_by_the_frequencies_themselves(ops):
    # base ** (-2 i / dim) to 50 digits, as square roots: dim 16 and base 10 ** 8 give powers of ten
    dim = 16
    table = ops.rotary_table(dim, base=1e8)
    at = [2 ** 31 - 1, -2 ** 31, 2 ** 36 + 12345, -(2 ** 38) + 1, 2 ** 40 + 7]
    x = torch.randn(len(at), 3, dim, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    y = ops.rotary(x, torch.tensor(at, device="cuda"), table).double()
    angle = []
    with decimal.localcontext(decimal.Context(prec=50)):
        for p in at:
            for i in range(dim // 2):
                turn = p / (decimal.Decimal(10) ** i * 2 * PI)
                angle.append(float(turn - turn.to_integral_value()) * 2 * math.pi)
    angle = torch.tensor(angle, dtype=torch.float64, device="cuda").view(len(at), 1, dim // 2)
    a, b = x[..., :dim // 2].double(), x[..., dim // 2:].double()
    want = torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1)
    # ten roundings of fp32 of the plane's size, and the frequency's own half unit of 2^-64 of a turn times the position
    far = 2 * math.pi * 2.0 ** -65 * torch.tensor(at, dtype=torch.float64, device="cuda").abs()[:, None, None]
    bound = (10 * 2.0 ** -24 + far) * (a.abs() + b.abs()).repeat(1, 1, 2) + 2.0 ** -24 * want.abs()
    off = (y - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
