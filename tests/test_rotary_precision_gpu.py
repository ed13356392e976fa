"""How small angles of rotary positions may be: the slow planes' sines at the first positions."""
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

