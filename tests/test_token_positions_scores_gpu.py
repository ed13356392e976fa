"""Rotary positions and scores of tokens against plain implementations in 64 bits (angles in whole numbers), at the sizes, layouts and masks where
they can go wrong. Tolerances are bounds of the arithmetic, derived beside their checks."""
import math

import pytest

torch = pytest.importorskip("torch")
from msnhnet_b200 import _ffi  # noqa: E402

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}         # half a unit in the last place, relative
TINY = {F32: 1e-45, F16: 2.0 ** -25, BF16: 1e-40}               # half of the smallest value
INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def ops():
    from msnhnet_b200 import tokens
    handle = tokens.TokenOps(0)
    yield handle
    handle.close()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed, dtype=F32):
    return torch.randn(*shape, generator=gen(seed), device="cuda").to(dtype)


# ---- rotary positions -----------------------------------------------------------------------------------------------

def check_rotary(y, x, positions, table):
    """Angles from the table's fractions in whole numbers of any length."""
    turns, half = table.turns.tolist(), table.turns.numel()
    fraction = [[(p * t) % 2 ** 64 / 2 ** 64 for t in turns] for p in positions.tolist()]
    angle = 2 * math.pi * torch.tensor(fraction, dtype=torch.float64, device="cuda").reshape(len(positions), 1, half)
    cos, sin = torch.cos(angle) * table.magnitude, torch.sin(angle) * table.magnitude
    xd = x.double()
    a, b = (xd[..., 0:2 * half:2], xd[..., 1:2 * half:2]) if table.interleaved else (xd[..., :half], xd[..., half:2 * half])
    one, two = a * cos - b * sin, a * sin + b * cos
    want, size = xd.clone(), torch.zeros_like(xd)
    for i, (v, w) in enumerate(((one, a.abs() + b.abs()), (two, a.abs() + b.abs()))):
        at = slice(i, 2 * half, 2) if table.interleaved else slice(i * half, (i + 1) * half)
        want[..., at], size[..., at] = v, w * abs(table.magnitude)
    # the fraction rounded to 24 bits (pi 2^-25), sine and cosine to a unit (2^-23), the magnitude (2^-24, and its own 2^-24), two products and a sum (3 * 2^-24)
    bound = U[y.dtype] * want.abs() + 10 * 2.0 ** -24 * size + TINY[y.dtype]
    bound[..., 2 * half:] = 0
    off = (y.double() - want).abs()
    assert y.dtype == x.dtype and bool((off <= bound).all()), float((off - bound).max())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 40, 128, 128), (1, 1, 2, 2), (3, 5, 80, 32), (7, 3, 20, 6), (130, 9, 64, 64), (33, 2, 256, 250), (1, 300, 128, 64), (2, 3, 96, 96),
                                                  (700, 6, 128, 128), (2, 2, 2080, 2048), (5, 4, 40, 16), (0, 4, 64, 64), (3, 0, 64, 64), (4000, 3, 64, 32)])
def test_rotary_matches_the_formula(ops, dtype, tokens, heads, dim, rot, interleaved):
    x = randn(tokens, heads, dim, seed=1, dtype=dtype)
    positions = torch.randint(0, 100000, (tokens,), generator=gen(2), dtype=torch.int32, device="cuda")
    table = ops.rotary_table(rot, interleaved=interleaved, magnitude=1.25)
    check_rotary(ops.rotary(x, positions, table), x, positions, table)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_of_far_and_negative_positions(ops, interleaved):
    x = randn(8, 3, 64, seed=3)
    positions = torch.tensor([0, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 40 + 7, -2 ** 62, 2 ** 63 - 1, 12345], dtype=torch.int64, device="cuda")
    table = ops.rotary_table(64, interleaved=interleaved)
    check_rotary(ops.rotary(x, positions, table), x, positions, table)
    near = positions[[0, 1, 7]].int()
    assert torch.equal(ops.rotary(x[:3], near, table), ops.rotary(x[:3], near.long(), table))
    # turned back
    again = ops.rotary(ops.rotary(x, positions[:8] // 2, table), -(positions[:8] // 2), table)
    assert bool(((again - x).abs() <= 2.0 ** -19 * x.abs().amax()).all())


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("extra,front", [(0, 0), (8, 0), (3, 0), (0, 1), (8, 8)])
def test_rotary_layouts(ops, dtype, heads_first, extra, front):
    # queries and keys in rows that hold more, unaligned ones, heads before tokens; beside, in place and into other strides
    tokens, heads, dim = 19, 6, 64
    raw = torch.full((front + tokens * heads * (dim + extra),), NAN, device="cuda").to(dtype)
    wide = raw[front:].view((heads, tokens, dim + extra) if heads_first else (tokens, heads, dim + extra))
    x = (wide.transpose(0, 1) if heads_first else wide)[..., :dim]
    x.copy_(randn(tokens, heads, dim, seed=4, dtype=dtype))
    positions = torch.arange(1000, 1000 + tokens, dtype=torch.int32, device="cuda")
    for rot in (64, 24):
        table = ops.rotary_table(rot)
        y = ops.rotary(x, positions, table)
        check_rotary(y, x, positions, table)
        other = torch.full((tokens, heads + 1, dim + 2), NAN, device="cuda").to(dtype)
        ops.rotary(x, positions, table, out=other[:, :heads, :dim])
        assert torch.equal(other[:, :heads, :dim], y) and bool(torch.isnan(other[:, heads]).all()) and bool(torch.isnan(other[..., dim:]).all())
        kept = x.clone()
        assert ops.rotary(x, positions, table, out=x) is x or True
        assert torch.equal(x, y)
        if extra:
            assert bool(torch.isnan(wide[..., dim:]).all())
        x.copy_(kept)
    one = randn(1, heads, dim, seed=5, dtype=dtype).expand(tokens, heads, dim)          # a row that all tokens share
    check_rotary(ops.rotary(one, positions, table), one, positions, table)


def test_rotary_of_infinity_and_nan_stays_in_its_plane(ops):
    x = randn(2, 2, 64, seed=6)
    x[0, 0, 3], x[1, 1, 40] = NAN, INF
    table = ops.rotary_table(64)
    y = ops.rotary(x, torch.tensor([5, 6], dtype=torch.int32, device="cuda"), table)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[0, 0, 3] = bad[0, 0, 35] = bad[1, 1, 8] = bad[1, 1, 40] = True
    assert torch.equal(~torch.isfinite(y), bad)


@pytest.mark.parametrize("stretch,factor", [(None, 1.0), ("all", 4.0), ("base", 8.0), ("slow", 16.0)])
@pytest.mark.parametrize("dim", [2, 64, 96])
def test_rotary_tables(ops, stretch, factor, dim):
    base, trained, low, high = 500000.0, 8192, 1.0, 4.0
    table = ops.rotary_table(dim, base=base, stretch=stretch, factor=factor, trained=trained, low=low, high=high)
    for i, got in enumerate(table.turns.tolist()):
        f = (base * factor ** (dim / max(dim - 2, 1)) if stretch == "base" else base) ** (-2 * i / dim)
        if stretch == "all":
            f /= factor
        if stretch == "slow":
            length = 2 * math.pi / f                                  # positions of one turn
            if length >= trained / low:
                f /= factor
            elif length > trained / high:
                kept = (trained / length - low) / (high - low)
                f = kept * f + (1 - kept) * f / factor
        assert abs(got / 2 ** 64 - f / (2 * math.pi)) <= 2.0 ** -48 * f + 2.0 ** -63
    if stretch == "base" and dim > 2:
        assert math.isclose(table.turns[-1].item() * factor, ops.rotary_table(dim, base=base).turns[-1].item(), rel_tol=1e-9)


def test_rotary_refuses(ops):
    x, positions, table = randn(3, 2, 32, seed=7), torch.arange(3, dtype=torch.int32, device="cuda"), ops.rotary_table(32)
    for bad in (x[0], x.double(), x.transpose(1, 2)):
        with pytest.raises(ValueError):
            ops.rotary(bad, positions, table)
    for bad in (positions[:2], positions.float(), positions.short()):
        with pytest.raises(ValueError, match="positions"):
            ops.rotary(x, bad, table)
    with pytest.raises(ValueError, match="out"):
        ops.rotary(x, positions, table, out=torch.empty(3, 2, 16, device="cuda"))
    with pytest.raises(_ffi.KernelError, match="planes"):
        ops.rotary(x, positions, ops.rotary_table(64))
    with pytest.raises(_ffi.KernelError, match="overlap"):
        ops.rotary(x, positions, table, out=torch.empty(1, 2, 32, device="cuda").expand(3, 2, 32))
    with pytest.raises(_ffi.KernelError, match="2048"):
        ops.rotary(randn(1, 1, 2050, seed=8), positions[:1], ops.rotary_table(2050))
    with pytest.raises(ValueError, match="gradient"):
        ops.rotary(x.clone().requires_grad_(), positions, table)
    a = _ffi.Rotary(x.data_ptr(), x.data_ptr(), None, table.turns.data_ptr(), 3, 2, 32, 32, _ffi.F32, 0, 0, 64, 32, 64, 32, 1.0)
    assert ops.lib.msnh_b200_rotary(ops.h, a, None) == 1 and "null" in ops.ctx.error()
    a.dtype = _ffi.E4M3
    assert ops.lib.msnh_b200_rotary(ops.h, a, None) == 2
    assert ops.lib.msnh_b200_rotary(None, a, None) == 1


def test_rotary_tells_torch_of_its_writes(ops):
    x, positions, table = randn(3, 2, 32, seed=9), torch.arange(3, dtype=torch.int32, device="cuda"), ops.rotary_table(32)
    before = x._version
    ops.rotary(x, positions, table)
    assert x._version == before
    ops.rotary(x, positions, table, out=x)
    assert x._version == before + 1


# ---- scores of tokens -----------------------------------------------------------------------------------------------

def check_scores(got, logits, ids, top, lanes=128):
    logprob, entropy, top_logprobs, top_ids = got
    z = logits.double()
    cols = z.shape[1]
    good = torch.isfinite(z.amax(-1)) & ~torch.isnan(z).any(-1)
    none = torch.zeros_like(z[:, 0])
    best = torch.where(good, z.amax(-1), none)[:, None]
    d = torch.where(good[:, None], (best - z), torch.zeros_like(z))
    log_s = torch.logsumexp(-d, -1)
    p = torch.exp(-d - log_s[:, None])
    far = torch.where(p > 0, d, torch.zeros_like(d))
    mean, square = (p * far).sum(-1), (p * far * far).sum(-1)
    # e^-d: the distance is rounded (2^-24 d), times log2 e (2^-24 d), 2^x to two units; a thread adds its logits one by one, at most one in `lanes` of them,
    # (and its maximum's growth rescales them, ten times at most in what is bound here); then the threads are joined (nine steps)
    n = 2.0 ** -24 * (cols / lanes + 60)
    rel = n + 2.0 ** -23 * (2 * mean + 4)
    bound_log = rel + 2.0 ** -22 * log_s

    def near(x, want, bound):
        same = (x == want.float()) | (torch.isnan(x) & torch.isnan(want))     # (what is beyond fp32's range is infinite)
        off = torch.where(same, torch.zeros_like(want), (x.double() - want).abs())
        assert bool((off <= bound).all()), float((off - bound).max())
    nan = torch.full_like(none, NAN)
    if ids is not None:
        there = good & (ids >= 0) & (ids < cols)
        x = -d.gather(1, ids.clamp(0, cols - 1)[:, None])[:, 0]
        near(logprob, torch.where(there, x - log_s, nan), bound_log + 2.0 ** -22 * torch.where(torch.isfinite(x), x.abs(), none))
    else:
        assert logprob is None
    near(entropy, torch.where(good, log_s + mean, nan), bound_log + mean * (rel + n) + 2.0 ** -23 * (2 * square + 4 * mean) + 2.0 ** -22 * (log_s + mean))
    if not top:
        assert top_logprobs is None and top_ids is None
        return
    order = torch.sort(z + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(top_ids, torch.where(good[:, None], order, torch.full_like(order, -1)))
    x = -d.gather(1, order)
    near(top_logprobs, torch.where(good[:, None], x - log_s[:, None], nan[:, None]), bound_log[:, None] + 2.0 ** -22 * torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols,top", [(1, 1, 1), (1, 2, 0), (3, 5, 5), (2, 31, 31), (2, 33, 32), (64, 1000, 5), (1, 1000, 32), (5, 4096, 8), (5, 4097, 8), (1, 8200, 20), (1, 40000, 32),
                                           (40, 16400, 4), (300, 9001, 3), (2, 131077, 20), (700, 5003, 1), (0, 100, 3), (1, 262144, 8)])
def test_scores_match_the_formula(ops, dtype, rows, cols, top):
    # (16-bit logits have many ties)
    z = (randn(rows, cols, seed=20) * 3).to(dtype)
    ids = torch.randint(0, cols, (rows,), generator=gen(21), device="cuda")
    check_scores(ops.token_scores(z, ids, top=top), z, ids, top)
    if cols == 1000:
        check_scores(ops.token_scores(z, top=top), z, None, top)
        check_scores(ops.token_scores(z, ids), z, ids, 0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols,top", [(1300, 1, 1), (1300, 30, 30), (1300, 128, 32), (1300, 129, 32), (1300, 257, 20), (1300, 512, 32), (1300, 513, 32), (1300, 1000, 8), (1300, 4096, 8), (1300, 4097, 8),
                                           (2000, 3001, 0), (4500, 1024, 32), (4500, 1025, 9), (4500, 8191, 8), (4500, 8192, 1), (4500, 8193, 8)])
def test_scores_of_many_narrow_rows(ops, dtype, rows, cols, top):
    z = (randn(rows, cols, seed=120) * 3).to(dtype)
    z[5::7, ::2] = -INF
    z[6::7, cols // 2] = NAN
    z[7::70] = -INF
    z[8::70] = 1.0
    ids = torch.randint(0, cols, (rows,), generator=gen(121), device="cuda")
    check_scores(ops.token_scores(z, ids, top=top), z, ids, top, lanes=32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [60, 500, 4000])
@pytest.mark.parametrize("extra,front", [(0, 1), (3, 0), (1, 5)])
def test_scores_of_many_narrow_rows_that_start_anywhere(ops, dtype, cols, extra, front):
    rows = 1100
    raw = torch.full((front + rows * (cols + extra),), NAN, device="cuda").to(dtype)
    z = raw[front:].view(rows, cols + extra)[:, :cols]
    z.copy_((randn(rows, cols, seed=122) * 2).to(dtype))
    z[::3, cols - 1] = 30.0
    ids = torch.randint(0, cols, (rows,), generator=gen(123), device="cuda")
    for top in (0, 1, 6):
        check_scores(ops.token_scores(z, ids, top=top), z, ids, top, lanes=32)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,cols", [(6, 100), (7, 1000), (5, 9000), (3, 70001)])
@pytest.mark.parametrize("extra,front", [(0, 1), (3, 0), (8, 0), (1, 5)])
def test_scores_take_strides_and_alignments(ops, dtype, rows, cols, extra, front):
    raw = torch.full((front + rows * (cols + extra),), NAN, device="cuda").to(dtype)
    z = raw[front:].view(rows, cols + extra)[:, :cols]
    z.copy_((randn(rows, cols, seed=22) * 2).to(dtype))
    ids = torch.randint(0, cols, (rows,), generator=gen(23), device="cuda")
    check_scores(ops.token_scores(z, ids, top=6), z, ids, 6)
    same = z[:1].expand(rows, cols)
    check_scores(ops.token_scores(same, ids, top=2), same, ids, 2)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cols", [40, 1000, 20000, 140000])
def test_scores_of_masks_ties_and_what_is_no_distribution(ops, dtype, cols):
    z = randn(16, cols, seed=24)
    lowest = torch.finfo(dtype).min
    z[0, ::2] = -INF                                              # half of them
    z[1, :] = -INF                                                # nothing is left
    z[2, :] = -INF
    z[2, cols // 2] = 3.0                                         # one is
    z[3, :cols - 1] = lowest
    z[4, :] = lowest                                              # all alike
    z[5, :] = 0.0                                                 # all alike
    z[6, cols // 3] = NAN
    z[7, cols - 1] = INF
    z[8, 1] = INF
    z[8, 2] = -INF
    z[9, ::2], z[9, 1::2] = 0.0, -0.0                             # equal numbers with other bits
    z[10] *= 1000 if dtype == F32 else 20
    z[11, :] = torch.arange(cols, device="cuda") * 1e-3           # the maximum grows all along
    z[12, :] = -torch.arange(cols, device="cuda") * 1e-3
    z[13, 0] = torch.finfo(dtype).max                             # further apart than the type goes
    z[13, 1:] = lowest
    z[14, :] = -INF
    z[14, -3:] = torch.tensor([1.0, 2.0, 1.0], device="cuda")
    z[15, : cols // 2] = torch.finfo(dtype).max
    z = z.to(dtype)
    ids = torch.randint(0, cols, (16,), generator=gen(25), device="cuda")
    ids[0], ids[2], ids[3], ids[13] = 0, cols // 2, cols - 1, cols - 1
    for top in (1, 7, 32):
        check_scores(ops.token_scores(z, ids, top=top), z, ids, top)


def test_scores_of_tokens_that_are_none(ops):
    z = randn(5, 900, seed=26)
    ids = torch.tensor([-1, 900, 899, 2 ** 40, -2 ** 62], device="cuda")
    got = ops.token_scores(z, ids, top=2)
    check_scores(got, z, ids, 2)
    assert torch.isnan(got[0]).tolist() == [True, True, False, True, True]


def test_scores_of_few_distinct_logits(ops):
    # long runs of equal logits: the lowest ids, whichever threads hold them
    for cols in (700, 5000, 100000):
        z = torch.randint(0, 3, (9, cols), generator=gen(27), device="cuda").half()
        z[4] = 0
        z[4, cols - 1] = 1
        ids = torch.zeros(9, dtype=torch.long, device="cuda")
        check_scores(ops.token_scores(z, ids, top=32), z, ids, 32)


def test_scores_of_rows_beyond_32_bits(ops):
    rows, cols = 17000, 131072                                    # 2.2e9 logits
    z = torch.zeros(rows, cols, dtype=F16, device="cuda")
    z[rows - 1, 77], z[0, cols - 1] = 9.0, 8.0
    ids = torch.full((rows,), 5, device="cuda")
    got = ops.token_scores(z, ids, top=1)
    some = torch.tensor([0, 1, 16383, 16384, rows - 1], device="cuda")
    check_scores([t[some] for t in got], z[some], ids[some], 1)


def test_scores_refuse(ops):
    z, ids = randn(3, 100, seed=28), torch.zeros(3, dtype=torch.long, device="cuda")
    for bad in (z[0], z.double(), z.t()):
        with pytest.raises(ValueError):
            ops.token_scores(bad, ids)
    for bad in (ids[:2], ids.int(), ids.float()):
        with pytest.raises(ValueError, match="ids"):
            ops.token_scores(z, bad)
    for top in (-1, 101):
        with pytest.raises(_ffi.KernelError, match="best"):
            ops.token_scores(z, ids, top=top)
    with pytest.raises(_ffi.KernelError, match="at most 32"):
        ops.token_scores(z, ids, top=33)
    with pytest.raises(_ffi.KernelError, match="0 logits"):
        ops.token_scores(z[:, :0], ids)
    with pytest.raises(ValueError, match="gradient"):
        ops.token_scores(z.clone().requires_grad_(), ids)
    a = _ffi.TokenScores(z.data_ptr(), None, z.data_ptr(), None, None, None, 3, 100, 100, _ffi.F32, 0)
    assert ops.lib.msnh_b200_token_scores(ops.h, a, None) == 1 and "null" in ops.ctx.error()
    a.dtype = _ffi.E4M3
    assert ops.lib.msnh_b200_token_scores(ops.h, a, None) == 2
    assert ops.lib.msnh_b200_token_scores(None, a, None) == 1


def test_positions_and_scores_on_another_stream_and_in_a_graph(ops):
    x, positions, table = randn(5, 4, 64, seed=29), torch.arange(5, dtype=torch.int32, device="cuda"), ops.rotary_table(64)
    z, ids = randn(5, 60000, seed=30), torch.arange(5, device="cuda")
    want = ops.rotary(x, positions, table), *ops.token_scores(z, ids, top=4)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.rotary(x, positions, table), *ops.token_scores(z, ids, top=4)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.rotary(x, positions, table), *ops.token_scores(z, ids, top=4)
    x.copy_(randn(5, 4, 64, seed=31))
    z.copy_(randn(5, 60000, seed=32))
    positions += 9
    graph.replay()
    torch.cuda.synchronize()
    again = ops.rotary(x, positions, table), *ops.token_scores(z, ids, top=4)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
