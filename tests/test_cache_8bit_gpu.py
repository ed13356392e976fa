"""The paged cache in 8 bits (codes of e4m3 with a scale for each block of tokens and head): what is written against a model in plain Python, code by
code, what is read back, and attention over it against the formula in 64 bits. Tolerances are bounds of the arithmetic, derived beside their checks."""
import math
import random

import pytest

torch = pytest.importorskip("torch")
from msnhnet_b200 import _ffi  # noqa: E402

pytestmark = pytest.mark.gpu

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
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


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---- the model ------------------------------------------------------------------------------------------------------

def scale_for(top):
    """The smallest power of two, from 2^-126 on, that brings `top` to 448 at most; 0 for 0."""
    if top == 0:
        return 0.0
    e = -126
    while top > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def codes_of(x, scale):
    """x (64 bits, on the CPU) over a scale as codes; what is not finite is NaN."""
    y = x / scale if scale else x * 0.0
    # (a quotient by a power of two that fp32 holds exactly, or rounds to what the codes round to, too: below 2^-10 it is 0 either way)
    return torch.where(torch.isfinite(x), y, torch.full_like(y, NAN)).float().to(E4M3)


class Model:
    """A cache's codes and scales, token by token. (The pages that a sequence takes are the cache's own: other tests hold those to a model.)"""

    def __init__(self, cache):
        self.cache, self.page, self.block = cache, cache.page_size, cache.scale_block
        self.codes = [t.cpu().clone() for t in (cache.k_pages, cache.v_pages)]
        self.scales = [t.cpu().double() for t in (cache.k_scales, cache.v_scales)]
        self.lengths = cache.lengths.tolist()

    def append(self, seqs, counts, k, v):
        table, first = self.cache.page_table.tolist(), 0
        for s, n in zip(seqs, counts):
            for codes, scales, new in zip(self.codes, self.scales, (k, v)):
                rows = new[first:first + n].cpu().double()
                at = self.lengths[s]
                for begin in range(at // self.block * self.block, at + n, self.block):
                    lo, hi = max(at, begin), min(at + n, begin + self.block)
                    page, b = table[s][lo // self.page], lo % self.page // self.block
                    place = [t % self.page for t in range(begin, hi)]
                    for h in range(rows.shape[1]):
                        mine = rows[lo - at:hi - at, h]
                        fine = mine[torch.isfinite(mine)].abs()
                        was = float(scales[page, h, b]) if lo > begin else 0.0
                        now = max(was, scale_for(float(fine.max()) if fine.numel() else 0.0))
                        if lo > begin and now != was:
                            old = codes[page, place[:lo - begin], h]
                            codes[page, place[:lo - begin], h] = (old.double() * was / now).float().to(E4M3)
                        codes[page, place[lo - begin:], h] = codes_of(mine, now)
                        scales[page, h, b] = now
            first += n
            self.lengths[s] += n

    def copy_page(self, a, b, rows):
        for codes, scales in zip(self.codes, self.scales):
            codes[b, :rows] = codes[a, :rows]
            scales[b, :, :-(-rows // self.block)] = scales[a, :, :-(-rows // self.block)]

    def same(self):
        assert self.cache.lengths.tolist() == self.lengths
        for mine, theirs in zip(self.codes, (self.cache.k_pages, self.cache.v_pages)):
            mine, theirs = mine.float(), theirs.cpu().float()
            assert torch.equal(torch.isnan(mine), torch.isnan(theirs))
            assert torch.equal(mine.nan_to_num(0.0), theirs.nan_to_num(0.0))
        for mine, theirs in zip(self.scales, (self.cache.k_scales, self.cache.v_scales)):
            assert torch.equal(mine, theirs.cpu().double())


def used_cache(n_pages, page, heads, dim, n_seqs, max_pages, block, seed, heads_first=False, front=0):
    """A cache whose pages and scales hold what others left there."""
    from msnhnet_b200 import tokens
    shape = (n_pages, heads, page, dim) if heads_first else (n_pages, page, heads, dim)
    sides = []
    for i in range(2):
        raw = torch.zeros(math.prod(shape) + front, device="cuda")
        raw.copy_(randn(raw.numel(), seed=seed + i) * 50)
        pages = raw.to(E4M3)[front:].view(shape)
        sides.append(pages.transpose(1, 2) if heads_first else pages)
    ints_ = [torch.zeros(*s, dtype=torch.int32, device="cuda") for s in ((n_seqs, max_pages), (n_seqs,), (n_pages,))]
    scales = [torch.exp2(torch.randint(-20, 20, (n_pages, heads, page // block), generator=gen(seed + 2 + i), device="cuda").float()) for i in range(2)]
    return tokens.PagedCache(*sides, *ints_, *scales)


# ---- writing --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("page,block,heads,dim,heads_first,front", [(16, 16, 2, 64, False, 0), (16, 4, 3, 128, False, 0), (8, 1, 2, 80, True, 0), (12, 6, 1, 24, False, 0), (64, 64, 1, 256, False, 0),
                                                                    (5, 5, 2, 7, False, 0), (16, 16, 2, 64, False, 3), (32, 8, 1, 40, True, 8), (1, 1, 4, 16, False, 0), (32, 32, 2, 12, False, 4), (16, 8, 1, 264, False, 0), (20, 20, 1, 1032, False, 0)])
def test_append_follows_the_model(ops, dtype, page, block, heads, dim, heads_first, front):
    rng = random.Random(page * 100 + block)
    cache = used_cache(90, page, heads, dim, 6, -(-150 // page), block, 1, heads_first, front)
    m = Model(cache)
    for step in range(12):
        one = rng.random() < 0.5
        seqs = rng.sample(range(6), rng.randint(1, 6))
        counts = [1 if one else rng.choice([0, 1, 2, 5, 17, 40]) for _ in seqs]
        if not one and len(seqs) > 1:
            counts[rng.randrange(len(counts))] = 0
        if any(m.lengths[s] + n > 150 for s, n in zip(seqs, counts)) or sum(-(-n // page) for n in m.lengths) + sum(-(-n // page) + 1 for n in counts) > 90:
            ops.kv_free(cache, ints(*range(6)))
            m.lengths = [0] * 6
            continue
        tokens = sum(counts)
        # magnitudes that grow and shrink from token to token, some tokens of zeros
        size = torch.exp2(torch.randint(-9, 9, (tokens, heads, 1), generator=gen(step), device="cuda").float())
        size[torch.rand(tokens, heads, 1, generator=gen(step + 50), device="cuda") < 0.1] = 0
        both = (randn(tokens, 2 * heads, dim + (8 if step % 2 else 3), seed=step + 100) * size.repeat(1, 2, 1)).to(dtype)
        k, v = both[:, :heads, :dim], both[:, heads:, :dim]
        starts = None if one else ints(*[sum(counts[:i]) for i in range(len(counts) + 1)])
        ops.kv_append(cache, k, v, seqs=ints(*seqs), starts=starts)
        m.append(seqs, counts, k, v)
        m.same()
    assert cache.refused() == 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [64, 10])
def test_append_of_numbers_at_the_ends(ops, dtype, dim):
    info = torch.finfo(dtype)
    rows = torch.zeros(14, 1, dim, device="cuda", dtype=dtype)
    rows[1] = info.max
    rows[2], rows[2, 0, 0] = 1.0, info.max
    rows[3] = info.tiny
    rows[4, 0, 3] = info.smallest_normal / 2                      # (a subnormal number)
    rows[5, 0, 1] = NAN
    rows[6] = INF
    rows[7], rows[7, 0, 2], rows[7, 0, 3], rows[7, 0, 4] = 3.0, -INF, NAN, -0.0
    rows[8] = torch.tensor(448.0)
    rows[9] = torch.tensor(449.0) if dtype != BF16 else torch.tensor(450.0)
    rows[10] = -1.75
    rows[11] = torch.linspace(-448, 448, dim)
    rows[12], rows[13] = 2.0 ** -9, -2.0 ** -10
    for block in (1, 2, 14):
        cache = used_cache(4, 14, 1, dim, 2, 2, block, 5)
        m = Model(cache)
        ops.kv_append(cache, rows, rows.flip(0), seqs=ints(1), starts=ints(0, 14))
        m.append([1], [14], rows, rows.flip(0))
        m.same()
        cache = used_cache(4, 14, 1, dim, 2, 2, block, 6)
        m = Model(cache)
        for i in range(14):                                       # token by token: a block's scale grows under its older codes
            ops.kv_append(cache, rows[i:i + 1], rows.flip(0)[i:i + 1], seqs=ints(0))
            m.append([0], [1], rows[i:i + 1], rows.flip(0)[i:i + 1])
            m.same()


def test_a_growing_scale_rounds_older_codes_once(ops):
    # scales are powers of two: codes of normal numbers are the same after the block has grown as if all had been written at once
    cache = ops.new_cache(8, 16, 2, 64, 2, 2, dtype=E4M3)
    assert cache.scale_block == 16
    x = randn(16, 2, 64, seed=7) * torch.exp2(torch.arange(16, device="cuda") / 8.0)[:, None, None]
    for i in range(16):
        ops.kv_append(cache, x[i:i + 1], x[i:i + 1], seqs=ints(0))
    ops.kv_append(cache, x, x, seqs=ints(1), starts=ints(0, 16))
    a, b = (cache.k_pages[cache.page_table[i, 0]].float() for i in (0, 1))
    assert torch.equal(cache.k_scales[cache.page_table[0, 0]], cache.k_scales[cache.page_table[1, 0]])
    normal = b.abs() >= 2.0 ** -6
    assert torch.equal(a[normal], b[normal]) and bool(((a - b).abs() <= 2.0 ** -9).all())


def test_append_to_blocks_whose_scale_is_the_callers(ops):
    cache = used_cache(3, 16, 1, 64, 1, 2, 16, 8)
    old = randn(4, 1, 64, seed=9)
    ops.kv_append(cache, old, old, seqs=ints(0), starts=ints(0, 4))
    page = int(cache.page_table[0, 0])
    cache.k_scales[page], cache.v_scales[page] = 0.3, 0.001        # no powers of two; the second one has to grow
    codes = cache.v_pages[page, :4, 0].double()
    kept = cache.k_pages[page, :4].view(torch.uint8).clone()
    new = randn(1, 1, 64, seed=10) * 5
    ops.kv_append(cache, new, new, seqs=ints(0))
    assert torch.equal(cache.k_pages[page, :4].view(torch.uint8), kept) and float(cache.k_scales[page, 0, 0]) == pytest.approx(0.3)
    s = float(cache.k_scales[page, 0, 0])
    exact = new[0, 0].double() / s                                # (the quotient is rounded to fp32 before it becomes a code)
    off = (cache.k_pages[page, 4, 0].double() - exact).abs()
    assert bool((off <= torch.maximum(exact.abs() * 2.0 ** -4, torch.full_like(exact, 2.0 ** -10)) * (1 + 2.0 ** -18)).all())
    now = float(cache.v_scales[page, 0, 0])
    assert now == scale_for(float(new.abs().max()))
    exact = codes * torch.tensor(0.001).double().item() / now
    off = (cache.v_pages[page, :4, 0].double() - exact).abs()
    assert bool((off <= torch.maximum(exact.abs() * 2.0 ** -4, torch.full_like(exact, 2.0 ** -10)) * (1 + 2.0 ** -18)).all())


@pytest.mark.parametrize("block,dim,heads_first", [(16, 64, False), (4, 128, True), (2, 9, False)])
def test_fork_copy_and_compact_take_scales_along(ops, block, dim, heads_first):
    cache = used_cache(20, 16, 2, dim, 5, 4, block, 11, heads_first)
    m = Model(cache)
    k = randn(60, 2, dim, seed=12, dtype=F16)
    ops.kv_append(cache, k, k, seqs=ints(0, 1), starts=ints(0, 37, 60))
    m.append([0, 1], [37, 23], k, k)
    ops.kv_fork(cache, ints(0, 0, 1), ints(2, 3, 4))
    table = cache.page_table.tolist()
    m.lengths = [37, 23, 37, 37, 23]
    for a, b, full, rows in ((0, 2, 2, 5), (0, 3, 2, 5), (1, 4, 1, 7)):
        assert table[b][:full] == table[a][:full] and table[b][full] != table[a][full]
        m.copy_page(table[a][full], table[b][full], rows)
    m.same()
    # the forks go on by themselves
    new = randn(3, 2, dim, seed=13, dtype=F16) * 100
    ops.kv_append(cache, new, new, seqs=ints(2, 3, 4))
    m.append([2, 3, 4], [1, 1, 1], new, new)
    m.same()
    ops.kv_copy_pages(cache, ints(table[0][0]), ints(19))
    m.copy_page(table[0][0], 19, 16)
    m.same()
    before = {s: ops.kv_read(cache, ints(0, m.lengths[s]), m.lengths[s], seqs=ints(s), dtype=F32) for s in (1, 3, 4)}
    ops.kv_free(cache, ints(0, 2))
    ops.kv_compact(cache)
    live = int((cache.refs != 0).sum())
    assert bool((cache.refs[:live] != 0).all()) and live == 6
    for s, kept in before.items():
        now = ops.kv_read(cache, ints(0, m.lengths[s]), m.lengths[s], seqs=ints(s), dtype=F32)
        assert torch.equal(now[0], kept[0]) and torch.equal(now[1], kept[1])


def test_append_and_read_of_many_sequences(ops):
    # more sequences than a warp looks through at once, and than the deciding block has threads; many without a token
    rng = random.Random(16)
    n = 3000
    cache = used_cache(6000, 8, 1, 16, n, 4, 4, 17)
    m = Model(cache)
    order = rng.sample(range(n), n)
    for _ in range(2):
        counts = [rng.choice([0, 0, 1, 2, 5, 9]) for _ in range(n)]
        tokens = sum(counts)
        k, v = randn(tokens, 1, 16, seed=18, dtype=F16), randn(tokens, 1, 16, seed=19, dtype=F16) * 8
        starts = ints(0, *torch.tensor(counts).cumsum(0).tolist())
        ops.kv_append(cache, k, v, seqs=ints(*order), starts=starts)
        m.append(order, counts, k, v)
    m.same()
    assert cache.refused() == 0
    lengths = [m.lengths[s] for s in order]
    starts = ints(0, *torch.tensor(lengths).cumsum(0).tolist())
    k, v = ops.kv_read(cache, starts, sum(lengths), seqs=ints(*order), dtype=F32)
    at, table = 0, cache.page_table.tolist()
    for s, length in zip(order, lengths):
        for t in range(length):
            page, place = table[s][t // 8], t % 8
            for side, out in ((0, k), (1, v)):
                if s % 50 == 0:
                    assert torch.equal(out[at + t, 0].cpu().double(), m.codes[side][page, place, 0].double() * m.scales[side][page, 0, place // 4])
        at += length


def test_append_refuses_on_the_device(ops):
    cache = used_cache(3, 4, 1, 16, 2, 2, 2, 14)
    m = Model(cache)
    x = randn(9, 1, 16, seed=15, dtype=BF16)
    ops.kv_append(cache, x, x, seqs=ints(0), starts=ints(0, 9))              # more than a table row takes
    ops.kv_append(cache, x[:2], x[:2], seqs=ints(-1, 2))
    ops.kv_append(cache, x, x, seqs=ints(0, 1), starts=ints(0, 7, 3))
    m.same()
    assert cache.refused() == 5
    ops.kv_append(cache, x[:5], x[:5], seqs=ints(0, 7, 1), starts=ints(0, 2, 3, 5))
    m.append([0], [2], x, x)
    m.append([1], [2], x[3:], x[3:])
    m.same()
    assert cache.refused() == 6


# ---- reading back ---------------------------------------------------------------------------------------------------

def fill(ops, cache, lengths, seed, dtype=F16):
    starts = ints(*[sum(lengths[:i]) for i in range(len(lengths) + 1)])
    k, v = (randn(sum(lengths), cache.n_kv_heads, cache.head_dim, seed=seed + i).to(cache.dtype if cache.dtype != E4M3 else dtype) for i in range(2))
    ops.kv_append(cache, k, v, starts=starts)
    return starts, k, v


@pytest.mark.parametrize("cache_type", [E4M3, F32, F16, BF16])
@pytest.mark.parametrize("out_type", [F32, F16, BF16])
@pytest.mark.parametrize("page,block,heads,dim", [(16, 4, 3, 64), (6, 3, 2, 10), (32, 32, 1, 256)])
def test_read_gives_what_the_cache_holds(ops, cache_type, out_type, page, block, heads, dim):
    lengths = [40, 0, 1, 33, 100]
    cache = ops.new_cache(60, page, heads, dim, 5, -(-100 // page), dtype=cache_type, **({"scale_block": block} if cache_type == E4M3 else {}))
    starts, k, v = fill(ops, cache, lengths, 20)
    got = ops.kv_read(cache, starts, sum(lengths), dtype=out_type)
    for new, out, pages, scales in ((k, got[0], cache.k_pages, cache.k_scales), (v, got[1], cache.v_pages, cache.v_scales)):
        want = []
        for s, n in enumerate(lengths):
            for t in range(n):
                at = int(cache.page_table[s, t // page])
                row = pages[at, t % page].double()
                want.append(row if scales is None else row * scales[at, :, t % page // block].double()[:, None])
        want = torch.stack(want)
        assert out.dtype == out_type and torch.equal(out, want.to(out_type))       # (scales are powers of two: one rounding)
        if cache_type == E4M3:
            # a code is off by half its step: 2^-4 of it, or 2^-10 of the scale; a scale is less than 2 / 448 of its block's largest value
            assert bool(((want - new.double()).abs() <= new.double().abs() * 2.0 ** -4 + new.abs().max().double() * 2.0 ** -9 / 448).all())
        else:
            assert torch.equal(want, new.double())
    assert ops.kv_read(cache, starts, sum(lengths))[0].dtype == (F16 if cache_type == E4M3 else cache_type)


def test_read_of_parts_holes_and_rows_of_nothing(ops):
    cache = ops.new_cache(60, 16, 2, 64, 5, 8, dtype=E4M3)
    lengths = [40, 0, 17, 33, 100]
    starts, _, _ = fill(ops, cache, lengths, 30)
    whole = [ops.kv_read(cache, ints(0, n), n, seqs=ints(s), dtype=F32) for s, n in enumerate(lengths)]
    hole = int(cache.page_table[4, 2])
    cache.page_table[4, 2] = -3
    for side in range(2):
        whole[4][side][32:48] = 0
    out = torch.full((2, 70, 2, 72), NAN, device="cuda")
    k, v = out[0, :, :, :64], out[1, :, :, :64]
    # ten rows of sequence 4 from 25 on, all of 2 and three beyond it, none of 0, five of none, from -2 of 3
    got = ops.kv_read(cache, ints(4, 34, 54, 54, 59, 64), 70, seqs=ints(4, 2, 0, 9, 3), first=ints(25, 0, 5, 0, -2), out=(k, v))
    assert got[0] is not None and got[0].data_ptr() == k.data_ptr()
    for side, rows in ((0, k), (1, v)):
        want = torch.zeros(70, 2, 64, device="cuda")
        want[4:34] = whole[4][side][25:55]
        want[34:51] = whole[2][side]
        want[61:64] = whole[3][side][:3]
        assert torch.equal(rows, want)
    assert bool(torch.isnan(out[..., 64:]).all())
    assert bool((ops.kv_read(cache, ints(0), 3)[0] == 0).all())
    assert ops.kv_read(cache, ints(0, 0), 0)[1].shape == (0, 2, 64)
    cache.page_table[4, 2] = hole


def test_read_of_values_beyond_the_output_type(ops):
    cache = ops.new_cache(2, 16, 1, 16, 1, 1, dtype=E4M3)
    x = torch.full((2, 1, 16), 1e6, device="cuda")
    x[1] = 1e-9
    ops.kv_append(cache, x, -x, starts=ints(0, 2))
    k, v = ops.kv_read(cache, ints(0, 2), 2, dtype=F16)
    assert bool((k[0] == INF).all()) and bool((v[0] == -INF).all()) and bool((k[1] == 0).all())
    assert bool(((ops.kv_read(cache, ints(0, 2), 2, dtype=F32)[0][0] - 1e6).abs() <= 1e6 / 16).all())


def test_read_back_and_append_again_gives_the_same_codes(ops):
    # values that the cache gave are codes times powers of two already
    cache = ops.new_cache(40, 16, 2, 80, 4, 8, dtype=E4M3, scale_block=8)
    starts, _, _ = fill(ops, cache, [50, 31], 40, F32)
    k, v = ops.kv_read(cache, starts, 81, dtype=F32)
    ops.kv_append(cache, k, v, seqs=ints(2, 3), starts=starts)
    again = ops.kv_read(cache, starts, 81, seqs=ints(2, 3), dtype=F32)
    assert torch.equal(again[0], k) and torch.equal(again[1], v)


# ---- attention ------------------------------------------------------------------------------------------------------

def code_cache(lengths, page, heads, dim, block, seed, width=None, heads_first=False, scales="powers"):
    """A cache whose sequences have `lengths` tokens, pages anywhere; what holds no token is NaN, its scales too. Also keys and values in 64 bits."""
    from msnhnet_b200 import tokens
    need = [-(-n // page) for n in lengths]
    total = sum(need) + 3
    shape = (total, heads, page, dim) if heads_first else (total, page, heads, dim)
    place = torch.randperm(total, generator=gen(seed), device="cuda").tolist()
    table = torch.full((len(lengths), max(max(need + [1]), width or 1)), -7, dtype=torch.int32)
    taken = iter(place)
    for i in range(len(lengths)):
        for j in range(need[i]):
            table[i, j] = next(taken)
    sides, all_scales, rows = [], [], []
    for side in range(2):
        pages = torch.full(shape, 127, dtype=torch.uint8, device="cuda").view(E4M3)
        pages = pages.transpose(1, 2) if heads_first else pages
        scale = torch.full((total, heads, page // block), NAN, device="cuda")
        mine = []
        for i, n in enumerate(lengths):
            codes = (randn(max(need[i], 1) * page, heads, dim, seed=seed + 10 + 2 * i + side) * 60).to(E4M3)
            some = torch.randint(-9, -5, (max(need[i], 1), heads, page // block), generator=gen(seed + 500 + 2 * i + side), device="cuda").float()
            some = torch.exp2(some)
            if scales == "any":
                some = some * (1 + torch.rand(some.shape, generator=gen(seed + 900 + 2 * i + side), device="cuda"))
            if scales == "wild":
                some = torch.exp2(torch.randint(-60, 20, some.shape, generator=gen(seed + 700 + 2 * i + side), device="cuda").float()) if side else some
            for j in range(need[i]):
                at, here = int(table[i, j]), min(page, n - j * page)
                pages.view(torch.uint8)[at, :here] = codes.view(torch.uint8)[j * page:j * page + here]
                scale[at, :, :-(-here // block)] = some[j, :, :-(-here // block)]
            by = some.transpose(1, 2).repeat_interleave(block, 1).reshape(-1, heads)
            mine.append((codes.double() * by.double()[..., None])[:n])
        sides.append(pages)
        all_scales.append(scale)
        rows.append(mine)
    refs = torch.zeros(total, dtype=torch.int32, device="cuda")
    cache = tokens.PagedCache(*sides, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), refs, *all_scales)
    return cache, rows[0], rows[1]


def check_attn(out, lse, q, keys, values, scale, window=0, absent=None):
    dim, heads = q.shape[2], q.shape[1]
    for i in range(q.shape[0]):
        n = keys[i].shape[0]
        first = max(0, n - window) if window else 0
        seen = torch.ones(n, dtype=torch.bool, device="cuda")
        seen[:first] = False
        if absent is not None:
            seen &= ~absent[i]
        k, v = keys[i][seen], values[i][seen]
        each = heads // keys[i].shape[1]
        if k.shape[0] == 0:
            assert bool((out[i] == 0).all()) and bool((lse[i] == -math.inf).all())
            continue
        k, v = k.repeat_interleave(each, 1), v.repeat_interleave(each, 1)
        x = q[i].double()
        scores = torch.einsum("hd,thd->ht", x, k) * scale
        size = torch.einsum("hd,thd->ht", x.abs(), k.abs()) * abs(scale)
        # what queries lose: 2^-24 of a value (in size, below) and 2^-39 of the head's largest
        lost = 2.0 ** -39 * x.abs().amax(-1)[:, None] * k.abs().sum(-1).T * abs(scale)
        p = torch.softmax(scores, -1)
        want = torch.einsum("ht,thd->hd", p, v)
        most = torch.einsum("ht,thd->hd", p, v.abs())
        # a tensor-core step of 16 products: 2^-22 of the sum of magnitudes; a query's two parts 2^-24; the score's three factors 2^-22
        off = 2.0 ** -22 * (dim / 16 + 5) * size.amax(-1, keepdim=True) + lost.amax(-1, keepdim=True) + 2.0 ** -21 * scores.abs().amax(-1, keepdim=True)
        # a factor p_t vs_t is two fp16 parts: 2^-22 of it, and where it is small 2^-38 of the largest factor, times codes of up to 448 (which a scale,
        # the largest code of a token being above 28 here or all of them 0, makes 16 of its value's largest magnitude)
        small = 2.0 ** -38 * 16 * (p.T * v.abs().amax(-1)).amax(0)[:, None] * k.shape[0]
        bound = U[out.dtype] * want.abs() * 1.01 + (2 * off + 2.0 ** -22 * (k.shape[0] / 16 + 34)) * most + small + TINY[out.dtype]
        none = torch.isnan(want).all(-1)                             # (an infinite query: no softmax)
        assert torch.equal(torch.isnan(out[i]), none[:, None].expand(heads, dim))
        fine = ~none
        assert bool(((out[i].double() - want).abs() <= bound)[fine].all()), (i, float(((out[i].double() - want).abs() / bound)[fine].max()))
        whole = torch.logsumexp(scores, -1)
        assert bool(((lse[i].double() - whole).abs() <= off[:, 0] + 2.0 ** -22 * (k.shape[0] / 16 + 32) + 2.0 ** -22 * whole.abs())[fine].all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lengths,page,block,kv_heads,each,dim", [
    ([1], 16, 16, 1, 1, 64), ([0], 16, 4, 2, 2, 64), ([1, 2, 3, 0, 15, 16, 17], 16, 16, 2, 4, 128), ([31, 33, 64, 65], 8, 8, 8, 4, 128), ([5, 127, 128, 129], 1, 1, 3, 5, 32),
    ([300, 7], 64, 32, 1, 8, 256), ([513], 128, 128, 4, 1, 96), ([100, 1000], 7, 7, 2, 16, 80), ([2500, 3, 0, 700], 16, 2, 2, 7, 128), ([60], 32, 16, 1, 20, 64),
    ([90, 40], 16, 1, 1, 40, 128), ([20000, 1], 16, 16, 1, 4, 128), ([33, 2], 16, 8, 2, 3, 16), ([50], 16, 16, 12, 1, 48), ([1] * 70, 4, 2, 1, 2, 64), ([77, 1300], 16, 16, 2, 2, 192),
    ([300, 40], 24, 12, 1, 16, 256), ([400], 20, 4, 2, 12, 208)])
def test_attention_matches_the_formula(ops, dtype, lengths, page, block, kv_heads, each, dim):
    cache, keys, values = code_cache(lengths, page, kv_heads, dim, block, 40)
    q = randn(len(lengths), kv_heads * each, dim, seed=41, dtype=dtype)
    out, lse = ops.attn_decode(q, cache, return_lse=True)
    assert out.dtype == dtype
    check_attn(out, lse, q, keys, values, dim ** -0.5)
    assert torch.equal(out, ops.attn_decode(q, cache))                # and the same again


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scales", ["any", "wild"])
@pytest.mark.parametrize("page,block", [(16, 16), (16, 1), (32, 4)])
def test_attention_with_scales_of_all_sizes(ops, dtype, scales, page, block):
    lengths = [5, 64, 700]
    cache, keys, values = code_cache(lengths, page, 2, 64, block, 50, scales=scales)
    q = randn(3, 6, 64, seed=51, dtype=dtype)
    out, lse = ops.attn_decode(q.float(), cache, return_lse=True)     # (fp16 has no place for the largest of them)
    check_attn(out, lse, q.float(), keys, values, 0.125)
    if scales == "any" or dtype == BF16:
        out, lse = ops.attn_decode(q, cache, return_lse=True)
        check_attn(out, lse, q, keys, values, 0.125)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("window", [1, 5, 16, 100, 5000])
def test_attention_window(ops, dtype, window):
    lengths = [1, 4, 5, 6, 99, 100, 101, 900, 0]
    cache, keys, values = code_cache(lengths, 16, 2, 64, 4, 60)
    for i, n in enumerate(lengths):
        cache.page_table[i, :max(0, n - window) // 16] = -1
    q = randn(len(lengths), 6, 64, seed=61, dtype=dtype)
    out, lse = ops.attn_decode(q, cache, window=window, scale=0.3, return_lse=True)
    check_attn(out, lse, q, keys, values, 0.3, window)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_holes(ops, dtype):
    lengths = [64, 70, 200, 16, 500]
    cache, keys, values = code_cache(lengths, 16, 2, 64, 16, 62)
    absent = [torch.zeros(n, dtype=torch.bool, device="cuda") for n in lengths]
    for i, j, mark in [(0, 1, -1), (1, 4, 10 ** 6), (2, 0, -1), (2, 5, cache.n_pages), (3, 0, -1), (4, 30, -1)] + [(4, j, -2) for j in range(3, 20)]:
        cache.page_table[i, j] = mark
        absent[i][16 * j:16 * (j + 1)] = True
    q = randn(5, 4, 64, seed=63, dtype=dtype)
    out, lse = ops.attn_decode(q, cache, return_lse=True)
    check_attn(out, lse, q, keys, values, 0.125, absent=absent)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads_first", [False, True])
def test_attention_layouts_and_rows(ops, dtype, heads_first):
    lengths = [40, 0, 333, 18]
    cache, keys, values = code_cache(lengths, 8, 3, 64, 8, 64, heads_first=heads_first)
    seqs = ints(2, 2, 0, 1, 3, 0, -1, 4, 2)
    q = randn(6, 9, 64 + 5, seed=65, dtype=dtype).transpose(0, 1)[:, :, 5:]
    out = torch.full((9, 6, 80), NAN, device="cuda", dtype=dtype)[:, :, 8:72]
    got, lse = ops.attn_decode(q, cache, seqs=seqs, out=out, return_lse=True)
    none = torch.zeros(0, 3, 64, device="cuda", dtype=torch.float64)
    pick = [s if 0 <= s < 4 else None for s in seqs.tolist()]
    check_attn(got, lse, q, [none if s is None else keys[s] for s in pick], [none if s is None else values[s] for s in pick], 0.125)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("front,stride", [(0, 64), (1, 64), (2, 64), (3, 65), (4, 64), (0, 66), (4, 68), (6, 70), (4, 67)])
@pytest.mark.parametrize("dim", [48, 64])
def test_attention_of_queries_that_start_anywhere(ops, dtype, front, stride, dim):
    cache, _, _ = code_cache([70, 5, 130], 16, 2, dim, 16, 68)
    q = randn(3, 6, dim, seed=69, dtype=dtype)
    room = torch.full((8 + 3 * 6 * stride,), NAN, device="cuda", dtype=dtype)
    there = room[front:].as_strided((3, 6, dim), (6 * stride, stride, 1))
    there.copy_(q)
    expected, lse = ops.attn_decode(q, cache, return_lse=True)
    got, got_lse = ops.attn_decode(there, cache, return_lse=True)
    assert torch.equal(got, expected) and torch.equal(got_lse, lse)


@pytest.mark.parametrize("dtype,size", [(F32, 1e30), (F32, 1e-30), (F32, 1.0), (BF16, 1e30), (BF16, 1e-30), (F16, 2.0 ** -20), (F16, 3e4)])
def test_attention_of_queries_of_all_sizes(ops, dtype, size):
    cache, keys, values = code_cache([90, 300], 16, 1, 64, 16, 66)
    q = (randn(2, 5, 64, seed=67) * size).to(dtype)
    q[1, 2] = 0
    q[0, 1, 5:] *= 2.0 ** -9                                         # some values far below the head's largest
    scale = 0.125 / size
    out, lse = ops.attn_decode(q, cache, scale=scale, return_lse=True)
    check_attn(out, lse, q, keys, values, scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_of_large_scores_and_of_what_is_no_number(ops, dtype):
    cache, keys, values = code_cache([200, 150, 80, 500], 16, 1, 64, 16, 68)
    q = randn(4, 2, 64, seed=69, dtype=dtype) * 30
    page = int(cache.page_table[2, 2])
    cache.k_pages.view(torch.uint8)[page, 5, 0, 7] = 0x7f
    page = int(cache.page_table[3, 30])
    cache.v_pages.view(torch.uint8)[page, 5, 0, 9] = 0xff
    out, lse = ops.attn_decode(q, cache, scale=1.0, return_lse=True)
    check_attn(out[:2], lse[:2], q[:2], keys[:2], values[:2], 1.0)
    assert bool(torch.isnan(out[2]).all())
    bad = torch.zeros_like(out[3], dtype=torch.bool)
    bad[:, 9] = True
    assert torch.equal(torch.isnan(out[3]), bad)                     # (a value that is no number: its column)
    cache.v_scales[page] = INF
    assert bool(torch.isnan(ops.attn_decode(q[3:], cache, seqs=ints(3), scale=1e-3)[0]).any())
    bad = randn(1, 2, 64, seed=70, dtype=dtype)
    bad[0, 1, 3] = NAN
    out = ops.attn_decode(bad, cache, seqs=ints(0))
    assert torch.isnan(out[0]).all(-1).tolist() == [False, True] and bool(torch.isfinite(out[0, 0]).all())


@pytest.mark.parametrize("longest", [60, 700])
def test_attention_of_many_rows(ops, longest):
    lengths = [(i * 37) % longest for i in range(90)]
    cache, keys, values = code_cache(lengths, 16, 2, 32, 8, 71)
    pick = [(i * 53) % 95 - 2 for i in range(600)]
    q = randn(600, 4, 32, seed=72, dtype=F16)
    out, lse = ops.attn_decode(q, cache, seqs=ints(*pick), return_lse=True)
    none = torch.zeros(0, 2, 32, device="cuda", dtype=torch.float64)
    check_attn(out, lse, q, [keys[s] if 0 <= s < 90 else none for s in pick], [values[s] if 0 <= s < 90 else none for s in pick], 32 ** -0.5)


@pytest.mark.parametrize("lengths,width", [([37], 300), ([500, 20], 300), ([4000], 300), ([60] * 5, 40), ([2000] * 20, 300)])
def test_attention_in_a_table_with_room(ops, lengths, width):
    cache, keys, values = code_cache(lengths, 16, 2, 128, 16, 73, width=width)
    q = randn(len(lengths), 8, 128, seed=74, dtype=BF16)
    out, lse = ops.attn_decode(q, cache, return_lse=True)
    check_attn(out, lse, q, keys, values, 128 ** -0.5)


def test_8_bit_cache_beyond_32_bits(ops):
    # the last pages of a cache of more than 2^32 codes a side
    from msnhnet_b200 import tokens
    pages, page, heads, dim = 66000, 64, 8, 128
    k = torch.zeros(pages, page, heads, dim, dtype=torch.uint8, device="cuda").view(E4M3)
    v = torch.zeros_like(k)
    scales = [torch.ones(pages, heads, 4, device="cuda") for _ in range(2)]
    refs = torch.ones(pages, dtype=torch.int32, device="cuda")
    refs[-3:] = 0
    cache = tokens.PagedCache(k, v, torch.zeros(2, 4, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), refs, *scales)
    new = randn(130, heads, dim, seed=75, dtype=F16)
    ops.kv_append(cache, new, new * 2, seqs=ints(1), starts=ints(0, 130))
    assert cache.page_table[1].tolist() == [pages - 3, pages - 2, pages - 1, 0] and cache.refused() == 0
    got = ops.kv_read(cache, ints(0, 130), 130, seqs=ints(1), dtype=F32)
    assert bool(((got[0] - new.float()).abs() <= new.float().abs() * 2.0 ** -4 + new.abs().max().float() * 2.0 ** -9 / 448).all())
    assert torch.equal(got[1], 2 * got[0])
    q = randn(1, 16, dim, seed=76, dtype=F16)
    out, lse = ops.attn_decode(q, cache, seqs=ints(1), return_lse=True)
    check_attn(out, lse, q, [got[0].double()], [got[1].double()], dim ** -0.5)


# ---- together -------------------------------------------------------------------------------------------------------

def test_on_another_stream_and_in_a_graph(ops):
    cache = ops.new_cache(64, 16, 2, 64, 4, 16, dtype=E4M3)
    fill(ops, cache, [30, 70, 5, 0], 80)
    q, k, v = randn(4, 6, 64, seed=81, dtype=F16), randn(4, 2, 64, seed=82, dtype=F16), randn(4, 2, 64, seed=83, dtype=F16)
    kept = [t.clone() for t in cache.tensors]

    def step():
        ops.kv_append(cache, k, v)
        return ops.attn_decode(q, cache), *ops.kv_read(cache, ints_starts, 12, first=firsts)
    ints_starts, firsts = ints(0, 3, 6, 9, 12), ints(28, 68, 3, 0)
    want = step()
    after = [t.clone() for t in cache.tensors]

    def back():
        for t, old in zip(cache.tensors, kept):
            t.copy_(old)
    back()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = step()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a.float(), b.float()) for a, b in zip(cache.tensors, after))
    back()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a.float(), b.float()) for a, b in zip(cache.tensors, after))
    graph.replay()                                                    # one more token each
    assert cache.lengths.tolist() == [32, 72, 7, 2]


def test_two_streams_at_once(ops):
    caches = []
    for i in range(2):
        cache = ops.new_cache(300, 16, 2, 128, 8, 40, dtype=E4M3)
        fill(ops, cache, [500, 3, 0, 77, 400, 1, 20, 600], 90 + i)
        caches.append(cache)
    q, new = randn(8, 8, 128, seed=92, dtype=F16), randn(8, 2, 128, seed=93, dtype=F16)
    logits = randn(8, 50000, seed=94)

    def step(cache):
        ops.kv_append(cache, new, new)
        return ops.attn_decode(q, cache), *ops.token_scores(logits, top=3)[1:]
    kept = [[t.clone() for t in c.tensors] for c in caches]
    want = [[step(c) for _ in range(5)] for c in caches]
    for c, old in zip(caches, kept):
        for t, o in zip(c.tensors, old):
            t.copy_(o)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in caches], [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(step(caches[i]))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for one, other in zip(a, b) for x, y in zip(one, other))


def test_writes_are_known_to_torch(ops):
    cache = ops.new_cache(8, 16, 1, 32, 2, 2, dtype=E4M3)
    before = [t._version for t in cache.tensors]
    x = randn(2, 1, 32, seed=84)
    ops.kv_append(cache, x, x)
    assert len(before) == 8 and all(t._version > b for t, b in zip(cache.tensors, before))
    out = torch.empty(2, 2, 1, 32, device="cuda")
    was = out._version
    ops.kv_read(cache, ints(0, 1, 2), 2, out=(out[0], out[1]))
    assert out._version > was


def test_8_bit_cache_refuses(ops):
    from msnhnet_b200 import tokens
    cache = ops.new_cache(8, 16, 2, 64, 2, 4, dtype=E4M3, scale_block=4)
    parts = cache.k_pages, cache.v_pages, cache.page_table, cache.lengths, cache.refs
    for scales in ((), (cache.k_scales,), (cache.k_scales, cache.v_scales[:, :1]), (cache.k_scales.double(), cache.v_scales.double()), (cache.k_scales[:, :, :3], cache.v_scales[:, :, :3]),
                   (torch.ones(8, 2, 3, device="cuda"),) * 2, (torch.ones(8, 2, 0, device="cuda"),) * 2):
        with pytest.raises(ValueError, match="scales"):
            tokens.PagedCache(*parts, *scales)
    plain = ops.new_cache(8, 16, 2, 64, 2, 4)
    with pytest.raises(ValueError, match="8-bit"):
        tokens.PagedCache(plain.k_pages, plain.v_pages, *parts[2:], cache.k_scales, cache.v_scales)
    with pytest.raises(ValueError, match="scales"):
        ops.new_cache(8, 16, 2, 64, 2, 4, dtype=E4M3, scale_block=5)
    with pytest.raises(ValueError, match="8-bit"):
        ops.new_cache(8, 16, 2, 64, 2, 4, scale_block=4)
    with pytest.raises(ValueError):
        ops.new_cache(8, 16, 2, 64, 2, 4, dtype=torch.float8_e5m2)
    x = randn(2, 2, 64, seed=85)
    for bad in (x.to(E4M3), x.double(), x[:, :1], x[..., :32]):
        with pytest.raises(ValueError, match="k, v"):
            ops.kv_append(cache, bad, bad)
    with pytest.raises(ValueError, match="k, v"):
        ops.kv_append(cache, x, x.half())
    q = randn(2, 4, 64, seed=86)
    for bad in (q.to(E4M3), q.double(), q[..., :32]):
        with pytest.raises(ValueError, match="q:"):
            ops.attn_decode(bad, cache)
    with pytest.raises(ValueError, match="out"):
        ops.attn_decode(q, cache, out=torch.empty(2, 4, 64, device="cuda", dtype=F16))
    odd = ops.new_cache(8, 16, 1, 24, 2, 4, dtype=E4M3)
    with pytest.raises(_ffi.KernelError, match="16 bytes"):
        ops.attn_decode(randn(2, 1, 24, seed=87), odd)
    starts = ints(0, 1, 2)
    for more in ({"dtype": E4M3}, {"dtype": torch.float64}, {"out": (torch.empty(2, 2, 64, device="cuda"), torch.empty(2, 2, 64, device="cuda", dtype=F16))}, {"seqs": ints(0)},
                 {"first": ints(0)}, {"out": (torch.empty(3, 2, 64, device="cuda"),) * 2}):
        with pytest.raises(ValueError):
            ops.kv_read(cache, starts, 2, **more)
    for bad in (starts.long(), starts[:0], starts[None]):
        with pytest.raises(ValueError, match="starts"):
            ops.kv_read(cache, bad, 2)
    with pytest.raises(ValueError):
        ops.kv_read(cache, starts, -1)
    with pytest.raises(_ffi.KernelError, match="sequences"):
        ops.kv_read(cache, ints(0, 1, 2, 3), 3)
    with pytest.raises(_ffi.KernelError, match="overlap"):
        ops.kv_read(cache, starts, 2, out=(torch.empty(1, 2, 64, device="cuda").expand(2, 2, 64),) * 2)
    lib, h = ops.lib, ops.h
    args = (None, None, 2, x.data_ptr(), x.data_ptr())
    space = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    rest = (128, 64, 2, space.data_ptr(), space.numel(), None)
    assert lib.msnh_b200_kv_append_as(h, cache.ref, *args, _ffi.E4M3, *rest) == 1 and "type" in ops.ctx.error()
    assert lib.msnh_b200_kv_append_as(h, plain.ref, *args, _ffi.F32, *rest) == 1 and "type" in ops.ctx.error()
    assert lib.msnh_b200_kv_append(h, cache.ref, *args, *rest) == 1 and "type" in ops.ctx.error()
    cache.args.scale_block = 3
    assert lib.msnh_b200_kv_free(h, cache.ref, cache.lengths.data_ptr(), 1, None) == 1 and "scales" in ops.ctx.error()
    cache.args.scale_block, cache.args.k_scales = 4, None
    assert lib.msnh_b200_kv_free(h, cache.ref, cache.lengths.data_ptr(), 1, None) == 1 and "scales" in ops.ctx.error()
