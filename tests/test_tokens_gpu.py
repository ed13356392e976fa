"""The operators for decoding tokens against plain implementations in 64 bits, at the sizes, masks and layouts where they can go wrong.

Tolerances are bounds of the arithmetic, from the formulas: a result rounded once to its type (`U`, half a unit in the last place), sums
of fp32 terms (2^-24 a term that a thread adds, 2^-22 a tensor-core step of 16 terms), softmax weights that may be rounded to the cache's type."""
import math

import pytest

torch = pytest.importorskip("torch")
from msnhnet_b200 import _ffi  # noqa: E402

pytestmark = pytest.mark.gpu

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
U = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}         # (bf16: eight bits with the leading one)
TINY = {F32: 1e-45, F16: 2.0 ** -25, BF16: 1e-40}               # half of the smallest value


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


def padded(t, extra, front=0):
    """t's values in rows that are `extra` values longer, `front` values into an allocation."""
    wide = torch.full((t.shape[0] * (t.shape[1] + extra) + front,), float("nan"), device="cuda").to(t.dtype)
    view = wide[front:].view(t.shape[0], t.shape[1] + extra)[:, :t.shape[1]]
    view.copy_(t)
    return view


# ---- norm -----------------------------------------------------------------------------------------------------------

def norm_ref(x, residual, weight, eps):
    h = x.double() + (residual.double() if residual is not None else 0)
    return h, h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * weight.double()


def check_norm(got, want, cols, dtype):
    rel = U[dtype] + 2.0 ** -24 * (cols / 64 + 12)
    assert bool(((got.double() - want).abs() <= rel * want.abs() + TINY[dtype]).all())


def check_codes(codes, scale, want, cols):
    rel = 2.0 ** -24 * (cols / 64 + 16)
    top = want.abs().amax(-1)
    assert bool(((scale.double() - top / 448).abs() <= rel * top / 448).all())
    exact = torch.where(top[:, None] > 0, want / (top / 448)[:, None], torch.zeros_like(want))
    half_step = torch.maximum(exact.abs() * 2.0 ** -4, torch.full_like(exact, 2.0 ** -10))
    assert bool(((codes.double() - exact).abs() <= half_step * (1 + 2.0 ** -12)).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (1, 64), (5, 100), (2, 1000), (33, 2048), (3, 2049), (4, 5120), (2, 12288), (1, 16392), (2, 40000), (300, 256), (0, 64)])
def test_norm_matches_the_formula(ops, dtype, rows, cols):
    x, r = randn(rows, cols, seed=1, dtype=dtype), randn(rows, cols, seed=2, dtype=dtype) * 4
    w = (1 + 0.3 * randn(cols, seed=3)).to(dtype)
    y, h = ops.rms_norm(x, w, eps=1e-5, residual=r)
    want_h, want = norm_ref(x, r, w, 1e-5)
    check_norm(y, want, cols, dtype)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    check_norm(ops.rms_norm(x, w, eps=1e-5), norm_ref(x, None, w, 1e-5)[1], cols, dtype)
    codes, scale, h8 = ops.rms_norm(x, w.float(), eps=1e-5, residual=r, out_dtype=E4M3)
    assert codes.dtype == E4M3 and torch.equal(h8, h)
    check_codes(codes, scale, norm_ref(x, r, w.float(), 1e-5)[1], cols)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cols", [1, 64, 250, 256, 512, 520, 1024, 2048, 2056, 5120, 8200, 12288, 16384])
def test_norm_of_many_rows(ops, dtype, cols):
    # more rows than the blocks that the device holds at once take together
    rows = 1300 if cols > 1024 else 5000
    x, r, w = randn(rows, cols, seed=15, dtype=dtype), randn(rows, cols, seed=16, dtype=dtype), randn(cols, seed=17, dtype=dtype)
    y, h = ops.rms_norm(x, w, residual=r)
    _, want = norm_ref(x, r, w, 1e-6)
    check_norm(y, want, cols, dtype)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    codes, scale = ops.rms_norm(x, w, residual=None, out_dtype=E4M3)
    check_codes(codes, scale, norm_ref(x, None, w, 1e-6)[1], cols)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("extra,front", [(8, 0), (3, 0), (0, 1), (8, 8)])
def test_norm_takes_strides_and_alignments(ops, dtype, extra, front):
    rows, cols = 5, 1024
    x, r, w = randn(rows, cols, seed=4, dtype=dtype), randn(rows, cols, seed=5, dtype=dtype), randn(cols, seed=6, dtype=dtype)
    _, want_h = ops.rms_norm(x, w, residual=r)
    out, rout = padded(torch.zeros_like(x), extra, front), padded(torch.zeros_like(x), extra, front)
    wv = padded(w[None], 0, front)[0]
    y, h = ops.rms_norm(padded(x, extra, front), wv, residual=padded(r, extra, front), residual_out=rout, out=out)
    assert torch.equal(h, want_h)
    check_norm(y, norm_ref(x, r, w, 1e-6)[1], cols, dtype)
    wide = torch.zeros(rows, cols + extra, device="cuda").to(E4M3)
    got, scale, _ = ops.rms_norm(padded(x, extra, front), wv, residual=padded(r, extra, front), out_dtype=E4M3, out=wide[:, :cols])
    check_codes(got, scale, norm_ref(x, r, w, 1e-6)[1], cols)


@pytest.mark.parametrize("cols", [100, 512, 4096, 24576])
def test_norm_in_place(ops, cols):
    x, r, w = randn(7, cols, seed=7, dtype=F16), randn(7, cols, seed=8, dtype=F16), randn(cols, seed=9, dtype=F16)
    y, h = ops.rms_norm(x, w, residual=r)
    x2, r2 = x.clone(), r.clone()
    ops.rms_norm(x2, w, residual=r2, residual_out=r2, out=x2)        # the residual and x make place for h and y
    assert torch.equal(r2, h) and torch.equal(x2, y)


def test_norm_rows_shared_by_all(ops):
    x, r, w = randn(1, 640, seed=10, dtype=F16).expand(6, 640), randn(6, 640, seed=11, dtype=F16), randn(640, seed=12, dtype=F16)
    y, h = ops.rms_norm(x, w, residual=r)
    check_norm(y, norm_ref(x, r, w, 1e-6)[1], 640, F16)


@pytest.mark.parametrize("cols", [96, 1024, 4097, 40000])
def test_norm_of_zeros_and_of_what_is_no_number(ops, cols):
    x = randn(6, cols, seed=13)
    x[1] = 0
    x[2, cols // 2] = float("nan")
    x[3, cols - 1] = float("inf")
    x[4] *= 1e-30
    x[5] *= 1e15
    w = torch.ones(cols, device="cuda")
    y = ops.rms_norm(x, w, eps=0.0)
    codes, scale = ops.rms_norm(x, w, eps=1e-6, out_dtype=E4M3)
    good = [0, 4, 5]
    check_norm(y[[0, 5]], norm_ref(x, None, w, 0.0)[1][[0, 5]], cols, F32)
    check_codes(codes[[0, 5]], scale[[0, 5]], norm_ref(x, None, w, 1e-6)[1][[0, 5]], cols)
    assert bool((codes[1].float() == 0).all()) and float(scale[1]) == 0
    assert bool((codes[2].float() == 0).all()) and math.isnan(float(scale[2]))
    assert bool((codes[3].float() == 0).all()) and math.isnan(float(scale[3]))
    assert math.isfinite(float(scale[good].sum())) and float(codes[4].float().abs().amax()) == 448
    assert bool(torch.isnan(y[2]).all())


def test_norm_refuses(ops):
    x, w = randn(2, 64, seed=14, dtype=F16), torch.ones(64, device="cuda", dtype=F16)
    with pytest.raises(ValueError):
        ops.rms_norm(x, w[:32])
    with pytest.raises(ValueError):
        ops.rms_norm(x, w, residual=x.float())
    with pytest.raises(ValueError):
        ops.rms_norm(x.t(), w)
    with pytest.raises(ValueError):
        ops.rms_norm(x, w, out_dtype=BF16)
    with pytest.raises(_ffi.KernelError, match="eps"):
        ops.rms_norm(x, w, eps=-1.0)
    with pytest.raises(_ffi.KernelError, match="overlap"):
        ops.rms_norm(x, w, out=torch.empty(1, 64, device="cuda", dtype=F16).expand(2, 64))
    a = _ffi.RmsNorm(x.data_ptr(), None, w.data_ptr(), None, x.data_ptr(), None, 2, 64, 7, 7, 7, 64, 0, 0, 64, 1e-6)
    assert ops.lib.msnh_b200_rms_norm(ops.h, a, None) == 2
    a.dtype = a.weight_dtype = a.out_dtype = _ffi.F16
    a.y = None
    assert ops.lib.msnh_b200_rms_norm(ops.h, a, None) == 1 and "null" in ops.ctx.error()
    assert ops.lib.msnh_b200_rms_norm(None, a, None) == 1
    a.rows = -1
    assert ops.lib.msnh_b200_rms_norm(ops.h, a, None) == 1


# ---- 4-bit products -------------------------------------------------------------------------------------------------

def w4_data(n, k, group, zeros, scale_dtype=F16, seed=20):
    groups = -(-k // group)
    codes = torch.randint(0, 256, (n, (k + 1) // 2), generator=gen(seed), dtype=torch.uint8, device="cuda")
    scales = ((0.5 + torch.rand(n, groups, generator=gen(seed + 1), device="cuda")) / (4.6 * math.sqrt(k))).to(scale_dtype)
    z = torch.randint(0, 16, (n, groups), generator=gen(seed + 2), dtype=torch.uint8, device="cuda") if zeros else None
    values = torch.stack([codes & 15, codes >> 4], -1).reshape(n, -1)[:, :k].double()
    column = torch.arange(k, device="cuda") // group
    w = (values - (z.double()[:, column] if zeros else 8)) * scales.double()[:, column]
    return codes, scales, z, w


def check_w4(y, x, w, x_scale, bias, k):
    xs = x.double() * (x_scale.double()[:, None] if x_scale is not None else 1)
    want = xs @ w.T + (bias.double() if bias is not None else 0)
    size = xs.abs() @ w.abs().T + (bias.double().abs() if bias is not None else 0)
    bound = U[y.dtype] * want.abs() * 1.01 + 2.0 ** -22 * (k / 16 + 24) * size + TINY[y.dtype]
    assert bool(((y.double() - want).abs() <= bound).all()), float(((y.double() - want).abs() / bound).max())


def w4_x(rows, k, dtype, seed):
    x = randn(rows, k, seed=seed)
    if dtype == E4M3:
        scale = x.abs().amax(-1) / 448
        return (x / scale[:, None]).to(E4M3), scale
    return x.to(dtype), None


@pytest.mark.parametrize("dtype", [F32, F16, BF16, E4M3])
@pytest.mark.parametrize("rows,k,n,group,zeros,bias", [
    (1, 1, 1, 32, True, True), (1, 64, 16, 32, False, False), (1, 100, 17, 32, True, False), (2, 130, 33, 64, False, True), (1, 512, 1000, 128, True, True),
    (3, 999, 50, 96, True, False), (8, 256, 64, 256, False, False), (9, 320, 48, 32, True, True), (16, 1024, 40, 128, True, False), (17, 192, 31, 64, False, False),
    (33, 640, 72, 128, True, True), (64, 448, 200, 32, True, True), (1, 4096, 4096, 128, True, False), (4, 8192, 24, 128, False, False), (5, 2050, 130, 2080, True, False),
    (1, 16384, 8, 128, True, False), (40, 3000, 5, 128, False, True), (0, 64, 16, 32, False, False)])
def test_w4_matches_the_formula(ops, dtype, rows, k, n, group, zeros, bias):
    codes, scales, z, w = w4_data(n, k, group, zeros)
    b = randn(n, seed=23) * 0.1 if bias else None
    x, x_scale = w4_x(rows, k, dtype, 24)
    y = ops.w4_linear(x, ops.w4_pack(codes, scales, z, k=k, group=group), bias=b, x_scale=x_scale)
    assert y.dtype == (F16 if dtype == E4M3 else dtype) and y.shape == (rows, n)
    check_w4(y, x, w, x_scale, b, k)


@pytest.mark.parametrize("dtype", [F32, F16, BF16, E4M3])
@pytest.mark.parametrize("rows,k,n,group,zeros", [(1, 130, 18960, 32, True), (2, 256, 19001, 128, False), (1, 900, 40000, 64, True), (3, 200, 19001, 32, True),
                                                  (24, 140, 20000, 64, False), (64, 256, 18944, 128, True)])
def test_w4_of_many_outputs(ops, dtype, rows, k, n, group, zeros):
    codes, scales, z, w = w4_data(n, k, group, zeros)
    x, x_scale = w4_x(rows, k, dtype, 32)
    check_w4(ops.w4_linear(x, ops.w4_pack(codes, scales, z, k=k, group=group), x_scale=x_scale), x, w, x_scale, None, k)


@pytest.mark.parametrize("dtype", [F32, F16, E4M3])
@pytest.mark.parametrize("rows,k,n", [(1, 5000, 3200), (7, 7100, 3200), (13, 5000, 3200), (20, 5000, 3200), (30, 5000, 4700), (64, 1000, 3200), (48, 4096, 2048)])
def test_w4_of_a_few_turns(ops, dtype, rows, k, n):
    # tiles and units in numbers that the warps of a block share in two or more sets
    codes, scales, z, w = w4_data(n, k, 128, True)
    x, x_scale = w4_x(rows, k, dtype, 34)
    check_w4(ops.w4_linear(x, ops.w4_pack(codes, scales, z, k=k, group=128), x_scale=x_scale), x, w, x_scale, None, k)


@pytest.mark.parametrize("rows", [1, 2])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_w4_values_of_all_sizes_times_many_outputs(ops, rows, dtype):
    k, n = 256, 9500
    codes, scales, z, w = w4_data(n, k, 64, True)
    weights = ops.w4_pack(codes, scales, z, k=k, group=64)
    x = randn(rows, k, seed=35) * torch.exp2(torch.randint(-12, 12, (rows, k), generator=gen(36), device="cuda").float())
    check_w4(ops.w4_linear(x.to(dtype), weights, out_dtype=F32), x.to(dtype), w, None, None, k)
    for at in (0, 1, 63, 64, 130, 255):                               # each weight by itself
        x = torch.zeros(rows, k, device="cuda", dtype=dtype)
        x[rows - 1, at] = 1
        y = ops.w4_linear(x, weights, out_dtype=F32)
        assert torch.equal(y[rows - 1].double(), w[:, at].float().double()) and bool((y[:rows - 1] == 0).all())
    x = randn(rows, k, seed=37, dtype=dtype)
    x[0, 200] = float("nan")
    y = ops.w4_linear(x, weights, out_dtype=F32)
    assert bool(torch.isnan(y[0]).all())
    check_w4(y[1:], x[1:], w, None, None, k)


@pytest.mark.parametrize("rows,k,n,dtype", [(1, 20000, 9600, F32), (2, 33000, 9500, F16), (2, 5000, 12000, E4M3)])
def test_w4_of_long_rows_times_many_outputs(ops, rows, k, n, dtype):
    codes, scales, z, w = w4_data(n, k, 128, True)
    x, x_scale = w4_x(rows, k, dtype, 38)
    check_w4(ops.w4_linear(x, ops.w4_pack(codes, scales, z, k=k, group=128), x_scale=x_scale, out_dtype=F32), x, w, x_scale, None, k)


@pytest.mark.parametrize("rows,k", [(1, 20000), (2, 33000), (3, 20000), (16, 12000), (64, 9000)])
def test_w4_of_long_rows(ops, rows, k):
    # operands that no block has room for, and units that many blocks share
    codes, scales, z, w = w4_data(100, k, 128, True)
    weights = ops.w4_pack(codes, scales, z, k=k, group=128)
    for dtype in (F32, F16, E4M3):
        x, x_scale = w4_x(rows, k, dtype, 33)
        y = ops.w4_linear(x, weights, x_scale=x_scale, out_dtype=F32)
        check_w4(y, x, w, x_scale, None, k)
        assert torch.equal(y, ops.w4_linear(x, weights, x_scale=x_scale, out_dtype=F32))


@pytest.mark.parametrize("scale_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("out_dtype", [F32, F16, BF16])
def test_w4_scale_and_output_types(ops, scale_dtype, out_dtype):
    codes, scales, z, w = w4_data(80, 352, 32, True, scale_dtype)
    weights = ops.w4_pack(codes, scales, z, k=352, group=32)
    for dtype in (F32, F16, BF16, E4M3):
        x, x_scale = w4_x(6, 352, dtype, 25)
        check_w4(ops.w4_linear(x, weights, x_scale=x_scale, out_dtype=out_dtype), x, w, x_scale, None, 352)


@pytest.mark.parametrize("dtype", [F32, F16, BF16, E4M3])
@pytest.mark.parametrize("extra,front", [(8, 0), (1, 0), (0, 1), (16, 16)])
def test_w4_takes_strides_and_alignments(ops, dtype, extra, front):
    codes, scales, z, w = w4_data(70, 416, 32, True)
    wide = torch.zeros(70, 250, dtype=torch.uint8, device="cuda")
    wide[:, :208] = codes
    weights = ops.w4_pack(wide[:, :208], scales, z, k=416, group=32)
    x, x_scale = w4_x(7, 416, dtype, 26)
    raw = torch.zeros(7 * (416 + extra) + front, device="cuda").to(dtype)
    view = raw[front:].view(7, 416 + extra)[:, :416]
    view.copy_(x)
    if dtype != E4M3:
        raw[front:].view(7, 416 + extra)[:, 416:] = float("nan")      # what lies between rows is not read into a sum
    out = torch.zeros(7, 70 + extra, device="cuda", dtype=F32)[:, :70]
    check_w4(ops.w4_linear(view, weights, x_scale=x_scale, out=out), x, w, x_scale, None, 416)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_w4_values_of_all_sizes(ops, dtype):
    # products are exact, so large and small values of x lose nothing to one another beyond the sum's own rounding
    codes, scales, z, w = w4_data(32, 256, 64, True)
    x = randn(4, 256, seed=27) * torch.exp2(torch.randint(-12, 12, (4, 256), generator=gen(28), device="cuda").float())
    x = x.to(dtype)
    check_w4(ops.w4_linear(x, ops.w4_pack(codes, scales, z, k=256, group=64), out_dtype=F32), x, w, None, None, 256)


@pytest.mark.parametrize("rows", [1, 8, 20])
def test_w4_one_value_at_a_time(ops, rows):
    # each weight by itself: a code, zero point or scale in the wrong place shows
    k, n, group = 200, 40, 32
    codes, scales, z, w = w4_data(n, k, group, True)
    weights = ops.w4_pack(codes, scales, z, k=k, group=group)
    for first in range(0, k, rows):
        x = torch.zeros(rows, k, device="cuda")
        for i in range(min(rows, k - first)):
            x[i, first + i] = 1
        y = ops.w4_linear(x, weights)
        m = min(rows, k - first)
        assert torch.equal(y[:m].double(), w.T[first:first + m].float().double())


def test_w4_infinity_and_nan_stay_in_their_row(ops):
    codes, scales, z, w = w4_data(48, 160, 32, True)
    weights = ops.w4_pack(codes, scales, z, k=160, group=32)
    for dtype in (F16, BF16, F32):
        x = randn(5, 160, seed=29, dtype=dtype)
        x[1, 3] = float("nan")
        x[3, 159] = float("nan")
        y = ops.w4_linear(x, weights)
        assert bool(torch.isnan(y[[1, 3]]).all())
        check_w4(y[[0, 2, 4]], x[[0, 2, 4]], w, None, None, 160)


def test_w4_refuses(ops):
    codes, scales, z, w = w4_data(16, 64, 32, True)
    weights = ops.w4_pack(codes, scales, z, k=64, group=32)
    x = randn(1, 64, seed=30, dtype=F16)
    with pytest.raises(_ffi.KernelError, match="rows"):
        ops.w4_linear(randn(65, 64, seed=31, dtype=F16), weights)
    with pytest.raises(_ffi.KernelError, match="group"):
        ops.w4_pack(codes, scales[:, :1].contiguous(), None, k=64, group=80)
    with pytest.raises(ValueError):
        ops.w4_pack(codes, scales, z, k=60, group=32)
    with pytest.raises(ValueError):
        ops.w4_linear(x[:, :32], weights)
    with pytest.raises(ValueError):
        ops.w4_linear(x, weights, out_dtype=E4M3)
    with pytest.raises(ValueError):
        ops.w4_linear(x, weights, bias=torch.zeros(16, device="cuda", dtype=F16))
    with pytest.raises(_ffi.KernelError, match="overlap"):
        ops.w4_linear(x.expand(2, 64), weights, out=torch.empty(1, 16, device="cuda", dtype=F16).expand(2, 16))
    import ctypes
    size = ctypes.c_size_t()
    for n, k, want in ((0, 64, 1), (16, 2 ** 27 + 1, 2), (2 ** 30 + 1, 64, 2), (16, 2 ** 27, 0)):
        shape = _ffi.W4(None, n, k, 32, _ffi.F16, 0)
        assert ops.lib.msnh_b200_w4_pack_bytes(ops.h, shape, ctypes.byref(size)) == want
    a = _ffi.W4Linear(x.data_ptr(), None, None, None, 1, _ffi.F16, _ffi.F16, 64, 16, None, 0)
    assert ops.lib.msnh_b200_w4_linear(ops.h, weights.ref, a, None) == 1
    a.y, a.dtype = x.data_ptr(), 9
    assert ops.lib.msnh_b200_w4_linear(ops.h, weights.ref, a, None) == 2


# ---- the cache and its attention ------------------------------------------------------------------------------------

def make_cache(lengths, page, kv_heads, dim, dtype, seed, heads_first=False, spare=3, width=None):
    """A cache whose sequences have `lengths` tokens, pages anywhere; what holds no token is NaN. Also the tokens' keys and values."""
    from msnhnet_b200 import tokens
    need = [-(-n // page) for n in lengths]
    total = sum(need) + spare
    shape = (total, kv_heads, page, dim) if heads_first else (total, page, kv_heads, dim)
    pages = [torch.full(shape, float("nan"), device="cuda", dtype=dtype) for _ in range(2)]
    if heads_first:
        pages = [p.transpose(1, 2) for p in pages]
    place = torch.randperm(total, generator=gen(seed), device="cuda").tolist()
    table = torch.full((len(lengths), max(max(need + [1]), width or 1)), -7, dtype=torch.int32)
    refs = torch.zeros(total, dtype=torch.int32)
    keys, values, used = [], [], 0
    for i, n in enumerate(lengths):
        k, v = randn(n, kv_heads, dim, seed=seed + 100 + 2 * i, dtype=dtype), randn(n, kv_heads, dim, seed=seed + 101 + 2 * i, dtype=dtype)
        for j in range(need[i]):
            at = place[used]
            used += 1
            table[i, j] = at
            refs[at] = 1
            rows = slice(j * page, min(n, (j + 1) * page))
            pages[0][at, :rows.stop - rows.start], pages[1][at, :rows.stop - rows.start] = k[rows], v[rows]
        keys.append(k)
        values.append(v)
    cache = tokens.PagedCache(pages[0], pages[1], table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), refs.cuda())
    return cache, keys, values


P_ROUND = {F32: 2.0 ** -23, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def check_attn(out, lse, q, keys, values, scale, window=0, absent=None):
    dim, heads = q.shape[2], q.shape[1]
    for i in range(q.shape[0]):
        n = keys[i].shape[0]
        first = max(0, n - window) if window else 0
        seen = torch.ones(n, dtype=torch.bool, device="cuda")
        seen[:first] = False
        if absent is not None:
            seen &= ~absent[i]
        k, v = keys[i][seen].double(), values[i][seen].double()
        each = heads // keys[i].shape[1]
        if k.shape[0] == 0:
            assert bool((out[i] == 0).all()) and bool((lse[i] == -math.inf).all())
            continue
        k, v = k.repeat_interleave(each, 1), v.repeat_interleave(each, 1)
        scores = torch.einsum("hd,thd->ht", q[i].double(), k) * scale
        size = torch.einsum("hd,thd->ht", q[i].double().abs(), k.abs()) * abs(scale)
        p = torch.softmax(scores, -1)
        want = torch.einsum("ht,thd->hd", p, v)
        most = torch.einsum("ht,thd->hd", p, v.abs())
        off = 2.0 ** -22 * (dim / 16 + 4) * size.amax(-1, keepdim=True) + 2.0 ** -21 * scores.abs().amax(-1, keepdim=True)
        bound = U[out.dtype] * want.abs() * 1.01 + (2 * off + P_ROUND[out.dtype] + 2.0 ** -22 * (k.shape[0] / 16 + 32)) * most + TINY[out.dtype]
        assert bool(((out[i].double() - want).abs() <= bound).all()), (i, float(((out[i].double() - want).abs() / bound).max()))
        whole = torch.logsumexp(scores, -1)
        assert bool(((lse[i].double() - whole).abs() <= off[:, 0] + 2.0 ** -22 * (k.shape[0] / 16 + 32) + 2.0 ** -22 * whole.abs()).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lengths,page,kv_heads,each,dim", [
    ([1], 16, 1, 1, 64), ([0], 16, 2, 2, 64), ([1, 2, 3, 0, 15, 16, 17], 16, 2, 4, 128), ([31, 33, 64, 65], 8, 8, 4, 128), ([5, 127, 128, 129], 1, 3, 5, 32),
    ([300, 7], 64, 1, 8, 256), ([513], 128, 4, 1, 96), ([100, 1000], 7, 2, 16, 80), ([2500, 3, 0, 700], 16, 2, 7, 128), ([60], 32, 1, 20, 64), ([90, 40], 16, 1, 40, 128),
    ([20000, 1], 16, 1, 4, 128), ([33, 2], 16, 2, 3, 8), ([50], 16, 12, 1, 40), ([1] * 70, 4, 1, 2, 64), ([77, 1300], 16, 2, 2, 192)])
def test_attention_matches_the_formula(ops, dtype, lengths, page, kv_heads, each, dim):
    cache, keys, values = make_cache(lengths, page, kv_heads, dim, dtype, 40)
    q = randn(len(lengths), kv_heads * each, dim, seed=41, dtype=dtype)
    out, lse = ops.attn_decode(q, cache, return_lse=True)
    check_attn(out, lse, q, keys, values, dim ** -0.5)
    assert torch.equal(out, ops.attn_decode(q, cache))                # and the same again


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("window", [1, 5, 16, 100, 5000])
def test_attention_window(ops, dtype, window):
    lengths = [1, 4, 5, 6, 99, 100, 101, 900, 0]
    cache, keys, values = make_cache(lengths, 16, 2, 64, dtype, 42)
    # pages that lie wholly before the window need not be there
    for i, n in enumerate(lengths):
        cache.page_table[i, :max(0, n - window) // 16] = -1
    q = randn(len(lengths), 6, 64, seed=43, dtype=dtype)
    out, lse = ops.attn_decode(q, cache, window=window, scale=0.3, return_lse=True)
    check_attn(out, lse, q, keys, values, 0.3, window)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_holes(ops, dtype):
    lengths = [64, 70, 200, 16, 500]
    cache, keys, values = make_cache(lengths, 16, 2, 64, dtype, 44)
    absent = [torch.zeros(n, dtype=torch.bool, device="cuda") for n in lengths]
    for i, j, mark in [(0, 1, -1), (1, 4, 10 ** 6), (2, 0, -1), (2, 5, cache.n_pages), (3, 0, -1), (4, 30, -1)] + [(4, j, -2) for j in range(3, 20)]:
        cache.page_table[i, j] = mark
        absent[i][16 * j:16 * (j + 1)] = True
    q = randn(5, 4, 64, seed=45, dtype=dtype)
    out, lse = ops.attn_decode(q, cache, return_lse=True)
    check_attn(out, lse, q, keys, values, 0.125, absent=absent)       # (sequence 3 has nothing left)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads_first", [False, True])
def test_attention_layouts_and_rows(ops, dtype, heads_first):
    lengths = [40, 0, 333, 18]
    cache, keys, values = make_cache(lengths, 8, 3, 64, dtype, 46, heads_first=heads_first)
    seqs = torch.tensor([2, 2, 0, 1, 3, 0, -1, 4, 2], dtype=torch.int32, device="cuda")
    q = randn(6, 9, 64 + 5, seed=47, dtype=dtype).transpose(0, 1)[:, :, 5:]          # nine rows of six heads, the heads farther apart
    out = torch.full((9, 6, 80), float("nan"), device="cuda", dtype=dtype)[:, :, 8:72]
    got, lse = ops.attn_decode(q, cache, seqs=seqs, out=out, return_lse=True)
    none = torch.zeros(0, 3, 64, device="cuda", dtype=dtype)
    pick = [s if 0 <= s < 4 else None for s in seqs.tolist()]
    check_attn(got, lse, q, [none if s is None else keys[s] for s in pick], [none if s is None else values[s] for s in pick], 0.125)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_of_large_scores(ops, dtype):
    # one token far above the rest; scores far below zero; an infinite key, which no softmax survives, in its own sequence only
    cache, keys, values = make_cache([200, 150, 80], 16, 1, 64, dtype, 48)
    q = randn(3, 2, 64, seed=49, dtype=dtype)
    for i, (token, factor) in enumerate([(130, 30.0), (3, -30.0)]):
        page, place = int(cache.page_table[i, token // 16]), token % 16
        keys[i][token] = (q[i, :1].float() * factor).to(dtype)
        cache.k_pages[page, place] = keys[i][token]
    cache.k_pages[int(cache.page_table[2, 2]), 5, 0, 7] = float("nan")
    out, lse = ops.attn_decode(q, cache, scale=1.0, return_lse=True)
    check_attn(out[:2], lse[:2], q[:2], keys[:2], values[:2], 1.0)
    assert bool(torch.isnan(out[2]).all())


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("longest", [60, 700])
def test_attention_of_many_rows(ops, dtype, longest):
    # more rows than one launch takes, in any order, some twice and some of no sequence
    lengths = [(i * 37) % longest for i in range(90)]
    cache, keys, values = make_cache(lengths, 16, 2, 32, dtype, 82)
    pick = [(i * 53) % 95 - 2 for i in range(600)]
    q = randn(600, 4, 32, seed=83, dtype=dtype)
    out, lse = ops.attn_decode(q, cache, seqs=ints(*pick), return_lse=True)
    none = torch.zeros(0, 2, 32, device="cuda", dtype=dtype)
    seen = [keys[s] if 0 <= s < 90 else none for s in pick], [values[s] if 0 <= s < 90 else none for s in pick]
    check_attn(out, lse, q, *seen, 32 ** -0.5)
    for part in (slice(0, 256), slice(300, 301)):                     # as much of it as one launch takes, and one row alone
        some, some_lse = ops.attn_decode(q[part], cache, seqs=ints(*pick[part]), return_lse=True)
        check_attn(some, some_lse, q[part], seen[0][part], seen[1][part], 32 ** -0.5)


def test_attention_beyond_32_bits(ops):
    # the last pages of a cache of more than 2^32 bytes a side (and 2^31 values)
    from msnhnet_b200 import tokens
    pages, page, heads, dim = 34000, 64, 8, 128
    k = torch.empty(pages, page, heads, dim, device="cuda", dtype=F16)
    v = torch.empty_like(k)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    cache = tokens.PagedCache(k, v, table, torch.tensor([150], dtype=torch.int32, device="cuda"), torch.zeros(pages, dtype=torch.int32, device="cuda"))
    for p in table[0].tolist():
        k[p], v[p] = randn(page, heads, dim, seed=50 + p % 7, dtype=F16), randn(page, heads, dim, seed=60 + p % 7, dtype=F16)
    keys = [torch.cat([k[p] for p in table[0].tolist()])[:150]]
    values = [torch.cat([v[p] for p in table[0].tolist()])[:150]]
    q = randn(1, 16, dim, seed=51, dtype=F16)
    out, lse = ops.attn_decode(q, cache, return_lse=True)
    check_attn(out, lse, q, keys, values, dim ** -0.5)
    # the same places through the cache's upkeep
    src = torch.tensor([pages - 1], dtype=torch.int32, device="cuda")
    dst = torch.tensor([pages - 3], dtype=torch.int32, device="cuda")
    ops.kv_copy_pages(cache, src, dst)
    assert torch.equal(k[pages - 3], k[pages - 1]) and torch.equal(v[pages - 3], v[pages - 1])


def test_attention_refuses(ops):
    cache, _, _ = make_cache([20, 20], 16, 2, 64, F16, 52)
    q = randn(2, 4, 64, seed=53, dtype=F16)
    with pytest.raises(ValueError):
        ops.attn_decode(q.float(), cache)
    with pytest.raises(ValueError):
        ops.attn_decode(q[:, :, :32], cache)
    with pytest.raises(ValueError):
        ops.attn_decode(q, cache, seqs=torch.tensor([0, 1], device="cuda"))
    with pytest.raises(_ffi.KernelError, match="heads"):
        ops.attn_decode(q[:, :3], cache)
    with pytest.raises(_ffi.KernelError, match="rows"):
        ops.attn_decode(randn(3, 4, 64, seed=54, dtype=F16), cache)
    with pytest.raises(_ffi.KernelError, match="window"):
        ops.attn_decode(q, cache, window=-1)
    odd, _, _ = make_cache([20], 16, 2, 20, F16, 55)
    with pytest.raises(_ffi.KernelError, match="16 bytes"):
        ops.attn_decode(randn(1, 2, 20, seed=56, dtype=F16), odd)
    wide, _, _ = make_cache([20], 16, 1, 264, F16, 57)
    with pytest.raises(_ffi.KernelError, match="256"):
        ops.attn_decode(randn(1, 2, 264, seed=58, dtype=F16), wide)
    args = _ffi.AttnDecode(q.data_ptr(), q.data_ptr(), None, None, 2, 4, 256, 64, 256, 64, 0.125, 0, None, 0)
    cache.args.max_pages = cache.args.table_stride = 64               # (long enough to be cut, so a workspace is wanted)
    assert ops.lib.msnh_b200_attn_decode(ops.h, cache.ref, args, None) == 1 and "workspace" in ops.ctx.error()
    cache.args.max_pages = cache.args.table_stride = 2 ** 27 - 1
    cache.args.n_kv_heads = args.n_heads = 16
    assert ops.lib.msnh_b200_attn_decode(ops.h, cache.ref, args, None) == 2 and "2^34" in ops.ctx.error()
    cache.args.max_pages = cache.args.table_stride = cache.max_pages
    cache.args.n_kv_heads = 2
    from msnhnet_b200 import tokens
    with pytest.raises(ValueError):
        tokens.PagedCache(cache.k_pages, cache.v_pages[:1], cache.page_table, cache.lengths, cache.refs)
    with pytest.raises(ValueError):
        tokens.PagedCache(cache.k_pages, cache.v_pages, cache.page_table.long(), cache.lengths, cache.refs)
    cache.args.n_pages = 0
    assert ops.lib.msnh_b200_kv_free(ops.h, cache.ref, cache.lengths.data_ptr(), 1, None) == 1


class Model:
    """The cache's upkeep in plain Python, to compare a real cache with."""

    def __init__(self, cache):
        self.page, self.max_pages, self.n_seqs = cache.page_size, cache.max_pages, cache.n_seqs
        self.table, self.lengths, self.refs = cache.page_table.tolist(), cache.lengths.tolist(), cache.refs.tolist()
        self.k, self.v, self.refused = cache.k_pages.clone(), cache.v_pages.clone(), 0

    def free_pages(self):
        return [i for i, r in enumerate(self.refs) if r == 0]

    def pages(self, s):
        return -(-self.lengths[s] // self.page)

    def append(self, seqs, counts, k, v):
        free, wanted, first, plans = self.free_pages(), 0, 0, []
        for s, n in zip(seqs, counts):
            rows, first = (first, first + n), first + n
            if not 0 <= s < self.n_seqs:
                self.refused += 1
                continue
            need = -(-(self.lengths[s] + n) // self.page) - self.pages(s)
            if self.pages(s) + need > self.max_pages:
                self.refused += 1
                continue
            mine, wanted = (wanted, wanted + need), wanted + need
            if need and mine[1] > len(free):
                self.refused += 1
                continue
            plans.append((s, n, rows, mine))
        for s, n, rows, mine in plans:
            at = self.pages(s)
            for j, page in enumerate(free[mine[0]:mine[1]]):
                self.table[s][at + j] = page
                self.refs[page] = 1
            for i in range(n):
                t = self.lengths[s] + i
                self.k[self.table[s][t // self.page], t % self.page] = k[rows[0] + i]
                self.v[self.table[s][t // self.page], t % self.page] = v[rows[0] + i]
            self.lengths[s] += n

    def fork(self, src, dst):
        free, taken, plans = self.free_pages(), 0, []
        for a, b in zip(src, dst):
            if not (0 <= a < self.n_seqs and 0 <= b < self.n_seqs and a != b and self.lengths[b] == 0):
                self.refused += 1
                continue
            wants = self.lengths[a] % self.page > 0
            mine, taken = taken, taken + wants
            if wants and mine >= len(free):
                self.refused += 1
                continue
            plans.append((a, b, free[mine] if wants else None))
        for a, b, new in plans:
            full, rest = divmod(self.lengths[a], self.page)
            self.table[b][:full] = self.table[a][:full]
            for page in self.table[b][:full]:
                self.refs[page] += 1
            if rest:
                old = self.table[a][full]
                self.table[b][full] = new
                self.refs[new] = 1
                self.k[new, :rest], self.v[new, :rest] = self.k[old, :rest], self.v[old, :rest]
            self.lengths[b] = self.lengths[a]

    def free(self, seqs):
        for s in seqs:
            if not 0 <= s < self.n_seqs:
                self.refused += 1
                continue
            for page in self.table[s][:self.pages(s)]:
                self.refs[page] -= 1
            self.lengths[s] = 0

    def compact(self):
        live = sum(r != 0 for r in self.refs)
        to = dict(zip([i for i in range(live, len(self.refs)) if self.refs[i]], [i for i in range(live) if not self.refs[i]]))
        for a, b in to.items():
            self.k[b], self.v[b] = self.k[a], self.v[a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        for s in range(self.n_seqs):
            for j in range(self.pages(s)):
                self.table[s][j] = to.get(self.table[s][j], self.table[s][j])

    def same(self, cache):
        assert cache.lengths.tolist() == self.lengths
        assert cache.refs.tolist() == self.refs
        assert cache.page_table.tolist() == self.table
        assert cache.refused() == self.refused
        # (bit patterns: unwritten places are NaN)
        kind = torch.int32 if cache.dtype == F32 else torch.int16
        for mine, theirs in ((self.k, cache.k_pages), (self.v, cache.v_pages)):
            assert torch.equal(mine.contiguous().view(kind), theirs.contiguous().view(kind))


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,page,dim,heads_first", [(F16, 4, 64, False), (F32, 3, 12, False), (BF16, 1, 7, False), (F16, 16, 64, True), (F16, 5, 3, True)])
def test_upkeep_follows_the_model(ops, dtype, page, dim, heads_first):
    import random
    rng = random.Random(70)
    cache, _, _ = make_cache([3, 0, 9, 0, 0, 21, 0, 0], page, 2, dim, dtype, 71, heads_first, spare=40, width=-(-48 // page))
    m = Model(cache)
    for step in range(40):
        what = rng.choice(["append", "append", "one", "fork", "free", "compact"])
        if what in ("append", "one"):
            seqs = rng.sample(range(8), rng.randint(1, 8))
            counts = [1 if what == "one" else rng.choice([0, 1, 2, 7, 20]) for _ in seqs]
            tokens = sum(counts)
            k, v = randn(tokens, 2, dim, seed=72 + step, dtype=dtype), randn(tokens, 2, dim, seed=172 + step, dtype=dtype)
            starts = None if what == "one" else ints(*[sum(counts[:i]) for i in range(len(counts) + 1)])
            ops.kv_append(cache, k, v, seqs=ints(*seqs), starts=starts)
            m.append(seqs, counts, k, v)
        elif what == "fork":
            src = rng.sample(range(8), 3)
            dst = [s for s in range(8) if s not in src][:rng.randint(1, 4)]
            src = [src[0], src[1], src[0], src[2]][:len(dst)]
            ops.kv_fork(cache, ints(*src), ints(*dst))
            m.fork(src, dst)
        elif what == "free":
            seqs = rng.sample(range(8), rng.randint(1, 3))
            ops.kv_free(cache, ints(*seqs))
            m.free(seqs)
        else:
            ops.kv_compact(cache)
            m.compact()
        m.same(cache)


def test_upkeep_refuses_on_the_device(ops):
    cache, _, _ = make_cache([16, 4, 0, 0], 4, 1, 16, F16, 73, spare=2, width=6)
    m = Model(cache)
    k = randn(30, 1, 16, seed=74, dtype=F16)
    # no such sequence; a table row too short; more pages than are free, of which the first two requests get theirs
    for seqs, counts in (([7, -1, 1], [1, 1, 1]), ([0], [9]), ([2, 3, 1], [4, 4, 5])):
        n = sum(counts)
        ops.kv_append(cache, k[:n], k[:n], seqs=ints(*seqs), starts=ints(*[sum(counts[:i]) for i in range(len(counts) + 1)]))
        m.append(seqs, counts, k, k)
        m.same(cache)
    for src, dst in (([0, 1], [1, 1]), ([9], [2]), ([1], [-1])):
        ops.kv_fork(cache, ints(*src), ints(*dst))
        m.fork(src, dst)
        m.same(cache)
    ops.kv_free(cache, ints(5, -3))
    m.free([5, -3])
    m.same(cache)
    # starts that leave the tokens
    ops.kv_append(cache, k[:2], k[:2], seqs=ints(2, 3), starts=ints(0, 1, 3))
    m.append([2], [1], k, k)
    m.refused += 1
    m.same(cache)


def test_upkeep_of_many_sequences_and_pages(ops):
    # more sequences and pages than the deciding block has threads
    n, page = 2600, 2
    lengths = [i % 5 for i in range(n)] + [0] * n
    cache, _, _ = make_cache(lengths, page, 1, 8, F16, 75, spare=3 * n, width=4)
    m = Model(cache)
    src, dst = list(range(n)), list(range(n, 2 * n))
    ops.kv_fork(cache, ints(*src), ints(*dst))
    m.fork(src, dst)
    m.same(cache)
    k = randn(n, 1, 8, seed=76, dtype=F16)
    ops.kv_append(cache, k, k, seqs=ints(*dst))
    m.append(dst, [1] * n, k, k)
    ops.kv_free(cache, ints(*src))
    m.free(src)
    m.same(cache)
    ops.kv_compact(cache)
    m.compact()
    m.same(cache)


def test_compact_beside_the_old_tables(ops):
    cache, _, _ = make_cache([30, 5, 17, 0, 44], 4, 2, 32, F16, 77, spare=30)
    ops.kv_free(cache, ints(0, 2))
    m = Model(cache)
    table, refs = torch.full_like(cache.page_table, 99), torch.full_like(cache.refs, 99)
    before = cache.page_table.clone(), cache.refs.clone()
    ops.kv_compact(cache, table_out=table, refs_out=refs)
    assert torch.equal(cache.page_table, before[0]) and torch.equal(cache.refs, before[1])
    m.compact()
    assert table.tolist() == m.table and refs.tolist() == m.refs


def test_fork_shares_what_attention_reads(ops):
    cache, keys, values = make_cache([37, 0, 0], 16, 2, 64, F16, 78, spare=6, width=4)
    ops.kv_fork(cache, ints(0, 0), ints(1, 2))
    k, v = randn(2, 2, 64, seed=79, dtype=F16), randn(2, 2, 64, seed=80, dtype=F16)
    ops.kv_append(cache, k, v, seqs=ints(1, 2))
    q = randn(3, 4, 64, seed=81, dtype=F16)
    out, lse = ops.attn_decode(q, cache, return_lse=True)
    grown = [torch.cat([keys[0], k[i:i + 1]]) for i in range(2)], [torch.cat([values[0], v[i:i + 1]]) for i in range(2)]
    check_attn(out, lse, q, [keys[0]] + grown[0], [values[0]] + grown[1], 0.125)
    assert cache.refs[cache.page_table[0, :2].long()].tolist() == [3, 3]


# ---- streams and graphs ---------------------------------------------------------------------------------------------

def step(ops, cache, x, r, norm, w, q_rows):
    y, h = ops.rms_norm(x, norm, residual=r)
    qkv = ops.w4_linear(y, w)
    rows, dim, hk = x.shape[0], cache.head_dim, cache.n_kv_heads
    q, k, v = qkv[:, :q_rows * dim].view(rows, q_rows, dim), qkv[:, q_rows * dim:(q_rows + hk) * dim].view(rows, hk, dim), qkv[:, (q_rows + hk) * dim:].view(rows, hk, dim)
    ops.kv_append(cache, k, v)
    return ops.attn_decode(q, cache), h


def test_on_another_stream_and_in_a_graph(ops):
    dim, hk, heads, rows, cols = 64, 2, 4, 3, 256
    x, r, norm = randn(rows, cols, seed=90, dtype=F16), randn(rows, cols, seed=91, dtype=F16), randn(cols, seed=92, dtype=F16)
    codes, scales, z, _ = w4_data((heads + 2 * hk) * dim, cols, 64, True)
    w = ops.w4_pack(codes, scales, z, k=cols, group=64)
    lengths = [40, 200, 15]
    plain, _, _ = make_cache(lengths, 16, hk, dim, F16, 93, spare=9, width=16)
    want, want_h = step(ops, plain, x, r, norm, w, heads)
    again, _ = step(ops, plain, x, r, norm, w, heads)
    other = torch.cuda.Stream()
    moved, _, _ = make_cache(lengths, 16, hk, dim, F16, 93, spare=9, width=16)
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got, got_h = step(ops, moved, x, r, norm, w, heads)
    other.synchronize()
    assert torch.equal(got, want) and torch.equal(got_h, want_h)
    kept, _, _ = make_cache(lengths, 16, hk, dim, F16, 93, spare=9, width=16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = step(ops, kept, x, r, norm, w, heads)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    graph.replay()                                                    # the second replay appends a second token
    torch.cuda.synchronize()
    assert torch.equal(out, again) and kept.lengths.tolist() == [n + 2 for n in lengths]


def test_upkeep_refuses_a_cache_of_another_device(ops):
    # (a tensor of the CPU stands for one of another GPU)
    cache, _, _ = make_cache([5, 0, 3], 4, 1, 8, F16, 94)
    before = cache.lengths.tolist(), cache.refs.tolist()
    cache.k_pages = cache.k_pages.cpu()
    for call in (lambda: ops.kv_fork(cache, ints(0), ints(1)), lambda: ops.kv_free(cache, ints(0)), lambda: ops.kv_copy_pages(cache, ints(0), ints(1)),
                 lambda: ops.kv_append(cache, cache.k_pages[0, :3], cache.k_pages[0, :3])):
        with pytest.raises(ValueError, match="cpu"):
            call()
    assert (cache.lengths.tolist(), cache.refs.tolist()) == before


def test_inputs_that_require_a_gradient(ops):
    x, r, w = randn(3, 64, seed=95), randn(3, 64, seed=96), randn(64, seed=97)
    codes, scales, z, _ = w4_data(32, 64, 32, True)
    weights = ops.w4_pack(codes, scales, z, k=64, group=32)
    cache, _, _ = make_cache([5, 9, 2], 4, 2, 16, F32, 98)
    q = randn(3, 4, 16, seed=99)
    calls = [(lambda a: ops.rms_norm(a, w), x), (lambda a: ops.rms_norm(x, a), w), (lambda a: ops.rms_norm(x, w, residual=a)[0], r), (lambda a: ops.w4_linear(a, weights), x),
             (lambda a: ops.w4_linear(x, weights, bias=a), randn(32, seed=100)), (lambda a: ops.attn_decode(a, cache), q),
             (lambda a: ops.w4_pack(codes, a, z, k=64, group=32).packed, scales)]
    for call, t in calls:
        want, t = call(t), t.detach().clone().requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            call(t)
        with torch.no_grad():
            assert torch.equal(call(t), want)


def test_writes_are_known_to_torch(ops):
    # what is written in place no longer counts as what was saved for a backward pass
    x, r, w, out = randn(3, 64, seed=101), randn(3, 64, seed=102), randn(64, seed=103), randn(3, 64, seed=104)
    codes, scales, z, _ = w4_data(64, 64, 32, True)
    weights = ops.w4_pack(codes, scales, z, k=64, group=32)
    cache, _, _ = make_cache([5, 9, 2, 0], 4, 2, 16, F32, 105)
    q, kv, o = randn(4, 4, 16, seed=106), randn(1, 2, 16, seed=107), randn(4, 4, 16, seed=108)
    table, refs = torch.zeros_like(cache.page_table), torch.zeros_like(cache.refs)
    calls = [(lambda: ops.rms_norm(x, w, residual=r, residual_out=r, out=out), [out, r], [x, w]), (lambda: ops.w4_linear(x, weights, out=out), [out], [x]),
             (lambda: ops.attn_decode(q, cache, out=o), [o], [q, cache.k_pages, cache.lengths]),
             (lambda: ops.kv_append(cache, kv, kv, seqs=ints(2)), [cache.k_pages, cache.v_pages, cache.lengths, cache.refs, cache.page_table], [kv]),
             (lambda: ops.kv_fork(cache, ints(0), ints(3)), [cache.k_pages, cache.v_pages, cache.lengths, cache.refs, cache.page_table], []),
             (lambda: ops.kv_free(cache, ints(0)), [cache.lengths, cache.refs], []), (lambda: ops.kv_copy_pages(cache, ints(0), ints(1)), [cache.k_pages, cache.v_pages], []),
             (lambda: ops.kv_compact(cache, table_out=table, refs_out=refs), [cache.k_pages, cache.v_pages, table, refs], [])]
    for call, written, read in calls:
        before = [t._version for t in written], [t._version for t in read]
        call()
        assert all(t._version > v for t, v in zip(written, before[0])) and [t._version for t in read] == before[1]
    with torch.no_grad():
        a = torch.ones(3, 64, device="cuda", requires_grad=True)
    y = a * out
    ops.rms_norm(x, w, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():                                      # tensors without such a count
        ops.rms_norm(x, w, out=torch.empty_like(x))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols", [(3, 96), (700, 256), (3, 1024), (700, 5120), (700, 12288), (3, 4097), (3, 40000)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_norm_to_8_bits_with_a_weight_that_is_no_number(ops, dtype, rows, cols, bad):
    # every row's y is not finite then; a value of 0 times an infinite weight is NaN, too
    x, w = randn(rows, cols, seed=109, dtype=dtype), randn(cols, seed=110, dtype=dtype)
    x[1, cols // 2] = 0
    w[cols // 2] = bad
    codes, scale = ops.rms_norm(x, w, out_dtype=E4M3)
    assert bool(torch.isnan(scale).all()) and bool((codes.float() == 0).all())


@pytest.mark.parametrize("rows,cols", [(3, 96), (700, 256), (700, 5120), (700, 12288), (3, 4097), (3, 40000)])
def test_norm_to_8_bits_of_zeros_without_an_eps(ops, rows, cols):
    x, w = randn(rows, cols, seed=111, dtype=BF16), randn(cols, seed=112, dtype=BF16)
    x[1] = 0
    codes, scale = ops.rms_norm(x, w, eps=0.0, out_dtype=E4M3)
    assert float(scale[1]) == 0 and bool((codes[1].float() == 0).all())
    others = [i for i in range(rows) if i != 1]
    check_codes(codes[others], scale[others], norm_ref(x[others], None, w, 0.0)[1], cols)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(5, 96), (700, 64), (700, 512), (5, 1024), (700, 5120), (700, 12288), (5, 16384), (5, 4097), (5, 40000)])
def test_norm_to_8_bits_of_rows_whose_squares_overflow(ops, dtype, rows, cols):
    # no zeros in the place of values that are none: the scale says so
    x, w = randn(rows, cols, seed=113), randn(cols, seed=115, dtype=dtype)
    x[0] *= 1e30
    x[2, cols // 2] = 1e25
    x = x.to(dtype)
    codes, scale = ops.rms_norm(x, w, out_dtype=E4M3)
    assert torch.isnan(scale).tolist() == [i in (0, 2) for i in range(rows)] and bool((codes[[0, 2]].float() == 0).all())
    others = [i for i in range(rows) if i not in (0, 2)]
    check_codes(codes[others], scale[others], norm_ref(x[others], None, w, 1e-6)[1], cols)


def test_norm_of_the_longest_row(ops):
    # (a thread's next place behind the row's end passes 2^31)
    cols = 2 ** 31 - 1
    x, y = torch.ones(1, cols, device="cuda", dtype=F16), torch.zeros(1, cols, device="cuda", dtype=F16)
    ops.rms_norm(x, x[0], eps=0.0, out=y)
    assert bool((y == 1).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k,n", [(1, 200, 48), (2, 200, 9500), (1, 200, 19001), (5, 200, 48), (2, 5000, 9500), (2, 200, 12001), (1, 2100, 9500), (2, 4200, 12001), (2, 5000, 19001), (13, 200, 9500), (40, 200, 48)])
@pytest.mark.parametrize("scale_dtype,group", [(F16, 64), (BF16, 32)])
def test_w4_infinities_are_infinities(ops, dtype, rows, k, n, scale_dtype, group):
    # in every kernel as in the formula: the infinity's sign times the weight's, NaN for a weight of 0 or infinities of both signs
    codes, scales, z, w = w4_data(n, k, group, True, scale_dtype)
    weights = ops.w4_pack(codes, scales, z, k=k, group=group)
    x = randn(rows, k, seed=117, dtype=dtype)
    last = rows - 1
    x[last, 3], x[last, k - 7] = float("inf"), float("-inf")
    y = ops.w4_linear(x, weights, out_dtype=F32)
    a, b = w[:, 3].sign(), -w[:, k - 7].sign()
    none = (a == 0) | (b == 0) | (a != b)
    assert torch.equal(torch.isnan(y[last]), none) and bool(none.any()) and bool((~none).any())
    assert torch.equal(y[last][~none].double(), a[~none] * math.inf)
    check_w4(y[:last], x[:last], w, None, None, k)
    x[last, k - 7] = 1
    x[last, 5] = float("inf")
    x[last, 6] = float("inf")
    y = ops.w4_linear(x, weights, out_dtype=F32)
    signs = w[:, [3, 5, 6]].sign()
    whole = (signs[:, 0] != 0) & (signs == signs[:, :1]).all(1)
    assert torch.equal(torch.isnan(y[last]), ~whole) and torch.equal(y[last][whole].double(), signs[whole, 0] * math.inf)
    x[last, 9] = float("nan")
    assert bool(torch.isnan(ops.w4_linear(x, weights, out_dtype=F32)[last]).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,k,n", [(1, 256, 48), (1, 256, 9500), (2, 256, 48), (2, 256, 9500), (5, 256, 48), (5, 256, 9500), (1, 2048, 9500), (2, 4096, 12001)])
@pytest.mark.parametrize("power", [-115, -100, -92, -60, 60, 100])
def test_w4_of_small_and_large_activations(ops, dtype, rows, k, n, power):
    # the same relative error, whatever the activations' exponent and the number of outputs
    codes, scales, z, w = w4_data(n, k, 64, True)
    weights = ops.w4_pack(codes, scales, z, k=k, group=64)
    x = (randn(rows, k, seed=116) * 2.0 ** power).to(dtype)
    check_w4(ops.w4_linear(x, weights, out_dtype=F32), x, w, None, None, k)
    x[:, :64] = 0                                                     # beside spans of zeros, and in one span of ordinary ones
    x[:, 64:128] = randn(rows, 64, seed=118, dtype=dtype)
    check_w4(ops.w4_linear(x, weights, out_dtype=F32), x, w, None, None, k)
    assert bool((ops.w4_linear(torch.zeros_like(x), weights, out_dtype=F32) == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,k,n", [(1, 256, 48), (1, 256, 9500), (2, 256, 9500), (1, 2048, 9500), (2, 4096, 12001), (5, 256, 48), (9, 256, 48), (13, 256, 9500), (20, 256, 100), (40, 256, 48), (64, 1000, 48)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_of_activations_near_the_largest(ops, dtype, rows, k, n, group):
    # products with codes pass the largest number, results do not
    codes, scales, z, w = w4_data(n, k, group, True)
    x = randn(rows, k, seed=119)
    x[:, 3:83:10] = (1 + torch.rand(rows, 8, generator=gen(120), device="cuda")) * 2.0 ** 124 * torch.tensor([1, -1, 1, 1, -1, 1, -1, -1], device="cuda")
    x = x.to(dtype)
    assert float((x.double().abs() @ w.abs().T).max()) < 3e38 and float(x.double().abs().max()) * 15 > 3.5e38
    check_w4(ops.w4_linear(x, ops.w4_pack(codes, scales, z, k=k, group=group), out_dtype=F32), x, w, None, None, k)


@pytest.mark.parametrize("rows,n", [(1, 48), (3, 9500), (6, 48), (20, 48)])
@pytest.mark.parametrize("value", [3.4028234663852886e38, -3.4e38, 3.39e38, 3.389e38, -3.31e38])
def test_w4_of_the_largest_activations(ops, rows, n, value):
    # fp32 values above the largest bf16 one, and just below it, are exact sums of their parts, too
    codes, scales, z, w = w4_data(n, 160, 32, True)
    x = randn(rows, 160, seed=121)
    x[rows - 1, 50] = value
    check_w4(ops.w4_linear(x, ops.w4_pack(codes, scales, z, k=160, group=32)), x, w, None, None, 160)


@pytest.mark.parametrize("rows,n", [(1, 48), (2, 9500), (7, 48), (40, 48)])
def test_w4_reports_a_wait_that_ran_out(rows, n):
    # the code is left by the host (no kernel waits in vain); the next call says what it was, and the one after it works
    from msnhnet_b200 import tokens
    ops = tokens.TokenOps(0)
    codes, scales, z, w = w4_data(n, 160, 32, True)
    weights, x = ops.w4_pack(codes, scales, z, k=160, group=32), randn(rows, 160, seed=122)
    ops.ctx.check(ops.lib.msnh_b200_ctx_set_error(ops.h, 6))
    with pytest.raises(_ffi.KernelError, match="status 5: a bounded wait inside an earlier 4-bit product"):
        ops.w4_linear(x, weights)
    check_w4(ops.w4_linear(x, weights), x, w, None, None, 160)
    ops.close()
    assert _ffi.kernel_lib().msnh_b200_ctx_set_error(None, 6) == 1


@pytest.mark.parametrize("starts", [[0, 5, 3, 8], [0, 2, 4, 3], [4, 0, 4, 8], [8, 6, 3, 0]])
def test_append_refuses_starts_that_are_not_in_order(ops, starts):
    # which sequence a token is of is not certain then: no sequence grows by tokens that nobody writes
    cache, _, _ = make_cache([3, 4, 0, 7], 4, 1, 16, F16, 123, spare=9, width=5)
    m = Model(cache)
    k = randn(8, 1, 16, seed=124, dtype=F16)
    ops.kv_append(cache, k, k, seqs=ints(0, 1, 2), starts=ints(*starts))
    m.refused = 3
    m.same(cache)
    ops.kv_append(cache, k, k, seqs=ints(0, 1, 2), starts=ints(1, 3, 3, 8))          # a gap at the front, none for one
    m.append([0, 1, 2], [2, 0, 5], k[1:], k[1:])
    m.same(cache)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lengths,each", [([40, 100, 70], 1), ([40, 100, 70], 4), ([300, 2000, 5000], 8), ([300, 2000, 5000], 20)])
def test_attention_of_infinite_keys_and_values(ops, dtype, lengths, each):
    cache, keys, values = make_cache(lengths, 16, 2, 64, dtype, 125, spare=6)
    q = randn(3, 2 * each, 64, seed=126, dtype=dtype) * 0.3
    q[:, :, 9] = 0.5
    inf = float("inf")
    # sequence 0: a key of -inf, a score of -inf: a token of weight 0; 1: an infinite value each in two columns, and both signs in a third;
    # 2: a key of +inf, which no softmax survives
    def put(pages, i, token, head, column, value):
        pages[int(cache.page_table[i, token // 16]), token % 16, head, column] = value
    put(cache.k_pages, 0, 17, 0, 9, -inf)
    for token, column, value in ((33, 3, inf), (99, 40, -inf), (5, 50, inf), (6, 50, -inf)):
        put(cache.v_pages, 1, token, 1, column, value)
    put(cache.k_pages, 2, 20, 1, 9, inf)
    out, lse = ops.attn_decode(q, cache, return_lse=True)
    absent = [torch.zeros(n, dtype=torch.bool, device="cuda") for n in lengths]
    absent[0][17] = True
    check_attn(out[:1, :each], lse[:1, :each], q[:1, :each], [keys[0][:, :1]], [values[0][:, :1]], 0.125, absent=absent)
    check_attn(out[:2, :each], lse[:2, :each], q[:2, :each], [k[:, :1] for k in keys], [v[:, :1] for v in values], 0.125, absent=absent)
    check_attn(out[:1, each:], lse[:1, each:], q[:1, each:], [keys[0][:, 1:]], [values[0][:, 1:]], 0.125)
    spoilt = out[1, each:]
    assert bool((spoilt[:, 3] == inf).all()) and bool((spoilt[:, 40] == -inf).all()) and bool(torch.isnan(spoilt[:, 50]).all())
    others = [c for c in range(64) if c not in (3, 40, 50)]
    check_attn(spoilt[None, :, others], lse[1:2, each:], q[1:2, each:], [keys[1][:, 1:]], [values[1][:, 1:, others]], 0.125)
    assert bool(torch.isnan(out[2, each:]).all()) and bool(torch.isfinite(out[2, :each]).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16, E4M3])
@pytest.mark.parametrize("n", [9457, 9472, 9488, 11825, 11840, 11856, 12288])
@pytest.mark.parametrize("rows,k", [(1, 2048), (1, 1920), (2, 2048), (2, 300), (2, 3968), (2, 4096)])
def test_w4_of_as_many_outputs_as_change_the_kernel(ops, dtype, n, rows, k):
    # four and five 16-row tiles for each of 148 SMs, and one tile more and less; 15 and 16, 31 and 32 pieces of k
    codes, scales, z, w = w4_data(n, k, 128, True)
    x, x_scale = w4_x(rows, k, dtype, 127)
    check_w4(ops.w4_linear(x, ops.w4_pack(codes, scales, z, k=k, group=128), x_scale=x_scale, out_dtype=F32), x, w, x_scale, None, k)


@pytest.mark.parametrize("dtype", [F32, F16, BF16, E4M3])
@pytest.mark.parametrize("rows,k,n,group", [(9, 515, 9500, 128), (13, 300, 19001, 64), (16, 420, 9500, 32), (12, 2100, 12000, 128)])
def test_w4_of_nine_to_sixteen_rows_of_many_outputs(ops, dtype, rows, k, n, group):
    codes, scales, z, w = w4_data(n, k, group, True)
    x, x_scale = w4_x(rows, k, dtype, 128)
    b = randn(n, seed=129) * 0.1
    check_w4(ops.w4_linear(x, ops.w4_pack(codes, scales, z, k=k, group=group), bias=b, x_scale=x_scale), x, w, x_scale, b, k)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cols", [64, 250, 512, 2048, 2056, 4104, 5120, 8200, 12288, 16384])
def test_norm_of_many_rows_to_8_bits_with_a_residual(ops, dtype, cols):
    # blocks that stay and copy rows ahead, x's and the residual's; beside the residual and in its place
    rows = 1300 if cols > 1024 else 5000
    x, r, w = randn(rows, cols, seed=130, dtype=dtype), randn(rows, cols, seed=131, dtype=dtype) * 2, randn(cols, seed=132, dtype=dtype)
    want_h, want = norm_ref(x, r, w, 1e-6)
    codes, scale, h = ops.rms_norm(x, w, residual=r, out_dtype=E4M3)
    check_codes(codes, scale, want, cols)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    r2 = r.clone()
    again, scale2, _ = ops.rms_norm(x, w, residual=r2, residual_out=r2, out_dtype=E4M3)
    assert torch.equal(again.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(scale2, scale) and torch.equal(r2, h)
    x2 = x.clone()
    again, scale2, _ = ops.rms_norm(x2, w, residual=r, residual_out=x2, out_dtype=E4M3)
    assert torch.equal(again.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(scale2, scale) and torch.equal(x2, h)
    x2, r2 = x.clone(), r.clone()
    y, _ = ops.rms_norm(x, w, residual=r)
    ops.rms_norm(x2, w, residual=r2, residual_out=r2, out=x2)
    assert torch.equal(x2, y) and torch.equal(r2, h)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lengths", [[1], [37], [500], [0, 5, 500, 17], [3000] + [20] * 30])
@pytest.mark.parametrize("width", [256, 4096])
def test_attention_in_a_table_with_room(ops, dtype, lengths, width):
    # whether a pair is cut, and how its parts are joined, is decided by what the table could hold
    cache, keys, values = make_cache(lengths, 16, 2, 64, dtype, 133, width=width)
    q = randn(len(lengths), 8, 64, seed=134, dtype=dtype)
    out, lse = ops.attn_decode(q, cache, return_lse=True)
    check_attn(out, lse, q, keys, values, 0.125)


@pytest.mark.parametrize("rows,k,n,dtype,group", [(1, 20000, 9600, F16, 128), (2, 33000, 11900, F16, 128), (2, 20000, 11850, BF16, 32), (1, 2050, 9600, E4M3, 64), (2, 4100, 19001, F16, 32)])
def test_w4_of_long_rows_in_whole_numbers(ops, rows, k, n, dtype, group):
    # 16- and 8-bit activations that are multiplied so: digits made apart, by clusters' blocks, by every block
    codes, scales, z, w = w4_data(n, k, group, True)
    weights = ops.w4_pack(codes, scales, z, k=k, group=group)
    x, x_scale = w4_x(rows, k, dtype, 135)
    y = ops.w4_linear(x, weights, x_scale=x_scale, out_dtype=F32)
    check_w4(y, x, w, x_scale, None, k)
    assert torch.equal(y, ops.w4_linear(x, weights, x_scale=x_scale, out_dtype=F32))
    if dtype != E4M3:
        x[rows - 1, k // 2] = float("nan")
        y = ops.w4_linear(x, weights, out_dtype=F32)
        assert bool(torch.isnan(y[rows - 1]).all())
        check_w4(y[:rows - 1], x[:rows - 1], w, None, None, k)
