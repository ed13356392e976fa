"""Outputs whose rows share memory are refused, with each other and with the input they are made of; layouts whose rows are apart are taken, however they lie."""
import pytest

torch = pytest.importorskip("torch")
from msnhnet_b200 import _ffi  # noqa: E402

pytestmark = pytest.mark.gpu

D = 32


@pytest.fixture(scope="module")
def ops():
    from msnhnet_b200 import tokens
    handle = tokens.TokenOps(0)
    yield handle
    handle.close()


def randn(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# strides of [3 tokens, 2 heads, D]: (token, head) and whether rows are apart
LAYOUTS = [((2 * D, D), True), ((D, 3 * D), True), ((5 * D, 2 * D), True), ((2 * D, 3 * D), True), ((D, D), False), ((2 * D, 2 * D), False), ((D, 2 * D), False), ((2 * D - 1, D), False),
           ((2 * D + 1, D), True), ((D, 3 * D - 1), False), ((3 * D, 3 * D // 2), True), ((2 * D + 15, 3 * D // 2), False), ((3 * D, 2 * D), True), ((3 * D, 2 * D + 1), False)]


@pytest.mark.parametrize("strides,apart", LAYOUTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rotary_into_any_layout(ops, dtype, strides, apart):
    x, positions, table = randn(3, 2, D, seed=1).to(dtype), ints(3, 4, 5), ops.rotary_table(D)
    out = torch.as_strided(torch.zeros(20 * D, device="cuda", dtype=dtype), (3, 2, D), (*strides, 1))
    if apart:
        ops.rotary(x, positions, table, out=out)
        assert torch.equal(out, ops.rotary(x, positions, table))
    else:
        with pytest.raises(_ffi.KernelError, match="overlap"):
            ops.rotary(x, positions, table, out=out)


# (offset, strides) of x and of out in one buffer, in values
PAIRS = [((0, (2 * D, D)), (0, (2 * D, D)), True),                    # in place
         ((0, (4 * D, D)), (2 * D, (4 * D, D)), True),                # beside each other in wider rows
         ((2 * D, (4 * D, D)), (0, (4 * D, D)), True),
         ((0, (4 * D, 2 * D)), (D, (4 * D, 2 * D)), True),            # every other head
         ((0, (4 * D, D)), (D, (4 * D, D)), False),
         ((0, (2 * D, D)), (2 * D, (2 * D, D)), False),
         ((0, (2 * D, D)), (1, (2 * D, D)), False),
         ((0, (2 * D, D)), (6 * D, (2 * D, D)), True),
         ((0, (2 * D, D)), (6 * D - 1, (2 * D, D)), False),
         ((0, (2 * D, D)), (0, (D, 3 * D)), False),                   # the same memory in another order
         ((0, (0, D)), (0, (2 * D, D)), False),                       # one token for all of them
         ((0, (0, D)), (2 * D, (2 * D, D)), True),
         ((0, (4 * D, 2 * D)), (D, (6 * D, 2 * D)), True),            # other strides, no row in common
         ((0, (4 * D, 2 * D)), (D - 1, (6 * D, 2 * D)), False)]


@pytest.mark.parametrize("one,other,apart", PAIRS)
def test_rotary_within_one_buffer(ops, one, other, apart):
    buffer, positions, table = randn(24 * D, seed=2), ints(3, 4, 5), ops.rotary_table(D)
    x, out = (torch.as_strided(buffer, (3, 2, D), (*strides, 1), at) for at, strides in (one, other))
    want = ops.rotary(x.clone(), positions, table)
    if apart:
        ops.rotary(x, positions, table, out=out)
        assert torch.equal(out, want)
    else:
        before = buffer.clone()
        with pytest.raises(_ffi.KernelError, match="overlap"):
            ops.rotary(x, positions, table, out=out)
        assert torch.equal(buffer, before)


def test_rotary_of_one_token_or_head_does_not_mind_its_strides(ops):
    buffer, table = randn(24 * D, seed=3), ops.rotary_table(D)
    for shape, strides, positions in (((1, 4, D), (1, D, 1), ints(7)), ((5, 1, D), (2 * D, 0, 1), ints(0, 1, 2, 3, 4))):
        x, out = (torch.as_strided(buffer, shape, strides, at) for at in (0, 12 * D))
        want = ops.rotary(x.clone(), positions, table)
        ops.rotary(x, positions, table, out=out)
        assert torch.equal(out, want)
        # in place, by a stride that no token but the first, or no head, uses
        ops.rotary(x, positions, table, out=torch.as_strided(buffer, shape, (7, D, 1) if shape[0] == 1 else (2 * D, 7, 1), 0))
        assert torch.equal(x, want)


@pytest.mark.parametrize("strides,apart", LAYOUTS)
@pytest.mark.parametrize("kind", [torch.float16, torch.float8_e4m3fn])
def test_reading_into_any_layout(ops, kind, strides, apart):
    cache = ops.new_cache(4, 4, 2, D, 2, 2, dtype=kind)
    k, v = (randn(3, 2, D, seed=s).half() for s in (4, 5))
    ops.kv_append(cache, k, v, seqs=ints(1), starts=ints(0, 3))
    want = ops.kv_read(cache, ints(0, 3), 3, seqs=ints(1))
    out = [torch.as_strided(torch.zeros(20 * D, device="cuda").half(), (3, 2, D), (*strides, 1)) for _ in range(2)]
    if apart:
        ops.kv_read(cache, ints(0, 3), 3, seqs=ints(1), out=out)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    else:
        with pytest.raises(_ffi.KernelError, match="overlap"):
            ops.kv_read(cache, ints(0, 3), 3, seqs=ints(1), out=out)


@pytest.mark.parametrize("strides,at,apart", [((4 * D, D), 2 * D, True), ((4 * D, 2 * D), D, True), ((2 * D, D), 6 * D, True), ((2 * D, D), 0, False), ((4 * D, D), D, False), ((2 * D, D), 2 * D, False),
                                              ((4 * D, D), 2 * D + 1, False)])
def test_keys_and_values_are_read_to_places_of_their_own(ops, strides, at, apart):
    cache = ops.new_cache(4, 4, 2, D, 2, 2)
    k, v = (randn(3, 2, D, seed=s).half() for s in (6, 7))
    ops.kv_append(cache, k, v, seqs=ints(1), starts=ints(0, 3))
    buffer = torch.zeros(20 * D, device="cuda").half()
    for first, second in ((0, at), (at, 0)):
        out = [torch.as_strided(buffer, (3, 2, D), (*strides, 1), i) for i in (first, second)]
        if apart:
            ops.kv_read(cache, ints(0, 3), 3, seqs=ints(1), out=out)
            assert torch.equal(out[0], k) and torch.equal(out[1], v)
        else:
            with pytest.raises(_ffi.KernelError, match="overlap"):
                ops.kv_read(cache, ints(0, 3), 3, seqs=ints(1), out=out)


@pytest.mark.parametrize("strides,apart", LAYOUTS)
@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.float8_e4m3fn])
def test_attention_into_any_layout(ops, kind, strides, apart):
    cache = ops.new_cache(6, 4, 2, D, 3, 2, dtype=kind)
    values = torch.float16 if kind == torch.float8_e4m3fn else kind
    k, v, q = (randn(3, 2, D, seed=s).to(values) for s in (8, 9, 10))
    ops.kv_append(cache, k, v)
    out = torch.as_strided(torch.zeros(20 * D, device="cuda", dtype=values), (3, 2, D), (*strides, 1))
    if apart:
        ops.attn_decode(q, cache, out=out)
        assert torch.equal(out, ops.attn_decode(q, cache))
    else:
        with pytest.raises(_ffi.KernelError, match="overlap"):
            ops.attn_decode(q, cache, out=out)


def test_outputs_that_are_given_are_what_comes_back(ops):
    x, positions, table = randn(3, 2, D, seed=11), ints(3, 4, 5), ops.rotary_table(D)
    want = ops.rotary(x, positions, table)
    out = torch.zeros_like(x)
    for given in (out, x):                                            # beside the input, then in its place
        got = ops.rotary(x, positions, table, out=given)
        assert got.data_ptr() == given.data_ptr() and got.stride() == given.stride() and torch.equal(got, want)
