"""What the operators of positions, scores and the 8-bit cache refuse before anything reaches a GPU. No device is needed: tensors of the CPU stand for
those of another device, and the handle has no context behind it."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")
from msnhnet_b200 import _ffi, tokens  # noqa: E402

E4M3 = torch.float8_e4m3fn


@pytest.fixture
def ops():
    """A handle of cuda:0 that every call must refuse to use."""
    handle = tokens.TokenOps.__new__(tokens.TokenOps)
    handle.device, handle._ctx, handle._index = torch.device("cuda", 0), 1, 0
    return handle


@pytest.fixture
def cache():
    """An 8-bit cache of another device than the handle's."""
    c = tokens.PagedCache.__new__(tokens.PagedCache)
    c.k_pages, c.v_pages = (torch.zeros(4, 2, 1, 16).to(E4M3) for _ in range(2))
    c.page_table, c.lengths, c.refs = (torch.zeros(*shape, dtype=torch.int32) for shape in ((2, 3), (2,), (4,)))
    c.k_scales, c.v_scales = torch.ones(4, 1, 1), torch.ones(4, 1, 1)
    c.tensors = c.k_pages, c.v_pages, c.page_table, c.lengths, c.refs, c.k_scales, c.v_scales
    c.args = _ffi.KvCache(c.k_pages.data_ptr(), c.v_pages.data_ptr(), 32, 16, 16, 32, 16, 16, c.page_table.data_ptr(), c.lengths.data_ptr(), c.refs.data_ptr(), None, 3, 4, 2, 1,
                          16, 2, 3, _ffi.E4M3, c.k_scales.data_ptr(), c.v_scales.data_ptr(), 2)
    c.address = ctypes.addressof(c.args)
    return c


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def table():
    return tokens.RotaryTable(torch.zeros(4, dtype=torch.int64), False, 1.0)


def test_tensors_of_another_device_are_refused(ops, cache):
    with pytest.raises(ValueError, match="x: a tensor on cpu"):
        ops.rotary(torch.zeros(2, 1, 8), ints(0, 1), table())
    with pytest.raises(ValueError, match="logits: a tensor on cpu"):
        ops.token_scores(torch.zeros(2, 8))
    for call in (lambda: ops.kv_read(cache, ints(0, 1), 1), lambda: ops.kv_append(cache, torch.zeros(2, 1, 16), torch.zeros(2, 1, 16))):
        with pytest.raises(ValueError, match="the cache: a tensor on cpu"):
            call()
    with pytest.raises(ValueError, match="one GPU"):
        tokens.PagedCache(cache.k_pages, cache.v_pages, cache.page_table, cache.lengths, cache.refs, cache.k_scales, cache.v_scales)


def test_tensors_that_require_a_gradient_are_refused(ops, cache):
    with pytest.raises(ValueError, match="gradient"):
        ops.rotary(torch.zeros(2, 1, 8, requires_grad=True), ints(0, 1), table())
    with pytest.raises(ValueError, match="gradient"):
        ops.token_scores(torch.zeros(2, 8, requires_grad=True))
    cache.k_scales.requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        tokens.PagedCache(cache.k_pages, cache.v_pages, cache.page_table, cache.lengths, cache.refs, cache.k_scales, cache.v_scales)


def test_scales_that_do_not_fit_are_refused(cache):
    parts = cache.k_pages, cache.v_pages, cache.page_table, cache.lengths, cache.refs
    for scales in ((), (cache.k_scales,), (torch.ones(4, 1, 3),) * 2, (torch.ones(4, 2, 1),) * 2, (torch.ones(4, 1, 1, dtype=torch.float64),) * 2, (torch.ones(1, 4, 1).transpose(0, 1),
                   torch.ones(4, 1, 2)), (torch.ones(4, 1, 4)[:, :, ::2],) * 2):
        with pytest.raises(ValueError, match="scales"):
            tokens.PagedCache(*parts, *scales)
    half = torch.zeros(4, 2, 1, 16).half()
    with pytest.raises(ValueError, match="8-bit"):
        tokens.PagedCache(half, half, *parts[2:], cache.k_scales, cache.v_scales)


def test_caches_that_do_not_fit_are_refused(ops):
    for more in ({"dtype": E4M3, "scale_block": 3}, {"dtype": E4M3, "scale_block": 0}, {"dtype": E4M3, "scale_block": 32}, {"scale_block": 4}):
        with pytest.raises(ValueError):
            ops.new_cache(4, 16, 1, 16, 2, 3, **more)


@pytest.mark.parametrize("dim,more", [(3, {}), (0, {}), (-2, {}), (8, {"base": 0.0}), (8, {"base": math.nan}), (8, {"factor": 0.0}), (8, {"stretch": "some"}), (8, {"low": 4.0, "high": 4.0}),
                                      (8, {"trained": 0})])
def test_rotary_tables_that_are_none_are_refused(ops, dim, more):
    ops.device = torch.device("cpu")
    with pytest.raises(ValueError):
        ops.rotary_table(dim, **more)


def test_rotary_tables_hold_whole_turns_as_fractions(ops):
    # (a base below 1 has planes that turn more than once a position: whole turns do not count)
    ops.device = torch.device("cpu")
    turns = ops.rotary_table(4, base=1e-4).turns.tolist()
    for i, got in enumerate(turns):
        f = (1e-4) ** (-i / 2) / (2 * math.pi)
        assert abs((got / 2 ** 64 - f + 0.5) % 1.0 - 0.5) < 2.0 ** -40
