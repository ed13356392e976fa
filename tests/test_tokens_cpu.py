"""What the token operators refuse before anything reaches a GPU. No device is needed: tensors of the CPU stand for those of another
device, and the handle has no context behind it."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
from msnhnet_b200 import _ffi, tokens  # noqa: E402


@pytest.fixture
def ops():
    """A handle of cuda:0 that every call must refuse to use."""
    handle = tokens.TokenOps.__new__(tokens.TokenOps)
    handle.device, handle._ctx, handle._index = torch.device("cuda", 0), 1, 0
    return handle


@pytest.fixture
def cache():
    """A cache of another device than the handle's."""
    c = tokens.PagedCache.__new__(tokens.PagedCache)
    c.k_pages, c.v_pages = torch.zeros(4, 2, 1, 8), torch.zeros(4, 2, 1, 8)
    c.page_table, c.lengths, c.refs = (torch.zeros(*shape, dtype=torch.int32) for shape in ((2, 3), (2,), (4,)))
    c.tensors = c.k_pages, c.v_pages, c.page_table, c.lengths, c.refs
    c.args = _ffi.KvCache(c.k_pages.data_ptr(), c.v_pages.data_ptr(), 16, 8, 8, 16, 8, 8, c.page_table.data_ptr(), c.lengths.data_ptr(), c.refs.data_ptr(), None, 3, 4, 2, 1, 8,
                          2, 3, _ffi.F32)
    c.address = ctypes.addressof(c.args)
    return c


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("call", [
    lambda ops, c: ops.kv_append(c, torch.zeros(2, 1, 8), torch.zeros(2, 1, 8)), lambda ops, c: ops.kv_fork(c, ints(0), ints(1)), lambda ops, c: ops.kv_free(c, ints(0)),
    lambda ops, c: ops.kv_copy_pages(c, ints(0), ints(1))], ids=["append", "fork", "free", "copy"])
def test_a_cache_of_another_device_is_refused(ops, cache, call):
    with pytest.raises(ValueError, match="the cache: a tensor on cpu"):
        call(ops, cache)


def test_tensors_of_another_device_are_refused(ops, cache):
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="x: a tensor on cpu"):
        ops.rms_norm(x, torch.ones(8))
    with pytest.raises(ValueError, match="q: a tensor on cpu"):
        ops.attn_decode(torch.zeros(2, 1, 8), cache)
    with pytest.raises(ValueError, match="the cache: a tensor on cpu"):
        ops.kv_compact(cache)
    with pytest.raises(ValueError, match="a tensor on cpu"):
        ops.w4_pack(torch.zeros(4, 16, dtype=torch.uint8), torch.ones(4, 1, dtype=torch.float16), k=32, group=32)


def test_tensors_that_require_a_gradient_are_refused(ops, cache):
    x, w = torch.zeros(2, 8), torch.ones(8, requires_grad=True)
    grad = {"match": "gradient"}
    with pytest.raises(ValueError, **grad):
        ops.rms_norm(x.requires_grad_(), torch.ones(8))
    with pytest.raises(ValueError, **grad):
        ops.attn_decode(torch.zeros(2, 1, 8, requires_grad=True), cache)
    cache.k_pages.requires_grad_()
    with pytest.raises(ValueError, **grad):
        ops.kv_free(cache, ints(0))
    with pytest.raises(ValueError, **grad):
        tokens.PagedCache(cache.k_pages, cache.v_pages, cache.page_table, cache.lengths, cache.refs)
    with torch.no_grad(), pytest.raises(ValueError, match="cpu"):    # (the next thing that is wrong)
        ops.rms_norm(x, w)
