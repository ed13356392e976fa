"""Appending to blocks whose scales the caller has written: any finite numbers, negative ones and such that are no powers of two."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from msnhnet_b200 import tokens
    handle = tokens.TokenOps(0)
    yield handle
    handle.close()


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def randn(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def held(ops, cache, n):
    return torch.stack(ops.kv_read(cache, ints(0, n), n, seqs=ints(1), dtype=torch.float32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 48, 20])                         # a head's columns in one warp, across warps, value by value
@pytest.mark.parametrize("times", [-1.0, -1.5, 1.5, -0.3])
def test_append_keeps_what_scales_of_the_caller_stand_for(ops, dtype, dim, times):
    cache = ops.new_cache(4, 16, 2, dim, 2, 2, dtype=E4M3, scale_block=16)
    first = randn(2, 5, 2, dim, seed=1).to(dtype)
    ops.kv_append(cache, *first, seqs=ints(1), starts=ints(0, 5))
    for scales in (cache.k_scales, cache.v_scales):
        scales.mul_(times)
    before, scales = held(ops, cache, 5), torch.stack([cache.k_scales, cache.v_scales]).clone()
    assert torch.equal(before.sign(), (first.float() * times).sign() * (before != 0))
    # zeros and small values: nothing has to grow
    for n, small in ((5, 0.0), (6, 1e-3)):
        new = (randn(2, 1, 2, dim, seed=2) * small).to(dtype)
        ops.kv_append(cache, *new, seqs=ints(1))
        after = held(ops, cache, n + 1)
        assert torch.equal(after[:, :5], before) and torch.equal(torch.stack([cache.k_scales, cache.v_scales]), scales)
        used = scales.abs()[:, :1, :, 0][..., None]
        assert bool(((after[:, n:] - new.float()).abs() <= 2.0 ** -4 * new.float().abs() + 2.0 ** -10 * used).all())
    # large ones: older codes are rounded again, once (half a step: 2^-4, or half of the smallest code), to the nearest of what the new scale has
    new = (randn(2, 1, 2, dim, seed=3) * 100).to(dtype)
    ops.kv_append(cache, *new, seqs=ints(1))
    after, used = held(ops, cache, 8), torch.stack([cache.k_scales, cache.v_scales])[:, :1, :, 0][..., None]
    assert bool((used > 0).all()) and bool((used.abs() >= scales.abs()[:, :1, :, 0][..., None]).all())
    assert bool(((after[:, :5] - before).abs() <= 2.0 ** -4 * (1 + 2.0 ** -20) * before.abs() + 2.0 ** -10 * used).all())
    assert bool(((after[:, 7:] - new.float()).abs() <= 2.0 ** -4 * new.float().abs() + 2.0 ** -10 * used).all())
