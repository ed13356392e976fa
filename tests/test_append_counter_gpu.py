"""An append of as many blocks of scales as a call may have: its launch counts to 2^31 - 2 and ends."""
import pytest

torch = pytest.importorskip("torch")
from msnhnet_b200 import _ffi  # noqa: E402

pytestmark = pytest.mark.gpu


def test_append_of_the_most_blocks_ends():
    from msnhnet_b200 import tokens
    ops = tokens.TokenOps(0)
    # a block of threads for each head of keys and of values, and a scale for every token: 2 * (tokens + 2 sequences' ends) items. The cache has no room for
    # them, so the sequence is refused and nothing is written; a token stands for all of them
    tokens_of_call = (2 ** 31 - 1) // 2 - 2
    cache = ops.new_cache(2, 1, 1, 512, 1, 2, dtype=torch.float8_e4m3fn, scale_block=1)
    one = torch.ones(1, 1, 512, device="cuda")
    ops.kv_append(cache, one, one)
    many = one.expand(tokens_of_call, 1, 512)
    ops.kv_append(cache, many, many, seqs=torch.zeros(1, dtype=torch.int32, device="cuda"), starts=torch.tensor([0, tokens_of_call], dtype=torch.int32, device="cuda"))
    assert cache.refused() == 1 and cache.lengths.tolist() == [1] and cache.refs.tolist() == [1, 0]
    more = one.expand(tokens_of_call + 1, 1, 512)
    with pytest.raises(_ffi.KernelError, match="2\\^31"):
        ops.kv_append(cache, more, more, seqs=torch.zeros(1, dtype=torch.int32, device="cuda"), starts=torch.tensor([0, tokens_of_call + 1], dtype=torch.int32, device="cuda"))
    ops.kv_append(cache, one, one)
    assert cache.lengths.tolist() == [2] and torch.equal(cache.k_pages.float() * cache.k_scales[..., None], torch.ones(2, 1, 1, 512, device="cuda"))
    ops.close()
