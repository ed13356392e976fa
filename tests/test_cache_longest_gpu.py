"""The longest sequence that a cache's table holds: its last tokens are 2^31 - 9 and before, and nothing behind them is looked at."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
PAGE = 1016                                                           # 8 * 127, and 2^28 - 1 is a multiple of 127


@pytest.fixture(scope="module")
def ops():
    from msnhnet_b200 import tokens
    handle = tokens.TokenOps(0)
    yield handle
    handle.close()


def cache_of(kind, dim, table, lengths, pages):
    from msnhnet_b200 import tokens
    scales = []
    if kind == E4M3:
        scales = [torch.exp2(torch.randint(-3, 3, (len(pages[0]), 1, PAGE // 8), generator=torch.Generator(device="cuda").manual_seed(s), device="cuda").float()) for s in (3, 4)]
    ints = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in (lengths, [1] * len(pages[0]))]
    return tokens.PagedCache(*pages, table, *ints, *scales)


@pytest.mark.parametrize("kind,dim", [(F16, 8), (BF16, 16), (F32, 4), (E4M3, 16), (E4M3, 128)])
def test_attention_ends_with_the_last_token(ops, kind, dim):
    longest = (2 ** 31 - 8) // PAGE
    pages = [(torch.randn(3, PAGE, 1, dim, generator=torch.Generator(device="cuda").manual_seed(s), device="cuda") * 2).to(kind) for s in (1, 2)]
    # the first sequence ends with page 1; what lies behind its row of the table is page 2
    table = torch.zeros(2, longest, dtype=torch.int32, device="cuda")
    table[0, longest - 1], table[1, 0] = 1, 2
    long = cache_of(kind, dim, table, [2 ** 31 - 8, PAGE], pages)
    short = cache_of(kind, dim, torch.tensor([[1], [2]], dtype=torch.int32, device="cuda"), [PAGE, PAGE], pages)
    q = torch.randn(2, 4, dim, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(F16 if kind == E4M3 else kind)
    for window in (40, 8, 1, 33, 200):
        # (the same tokens at the same places of a tile)
        for got, want in zip(ops.attn_decode(q, long, window=window, return_lse=True), ops.attn_decode(q, short, window=window, return_lse=True)):
            assert torch.equal(got, want)
    k, v = (torch.zeros(PAGE, 1, dim, dtype=F32, device="cuda") for _ in range(2))
    ops.kv_read(long, torch.tensor([0, PAGE], dtype=torch.int32, device="cuda"), PAGE, first=torch.tensor([2 ** 31 - 8 - PAGE + 1], dtype=torch.int32, device="cuda"), out=(k, v))
    for got, want in zip((k, v), ops.kv_read(short, torch.tensor([0, PAGE], dtype=torch.int32, device="cuda"), PAGE, first=torch.tensor([1], dtype=torch.int32, device="cuda"), dtype=F32)):
        assert torch.equal(got, want) and bool((got[-1] == 0).all())
