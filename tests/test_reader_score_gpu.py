"""What Reader.score says of a text with a token that is none: that one, and all behind it, have no probability."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from msnhnet_b200 import tokens
    handle = tokens.TokenOps(0)
    yield handle
    handle.close()


@pytest.mark.parametrize("ids,first_bad", [([1, -1, 2, 3, 4], 1), ([5, 6, 1000, 7, 8, 9], 2), ([-7, 1, 2], 0), ([4, 77, 2 ** 40, -1, 5], 2), ([3, 4, -1], 2), ([3, 4, 5], 3)])
@pytest.mark.parametrize("positions", ["learned", "rotary"])
def test_nothing_follows_a_token_that_is_none(ops, positions, ids, first_bad):
    from msnhnet_b200.reader import Reader
    reader = Reader(ops, n_seqs=2, positions=positions)
    f = torch.randn(9, 512, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    logprobs, entropies, top, best = reader.score(f, torch.tensor(ids), alternatives=2)
    # (the token that is none has no probability itself, but what could stand in its place has)
    assert torch.isnan(logprobs).tolist() == [i >= first_bad for i in range(len(ids))]
    assert torch.isnan(entropies).tolist() == [i > first_bad for i in range(len(ids))]
    assert torch.isnan(top).any(-1).tolist() == (best < 0).all(-1).tolist() == [i > first_bad for i in range(len(ids))]
    # what stands before it is as without the rest
    if first_bad:
        alone = reader.score(f, torch.tensor(ids[:first_bad]), alternatives=2)
        for got, want in zip((logprobs, entropies, top, best), alone):
            assert torch.equal(got[:first_bad], want)
    for cache in reader.caches:
        assert int(cache.refs.sum()) == 0
