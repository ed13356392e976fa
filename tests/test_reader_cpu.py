"""What the reader refuses before anything reaches a GPU: its operators are stand-ins that must not be called."""
import types

import pytest

torch = pytest.importorskip("torch")
from msnhnet_b200.reader import Reader  # noqa: E402


class NoOps:
    device = torch.device("cpu")

    def w4_pack(self, *args, **kwargs):
        return None

    def new_cache(self, n_pages, page, kv_heads, head_dim, n_seqs, pages):
        return types.SimpleNamespace(lengths=torch.zeros(n_seqs, dtype=torch.int32))

    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


def reader(n_seqs=3, max_tokens=64):
    return Reader(NoOps(), channels=64, width=64, layers=2, heads=2, kv_heads=1, head_dim=32, ffn=64, vocab=10, n_seqs=n_seqs, max_tokens=max_tokens)


def maps(*cells):
    return [torch.zeros(n, 64) for n in cells]


@pytest.mark.parametrize("features,tokens", [(maps(49), 17), (maps(49, 20), 40), (maps(10, 10, 10, 10), 2), (maps(65), 1), (maps(0), 1), (maps(5), 0), ([], 3)])
def test_read_refuses_what_does_not_fit(features, tokens):
    with pytest.raises(ValueError):
        reader().read(features, tokens)


def test_look_refuses_what_does_not_fit():
    r = reader()
    for cells, seq in ((10, 3), (10, -1), (65, 0), (0, 0)):
        with pytest.raises(ValueError):
            r.look(torch.zeros(cells, 64), seq)
    r.most[1] = 60
    r.caches[0].lengths[1] = 60
    with pytest.raises(ValueError, match="more tokens"):
        r.look(torch.zeros(10, 64), 1)


def test_step_refuses_a_token_too_many():
    r = reader()
    r.most = [64, 64, 64]
    r.caches[0].lengths[:] = torch.tensor([5, 64, 63], dtype=torch.int32)
    one = torch.tensor([1])
    with pytest.raises(ValueError, match=r"sequences \[1\]"):
        r.step(one, torch.tensor([1], dtype=torch.int32))
    assert r.most == [5, 64, 63]                                     # what was looked up
    with pytest.raises(AssertionError, match="reached"):             # the others have room
        r.step(torch.tensor([1, 1]), torch.tensor([0, 2], dtype=torch.int32))
    assert r.most == [6, 64, 64]


def test_step_refuses_too_many_rows():
    r = reader(n_seqs=70)
    with pytest.raises(ValueError, match="64"):
        r.step(torch.zeros(65, dtype=torch.long), torch.arange(65, dtype=torch.int32))
    with pytest.raises(ValueError, match="sequences"):
        r.step(torch.zeros(2, dtype=torch.long), torch.arange(3, dtype=torch.int32))


def test_a_fork_may_be_as_long_as_the_longest():
    class Forks(NoOps):
        def kv_fork(self, cache, src, dst):
            pass

    r = Reader(Forks(), channels=64, width=64, layers=2, heads=2, kv_heads=1, head_dim=32, ffn=64, vocab=10, n_seqs=3, max_tokens=64)
    r.most = [60, 0, 3]
    r.fork(torch.tensor([0], dtype=torch.int32), torch.tensor([1], dtype=torch.int32))
    for cache in r.caches:
        cache.lengths[:] = torch.tensor([0, 60, 3], dtype=torch.int32)                # (the first one has been forgotten since)
    with pytest.raises(ValueError, match="more tokens"):
        r.look(torch.zeros(10, 64), 1)


def test_features_are_the_first_tokens():
    r = reader()
    r.most, r.caches[0].lengths[1] = [0, 5, 7], 5
    with pytest.raises(ValueError, match=r"\[1\] are not empty"):
        r.look(torch.zeros(10, 64), 1)
    with pytest.raises(ValueError, match=r"\[1\] are not empty"):
        r.read(maps(10, 10), 3)
    with pytest.raises(AssertionError, match="reached"):             # (the third one has been forgotten since it was counted)
        r.look(torch.zeros(10, 64), 2)
