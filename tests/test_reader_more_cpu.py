"""What the reader's scores, saved sequences, positions and caches refuse before anything reaches a GPU: its operators are stand-ins that must not be called."""
import types

import pytest

torch = pytest.importorskip("torch")
from msnhnet_b200.reader import Reader  # noqa: E402

E4M3 = torch.float8_e4m3fn


class NoOps:
    device = torch.device("cpu")

    def __init__(self):
        self.made = []

    def w4_pack(self, *args, **kwargs):
        return None

    def new_cache(self, n_pages, page, kv_heads, head_dim, n_seqs, pages, **more):
        self.made.append(more)
        return types.SimpleNamespace(lengths=torch.zeros(n_seqs, dtype=torch.int32), dtype=more.get("dtype", torch.float16))

    def rotary_table(self, dim, **more):
        self.table = dim, more
        return object()

    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


def reader(ops=None, **more):
    return Reader(ops or NoOps(), channels=64, width=64, layers=2, heads=2, kv_heads=1, head_dim=32, ffn=64, vocab=10, n_seqs=3, max_tokens=64, **more)


def test_caches_and_positions_are_as_asked():
    ops = NoOps()
    assert reader(ops).turns is None and ops.made == [{}, {}]
    ops = NoOps()
    r = reader(ops, cache_dtype=E4M3, positions="rotary", rotary={"base": 5e5, "stretch": "slow"})
    assert r.turns is not None and ops.made == [{"dtype": E4M3}] * 2 and ops.table == (32, {"base": 5e5, "stretch": "slow"})
    with pytest.raises(ValueError, match="positions"):
        reader(positions="none")
    with pytest.raises(ValueError, match="positions"):
        reader(rotary={"base": 5e5})


@pytest.mark.parametrize("cells,ids,alternatives", [(0, [1], 0), (65, [1], 0), (30, [1] * 36, 0), (5, [], 0), (5, [[1]], 0), (5, [1], -1), (5, [1], 11)])
def test_score_refuses_what_does_not_fit(cells, ids, alternatives):
    with pytest.raises(ValueError):
        reader().score(torch.zeros(cells, 64), torch.tensor(ids, dtype=torch.int64), alternatives)


def test_score_and_restore_want_an_empty_sequence():
    r = reader()
    r.most, r.caches[0].lengths[0] = [5, 0, 0], 5
    with pytest.raises(ValueError, match="not empty"):
        r.score(torch.zeros(5, 64), torch.tensor([1]))
    with pytest.raises(ValueError, match="not empty"):
        r.restore(0, [(torch.zeros(3, 1, 32),) * 2] * 2)
    with pytest.raises(AssertionError, match="reached"):
        r.restore(1, [(torch.zeros(3, 1, 32),) * 2] * 2)


def test_save_and_restore_refuse_what_does_not_fit():
    r = reader()
    for seq in (-1, 3):
        with pytest.raises(ValueError):
            r.save(seq)
        with pytest.raises(ValueError):
            r.restore(seq, [(torch.zeros(3, 1, 32),) * 2] * 2)
    one = torch.zeros(3, 1, 32)
    for saved in ([(one, one)], [(one, one), (one, one[:2])], [(one, one), (one[..., :16], one)], [(torch.zeros(65, 1, 32),) * 2] * 2):
        with pytest.raises(ValueError):
            r.restore(1, saved)
