"""The token operators together: the reader behind an image net, against the same decoder in 64 bits, and its cache under forks."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import helpers as H  # noqa: E402
from msnhnet_b200 import _ffi, synth  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from msnhnet_b200 import tokens
    handle = tokens.TokenOps(0)
    yield handle
    handle.close()


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def dense(plain):
    codes, scales, zeros, group = plain
    values = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1).double()
    column = torch.arange(values.shape[1], device="cuda") // group
    return (values - zeros.double()[:, column]) * scales.double()[:, column]


class Plain:
    """The decoder in 64 bits, nothing rounded on the way."""

    def __init__(self, reader):
        self.r = reader
        self.w = {k: dense(v) for k, v in reader.plain.items()}
        self.keys = [[] for _ in range(reader.layers)]
        self.values = [[] for _ in range(reader.layers)]

    @staticmethod
    def norm(h, w):
        return h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w.double()

    def decode(self, x):
        r, h = self.r, x
        d = r.head_dim
        for i, w in enumerate(r.weights):
            qkv = (self.norm(h, w["norm1"]) @ self.w[i, "qkv"].T).view(len(x), -1, d)
            self.keys[i].append(qkv[:, r.heads:r.heads + r.kv_heads])
            self.values[i].append(qkv[:, r.heads + r.kv_heads:])
            k, v = (torch.cat(t).repeat_interleave(r.heads // r.kv_heads, 1) for t in (self.keys[i], self.values[i]))
            p = torch.softmax(torch.einsum("nhd,thd->nht", qkv[:, :r.heads], k) / d ** 0.5, -1)
            h = h + torch.einsum("nht,thd->nhd", p, v).reshape(len(x), -1) @ self.w[i, "out"].T
            h = h + torch.nn.functional.silu(self.norm(h, w["norm2"]) @ self.w[i, "up"].T) @ self.w[i, "down"].T
        return self.norm(h, r.last_norm) @ self.w["head"].T

    def look(self, features):
        return self.decode(features.double() @ self.w["project"].T + self.r.position[:len(features)].double())

    def step(self, token, at):
        return self.decode(self.r.embedding[token:token + 1].double() + self.r.position[at:at + 1].double())


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


def test_reader_follows_the_decoder_in_64_bits(ops):
    from msnhnet_b200.reader import Reader
    reader = Reader(ops, n_seqs=3)
    features = torch.randn(49, 512, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    plain = Plain(reader)
    # Activations in 8 bits have a relative rounding error of at most 2^-4, 2^-4 / sqrt(12) times a binade's mean (about 2 %) as the root of
    # its mean square; five norms lie between the features and the logits, and what they add is at most their sum: under 15 % of the norm.
    assert off(reader.look(features, 1), plain.look(features)) < 0.15
    for at, token in enumerate([5, 999, 0, 17]):
        got = reader.step(torch.tensor([token], device="cuda"), ints(1))
        assert off(got, plain.step(token, 49 + at)) < 0.15
    assert [c.refused() for c in reader.caches] == [0, 0]


def test_reader_forks_and_forgets(ops):
    from msnhnet_b200.reader import Reader
    reader = Reader(ops, n_seqs=4, max_tokens=80)
    g = torch.Generator(device="cuda").manual_seed(4)
    first, second = (torch.randn(n, 512, generator=g, device="cuda") for n in (49, 33))
    alone = []
    for token in (7, 8):                                              # each way by itself
        reader.look(first, 0)
        reader.step(torch.tensor([3], device="cuda"), ints(0))
        reader.step(torch.tensor([token], device="cuda"), ints(0))
        alone.append(reader.step(torch.tensor([token + 1], device="cuda"), ints(0)))
        reader.forget(ints(0))
    # both ways as forks of one, beside another sequence, before and after pages are moved together
    reader.look(second, 2)
    reader.look(first, 0)
    reader.step(torch.tensor([3], device="cuda"), ints(0))
    reader.fork(ints(0), ints(1))
    reader.forget(ints(2))
    reader.step(torch.tensor([7, 8], device="cuda"), ints(0, 1))
    reader.tidy()
    both = reader.step(torch.tensor([8, 9], device="cuda"), ints(0, 1))
    for i in range(2):
        assert off(both[i:i + 1], alone[i].double()) < 0.15           # (other tile shapes: other last bits, and 8-bit roundings that follow them)
    reader.forget(ints(0, 1))
    for cache in reader.caches:
        assert int(cache.refs.sum()) == 0 and cache.refused() == 0


def test_reader_behind_a_net(ops):
    from msnhnet_b200.reader import Reader, features_of
    text = H.net_text("resnet18", 224)
    net = H.GpuNet(text, H.net_blob("resnet18", text), fp16=True, batch=2, flags=_ffi.PLAN_KEEP_ALL)
    features = features_of(net, synth.make_images(2, 3, 224, 224))
    net.close()
    assert features.shape == (2, 49, 512) and bool(torch.isfinite(features).all())
    reader = Reader(ops, n_seqs=2)
    said = reader.read(list(features), 5)
    assert said.shape == (2, 5) and np.array_equal(said.cpu().numpy(), reader.read(list(features), 5).cpu().numpy())


def test_reader_fills_a_sequence_and_refuses_more(ops):
    from msnhnet_b200.reader import Reader
    reader = Reader(ops, n_seqs=2, max_tokens=52)
    g = torch.Generator(device="cuda").manual_seed(5)
    first, second = (torch.randn(n, 512, generator=g, device="cuda") for n in (49, 10))
    reader.look(first, 0)
    reader.look(second, 1)
    for token in (4, 5, 6):
        reader.step(torch.tensor([token], device="cuda"), ints(0))
    with pytest.raises(ValueError, match="52"):
        reader.step(torch.tensor([7], device="cuda"), ints(0))
    assert reader.caches[0].lengths.tolist() == [52, 10]
    assert bool(torch.isfinite(reader.step(torch.tensor([7], device="cuda"), ints(1))).all())
    assert reader.caches[1].lengths.tolist() == [52, 11]
    reader.forget(ints(0, 1))
    said = reader.read([first, second], 4)
    assert torch.equal(said, reader.read([first, second], 4))
    with pytest.raises(ValueError):
        reader.read([first, second], 5)


def test_reader_leaves_out_rows_of_no_sequence_and_no_token(ops):
    from msnhnet_b200.reader import Reader
    reader = Reader(ops, n_seqs=3)
    features = torch.randn(20, 512, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    for seq in range(3):
        reader.look(features, seq)
    logits = reader.step(torch.tensor([5, 1000, 5, -1, 5], device="cuda"), ints(0, 1, 3, 2, -1))
    assert torch.isnan(logits).all(-1).tolist() == [False, True, True, True, True] and bool(torch.isfinite(logits[0]).all())
    assert [c.lengths.tolist() for c in reader.caches] == [[21, 20, 20]] * 2
    assert [c.refused() for c in reader.caches] == [4, 4]


def test_reader_takes_tokens_from_the_host(ops):
    from msnhnet_b200.reader import Reader
    reader = Reader(ops, n_seqs=3)
    features = torch.randn(20, 512, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    for seq in range(3):
        reader.look(features, seq)
    want = reader.step(torch.tensor([5], device="cuda"), ints(0))
    assert torch.equal(reader.step(torch.tensor([5]), ints(1)), want) and torch.equal(reader.step([5], ints(2)), want)
