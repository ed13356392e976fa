"""The operators of positions, scores and the 8-bit cache together: the reader with rotary positions and an 8-bit cache against the same decoder in 64
bits, what it reads with scores, how it scores a text, and sequences that are kept elsewhere."""
import math

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


def features(n, seed):
    return torch.randn(n, 512, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def dense(plain):
    codes, scales, zeros, group = plain
    values = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1).double()
    column = torch.arange(values.shape[1], device="cuda") // group
    return (values - zeros.double()[:, column]) * scales.double()[:, column]


class Plain:
    """The decoder with rotary positions in 64 bits, nothing rounded on the way."""

    def __init__(self, reader):
        self.r = reader
        self.w = {k: dense(v) for k, v in reader.plain.items()}
        self.keys = [[] for _ in range(reader.layers)]
        self.values = [[] for _ in range(reader.layers)]

    @staticmethod
    def norm(h, w):
        return h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w.double()

    def turned(self, x, at):
        half = self.r.head_dim // 2
        f = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        z = torch.complex(x[..., :half], x[..., half:]) * torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), at.double()[:, None] * f)[:, None]
        return torch.cat([z.real, z.imag], -1)

    def decode(self, x, at):
        r, h = self.r, x
        d = r.head_dim
        for i, w in enumerate(r.weights):
            qkv = (self.norm(h, w["norm1"]) @ self.w[i, "qkv"].T).view(len(x), -1, d)
            both = self.turned(qkv[:, :r.heads + r.kv_heads], at)
            self.keys[i].append(both[:, r.heads:])
            self.values[i].append(qkv[:, r.heads + r.kv_heads:])
            k, v = (torch.cat(t).repeat_interleave(r.heads // r.kv_heads, 1) for t in (self.keys[i], self.values[i]))
            p = torch.softmax(torch.einsum("nhd,thd->nht", both[:, :r.heads], k) / d ** 0.5, -1)
            h = h + torch.einsum("nht,thd->nhd", p, v).reshape(len(x), -1) @ self.w[i, "out"].T
            h = h + torch.nn.functional.silu(self.norm(h, w["norm2"]) @ self.w[i, "up"].T) @ self.w[i, "down"].T
        return self.norm(h, r.last_norm) @ self.w["head"].T

    def look(self, f):
        return self.decode(f.double() @ self.w["project"].T, torch.arange(len(f), device="cuda"))

    def step(self, token, at):
        return self.decode(self.r.embedding[token:token + 1].double(), torch.tensor([at], device="cuda"))


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("cache_dtype", [torch.float16, E4M3])
def test_reader_with_rotary_positions_follows_the_decoder_in_64_bits(ops, cache_dtype):
    from msnhnet_b200.reader import Reader
    reader = Reader(ops, n_seqs=3, positions="rotary", cache_dtype=cache_dtype)
    f, plain = features(49, 5), Plain(reader)
    # An 8-bit rounding is off by at most 2^-4, by 2^-4 / sqrt(12) times a binade's mean (about 2 %) in the root of its mean square. Five norms lie between the
    # features and the logits: under 15 % of the norm together. In an 8-bit cache a layer's keys and values are two more: under 25 %.
    bound = 0.15 if cache_dtype == torch.float16 else 0.25
    assert off(reader.look(f, 1), plain.look(f)) < bound
    for at, token in enumerate([5, 999, 0, 17]):
        got = reader.step(torch.tensor([token], device="cuda"), ints(1))
        assert off(got, plain.step(token, 49 + at)) < bound
    assert [c.refused() for c in reader.caches] == [0, 0]


@pytest.mark.parametrize("positions", ["learned", "rotary"])
@pytest.mark.parametrize("cache_dtype", [torch.float16, E4M3])
def test_reader_reads_with_scores(ops, positions, cache_dtype):
    from msnhnet_b200.reader import Reader
    reader = Reader(ops, n_seqs=3, positions=positions, cache_dtype=cache_dtype)
    maps = [features(49, 6), features(33, 7), features(1, 8)]
    said = reader.read(maps, 9)
    tokens, logprobs, entropies = reader.read(maps, 9, scores=True)
    assert torch.equal(said, tokens) and logprobs.shape == entropies.shape == (3, 9)
    assert bool((logprobs < 0).all()) and bool((entropies > 0).all()) and bool((entropies <= math.log(1000) + 1e-5).all())
    # the likeliest token has at least the share of a uniform choice among e^entropy tokens
    assert bool((logprobs >= -entropies - 1e-4).all())
    # the same texts, scored: each map's tokens at once by one sequence (other rows in a call: other tile shapes, whose last bits the 8-bit roundings
    # that follow may magnify), so only the first token's logits, which no step has touched, are the same
    for i, f in enumerate(maps):
        got, entropy, top, ids = reader.score(f, tokens[i], alternatives=4)
        assert torch.equal(got[0], logprobs[i, 0]) and torch.equal(entropy[0], entropies[i, 0]) and int(ids[0, 0]) == int(tokens[i, 0])
        assert torch.equal(top[0, 0], got[0]) and bool((top[:, 0] >= got).all()) and bool((top[:, :-1] >= top[:, 1:]).all())
        assert off(got, logprobs[i].double()) < 0.25
    for cache in reader.caches:
        assert int(cache.refs.sum()) == 0 and cache.refused() == 0


def test_reader_scores_a_text_like_its_own_steps(ops):
    from msnhnet_b200.reader import Reader
    reader = Reader(ops, n_seqs=2, positions="rotary", cache_dtype=E4M3)
    f, ids = features(20, 9), torch.tensor([4, 77, 999, 0, 123])
    got, entropy, _, _ = reader.score(f, ids)
    rows = [reader.look(f, 0)[-1:]]
    for i in range(4):
        rows.append(reader.step(ids[i:i + 1], ints(0)))
    log_p = torch.log_softmax(torch.cat(rows).double(), -1)
    want = log_p.gather(1, ids.cuda()[:, None])[:, 0]
    # (fp32 sums over 1000 logits: 2^-24 for each of a thread's, and for the distances' roundings)
    assert bool(((got.double() - want).abs() <= 2e-5).all())
    assert bool(((entropy.double() + (log_p.exp() * log_p).sum(-1)).abs() <= 5e-5).all())
    reader.forget(ints(0))
    bad = reader.score(features(3, 10), torch.tensor([1, -1, 2]))[0]
    assert torch.isnan(bad).tolist() == [False, True, True]          # no such token, and nothing follows it


@pytest.mark.parametrize("cache_dtype", [torch.float16, E4M3])
@pytest.mark.parametrize("positions", ["learned", "rotary"])
def test_reader_keeps_sequences_elsewhere(ops, cache_dtype, positions):
    from msnhnet_b200.reader import Reader
    reader = Reader(ops, n_seqs=3, positions=positions, cache_dtype=cache_dtype)
    reader.look(features(37, 11), 1)
    reader.step(torch.tensor([3]), ints(1))
    kept = [tuple(t.cpu() for t in pair) for pair in reader.save(1)]
    assert kept[0][0].shape == (38, 2, 64)
    want = reader.step(torch.tensor([8]), ints(1))
    reader.forget(ints(1))
    reader.restore(2, kept)
    assert torch.equal(reader.step(torch.tensor([8]), ints(2)), want)   # (codes times powers of two are the same codes again)
    assert reader.caches[0].lengths.tolist() == [0, 0, 39]
    assert reader.save(0)[1][0].shape == (0, 2, 64)
    reader.restore(0, reader.save(1))
    reader.forget(ints(0, 2))
    for cache in reader.caches:
        assert int(cache.refs.sum()) == 0 and cache.refused() == 0


def test_reader_forks_in_an_8_bit_cache(ops):
    from msnhnet_b200.reader import Reader
    reader = Reader(ops, n_seqs=4, max_tokens=80, positions="rotary", cache_dtype=E4M3)
    first, second = features(49, 12), features(33, 13)
    alone = []
    for token in (7, 8):
        reader.look(first, 0)
        reader.step(torch.tensor([3]), ints(0))
        reader.step(torch.tensor([token]), ints(0))
        alone.append(reader.step(torch.tensor([token + 1]), ints(0)))
        reader.forget(ints(0))
    reader.look(second, 2)
    reader.look(first, 0)
    reader.step(torch.tensor([3]), ints(0))
    reader.fork(ints(0), ints(1))
    reader.forget(ints(2))
    reader.step(torch.tensor([7, 8]), ints(0, 1))
    reader.tidy()
    both = reader.step(torch.tensor([8, 9]), ints(0, 1))
    for i in range(2):
        assert off(both[i:i + 1], alone[i].double()) < 0.25           # (other tile shapes: other last bits, and 8-bit roundings that follow them)
    reader.forget(ints(0, 1))
    for cache in reader.caches:
        assert int(cache.refs.sum()) == 0 and cache.refused() == 0


def test_reader_command(ops, capsys, monkeypatch):
    from msnhnet_b200 import reader
    monkeypatch.setattr("sys.argv", ["reader", "--images", "1", "--tokens", "3", "--cache", "e4m3", "--positions", "rotary", "--scores"])
    reader.main()
    out = capsys.readouterr().out
    assert "image 0:" in out and "log p:" in out and "entropy:" in out
