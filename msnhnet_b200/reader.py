"""A reader of image features: the token operators (tokens.py) as one decoder behind a net.

The net's last feature map is the prefix, one token a cell; every cell sees every other. Then tokens follow one at a time, each over all
before it: norm (with the residual's addition, activations in 8 bits), 4-bit products, the cache, attention. Weights are seeded stand-ins, as the
nets' are.

    python -m msnhnet_b200.reader [--images N] [--tokens N] [--cache f16|e4m3] [--positions learned|rotary] [--scores]
                                                                 # reads the features of ResNet-18, 224 x 224
"""
import argparse
import time

import torch

from . import tokens

E4M3 = torch.float8_e4m3fn


class Reader:
    """A decoder of `layers` layers: width features, heads query heads over kv_heads key heads of head_dim, ffn hidden values, vocab tokens.
    At most n_seqs sequences of max_tokens (features and tokens) each, MAX_ROWS of them in a call. What cannot fit raises ValueError
    before anything is launched. cache_dtype: float16, or float8_e4m3fn for half the memory. positions: "learned" ones, added to what is looked at
    and read, or "rotary": queries and keys are turned by where they are (rotary: further arguments of TokenOps.rotary_table)."""

    MAX_ROWS = 64                            # of w4_linear

    def __init__(self, ops, channels=512, width=512, layers=2, heads=8, kv_heads=2, head_dim=64, ffn=1024, vocab=1000, n_seqs=8, max_tokens=256, page=16, seed=1,
                 cache_dtype=torch.float16, positions="learned", rotary=None):
        if positions not in ("learned", "rotary") or (rotary and positions != "rotary"):
            raise ValueError(f"positions {positions!r}: 'learned', or 'rotary' with arguments of its own")
        self.ops, self.width, self.heads, self.kv_heads, self.head_dim, self.layers = ops, width, heads, kv_heads, head_dim, layers
        self.vocab, self.n_seqs, self.max_tokens = vocab, n_seqs, max_tokens
        # Tokens of each sequence, at most: the sequences' numbers lie on the GPU, so a step counts for all of them. Where a count reaches
        # max_tokens the lengths are looked up.
        self.most = [0] * n_seqs
        g = torch.Generator(device=ops.device).manual_seed(seed)

        def normal(*shape):
            return torch.randn(*shape, generator=g, device=ops.device)

        def linear(n, k, group=64):
            codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8, device=ops.device)
            scales = ((0.5 + torch.rand(n, k // group, generator=g, device=ops.device)) / (4.6 * k ** 0.5)).half()
            zeros = torch.randint(6, 10, (n, k // group), generator=g, dtype=torch.uint8, device=ops.device)
            return ops.w4_pack(codes, scales, zeros, group=group), (codes, scales, zeros, group)

        def norm():
            return (1 + 0.1 * normal(width)).half()

        shapes = {"qkv": ((heads + 2 * kv_heads) * head_dim, width), "out": (width, heads * head_dim), "up": (ffn, width), "down": (width, ffn)}
        # (.plain: codes, scales, zeros and group of every product, for those who want to check one)
        self.plain = {}
        self.weights = []
        for i in range(layers):
            one = {}
            for name, (n, k) in shapes.items():
                one[name], self.plain[i, name] = linear(n, k)
            one["norm1"], one["norm2"] = norm(), norm()
            self.weights.append(one)
        self.project, self.plain["project"] = linear(width, channels)
        self.head, self.plain["head"] = linear(vocab, width)
        self.last_norm = norm()
        self.embedding = (0.5 * normal(vocab, width)).half()
        self.position = (0.5 * normal(max_tokens, width)).half()
        # (rotary positions turn keys and queries, and nothing is added to what is looked at and read)
        self.turns = ops.rotary_table(head_dim, **(rotary or {})) if positions == "rotary" else None
        pages = -(-max_tokens // page)
        more = {} if cache_dtype == torch.float16 else {"dtype": cache_dtype}
        self.caches = [ops.new_cache(n_seqs * pages, page, kv_heads, head_dim, n_seqs, pages, **more) for _ in range(layers)]

    def _placed(self, x, at):
        """Rows of values with their learned positions; as they are where positions are rotary."""
        return x + self.position[at] if self.turns is None else x

    def _decode(self, x, seqs, append, at):
        """Rows of values at positions `at` (int32) through the layers; append(cache, k, v) puts their keys and values down. Returns the logits."""
        ops, rows, h = self.ops, x.shape[0], x
        delta = None
        for w, cache in zip(self.weights, self.caches):
            if delta is None:
                y, scale = ops.rms_norm(h, w["norm1"], out_dtype=E4M3)
            else:
                y, scale, h = ops.rms_norm(delta, w["norm1"], residual=h, residual_out=h, out_dtype=E4M3)
            qkv = ops.w4_linear(y, w["qkv"], x_scale=scale).view(rows, -1, self.head_dim)
            if self.turns is not None:
                turned = qkv[:, :self.heads + self.kv_heads]
                ops.rotary(turned, at, self.turns, out=turned)
            append(cache, qkv[:, self.heads:self.heads + self.kv_heads], qkv[:, self.heads + self.kv_heads:])
            seen = ops.attn_decode(qkv[:, :self.heads], cache, seqs=seqs)
            delta = ops.w4_linear(seen.view(rows, -1), w["out"])
            y, scale, h = ops.rms_norm(delta, w["norm2"], residual=h, residual_out=h, out_dtype=E4M3)
            delta = ops.w4_linear(torch.nn.functional.silu(ops.w4_linear(y, w["up"], x_scale=scale)), w["down"])
        y, scale, _ = ops.rms_norm(delta, self.last_norm, residual=h, residual_out=h, out_dtype=E4M3)
        return ops.w4_linear(y, self.head, x_scale=scale, out_dtype=torch.float32)

    def _take(self, n, seqs, named=None):
        """Counts n tokens more for sequences `named` (seqs on the GPU without it); ValueError where one of them has no place for them."""
        known = range(self.n_seqs) if named is None else named
        if max((self.most[i] for i in known), default=0) + n > self.max_tokens:
            self.most = self.caches[0].lengths.tolist()              # (waits for the GPU)
            if named is None:
                known = [i for i in seqs.tolist() if 0 <= i < self.n_seqs]
            full = [i for i in known if self.most[i] + n > self.max_tokens]
            if full:
                raise ValueError(f"sequences {full}: {n} more tokens would pass {self.max_tokens}")
        for i in known:
            self.most[i] += n

    def _empty(self, named):
        """ValueError where one of the sequences has tokens."""
        if any(self.most[i] for i in named):
            self.most = self.caches[0].lengths.tolist()              # (waits for the GPU)
            full = [i for i in named if self.most[i]]
            if full:
                raise ValueError(f"sequences {full} are not empty: no more tokens can be their first ones")

    def look(self, features, seq):
        """features [cells, channels] (at most 64 cells) become the first tokens of the empty sequence `seq`; logits of every cell."""
        n = features.shape[0]
        if not 0 <= seq < self.n_seqs or not 0 < n <= self.MAX_ROWS:
            raise ValueError(f"{n} cells for sequence {seq}: 1 to {self.MAX_ROWS} cells, {self.n_seqs} sequences")
        self._empty([seq])
        self._take(n, None, [seq])
        x = self._placed(self.ops.w4_linear(features.half(), self.project), slice(n))
        at = None if self.turns is None else torch.arange(n, dtype=torch.int32, device=x.device)
        one = torch.tensor([seq], dtype=torch.int32, device=x.device)
        starts = torch.tensor([0, n], dtype=torch.int32, device=x.device)
        return self._decode(x, one.expand(n).contiguous(), lambda cache, k, v: self.ops.kv_append(cache, k, v, seqs=one, starts=starts), at)

    def step(self, ids, seqs):
        """One token (ids: int64 [n], at most 64) behind each of the sequences seqs (int32 [n]); the logits of what follows. A row whose
        token or sequence is none leaves every sequence as it was; its logits are NaN."""
        return self._step(torch.as_tensor(ids, device=self.position.device), seqs)

    def _step(self, ids, seqs, named=None):
        if len(ids) != len(seqs) or len(ids) > self.MAX_ROWS:
            raise ValueError(f"{len(ids)} tokens for {len(seqs)} sequences: as many, and at most {self.MAX_ROWS}")
        self._take(1, seqs, named)
        if named is not None:                                        # (all of them known to be in range)
            at = self.caches[0].lengths[seqs.long()]
            return self._decode(self._placed(self.embedding[ids], at.long()), seqs, lambda cache, k, v: self.ops.kv_append(cache, k, v, seqs=seqs), at)
        # (indexes are kept in range: one that is not would end the process's use of the GPU)
        seq, token = seqs.clamp(0, self.n_seqs - 1), ids.clamp(0, self.vocab - 1)
        there = (seq == seqs) & (token == ids)
        at = self.caches[0].lengths.index_select(0, seq).clamp_(0, self.max_tokens - 1)
        seqs = torch.where(there, seqs, -1)
        logits = self._decode(self._placed(self.embedding.index_select(0, token), at), seqs, lambda cache, k, v: self.ops.kv_append(cache, k, v, seqs=seqs), at)
        return torch.where(there[:, None], logits, float("nan"))

    def fork(self, src, dst):
        """Sequences dst become copies of sequences src. One that is not empty stays as it is, and every cache counts it as refused."""
        for cache in self.caches:
            self.ops.kv_fork(cache, src, dst)
        self.most = [max(self.most)] * self.n_seqs                    # (which of them are copies, and of which, is known to the GPU only)

    def forget(self, seqs):
        for cache in self.caches:
            self.ops.kv_free(cache, seqs)

    def tidy(self):
        for cache in self.caches:
            self.ops.kv_compact(cache)

    def read(self, features, n_tokens, scores=False):
        """The likeliest tokens, one after the other, for each of a list of feature maps [cells, channels]: int64 [maps, n_tokens]. Takes
        sequences 0, 1, ..., which have to be empty, and forgets them again. With scores: (tokens, logprobs, entropies), both float32
        [maps, n_tokens]: how likely each token was among all, and how undecided the reader (a token is -1, and its scores NaN, where logits are no
        numbers)."""
        if not 0 < len(features) <= min(self.n_seqs, self.MAX_ROWS) or n_tokens < 1:
            raise ValueError(f"{n_tokens} tokens for {len(features)} maps: at least one of each, {min(self.n_seqs, self.MAX_ROWS)} maps at most")
        for f in features:
            self._fits(f.shape[0], n_tokens)
        named = list(range(len(features)))
        self._empty(named)
        seqs = torch.arange(len(features), dtype=torch.int32, device=self.position.device)
        logits = torch.stack([self.look(f, i)[-1] for i, f in enumerate(features)])
        said = []
        for i in range(n_tokens):
            if i:
                logits = self._step(ids, seqs, named)
            if scores:
                _, entropy, logprob, best = self.ops.token_scores(logits, top=1)
                ids = best[:, 0].clamp(min=0)                        # (one that is none is no index)
                said.append((best[:, 0], logprob[:, 0], entropy))
            else:
                ids = logits.argmax(-1)
                said.append((ids,))
        self._forgotten(seqs, named)
        out = tuple(torch.stack(column, 1) for column in zip(*said))
        return out if scores else out[0]

    def score(self, features, ids, alternatives=0):
        """How likely the reader takes a text to be: ids [n] behind a feature map [cells, channels]. (logprobs float32 [n], entropies float32
        [n], top_logprobs, top_ids [n, alternatives] or None), as TokenOps.token_scores gives them. An id that is no token has a log probability of NaN, and
        whatever follows it has NaN throughout (and ids of -1). Takes sequence 0, which has to be empty, and forgets it again."""
        ids = torch.as_tensor(ids, dtype=torch.int64, device=self.position.device)
        if ids.dim() != 1 or len(ids) < 1:
            raise ValueError("ids: [n], one token at least")
        if not 0 <= alternatives <= min(tokens.TokenOps.MAX_TOP, self.vocab):
            raise ValueError(f"{alternatives} alternatives: at most {min(tokens.TokenOps.MAX_TOP, self.vocab)}")
        self._fits(features.shape[0], len(ids))
        self._empty([0])
        seqs = torch.zeros(1, dtype=torch.int32, device=self.position.device)
        rows = [self.look(features, 0)[-1:]]
        for i in range(len(ids) - 1):
            rows.append(self.step(ids[i:i + 1], seqs))
        self._forgotten(seqs, [0])
        # (a step leaves the sequence as it was where a token is none: what came behind it would be scored as if it were not there)
        follows = ((ids >= 0) & (ids < self.vocab)).roll(1).index_fill(0, ids.new_zeros(1), True).cumprod(0).bool()
        logits = torch.where(follows[:, None], torch.cat(rows), float("nan"))
        return self.ops.token_scores(logits, ids, top=alternatives)

    def save(self, seq):
        """What the caches hold of a sequence, to be kept elsewhere: a list of (keys, values) [tokens, kv_heads, head_dim], one of each layer
        (waits for the GPU). Values of an 8-bit cache are float32, which holds them as they are."""
        if not 0 <= seq < self.n_seqs:
            raise ValueError(f"sequence {seq} of {self.n_seqs}")
        n = int(self.caches[0].lengths[seq])
        device = self.position.device
        one, starts = (torch.tensor(v, dtype=torch.int32, device=device) for v in ([seq], [0, n]))
        kept = torch.float32 if self.caches[0].dtype == E4M3 else None
        return [self.ops.kv_read(cache, starts, n, seqs=one, dtype=kept) for cache in self.caches]

    def restore(self, seq, saved):
        """Makes the empty sequence `seq` what save gave (of this reader or one of the same shape; on any device). Keys and values are the same ones; in an
        8-bit cache a last block that is not full may have half the scale it had, where its largest value was rounded down to 224 of it, and tokens that
        follow are then rounded by that."""
        if not 0 <= seq < self.n_seqs or len(saved) != self.layers:
            raise ValueError(f"{len(saved)} layers for sequence {seq}: {self.layers} layers, {self.n_seqs} sequences")
        n = saved[0][0].shape[0]
        if any(t.shape != (n, self.kv_heads, self.head_dim) for pair in saved for t in pair):
            raise ValueError("keys and values of all layers: as many tokens, and the reader's heads")
        self._empty([seq])
        self._take(n, None, [seq])
        device = self.position.device
        one, starts = (torch.tensor(v, dtype=torch.int32, device=device) for v in ([seq], [0, n]))
        kind = torch.float32 if self.caches[0].dtype == E4M3 else self.caches[0].dtype
        for cache, (k, v) in zip(self.caches, saved):
            self.ops.kv_append(cache, k.to(device, kind).contiguous(), v.to(device, kind).contiguous(), seqs=one, starts=starts)

    def _fits(self, cells, n_tokens):
        if not 0 < cells <= self.MAX_ROWS or cells + n_tokens - 1 > self.max_tokens:
            raise ValueError(f"{cells} cells and {n_tokens} tokens: at most {self.MAX_ROWS} cells, {self.max_tokens} of both")

    def _forgotten(self, seqs, named):
        self.forget(seqs)
        for i in named:
            self.most[i] = 0


def features_of(net, images, cells=49):
    """The last feature map of `cells` cells of a net that keeps its layers, [images, cells, channels] on the GPU."""
    net.forward(images)
    for layer in range(net.n_layers - 1, -1, -1):
        out = net.layer_output(layer, len(images))
        if out.shape[2] * out.shape[3] == cells:
            return torch.from_numpy(out).cuda().flatten(2).transpose(1, 2).contiguous()
    raise ValueError(f"no layer of {cells} cells")


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--images", type=int, default=2)
    ap.add_argument("--tokens", type=int, default=24)
    ap.add_argument("--cache", choices=["f16", "e4m3"], default="f16")
    ap.add_argument("--positions", choices=["learned", "rotary"], default="learned")
    ap.add_argument("--scores", action="store_true", help="how likely each token was, and how undecided the reader")
    a = ap.parse_args()
    from . import _ffi, synth, topologies
    from .net import Net
    text = topologies.NETS["resnet18"](size=224)
    net = Net(text, synth.make_blob(text, synth.load_factors("resnet18")), fp16=True, batch=a.images, flags=_ffi.PLAN_KEEP_ALL)
    features = features_of(net, synth.make_images(a.images, 3, 224, 224))
    net.close()
    reader = Reader(tokens.TokenOps(), n_seqs=a.images, max_tokens=max(256, features.shape[1] + a.tokens),
                    cache_dtype=E4M3 if a.cache == "e4m3" else torch.float16, positions=a.positions)
    reader.read(list(features), 2)
    torch.cuda.synchronize()
    began = time.perf_counter()
    said = reader.read(list(features), a.tokens, scores=a.scores)
    torch.cuda.synchronize()
    took = time.perf_counter() - began
    for i, ids in enumerate((said[0] if a.scores else said).tolist()):
        print(f"image {i}:", *ids)
        if a.scores:
            print("   log p:", *(f"{x:.2f}" for x in said[1][i].tolist()))
            print("   entropy:", *(f"{x:.2f}" for x in said[2][i].tolist()))
    print(f"{took / a.tokens * 1e3:.2f} ms a token and image batch")


if __name__ == "__main__":
    main()
