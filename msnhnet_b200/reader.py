"""A reader of image features: the token operators (tokens.py) as one decoder behind a net.

The net's last feature map is the prefix, one token a cell; every cell sees every other. Then tokens follow one at a time, each over all
before it: norm (with the residual's addition, activations in 8 bits), 4-bit products, the cache, attention. Weights are seeded stand-ins, as the
nets' are.

    python -m msnhnet_b200.reader [--images N] [--tokens N]      # reads the features of ResNet-18, 224 x 224
"""
import argparse
import time

import torch

from . import tokens

E4M3 = torch.float8_e4m3fn


class Reader:
    """A decoder of `layers` layers: width features, heads query heads over kv_heads key heads of head_dim, ffn hidden values, vocab tokens.
    At most n_seqs sequences of max_tokens (features and tokens) each, MAX_ROWS of them in a call. What cannot fit raises ValueError
    before anything is launched."""

    MAX_ROWS = 64                            # of w4_linear

    def __init__(self, ops, channels=512, width=512, layers=2, heads=8, kv_heads=2, head_dim=64, ffn=1024, vocab=1000, n_seqs=8, max_tokens=256, page=16, seed=1):
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
        pages = -(-max_tokens // page)
        self.caches = [ops.new_cache(n_seqs * pages, page, kv_heads, head_dim, n_seqs, pages) for _ in range(layers)]

    def _decode(self, x, seqs, append):
        """Rows of values through the layers; append(cache, k, v) puts their keys and values down. Returns the logits."""
        ops, rows, h = self.ops, x.shape[0], x
        delta = None
        for w, cache in zip(self.weights, self.caches):
            if delta is None:
                y, scale = ops.rms_norm(h, w["norm1"], out_dtype=E4M3)
            else:
                y, scale, h = ops.rms_norm(delta, w["norm1"], residual=h, residual_out=h, out_dtype=E4M3)
            qkv = ops.w4_linear(y, w["qkv"], x_scale=scale).view(rows, -1, self.head_dim)
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
        x = self.ops.w4_linear(features.half(), self.project) + self.position[:n]
        one = torch.tensor([seq], dtype=torch.int32, device=x.device)
        starts = torch.tensor([0, n], dtype=torch.int32, device=x.device)
        return self._decode(x, one.expand(n).contiguous(), lambda cache, k, v: self.ops.kv_append(cache, k, v, seqs=one, starts=starts))

    def step(self, ids, seqs):
        """One token (ids: int64 [n], at most 64) behind each of the sequences seqs (int32 [n]); the logits of what follows. A row whose
        token or sequence is none leaves every sequence as it was; its logits are NaN."""
        return self._step(torch.as_tensor(ids, device=self.position.device), seqs)

    def _step(self, ids, seqs, named=None):
        if len(ids) != len(seqs) or len(ids) > self.MAX_ROWS:
            raise ValueError(f"{len(ids)} tokens for {len(seqs)} sequences: as many, and at most {self.MAX_ROWS}")
        self._take(1, seqs, named)
        if named is not None:                                        # (all of them known to be in range)
            return self._decode(self.embedding[ids] + self.position[self.caches[0].lengths[seqs.long()].long()], seqs,
                                lambda cache, k, v: self.ops.kv_append(cache, k, v, seqs=seqs))
        # (indexes are kept in range: one that is not would end the process's use of the GPU)
        seq, token = seqs.clamp(0, self.n_seqs - 1), ids.clamp(0, self.vocab - 1)
        there = (seq == seqs) & (token == ids)
        at = self.caches[0].lengths.index_select(0, seq).clamp_(0, self.max_tokens - 1)
        seqs = torch.where(there, seqs, -1)
        logits = self._decode(self.embedding.index_select(0, token) + self.position.index_select(0, at), seqs, lambda cache, k, v: self.ops.kv_append(cache, k, v, seqs=seqs))
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

    def read(self, features, n_tokens):
        """The likeliest tokens, one after the other, for each of a list of feature maps [cells, channels]: int64 [maps, n_tokens]. Takes
        sequences 0, 1, ..., which have to be empty, and forgets them again."""
        if not 0 < len(features) <= min(self.n_seqs, self.MAX_ROWS) or n_tokens < 1:
            raise ValueError(f"{n_tokens} tokens for {len(features)} maps: at least one of each, {min(self.n_seqs, self.MAX_ROWS)} maps at most")
        for f in features:
            if not 0 < f.shape[0] <= self.MAX_ROWS or f.shape[0] + n_tokens - 1 > self.max_tokens:
                raise ValueError(f"{f.shape[0]} cells and {n_tokens} tokens: at most {self.MAX_ROWS} cells, {self.max_tokens} of both")
        named = list(range(len(features)))
        self._empty(named)
        seqs = torch.arange(len(features), dtype=torch.int32, device=self.position.device)
        ids = torch.stack([self.look(f, i)[-1].argmax() for i, f in enumerate(features)])
        said = [ids]
        for _ in range(n_tokens - 1):
            ids = self._step(ids, seqs, named).argmax(-1)
            said.append(ids)
        self.forget(seqs)
        for i in named:
            self.most[i] = 0
        return torch.stack(said, 1)


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
    a = ap.parse_args()
    from . import _ffi, synth, topologies
    from .net import Net
    text = topologies.NETS["resnet18"](size=224)
    net = Net(text, synth.make_blob(text, synth.load_factors("resnet18")), fp16=True, batch=a.images, flags=_ffi.PLAN_KEEP_ALL)
    features = features_of(net, synth.make_images(a.images, 3, 224, 224))
    net.close()
    reader = Reader(tokens.TokenOps(), n_seqs=a.images, max_tokens=max(256, features.shape[1] + a.tokens))
    reader.read(list(features), 2)
    torch.cuda.synchronize()
    began = time.perf_counter()
    said = reader.read(list(features), a.tokens).tolist()
    for i, ids in enumerate(said):
        print(f"image {i}:", *ids)
    print(f"{(time.perf_counter() - began) / a.tokens * 1e3:.2f} ms a token and image batch")


if __name__ == "__main__":
    main()
