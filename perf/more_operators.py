"""What is timed of the operators that a decoding step has beside its norm, products and attention in 16 bits (msnhnet_b200/tokens.py): rotary
positions, a paged cache in 8 bits with a scale for each block of tokens and head, attention over it, and scores of tokens.

A case names the operator in "op":

    rotary   queries and keys are turned by their positions: `rot` of a head's `dim` values, in planes (2i, 2i + 1) or (i, i + rot / 2)
    write    prompts of 1 to `longest` tokens are quantised into the pages of an 8-bit cache, and their sequences are given up again
    beams    every sequence of an 8-bit cache is forked "fanout" times, each fork gets one token, and the forks are given up again
    read     keys and values of whole sequences come back from an 8-bit cache in the element type
    attn     one query token for each sequence over its pages of 8-bit keys and values; lengths from one token to "longest"
    scores   of rows of logits: log probability of a given token, entropy, and the `top` likeliest tokens with theirs

Element types: f32, f16, bf16. Where `own` is false the operators are computed in elementary torch operations in 32 bits, angles in 64.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
E4M3 = torch.float8_e4m3fn


def rotary(tokens, heads, dim, rot, dtype, interleaved, far, stretch, factor):
    return {"op": "rotary", "tokens": tokens, "heads": heads, "dim": dim, "rot": rot, "type": dtype, "interleaved": interleaved, "far": far,
            "stretch": stretch, "factor": factor}


def write(seqs, longest, kv_heads, dim, page, block, dtype):
    return {"op": "write", "seqs": seqs, "longest": longest, "kv_heads": kv_heads, "dim": dim, "page": page, "block": block, "type": dtype}


def beams(seqs, longest, fanout, kv_heads, dim, page, block, dtype):
    return {"op": "beams", "seqs": seqs, "longest": longest, "fanout": fanout, "kv_heads": kv_heads, "dim": dim, "page": page, "block": block, "type": dtype}


def read(seqs, longest, kv_heads, dim, page, block, dtype):
    return {"op": "read", "seqs": seqs, "longest": longest, "kv_heads": kv_heads, "dim": dim, "page": page, "block": block, "type": dtype}


def attn(seqs, longest, empty, heads, kv_heads, dim, page, block, dtype, window=0):
    return {"op": "attn", "seqs": seqs, "longest": longest, "empty": empty, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "block": block, "type": dtype, "window": window}


def scores(rows, cols, top, dtype, masked):
    return {"op": "scores", "rows": rows, "cols": cols, "top": top, "type": dtype, "masked": masked}


def listed():
    return [
        # one token of one caller, where the call itself is what counts
        dict(rotary(1, 40, 128, 128, "f16", False, 4096, "none", 1.0), name="rotary f16 one token"),                    # 32 query and 8 key heads
        dict(attn(1, 37, 0, 32, 8, 128, 16, 16, "f16"), name="attn f16 37 tokens"),                                     # the start of an answer
        dict(scores(1, 1000, 5, "f32", False), name="scores f32 one row"),                                              # as many as ResNet-18's classes
        dict(read(1, 300, 2, 64, 16, 16, "f16"), name="read f16 one sequence"),                                         # an image's cells and an answer
        # ordinary steps
        dict(beams(64, 2048, 4, 8, 128, 16, 16, "f16"), name="beams f16 64x4"),                                         # a beam search's step
        dict(scores(3, 128000, 20, "f16", True), name="scores f16 wide rows"),                                          # a step over a large vocabulary, some tokens forbidden
        # large ones: prompts, many or long sequences
        dict(rotary(4100, 40, 128, 128, "bf16", False, 131072, "slow", 8.0), name="rotary bf16 prompt"),                # a prompt far into a stretched context
        dict(write(24, 8192, 8, 128, 16, 16, "bf16"), name="write bf16 prompts"),
        dict(read(24, 8192, 8, 128, 16, 16, "bf16"), name="read bf16 24 sequences"),
        dict(attn(48, 8192, 2, 32, 8, 128, 16, 16, "bf16"), name="attn bf16 48 callers"),
        dict(attn(2, 131072, 0, 32, 8, 128, 64, 32, "f16"), name="attn f16 long"),                                      # a long document beside a short one
        dict(scores(2000, 50000, 8, "bf16", False), name="scores bf16 2000 rows"),                                      # a text scored token by token
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "write", "beams", "read", "attn", "attn", "attn", "scores", "scores"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "rotary":
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        heads = rng.randint(1, 48)
        rot = rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)])
        tokens = _spread(rng, 1, min(8192, 40_000_000 // (heads * dim * SIZE[dtype])))
        return rotary(tokens, heads, dim, rot, dtype, rng.random() < 0.5, _spread(rng, 1, 1_000_000), rng.choice(["none", "all", "base", "slow"]),
                      rng.choice([2.0, 4.0, 8.0, 32.0]))
    if op == "scores":
        cols = _spread(rng, 2, 262144)
        rows = _spread(rng, 1, max(1, min(4096, 100_000_000 // (cols * SIZE[dtype]))))
        return scores(rows, cols, min(cols // 2, rng.choice([0, 1, 5, 8, 20, 32])), dtype, rng.random() < 0.3)
    page = rng.choice([8, 16, 32, 64])
    block = rng.choice([b for b in (1, 2, 4, 8, 16, 16, 16, 32, 64) if b <= page])
    kv_heads = rng.choice([1, 2, 4, 8])
    if op == "attn":
        seqs, longest = _spread(rng, 1, 64), _spread(rng, 1, 65536)
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        longest = min(longest, max(1, 400_000 // seqs), 100_000_000 // (kv_heads * dim * 2))
        return attn(seqs, longest, rng.choice([0, 0, 1]) if seqs > 1 else 0, kv_heads * rng.choice([1, 2, 4, 5, 8, 16]), kv_heads, dim, page, block, dtype,
                    rng.choice([0, 0, 0, _spread(rng, 1, 2048)]))
    dim = rng.choice([64, 80, 96, 128])
    seqs, longest = _spread(rng, 1, 64), _spread(rng, 16, 4096)
    if op == "beams":
        return beams(seqs, longest, rng.choice([1, 2, 3, 4]), kv_heads, dim, page, block, dtype)
    most = 20_000_000 // (kv_heads * dim * SIZE[dtype])
    while sum(_lengths(seqs, longest, 0)) > most:
        longest = longest * 3 // 4
    return (write if op == "write" else read)(seqs, longest, kv_heads, dim, page, block, dtype)


def _lengths(count, longest, empty):
    """Tokens of each sequence, spread over the logarithm; the first `empty` ones have none."""
    return [0 if i < empty else max(1, round(longest ** ((i + 1) / count))) for i in range(count)]


def _pages_of(lengths, page):
    return sum(-(-n // page) for n in lengths)


def work(case):
    c = case
    if c["op"] == "rotary":
        n = c["tokens"] * c["heads"] * c["dim"]
        return {"bytes": 2 * n * SIZE[c["type"]] + 4 * c["tokens"], "flops": 3 * c["tokens"] * c["heads"] * c["rot"]}
    if c["op"] == "scores":
        n = c["rows"] * c["cols"]
        return {"bytes": n * SIZE[c["type"]] + c["rows"] * (16 + 12 * c["top"]), "flops": 5 * n}
    codes = c["kv_heads"] * c["dim"]                             # bytes of a token's keys
    lengths = _lengths(c["seqs"], c["longest"], c.get("empty", 0))

    def scale_bytes(n):
        return 4 * c["kv_heads"] * -(-n // c["block"])
    if c["op"] == "attn":
        seen = [min(n, c["window"]) if c["window"] else n for n in lengths]
        return {"bytes": 2 * sum(n * codes + scale_bytes(n) for n in seen) + 2 * c["seqs"] * c["heads"] * c["dim"] * SIZE[c["type"]] +
                4 * sum(-(-n // c["page"]) for n in seen), "flops": 4 * sum(seen) * c["heads"] * c["dim"]}
    if c["op"] in ("write", "read"):
        return {"bytes": 2 * sum(n * codes * (1 + SIZE[c["type"]]) + scale_bytes(n) for n in lengths) + 4 * _pages_of(lengths, c["page"]),
                "flops": 4 * sum(lengths) * codes}
    # beams: rows of the last page copied with their scales, one token's rows read and its codes written; a table entry read and written, a page's count up and down
    copied = sum(2 * (n % c["page"]) * codes + 2 * scale_bytes(n % c["page"]) for n in lengths) * c["fanout"] * 2
    shared = sum(n // c["page"] for n in lengths) * c["fanout"]
    return {"bytes": copied + 2 * codes * (1 + SIZE[c["type"]]) * c["seqs"] * c["fanout"] + 24 * shared, "flops": 4 * codes * c["seqs"] * c["fanout"]}


_ops = None


def _token_ops():
    """The handle that a program makes once."""
    global _ops
    if _ops is None:
        from msnhnet_b200 import tokens
        _ops = tokens.TokenOps()
    return _ops


BASE, TRAINED, LOW, HIGH = 10000.0, 8192, 1.0, 4.0


def _magnitude(c):
    return 1.0 if c["stretch"] == "none" else 0.1 * math.log(c["factor"]) + 1.0


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = {"device": "cuda"}

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, dtype=dtype, **dev)

    state = {"case": c}
    if own:
        state["ops"] = _token_ops()
    if c["op"] == "rotary":
        # queries and keys as a product leaves them, the values behind them
        both = normal(c["tokens"], c["heads"] + max(1, c["heads"] // 5), c["dim"]).to(TYPES[c["type"]])
        state["x"] = both[:, :c["heads"]]
        first = torch.randint(0, max(1, c["far"] - c["tokens"] + 1), (), generator=g, **dev)
        state["positions"] = (first + torch.arange(c["tokens"], **dev)).to(torch.int32)
        if own:
            state["table"] = state["ops"].rotary_table(c["rot"], base=BASE, interleaved=c["interleaved"], stretch=None if c["stretch"] == "none" else c["stretch"],
                                                       factor=c["factor"], trained=TRAINED, low=LOW, high=HIGH, magnitude=_magnitude(c))
        else:
            state["frequencies"] = _frequencies(c)
    elif c["op"] == "scores":
        z = normal(c["rows"], c["cols"]) * (1 + 2 * torch.rand(c["rows"], 1, generator=g, **dev))
        state["ids"] = torch.randint(0, c["cols"], (c["rows"],), generator=g, **dev)
        if c["masked"]:
            # a quarter of the tokens is forbidden, and the given one is not
            z[:, torch.rand(c["cols"], generator=g, **dev) < 0.25] = -math.inf
            z[torch.arange(c["rows"], **dev), state["ids"]] = 2.0
        state["logits"] = z.to(TYPES[c["type"]])
    else:
        state.update(_prepare_cache(c, g, normal))
    return state


def _prepare_cache(c, g, normal):
    page, heads, dim, block = c["page"], c["kv_heads"], c["dim"], c["block"]
    fanout = c.get("fanout", 0)
    lengths = _lengths(c["seqs"], c["longest"], c.get("empty", 0))
    live = _pages_of(lengths, page)
    # room for the forks' own pages: the copied one and one more where the new token opens it
    total = live + 2 * c["seqs"] * fanout + 7
    order = torch.randperm(len(lengths), generator=g, device="cuda")
    length = torch.tensor(lengths, dtype=torch.int32, device="cuda")[order]
    width = -(-c["longest"] // page) + (1 if fanout else 0)
    # pages were taken and given back for a while: a sequence's pages lie anywhere in the pool
    place = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    count = (length + page - 1) // page
    first = torch.cumsum(count, 0) - count
    column = torch.arange(width, device="cuda")
    index = first[:, None] + column[None]
    table = torch.where(column[None] < count[:, None], place[index.clamp(max=total - 1)], torch.zeros((), dtype=torch.int32, device="cuda"))
    refs = torch.zeros(total, dtype=torch.int32, device="cuda")
    refs[place[:live].long()] = 1
    forks = c["seqs"] * fanout
    channel = torch.exp(0.5 * normal(heads, dim))                # some channels are larger than others
    sides = {}
    for side in ("k", "v"):
        codes = torch.empty(total, page, heads, dim, dtype=E4M3, device="cuda")
        scales = torch.empty(total, heads, page // block, device="cuda")
        for at in range(0, total, 1 << 12):
            x = (normal(min(total - at, 1 << 12), page, heads, dim) * channel).unflatten(1, (page // block, block))
            scale = _scale_for(x.abs().amax((2, 4)))
            codes[at:at + (1 << 12)] = (x / scale[:, :, None, :, None]).flatten(1, 2).to(E4M3)
            scales[at:at + (1 << 12)] = scale.transpose(1, 2)
        sides[side + "_pages"], sides[side + "_scales"] = codes, scales
    state = {
        **sides,
        "table": torch.cat([table, torch.zeros(forks, width, dtype=torch.int32, device="cuda")]).contiguous(),
        "lengths": torch.cat([length, torch.zeros(forks, dtype=torch.int32, device="cuda")]).contiguous(),
        "refs": refs,
    }
    dtype = TYPES[c["type"]]

    def fresh(n):
        # keys and values as a product leaves them, behind as many queries
        qkv = (normal(n, 3 * heads, dim) * channel.repeat(3, 1)).to(dtype)
        return {"k_new": qkv[:, heads:2 * heads], "v_new": qkv[:, 2 * heads:]}

    def offsets():
        return torch.nn.functional.pad(torch.cumsum(length, 0), (1, 0)).to(torch.int32)
    if c["op"] == "attn":
        state["queries"] = normal(c["seqs"], c["heads"], dim).to(dtype)
    elif c["op"] == "beams":
        state["src"] = torch.arange(c["seqs"], dtype=torch.int32, device="cuda").repeat_interleave(fanout)
        state["dst"] = torch.arange(c["seqs"], c["seqs"] + forks, dtype=torch.int32, device="cuda")
        state.update(fresh(forks))
    elif c["op"] == "read":
        state["starts"], state["tokens"] = offsets(), sum(lengths)
    else:
        # a pool that others have used: what they left in pages and scales is still there
        state["starts"], state["seqs"] = offsets(), torch.arange(c["seqs"], dtype=torch.int32, device="cuda")
        state["table"].zero_(), state["lengths"].zero_(), state["refs"].zero_()
        state.update(fresh(sum(lengths)))
    if own:
        from msnhnet_b200 import tokens
        state["ops"] = _token_ops()
        state["cache"] = tokens.PagedCache(state["k_pages"], state["v_pages"], state["table"], state["lengths"], state["refs"], state["k_scales"], state["v_scales"])
    return state


def run(state):
    c = state["case"]
    return (_run_own if own else _run_plain)[c["op"]](state, c)


# ---- the framework's operators --------------------------------------------------------------------------------------

def _own_rotary(s, c):
    return s["ops"].rotary(s["x"], s["positions"], s["table"])


def _own_write(s, c):
    s["ops"].kv_append(s["cache"], s["k_new"], s["v_new"], starts=s["starts"])
    s["ops"].kv_free(s["cache"], s["seqs"])
    return s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["table"], s["lengths"], s["refs"]


def _own_beams(s, c):
    ops, cache = s["ops"], s["cache"]
    ops.kv_fork(cache, s["src"], s["dst"])
    ops.kv_append(cache, s["k_new"], s["v_new"], seqs=s["dst"])
    ops.kv_free(cache, s["dst"])
    return s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["table"], s["lengths"], s["refs"]


def _own_read(s, c):
    return s["ops"].kv_read(s["cache"], s["starts"], s["tokens"], dtype=TYPES[c["type"]])


def _own_attn(s, c):
    return s["ops"].attn_decode(s["queries"], s["cache"], window=c["window"])


def _own_scores(s, c):
    return tuple(t for t in s["ops"].token_scores(s["logits"], s["ids"], top=c["top"]) if t is not None)


_run_own = {"rotary": _own_rotary, "write": _own_write, "beams": _own_beams, "read": _own_read, "attn": _own_attn, "scores": _own_scores}


# ---- their plain forms ----------------------------------------------------------------------------------------------

def _frequencies(c):
    """Radians a position of each plane, in 64 bits."""
    i = torch.arange(c["rot"] // 2, dtype=torch.float64, device="cuda")
    base = BASE
    if c["stretch"] == "base":
        base = BASE * c["factor"] ** (c["rot"] / max(c["rot"] - 2, 1))
    f = base ** (-2 * i / c["rot"])
    if c["stretch"] == "all":
        f = f / c["factor"]
    if c["stretch"] == "slow":
        # planes that turn LOW times or less within what a model was trained on are slowed down, those that turn HIGH times or more are not
        keep = ((TRAINED * f / (2 * math.pi) - LOW) / (HIGH - LOW)).clamp(0, 1)
        f = f * (keep + (1 - keep) / c["factor"])
    return f


def _plain_rotary(s, c):
    x, half = s["x"].float(), c["rot"] // 2
    angle = s["positions"].double()[:, None, None] * s["frequencies"]
    cos, sin = (torch.cos(angle) * _magnitude(c)).float(), (torch.sin(angle) * _magnitude(c)).float()
    turned = x[..., :c["rot"]]
    if c["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, x[..., c["rot"]:]], -1).to(s["x"].dtype)


def _scale_for(top):
    """The smallest power of two that takes values of up to `top` to 448 at most; 0 for 0."""
    m, e = torch.frexp(top)
    e = (e - 9 + (m > 0.875).int()).clamp(min=-126)
    return torch.where(top > 0, ((e + 127) << 23).view(torch.float32), torch.zeros_like(top))


def _codes(x, scale):
    return torch.where(scale > 0, x / scale, torch.zeros_like(x)).to(E4M3)


def _plain_write(s, c):
    table, lengths, refs, starts = s["table"], s["lengths"], s["refs"], s["starts"].long()
    page, block, heads = c["page"], c["block"], c["kv_heads"]
    counts = starts[1:] - starts[:-1]
    need = (counts + page - 1) // page
    first = torch.cumsum(need, 0) - need
    free = torch.argsort((refs != 0).int(), stable=True)
    column = torch.arange(table.shape[1], device="cuda")
    rows = free[(first[:, None] + column[None]).clamp(max=refs.shape[0] - 1)]
    table.copy_(torch.where(column[None] < need[:, None], rows.to(table.dtype), table))
    token = torch.arange(s["k_new"].shape[0], device="cuda")
    seq = torch.searchsorted(starts[1:], token, right=True)
    at = token - starts[seq]
    where, place = table[seq, at // page].long(), at % page
    for side in ("k", "v"):
        x, scales = s[side + "_new"].float(), s[side + "_scales"]
        flat = (where[:, None] * heads + torch.arange(heads, device="cuda")) * scales.shape[2] + (place // block)[:, None]
        top = torch.zeros(scales.numel(), device="cuda").scatter_reduce(0, flat.flatten(), x.abs().amax(-1).flatten(), "amax")
        scale = _scale_for(top)[flat]
        scales.view(-1)[flat] = scale
        s[side + "_pages"].view(torch.uint8)[where, place] = _codes(x, scale[..., None]).view(torch.uint8)
    # the sequences are given up: pages taken are free again
    lengths.zero_()
    return s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], table, lengths, refs


def _plain_beams(s, c):
    table, lengths, refs = s["table"], s["lengths"], s["refs"]
    src, dst, page, block = s["src"].long(), s["dst"].long(), c["page"], c["block"]
    one = torch.ones((), dtype=refs.dtype, device="cuda")
    # fork: full pages are shared, the rows of a page that is not full go to the lowest free page, with the scales of their blocks
    length = lengths[src]
    full, rest = (length // page).long(), length % page
    free = torch.argsort((refs != 0).int(), stable=True)
    wants = rest > 0
    new = free[torch.cumsum(wants, 0) - 1]
    column = torch.arange(table.shape[1], device="cuda")
    shared = column[None] < full[:, None]
    rows = torch.where(shared, table[src], table[dst])
    last = full.clamp(max=table.shape[1] - 1)
    old = table[src, torch.where(wants, last, (full - 1).clamp(min=0))].long()
    rows = torch.where(wants[:, None] & (column[None] == last[:, None]), new[:, None].to(table.dtype), rows)
    table[dst] = rows
    refs.index_add_(0, torch.where(shared, rows, torch.zeros_like(rows)).reshape(-1).long(), shared.reshape(-1).to(refs.dtype))
    refs.index_add_(0, new, wants.to(refs.dtype))
    keep = (torch.arange(page, device="cuda")[None] < rest[:, None])[..., None, None]
    blocks = torch.arange(page // block, device="cuda")
    held = (blocks[None] * block < rest[:, None])[:, None]
    # (a fork with nothing to copy writes its parent's page back to where it is)
    to = torch.where(wants, new, old)
    for side in ("k", "v"):
        pages, scales = s[side + "_pages"].view(torch.uint8), s[side + "_scales"]
        pages[to] = torch.where(keep, pages[old], pages[to])
        scales[to] = torch.where(held, scales[old], scales[to])
    lengths[dst] = length
    # append: one token each; a page is opened where the last one is full
    opens = rest == 0
    free = torch.argsort((refs != 0).int(), stable=True)
    opened = free[torch.cumsum(opens, 0) - 1]
    table[dst, full] = torch.where(opens, opened.to(table.dtype), table[dst, full])
    refs.index_add_(0, opened, opens.to(refs.dtype))
    at, mine = table[dst, full].long(), (rest // block).long()
    place = mine[:, None] * block + torch.arange(block, device="cuda")[None]
    before = rest % block
    for side in ("k", "v"):
        x, pages, scales = s[side + "_new"].float(), s[side + "_pages"].view(torch.uint8), s[side + "_scales"]
        was = torch.where((before > 0)[:, None], scales[at, :, mine], torch.zeros((), device="cuda"))
        now = torch.maximum(was, _scale_for(x.abs().amax(-1)))
        # the block's older codes by the new scale, the token's own behind them
        codes = pages[at[:, None], place]
        again = _codes(codes.view(E4M3).float() * was[:, None, :, None], now[:, None, :, None]).view(torch.uint8)
        i = torch.arange(block, device="cuda")[None, :, None, None]
        behind = before[:, None, None, None]
        pages[at[:, None], place] = torch.where(i < behind, again, torch.where(i == behind, _codes(x, now[..., None]).view(torch.uint8)[:, None], codes))
        scales[at, :, mine] = now
    lengths[dst] = length + 1
    # free
    held = column[None] < (full + 1)[:, None]
    mine = table[dst]
    refs.index_add_(0, torch.where(held, mine, torch.zeros_like(mine)).reshape(-1).long(), -one * held.reshape(-1).to(refs.dtype))
    lengths[dst] = 0
    return s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], table, lengths, refs


def _values(s, side, pages, place, block):
    """Keys or values at places of pages, in 32 bits."""
    x = s[side + "_pages"].view(torch.uint8)[pages, place].view(E4M3).float()
    return x * s[side + "_scales"][pages, :, place // block][..., None]


def _plain_read(s, c):
    starts = s["starts"].long()
    token = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(starts[1:], token, right=True)
    at = token - starts[seq]
    pages, place = s["table"][seq, at // c["page"]].long(), at % c["page"]
    return tuple(_values(s, side, pages, place, c["block"]).to(TYPES[c["type"]]) for side in ("k", "v"))


def _plain_attn(s, c):
    b, hk, d = c["seqs"], c["kv_heads"], c["dim"]
    at = s["table"].long()[:, :, None]
    place = torch.arange(c["page"], device="cuda")[None, None]
    k = _values(s, "k", at, place, c["block"]).reshape(b, -1, hk, d)
    v = _values(s, "v", at, place, c["block"]).reshape(b, -1, hk, d)
    q = s["queries"].float().reshape(b, hk, -1, d)
    z = torch.matmul(q, k.permute(0, 2, 3, 1)) * (d ** -0.5)                            # sequence, kv head, query head, position
    position = torch.arange(k.shape[1], device="cuda")
    length = s["lengths"][:, None]
    seen = position < length
    if c["window"]:
        seen &= position >= length - c["window"]
    z = z.masked_fill(~seen[:, None, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    return torch.matmul(p, v.permute(0, 2, 1, 3)).reshape(b, -1, d).to(s["queries"].dtype)


def _plain_scores(s, c):
    z = s["logits"].float()
    top = z.amax(-1, keepdim=True)
    d = z - top
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    log_p = d - torch.log(total)
    entropy = -(torch.where(e > 0, log_p, torch.zeros_like(log_p)) * e).sum(-1) / total[:, 0]
    given = log_p.gather(1, s["ids"][:, None])[:, 0]
    if not c["top"]:
        return given, entropy
    # keys in the numbers' order, the lowest column first among equal ones
    bits = (z + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    keys = (order << 32) | (c["cols"] - 1 - torch.arange(c["cols"], device="cuda"))
    ids = c["cols"] - 1 - (torch.topk(keys, c["top"], -1).values & 0xffffffff)
    return given, entropy, log_p.gather(1, ids), ids


_run_plain = {"rotary": _plain_rotary, "write": _plain_write, "beams": _plain_beams, "read": _plain_read, "attn": _plain_attn, "scores": _plain_scores}


# ---- from the definitions, in 64 bits -------------------------------------------------------------------------------

def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return {"rotary": _exact_rotary, "write": _exact_write, "beams": _exact_beams, "read": _exact_read, "attn": _exact_attn, "scores": _exact_scores}[case["op"]](s, case)


def _exact_rotary(s, c):
    f = []
    for i in range(c["rot"] // 2):
        base = BASE if c["stretch"] != "base" else BASE * c["factor"] ** (c["rot"] / max(c["rot"] - 2, 1))
        one = base ** (-2 * i / c["rot"])
        if c["stretch"] == "all":
            one /= c["factor"]
        if c["stretch"] == "slow":
            turns = TRAINED * one / (2 * math.pi)
            share = min(max((turns - LOW) / (HIGH - LOW), 0.0), 1.0)
            one = share * one + (1 - share) * one / c["factor"]
        f.append(one)
    angle = torch.outer(s["positions"].double(), torch.tensor(f, dtype=torch.float64, device="cuda"))
    turn = torch.polar(torch.full_like(angle, _magnitude(c)), angle)[:, None]
    y = s["x"].double()
    if c["interleaved"]:
        y[..., :c["rot"]] = torch.view_as_real(torch.view_as_complex(y[..., :c["rot"]].reshape(*y.shape[:2], -1, 2).contiguous()) * turn).flatten(-2)
    else:
        z = torch.complex(y[..., :c["rot"] // 2], y[..., c["rot"] // 2:c["rot"]]) * turn
        y = torch.cat([z.real, z.imag, y[..., c["rot"]:]], -1)
    return y


def _round_e4m3(z):
    """Three bits behind the leading one, down to 2^-9 in the lowest binade; halves to even."""
    step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(z / step) * step


def _power(top):
    """The scale of a block whose largest value is `top`, by trying powers of two around its logarithm."""
    scale = torch.zeros_like(top)
    guess = torch.floor(torch.log2(top.clamp(min=1e-300) / 448))
    for more in (3, 2, 1, 0, -1):
        p = torch.exp2((guess + more).clamp(min=-126))
        scale = torch.where((top > 0) & (top <= 448 * p), p, scale)
    return scale


def _put(codes, scales, page, first, rows, block):
    """Token by token groups: rows [n, heads, dim] from place `first` on of one page, as one call writes them."""
    n = rows.shape[0]
    for b in range(first // block, (first + n - 1) // block + 1):
        lo, hi = max(first, b * block), min(first + n, (b + 1) * block)
        mine = rows[lo - first:hi - first]
        was = scales[page, :, b] if lo > b * block else torch.zeros(rows.shape[1], dtype=torch.float64, device="cuda")
        now = torch.maximum(was, _power(mine.abs().amax((0, 2))))
        by = now.clamp(min=1e-300)[:, None]
        codes[page, b * block:lo] = _round_e4m3(codes[page, b * block:lo] * was[:, None] / by)
        codes[page, lo:hi] = _round_e4m3(mine / by)
        scales[page, :, b] = now


def _exact_write(s, c):
    codes = {side: s[side + "_pages"].double() for side in "kv"}
    scales = {side: s[side + "_scales"].double() for side in "kv"}
    table, taken = s["table"].tolist(), 0
    starts = s["starts"].tolist()
    for i, (a, b) in enumerate(zip(starts, starts[1:])):
        n_pages = -(-(b - a) // c["page"])
        table[i][:n_pages] = range(taken, taken + n_pages)
        taken += n_pages
    # whole pages of all sequences together, block by block; the ragged last ones each by itself
    for side in "kv":
        rows = s[side + "_new"].double()
        page = 0
        for a, b in zip(starts, starts[1:]):
            whole = (b - a) // c["page"]
            if whole:
                x = rows[a:a + whole * c["page"]].reshape(whole, c["page"] // c["block"], c["block"], *rows.shape[1:])
                now = _power(x.abs().amax((2, 4)))
                codes[side][page:page + whole] = _round_e4m3(x / now.clamp(min=1e-300)[:, :, None, :, None]).flatten(1, 2)
                scales[side][page:page + whole] = now.transpose(1, 2)
            if (b - a) % c["page"]:
                _put(codes[side], scales[side], page + whole, 0, rows[a + whole * c["page"]:b], c["block"])
            page += -(-(b - a) // c["page"])
    return codes["k"], codes["v"], scales["k"], scales["v"], torch.tensor(table, dtype=torch.int32), s["lengths"], s["refs"]


def _exact_beams(s, c):
    """The upkeep page by page."""
    page, block = c["page"], c["block"]
    codes = {side: s[side + "_pages"].double() for side in "kv"}
    scales = {side: s[side + "_scales"].double() for side in "kv"}
    table, lengths, refs = s["table"].tolist(), s["lengths"].tolist(), s["refs"].tolist()
    free = [i for i, r in enumerate(refs) if not r]
    taken = 0
    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
        n = lengths[a]
        table[b][:n // page] = table[a][:n // page]
        lengths[b] = n
        if n % page:
            old, new, taken = table[a][n // page], free[taken], taken + 1
            table[b][n // page] = new
            some = -(-(n % page) // block)
            for side in "kv":
                codes[side][new, :n % page] = codes[side][old, :n % page]
                scales[side][new, :, :some] = scales[side][old, :, :some]
    for i, b in enumerate(s["dst"].tolist()):
        n = lengths[b]
        if n % page == 0:
            table[b][n // page], taken = free[taken], taken + 1
        for side in "kv":
            _put(codes[side], scales[side], table[b][n // page], n % page, s[side + "_new"][i:i + 1].double(), block)
        lengths[b] = 0
    return codes["k"], codes["v"], scales["k"], scales["v"], torch.tensor(table, dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32), s["refs"]


def _sequence(s, c, i, side):
    """All keys or values of a sequence, in 64 bits."""
    n = int(s["lengths"][i])
    pages = s["table"][i, :-(-n // c["page"])].long()
    x = s[side + "_pages"].view(torch.uint8)[pages].view(E4M3).double()
    scale = s[side + "_scales"][pages].double().transpose(1, 2).repeat_interleave(c["block"], 1)
    return (x * scale[..., None]).flatten(0, 1)[:n]


def _exact_read(s, c):
    return tuple(torch.cat([_sequence(s, c, i, side) for i in range(c["seqs"])]) for side in "kv")


def _exact_attn(s, c):
    out = torch.zeros(c["seqs"], c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    each = c["heads"] // c["kv_heads"]
    for i, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        first = max(0, n - c["window"]) if c["window"] else 0
        k, v = _sequence(s, c, i, "k")[first:], _sequence(s, c, i, "v")[first:]
        for h in range(c["kv_heads"]):
            q = s["queries"][i, h * each:(h + 1) * each].double()
            out[i, h * each:(h + 1) * each] = torch.softmax(q @ k[:, h].T / math.sqrt(c["dim"]), -1) @ v[:, h]
    return out


def _exact_scores(s, c):
    given, entropy, values, ids = [], [], [], []
    some = max(1, 20_000_000 // c["cols"])
    for at in range(0, c["rows"], some):
        z = s["logits"][at:at + some].double()
        log_p = torch.log_softmax(z, -1)
        p = torch.exp(log_p)
        given.append(log_p.gather(1, s["ids"][at:at + some, None])[:, 0])
        entropy.append(-torch.special.xlogy(p, p).sum(-1))
        if c["top"]:
            order = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
            ids.append(order)
            values.append(log_p.gather(1, order))
    out = torch.cat(given), torch.cat(entropy)
    return out if not c["top"] else out + (torch.cat(values), torch.cat(ids))
