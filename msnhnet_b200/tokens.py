"""Operators for decoding tokens, on torch tensors of the GPU (the C ABI's "operators for decoding tokens", include/msnh_b200.h).

    ops = TokenOps()                                     # a handle for one device, used by one host thread at a time
    y, h = ops.rms_norm(x, weight, residual=h)           # h: the sum, for the next residual
    w = ops.w4_pack(codes, scales)                       # once; then, every step:
    qkv = ops.w4_linear(y, w)
    cache = ops.new_cache(n_pages, page_size, n_kv_heads, head_dim, n_seqs, max_pages, dtype)     # float8_e4m3fn: half the memory
    ops.rotary(x, positions, table, out=x)               # queries and keys by their positions; table = ops.rotary_table(head_dim)
    ops.kv_append(cache, k, v)
    out = ops.attn_decode(q, cache)
    logprob, entropy, best, ids = ops.token_scores(logits, top=5)

Calls enqueue on torch's current stream of the tensors' device and do not wait; nothing here computes anything. Wrong types, shapes or
devices raise ValueError before the call, and so does a tensor that requires a gradient where torch records gradients: the operators have
none, and their results would be cut off unnoticed. What the library refuses raises _ffi.KernelError. The checks and the C call are native
(host/tokens_torch.cpp): in Python they took longer than the kernels of one token.
"""
import ctypes as C
import decimal
import math

import torch

from . import _ffi

_ffi.kernel_lib()
from . import _tokens  # noqa: E402  (needs torch's and the kernel library's symbols)

_DTYPE = {torch.float32: _ffi.F32, torch.float16: _ffi.F16, torch.bfloat16: _ffi.BF16, torch.float8_e4m3fn: _ffi.E4M3}
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
# (rotary tables: a fraction of 64 bits takes more than a float's 53)
_TWO_PI = decimal.Decimal("6.28318530717958647692528676655900576839433879875021164194989")


def _no_gradient(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("a tensor requires a gradient, and these operators have none (torch.no_grad() takes it as it is)")


class W4Weights:
    """4-bit weights as the kernels read them (TokenOps.w4_pack): [n, k] with a scale for every `group` values of a row."""

    def __init__(self, packed, n, k, group, scale_dtype, has_zeros):
        self.packed, self.n, self.k, self.group = packed, n, k, group
        self.args = _ffi.W4(packed.data_ptr() if packed is not None else None, n, k, group, _DTYPE[scale_dtype], int(has_zeros))
        self.ref = C.byref(self.args)
        self.address = C.addressof(self.args)


class RotaryTable:
    """What TokenOps.rotary turns by (TokenOps.rotary_table): `turns`, the whole turns a position of each plane as 64-bit fractions (int64 on the
    GPU; the nearest ones: off by 2^-65 of a turn, times the position for an angle), whether planes are interleaved, and the factor of what is turned."""

    def __init__(self, turns, interleaved, magnitude):
        self.turns, self.interleaved, self.magnitude = turns, interleaved, magnitude


class PagedCache:
    """Keys and values in pages (MsnhB200KvCache), over tensors of the caller:

    k_pages, v_pages  [n_pages, page_size, n_kv_heads, head_dim] (any strides but the last), float32, float16, bfloat16 or float8_e4m3fn
    page_table        int32 [n_seqs, max_pages]; lengths int32 [n_seqs]; refs int32 [n_pages]; all of them 0 in a fresh cache
    k_scales, v_scales  for pages of float8_e4m3fn: float32 [n_pages, n_kv_heads, page_size / scale_block], what a code of a block of
                      scale_block tokens of a page and head is taken times
    """

    def __init__(self, k_pages, v_pages, page_table, lengths, refs, k_scales=None, v_scales=None):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype or k_pages.dtype not in _DTYPE:
            raise ValueError("k_pages and v_pages: [n_pages, page_size, n_kv_heads, head_dim] of one floating type")
        if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
            raise ValueError("k_pages and v_pages: the values of a head lie side by side")
        if page_table.dim() != 2 or page_table.stride(1) != 1 or lengths.shape != page_table.shape[:1] or refs.shape != k_pages.shape[:1]:
            raise ValueError("page_table [n_seqs, max_pages], lengths [n_seqs], refs [n_pages]")
        for t in (page_table, lengths, refs):
            if t.dtype != torch.int32:
                raise ValueError("page_table, lengths and refs are int32")
        if not lengths.is_contiguous() or not refs.is_contiguous():
            raise ValueError("lengths and refs are contiguous")
        scales = (k_scales, v_scales)
        self.scale_block = 0
        if k_pages.dtype not in _FLOATS:
            n_pages, page_size, heads, _ = k_pages.shape
            if any(t is None or t.dim() != 3 or t.shape[:2] != (n_pages, heads) or t.shape != k_scales.shape or t.dtype != torch.float32 or not t.is_contiguous() for t in scales):
                raise ValueError("k_scales and v_scales: contiguous float32 [n_pages, n_kv_heads, blocks of a page] beside 8-bit pages")
            blocks = k_scales.shape[2]
            if blocks < 1 or page_size % blocks:
                raise ValueError(f"k_scales and v_scales: {blocks} blocks in pages of {page_size} tokens")
            self.scale_block = page_size // blocks
        elif any(t is not None for t in scales):
            raise ValueError("k_scales and v_scales are of 8-bit pages")
        scales = tuple(t for t in scales if t is not None)
        _no_gradient(k_pages, v_pages, *scales)
        self.device = k_pages.device
        if not k_pages.is_cuda or any(t.device != self.device for t in (v_pages, page_table, lengths, refs, *scales)):
            raise ValueError("the cache's tensors are on one GPU")
        self.k_pages, self.v_pages, self.page_table, self.lengths, self.refs = k_pages, v_pages, page_table, lengths, refs
        self.k_scales, self.v_scales = k_scales, v_scales
        self.refused_count = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.tensors = k_pages, v_pages, page_table, lengths, refs, self.refused_count, *scales
        self.dtype = k_pages.dtype
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = k_pages.shape
        self.n_seqs, self.max_pages = page_table.shape
        self.args = _ffi.KvCache(k_pages.data_ptr(), v_pages.data_ptr(), *k_pages.stride()[:3], *v_pages.stride()[:3], page_table.data_ptr(),
                                 lengths.data_ptr(), refs.data_ptr(), self.refused_count.data_ptr(), page_table.stride(0), self.n_pages,
                                 self.page_size, self.n_kv_heads, self.head_dim, self.n_seqs, self.max_pages, _DTYPE[self.dtype],
                                 *((k_scales.data_ptr(), v_scales.data_ptr(), self.scale_block) if scales else (None, None, 0)))
        self.ref = C.byref(self.args)
        self.address = C.addressof(self.args)

    def refused(self):
        """How many sequences operations on this cache have refused so far (waits for the GPU)."""
        return int(self.refused_count)


class TokenOps:
    """The operators of one device (a context of the kernel library)."""

    MAX_TOP = 32                             # of token_scores

    def __init__(self, device=None):
        self.device = torch.device("cuda", torch.cuda.current_device() if device is None else device)
        self.ctx = _ffi.Context(self.device.index)
        self.lib, self.h = self.ctx.lib, self.ctx.h
        self._index, self._ctx = self.device.index, self.h.value

    def close(self):
        self.ctx.close()
        self.h, self._ctx = None, 0

    def rms_norm(self, x, weight, eps=1e-6, residual=None, out_dtype=None, residual_out=None, out=None):
        """(y, h) with a residual, y without one; with out_dtype float8_e4m3fn (y, scale of each row, h) and (y, scale).

        x [rows, cols]; residual, residual_out: the same type and shape (residual_out may be residual: added in place). weight: [cols] of
        x's type or float32."""
        return _tokens.rms_norm(self._ctx, self._index, x, weight, eps, residual, out_dtype, residual_out, out)

    def w4_pack(self, codes, scales, zeros=None, k=None, group=128):
        """Lays weights out for w4_linear: codes uint8 [n, ceil(k / 2)] (value 2i in the low half of byte i), scales [n, ceil(k / group)],
        zeros uint8 of the same shape or None (zero point 8)."""
        if codes.dim() != 2 or codes.dtype != torch.uint8 or codes.stride(1) != 1:
            raise ValueError("codes: uint8 [n, ceil(k / 2)]")
        n = codes.shape[0]
        k = 2 * codes.shape[1] if k is None else k
        groups = -(-k // group)
        if codes.shape[1] != (k + 1) // 2 or scales.shape != (n, groups) or scales.dtype not in _FLOATS or not scales.is_contiguous():
            raise ValueError(f"codes [n, {(k + 1) // 2}] and scales [n, {groups}] are wanted for k = {k} in groups of {group}")
        if zeros is not None and (zeros.shape != scales.shape or zeros.dtype != torch.uint8 or not zeros.is_contiguous()):
            raise ValueError("zeros: uint8, the scales' shape")
        for t in (codes, scales, zeros):
            if t is not None and t.device != self.device:
                raise ValueError(f"a tensor on {t.device} in a call of {self.device}")
        _no_gradient(scales)
        w = W4Weights(None, n, k, group, scales.dtype, zeros is not None)
        size = C.c_size_t()
        self.ctx.check(self.lib.msnh_b200_w4_pack_bytes(self.h, w.ref, C.byref(size)))
        w.packed = torch.empty(size.value, dtype=torch.uint8, device=self.device)
        w.args.packed = w.packed.data_ptr()
        self.ctx.check(self.lib.msnh_b200_w4_pack(self.h, w.ref, codes.data_ptr(), codes.stride(0), scales.data_ptr(), zeros.data_ptr() if zeros is not None else None,
                                                  w.packed.data_ptr(), torch.cuda.current_stream(self.device).cuda_stream))
        return w

    def w4_linear(self, x, weights, bias=None, x_scale=None, out_dtype=None, out=None):
        """x [rows, k] times the weights' transpose: [rows, n], at most 64 rows. x of float8_e4m3fn gives float16 unless out_dtype says
        otherwise; x_scale: float32 [rows]; bias: float32 [n]."""
        return _tokens.w4_linear(self._ctx, self._index, x, weights.address, weights.packed, bias, x_scale, out_dtype, out)

    def rotary_table(self, dim, base=10000.0, interleaved=False, stretch=None, factor=1.0, trained=8192, low=1.0, high=4.0, magnitude=1.0):
        """Frequencies for rotary: the first `dim` values of a head are turned, plane i by base ** (-2 i / dim) radians a position; planes are
        the values (i, i + dim / 2) or, interleaved, (2i, 2i + 1). What is turned is taken times `magnitude`.

        For texts `factor` times as long as the `trained` positions a model knows, stretch slows planes down: "all" of them by the factor; by a
        larger "base" (base * factor ** (dim / (dim - 2)): the slowest plane by the factor, the fastest not at all); or "slow" ones: those that
        turn `low` times or less within the trained positions by the factor, those that turn `high` times or more not, in between a mixture."""
        if dim < 2 or dim % 2 or not base > 0 or not factor > 0 or not high > low or trained < 1:
            raise ValueError(f"rotary_table: dim {dim} (even, 2 at least), base {base}, factor {factor}, {low} to {high} turns of {trained} positions")
        if stretch not in (None, "all", "base", "slow"):
            raise ValueError(f"stretch {stretch!r}: None, 'all', 'base' or 'slow'")
        turns = []
        # (without traps: infinite bases and factors are what they are in floats)
        with decimal.localcontext(decimal.Context(prec=40, traps=[])) as numbers:
            base, factor, trained, low, high, dim = (decimal.Decimal(float(v)) for v in (base, factor, trained, low, high, dim))
            if stretch == "base":
                base = base * factor ** (dim / max(dim - 2, 1))
            # bases and factors below 1 give whole turns, whose digits come in front of the fraction's
            numbers.prec += max(-base.adjusted(), 0) + max(-factor.adjusted(), 0)
            ratio, plane = (base.ln() * -2 / dim).exp(), 1 / _TWO_PI
            for _ in range(int(dim) // 2):
                turn = plane
                plane *= ratio
                if stretch == "all":
                    turn /= factor
                elif stretch == "slow":
                    kept = min(max((trained * turn - low) / (high - low), 0), 1)
                    turn *= kept + (1 - kept) / factor
                turns.append((int((turn * 2 ** 64).to_integral_value()) + 2 ** 63) % 2 ** 64 - 2 ** 63)
        return RotaryTable(torch.tensor(turns, dtype=torch.int64, device=self.device), bool(interleaved), float(magnitude))

    def rotary(self, x, positions, table, out=None):
        """Turns the heads of x [tokens, heads, head_dim] (queries and keys side by side, if you like) by positions [tokens] (int32 or int64, of any
        size and sign) and a table of rotary_table. out may be x: turned in place."""
        return _tokens.rotary(self._ctx, self._index, x, positions, table.turns, table.interleaved, table.magnitude, out)

    def token_scores(self, logits, ids=None, top=0):
        """(logprob, entropy, top_logprobs, top_ids) of softmax(logits), for rows of logits; what is not asked for is None.

        logprob: float32 [rows], of the tokens ids (int64 [rows]; NaN where one is none). entropy: float32 [rows]. top_logprobs, top_ids:
        float32 and int64 [rows, top], the likeliest tokens (at most 32), the lowest id first among equal ones. A row that is no distribution
        (a NaN, +infinity, or only -infinity) has NaN throughout, and ids of -1."""
        return _tokens.token_scores(self._ctx, self._index, logits, ids, top)

    def new_cache(self, n_pages, page_size, n_kv_heads, head_dim, n_seqs, max_pages, dtype=torch.float16, scale_block=None):
        """A fresh cache with memory of its own. dtype float8_e4m3fn: half the memory, with a scale for each scale_block tokens of a page and head
        (a divisor of page_size; without it the largest one of 16 that is)."""
        if dtype == torch.float8_e4m3fn:
            scale_block = math.gcd(16, page_size) if scale_block is None else scale_block
            if scale_block < 1 or page_size % scale_block:
                raise ValueError(f"scales of {scale_block} tokens in pages of {page_size}")
        elif scale_block is not None:
            raise ValueError("scale_block is of 8-bit pages")
        pages = [torch.zeros(n_pages, page_size, n_kv_heads, head_dim, dtype=dtype, device=self.device) for _ in range(2)]
        ints = [torch.zeros(*shape, dtype=torch.int32, device=self.device) for shape in ((n_seqs, max_pages), (n_seqs,), (n_pages,))]
        if dtype != torch.float8_e4m3fn:
            return PagedCache(*pages, *ints)
        return PagedCache(*pages, *ints, *(torch.zeros(n_pages, n_kv_heads, page_size // scale_block, device=self.device) for _ in range(2)))

    def attn_decode(self, q, cache, seqs=None, scale=None, window=0, out=None, return_lse=False):
        """One query token a row: q [rows, n_heads, head_dim] over the cached tokens of sequence seqs[row] (int32; row without seqs); its last
        `window` ones only where that is not 0. scale: 1 / sqrt(head_dim). Returns out, or (out, lse float32 [rows, n_heads]). q has the cache's
        type; over 8 bits it may have any floating one, and out is of the same."""
        return _tokens.attn_decode(self._ctx, self._index, q, cache.address, cache.k_pages, seqs, scale, window, out, return_lse)

    def kv_append(self, cache, k, v, seqs=None, starts=None):
        """Tokens behind their sequences' own: k, v [tokens, n_kv_heads, head_dim]; one token for each of seqs (int32; without it for
        sequences 0, 1, ...), or rows starts[i] to starts[i + 1] (int32, one more than sequences) for sequence seqs[i]. k and v have the cache's
        type; for 8 bits any floating one: they are quantised, by the smallest power of two that brings the values of a block of tokens and head
        to 448 at most. A block that was begun keeps its scale, or takes a larger one with its older codes rounded again."""
        _tokens.kv_append(self._ctx, self._index, cache.address, cache.k_pages, cache.tensors, k, v, seqs, starts)

    def kv_read(self, cache, starts, tokens, seqs=None, first=None, dtype=None, out=None):
        """Keys and values as the cache holds them, (k, v) [tokens, n_kv_heads, head_dim]: rows starts[i] to starts[i + 1] (int32, one more than
        sequences) are those of sequence seqs[i] (int32; i without it) from its token first[i] (int32; 0 without it) on. Rows of no sequence or
        token are 0. dtype: the cache's, float16 for 8 bits (what is beyond a type's range is infinite); out: (k, v) to write into."""
        k, v = (None, None) if out is None else out
        return _tokens.kv_read(self._ctx, self._index, cache.address, cache.k_pages, starts, tokens, seqs, first, dtype, k, v)

    def kv_fork(self, cache, src, dst):
        """Sequences dst (int32, empty before) become copies of sequences src."""
        _tokens.kv_fork(self._ctx, self._index, cache.address, cache.k_pages, cache.tensors, src, dst)

    def kv_free(self, cache, seqs):
        """Sequences seqs (int32) give their pages back."""
        _tokens.kv_free(self._ctx, self._index, cache.address, cache.k_pages, cache.tensors, seqs)

    def kv_compact(self, cache, table_out=None, refs_out=None):
        """Moves live pages together: afterwards they are the first ones. table_out, refs_out: where the new table and counts go
        (the cache's own without them)."""
        _tokens.kv_compact(self._ctx, self._index, cache.address, cache.page_table, cache.tensors, cache.page_table if table_out is None else table_out,
                           cache.refs if refs_out is None else refs_out)

    def kv_copy_pages(self, cache, src, dst):
        """Contents of pages src (int32) to pages dst."""
        _tokens.kv_copy_pages(self._ctx, self._index, cache.address, cache.k_pages, cache.tensors, src, dst)
