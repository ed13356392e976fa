"""Operators for decoding tokens, on torch tensors of the GPU (the C ABI's "operators for decoding tokens", include/msnh_b200.h).

    ops = TokenOps()                                     # a handle for one device, used by one host thread at a time
    y, h = ops.rms_norm(x, weight, residual=h)           # h: the sum, for the next residual
    w = ops.w4_pack(codes, scales)                       # once; then, every step:
    qkv = ops.w4_linear(y, w)
    cache = ops.new_cache(n_pages, page_size, n_kv_heads, head_dim, n_seqs, max_pages, dtype)
    ops.kv_append(cache, k, v)
    out = ops.attn_decode(q, cache)

Calls enqueue on torch's current stream of the tensors' device and do not wait; nothing here computes anything. Wrong types, shapes or
devices raise ValueError before the call, and so does a tensor that requires a gradient where torch records gradients: the operators have
none, and their results would be cut off unnoticed. What the library refuses raises _ffi.KernelError. The checks and the C call are native
(host/tokens_torch.cpp): in Python they took longer than the kernels of one token.
"""
import ctypes as C

import torch

from . import _ffi

_ffi.kernel_lib()
from . import _tokens  # noqa: E402  (needs torch's and the kernel library's symbols)

_DTYPE = {torch.float32: _ffi.F32, torch.float16: _ffi.F16, torch.bfloat16: _ffi.BF16, torch.float8_e4m3fn: _ffi.E4M3}
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


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


class PagedCache:
    """Keys and values in pages (MsnhB200KvCache), over tensors of the caller:

    k_pages, v_pages  [n_pages, page_size, n_kv_heads, head_dim] (any strides but the last), float32, float16 or bfloat16
    page_table        int32 [n_seqs, max_pages]; lengths int32 [n_seqs]; refs int32 [n_pages]; all of them 0 in a fresh cache
    """

    def __init__(self, k_pages, v_pages, page_table, lengths, refs):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype or k_pages.dtype not in _FLOATS:
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
        _no_gradient(k_pages, v_pages)
        self.device = k_pages.device
        if not k_pages.is_cuda or any(t.device != self.device for t in (v_pages, page_table, lengths, refs)):
            raise ValueError("the cache's tensors are on one GPU")
        self.k_pages, self.v_pages, self.page_table, self.lengths, self.refs = k_pages, v_pages, page_table, lengths, refs
        self.refused_count = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.tensors = k_pages, v_pages, page_table, lengths, refs, self.refused_count
        self.dtype = k_pages.dtype
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = k_pages.shape
        self.n_seqs, self.max_pages = page_table.shape
        self.args = _ffi.KvCache(k_pages.data_ptr(), v_pages.data_ptr(), *k_pages.stride()[:3], *v_pages.stride()[:3], page_table.data_ptr(),
                                 lengths.data_ptr(), refs.data_ptr(), self.refused_count.data_ptr(), page_table.stride(0), self.n_pages,
                                 self.page_size, self.n_kv_heads, self.head_dim, self.n_seqs, self.max_pages, _DTYPE[self.dtype])
        self.ref = C.byref(self.args)
        self.address = C.addressof(self.args)

    def refused(self):
        """How many sequences operations on this cache have refused so far (waits for the GPU)."""
        return int(self.refused_count)


class TokenOps:
    """The operators of one device (a context of the kernel library)."""

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

    def new_cache(self, n_pages, page_size, n_kv_heads, head_dim, n_seqs, max_pages, dtype=torch.float16):
        """A fresh cache with memory of its own."""
        pages = [torch.zeros(n_pages, page_size, n_kv_heads, head_dim, dtype=dtype, device=self.device) for _ in range(2)]
        ints = [torch.zeros(*shape, dtype=torch.int32, device=self.device) for shape in ((n_seqs, max_pages), (n_seqs,), (n_pages,))]
        return PagedCache(*pages, *ints)

    def attn_decode(self, q, cache, seqs=None, scale=None, window=0, out=None, return_lse=False):
        """One query token a row: q [rows, n_heads, head_dim] over the cached tokens of sequence seqs[row] (int32; row without seqs); its last
        `window` ones only where that is not 0. scale: 1 / sqrt(head_dim). Returns out, or (out, lse float32 [rows, n_heads])."""
        return _tokens.attn_decode(self._ctx, self._index, q, cache.address, cache.k_pages, seqs, scale, window, out, return_lse)

    def kv_append(self, cache, k, v, seqs=None, starts=None):
        """Tokens behind their sequences' own: k, v [tokens, n_kv_heads, head_dim]; one token for each of seqs (int32; without it for
        sequences 0, 1, ...), or rows starts[i] to starts[i + 1] (int32, one more than sequences) for sequence seqs[i]."""
        _tokens.kv_append(self._ctx, self._index, cache.address, cache.k_pages, cache.tensors, k, v, seqs, starts)

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
