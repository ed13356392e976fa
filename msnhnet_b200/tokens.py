"""Operators for decoding tokens, on torch tensors of the GPU (the C ABI's "operators for decoding tokens", include/msnh_b200.h).

    ops = TokenOps()                                     # a handle for one device, used by one host thread at a time
    y, h = ops.rms_norm(x, weight, residual=h)           # h: the sum, for the next residual
    w = ops.w4_pack(codes, scales)                       # once; then, every step:
    qkv = ops.w4_linear(y, w)
    cache = ops.new_cache(n_pages, page_size, n_kv_heads, head_dim, n_seqs, max_pages, dtype)
    ops.kv_append(cache, k, v)
    out = ops.attn_decode(q, cache)

Calls enqueue on torch's current stream of the tensors' device and do not wait; nothing here computes anything. Wrong types, shapes or
devices raise ValueError before the call, what the library refuses raises _ffi.KernelError.
"""
import ctypes as C

import torch

from . import _ffi

_DTYPE = {torch.float32: _ffi.F32, torch.float16: _ffi.F16, torch.bfloat16: _ffi.BF16, torch.float8_e4m3fn: _ffi.E4M3}
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_current_stream = torch._C._cuda_getCurrentRawStream


class W4Weights:
    """4-bit weights as the kernels read them (TokenOps.w4_pack): [n, k] with a scale for every `group` values of a row."""

    def __init__(self, packed, n, k, group, scale_dtype, has_zeros):
        self.packed, self.n, self.k, self.group = packed, n, k, group
        self.args = _ffi.W4(packed.data_ptr() if packed is not None else None, n, k, group, _DTYPE[scale_dtype], int(has_zeros))
        self.ref = C.byref(self.args)


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
        self.device = k_pages.device
        if not k_pages.is_cuda or any(t.device != self.device for t in (v_pages, page_table, lengths, refs)):
            raise ValueError("the cache's tensors are on one GPU")
        self.k_pages, self.v_pages, self.page_table, self.lengths, self.refs = k_pages, v_pages, page_table, lengths, refs
        self.refused_count = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.dtype = k_pages.dtype
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = k_pages.shape
        self.n_seqs, self.max_pages = page_table.shape
        self.args = _ffi.KvCache(k_pages.data_ptr(), v_pages.data_ptr(), *k_pages.stride()[:3], *v_pages.stride()[:3], page_table.data_ptr(),
                                 lengths.data_ptr(), refs.data_ptr(), self.refused_count.data_ptr(), page_table.stride(0), self.n_pages,
                                 self.page_size, self.n_kv_heads, self.head_dim, self.n_seqs, self.max_pages, _DTYPE[self.dtype])
        self.ref = C.byref(self.args)

    def refused(self):
        """How many sequences operations on this cache have refused so far (waits for the GPU)."""
        return int(self.refused_count)


def _rows(t, cols, what, dtype=None):
    if t.dim() != 2 or t.shape[1] != cols or (t.stride(1) != 1 and cols > 1) or (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{what}: rows of {cols} values side by side" + (f" of type {dtype}" if dtype is not None else ""))


class TokenOps:
    """The operators of one device (a context of the kernel library)."""

    def __init__(self, device=None):
        self.device = torch.device("cuda", torch.cuda.current_device() if device is None else device)
        self.ctx = _ffi.Context(self.device.index)
        self.lib, self.h = self.ctx.lib, self.ctx.h
        self._index = self.device.index

    def close(self):
        self.ctx.close()
        self.h = None

    def _here(self, *tensors):
        for t in tensors:
            if t is not None and t.device != self.device:
                raise ValueError(f"a tensor on {t.device} in a call of {self.device}")

    def _run(self, rc):
        if rc:
            self.ctx.check(rc)

    def rms_norm(self, x, weight, eps=1e-6, residual=None, out_dtype=None, residual_out=None, out=None):
        """(y, h) with a residual, y without one; with out_dtype float8_e4m3fn (y, scale of each row, h) and (y, scale).

        x [rows, cols]; residual, residual_out: the same type and shape (residual_out may be residual: added in place)."""
        dtype, (rows, cols) = x.dtype, x.shape if x.dim() == 2 else (-1, 1)
        out_dtype = out_dtype or dtype
        _rows(x, cols, "x")
        if dtype not in _FLOATS or (out_dtype != dtype and out_dtype != torch.float8_e4m3fn):
            raise ValueError(f"rms_norm: {dtype} to {out_dtype}")
        if weight.shape != (cols,) or weight.dtype not in (dtype, torch.float32) or not weight.is_contiguous():
            raise ValueError(f"weight: {cols} values of x's type or float32")
        self._here(x, weight, residual, residual_out, out)
        if residual is not None:
            _rows(residual, cols, "residual", dtype)
            if residual_out is None:
                residual_out = torch.empty((rows, cols), dtype=dtype, device=self.device)
        if residual_out is not None:
            _rows(residual_out, cols, "residual_out", dtype)
        if out is None:
            out = torch.empty((rows, cols), dtype=out_dtype, device=self.device)
        else:
            _rows(out, cols, "out", out_dtype)
        for t in (residual, residual_out, out):
            if t is not None and t.shape[0] != rows:
                raise ValueError(f"rms_norm: {t.shape[0]} rows beside {rows}")
        scale = torch.empty(rows, dtype=torch.float32, device=self.device) if out_dtype != dtype else None
        a = _ffi.RmsNorm(x.data_ptr(), residual.data_ptr() if residual is not None else None, weight.data_ptr(),
                         residual_out.data_ptr() if residual_out is not None else None, out.data_ptr(), scale.data_ptr() if scale is not None else None,
                         rows, cols, _DTYPE[dtype], _DTYPE[weight.dtype], _DTYPE[out_dtype], x.stride(0), residual.stride(0) if residual is not None else 0,
                         residual_out.stride(0) if residual_out is not None else 0, out.stride(0), eps)
        self._run(self.lib.msnh_b200_rms_norm(self.h, C.byref(a), _current_stream(self._index)))
        got = (out,) + ((scale,) if scale is not None else ()) + ((residual_out,) if residual_out is not None else ())
        return got if len(got) > 1 else out

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
        self._here(codes, scales, zeros)
        w = W4Weights(None, n, k, group, scales.dtype, zeros is not None)
        size = C.c_size_t()
        self._run(self.lib.msnh_b200_w4_pack_bytes(self.h, w.ref, C.byref(size)))
        w.packed = torch.empty(size.value, dtype=torch.uint8, device=self.device)
        w.args.packed = w.packed.data_ptr()
        self._run(self.lib.msnh_b200_w4_pack(self.h, w.ref, codes.data_ptr(), codes.stride(0), scales.data_ptr(), zeros.data_ptr() if zeros is not None else None,
                                             w.packed.data_ptr(), _current_stream(self._index)))
        return w

    def w4_linear(self, x, weights, bias=None, x_scale=None, out_dtype=None, out=None):
        """x [rows, k] times the weights' transpose: [rows, n], at most 64 rows. x of float8_e4m3fn gives float16 unless out_dtype says
        otherwise; x_scale: float32 [rows]; bias: float32 [n]."""
        _rows(x, weights.k, "x")
        rows, dtype = x.shape[0], x.dtype
        if out is not None:
            out_dtype = out.dtype
        elif out_dtype is None:
            out_dtype = dtype if dtype in _FLOATS else torch.float16
        if dtype not in _DTYPE or out_dtype not in _FLOATS:
            raise ValueError(f"w4_linear: {dtype} to {out_dtype}")
        for t, n, what in ((bias, weights.n, "bias"), (x_scale, rows, "x_scale")):
            if t is not None and (t.shape != (n,) or t.dtype != torch.float32 or not t.is_contiguous()):
                raise ValueError(f"{what}: float32, {n} values")
        self._here(x, weights.packed, bias, x_scale, out)
        if out is None:
            out = torch.empty((rows, weights.n), dtype=out_dtype, device=self.device)
        else:
            _rows(out, weights.n, "out")
            if out.shape[0] != rows:
                raise ValueError(f"out: {out.shape[0]} rows beside {rows}")
        a = _ffi.W4Linear(x.data_ptr(), out.data_ptr(), x_scale.data_ptr() if x_scale is not None else None, bias.data_ptr() if bias is not None else None,
                          rows, _DTYPE[dtype], _DTYPE[out_dtype], x.stride(0), out.stride(0), None, 0)
        ref = C.byref(a)
        scratch = self._scratch(self.lib.msnh_b200_w4_linear_workspace, weights.ref, ref, a)
        self._run(self.lib.msnh_b200_w4_linear(self.h, weights.ref, ref, _current_stream(self._index)))
        del scratch
        return out

    def _scratch(self, ask, first, second, args):
        size = C.c_size_t()
        self._run(ask(self.h, first, second, C.byref(size)))
        if not size.value:
            return None
        # from torch's allocator: it belongs to the current stream, and what runs there later may take it over
        scratch = torch.empty(size.value, dtype=torch.uint8, device=self.device)
        args.workspace, args.workspace_bytes = scratch.data_ptr(), size.value
        return scratch

    def new_cache(self, n_pages, page_size, n_kv_heads, head_dim, n_seqs, max_pages, dtype=torch.float16):
        """A fresh cache with memory of its own."""
        pages = [torch.zeros(n_pages, page_size, n_kv_heads, head_dim, dtype=dtype, device=self.device) for _ in range(2)]
        ints = [torch.zeros(*shape, dtype=torch.int32, device=self.device) for shape in ((n_seqs, max_pages), (n_seqs,), (n_pages,))]
        return PagedCache(*pages, *ints)

    def attn_decode(self, q, cache, seqs=None, scale=None, window=0, out=None, return_lse=False):
        """One query token a row: q [rows, n_heads, head_dim] over the cached tokens of sequence seqs[row] (row without seqs); its last
        `window` ones only where that is not 0. scale: 1 / sqrt(head_dim). Returns out, or (out, lse float32 [rows, n_heads])."""
        if q.dim() != 3 or q.shape[2] != cache.head_dim or q.dtype != cache.dtype or q.stride(2) != 1:
            raise ValueError(f"q: [rows, n_heads, {cache.head_dim}] of the cache's type {cache.dtype}")
        rows, heads, dim = q.shape
        self._here(q, cache.k_pages, seqs, out)
        if seqs is not None:
            _int_vector(seqs, rows, "seqs")
        if out is None:
            out = torch.empty((rows, heads, dim), dtype=q.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
            raise ValueError("out: q's shape and type")
        lse = torch.empty((rows, heads), dtype=torch.float32, device=self.device) if return_lse else None
        a = _ffi.AttnDecode(q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else None, seqs.data_ptr() if seqs is not None else None, rows, heads,
                            q.stride(0), q.stride(1), out.stride(0), out.stride(1), dim ** -0.5 if scale is None else scale, window, None, 0)
        ref = C.byref(a)
        scratch = self._scratch(self.lib.msnh_b200_attn_decode_workspace, cache.ref, ref, a)
        self._run(self.lib.msnh_b200_attn_decode(self.h, cache.ref, ref, _current_stream(self._index)))
        del scratch
        return (out, lse) if return_lse else out

    def _kv_scratch(self, cache, n):
        size = C.c_size_t()
        self._run(self.lib.msnh_b200_kv_workspace(self.h, cache.ref, n, C.byref(size)))
        return torch.empty(size.value, dtype=torch.uint8, device=self.device)

    def kv_append(self, cache, k, v, seqs=None, starts=None):
        """Tokens behind their sequences' own: k, v [tokens, n_kv_heads, head_dim]; one token for each of seqs (int32; without it for
        sequences 0, 1, ...), or rows starts[i] to starts[i + 1] (int32, one more than sequences) for sequence seqs[i]."""
        if k.shape != v.shape or k.dim() != 3 or k.shape[1:] != cache.k_pages.shape[2:] or k.dtype != cache.dtype or v.dtype != cache.dtype:
            raise ValueError(f"k, v: [tokens, {cache.n_kv_heads}, {cache.head_dim}] of the cache's type {cache.dtype}")
        if k.stride() != v.stride() or k.stride(2) != 1:
            raise ValueError("k, v: the same strides, the values of a head side by side")
        tokens = k.shape[0]
        n = tokens if starts is None else starts.shape[0] - 1
        if starts is not None:
            _int_vector(starts, max(n, 0) + 1, "starts")
        if seqs is not None:
            _int_vector(seqs, n, "seqs")
        self._here(cache.k_pages, k, v, seqs, starts)
        scratch = self._kv_scratch(cache, n)
        self._run(self.lib.msnh_b200_kv_append(self.h, cache.ref, seqs.data_ptr() if seqs is not None else None, starts.data_ptr() if starts is not None else None,
                                               n, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), tokens, scratch.data_ptr(), scratch.numel(),
                                               _current_stream(self._index)))

    def kv_fork(self, cache, src, dst):
        """Sequences dst (int32, empty before) become copies of sequences src."""
        _int_vector(src, src.shape[0], "src")
        _int_vector(dst, src.shape[0], "dst")
        self._here(cache.k_pages, src, dst)
        scratch = self._kv_scratch(cache, src.shape[0])
        self._run(self.lib.msnh_b200_kv_fork(self.h, cache.ref, src.data_ptr(), dst.data_ptr(), src.shape[0], scratch.data_ptr(), scratch.numel(),
                                             _current_stream(self._index)))

    def kv_free(self, cache, seqs):
        """Sequences seqs (int32) give their pages back."""
        _int_vector(seqs, seqs.shape[0], "seqs")
        self._here(cache.k_pages, seqs)
        self._run(self.lib.msnh_b200_kv_free(self.h, cache.ref, seqs.data_ptr(), seqs.shape[0], _current_stream(self._index)))

    def kv_compact(self, cache, table_out=None, refs_out=None):
        """Moves live pages together: afterwards they are the first ones. table_out, refs_out: where the new table and counts go
        (the cache's own without them)."""
        table_out = cache.page_table if table_out is None else table_out
        refs_out = cache.refs if refs_out is None else refs_out
        if table_out.shape != cache.page_table.shape or table_out.stride() != cache.page_table.stride() or table_out.dtype != torch.int32:
            raise ValueError("table_out: int32, the page table's shape and strides")
        _int_vector(refs_out, cache.n_pages, "refs_out")
        self._here(cache.k_pages, table_out, refs_out)
        scratch = self._kv_scratch(cache, 0)
        self._run(self.lib.msnh_b200_kv_compact(self.h, cache.ref, table_out.data_ptr(), refs_out.data_ptr(), scratch.data_ptr(), scratch.numel(),
                                                _current_stream(self._index)))

    def kv_copy_pages(self, cache, src, dst):
        """Contents of pages src (int32) to pages dst."""
        _int_vector(src, src.shape[0], "src")
        _int_vector(dst, src.shape[0], "dst")
        self._here(cache.k_pages, src, dst)
        self._run(self.lib.msnh_b200_kv_copy_pages(self.h, cache.ref, src.data_ptr(), dst.data_ptr(), src.shape[0], _current_stream(self._index)))


def _int_vector(t, n, what):
    if t.shape != (n,) or t.dtype != torch.int32 or not t.is_contiguous():
        raise ValueError(f"{what}: int32, {n} values")
