// The token operators (include/msnh_b200.h) on torch tensors: what msnhnet_b200/tokens.py calls. Checks of types, shapes, strides and
// devices, outputs and workspaces from torch's allocator (they belong to the current stream, and what runs there later may take them over),
// the C call, its status. A call for one token takes the GPU two or three microseconds, and as much again in Python for every object it
// looks at, so that is done here. Computes nothing.
//
// A module of plain positional functions; arguments that may be None are marked in their lists below. Raises ValueError for arguments that
// do not fit, _ffi.KernelError for what the library refuses.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cmath>
#include <exception>
#include <string>
#include <vector>

#include "msnh_b200.h"

namespace {

struct Refused : std::exception {                                // a Python error is set
};

[[noreturn]] void wrong(const std::string &what) {
    PyErr_SetString(PyExc_ValueError, what.c_str());
    throw Refused();
}

void check(MsnhB200Ctx *ctx, int status) {
    if (status == MSNH_B200_OK) return;
    PyObject *ffi = PyImport_ImportModule("msnhnet_b200._ffi");
    PyObject *kind = ffi ? PyObject_GetAttrString(ffi, "KernelError") : nullptr;
    if (kind) PyErr_Format(kind, "status %d: %s", status, msnh_b200_last_error(ctx));
    Py_XDECREF(kind);
    Py_XDECREF(ffi);
    throw Refused();
}

int type_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return MSNH_B200_F32;
        case at::kHalf: return MSNH_B200_F16;
        case at::kBFloat16: return MSNH_B200_BF16;
        case at::kFloat8_e4m3fn: return MSNH_B200_E4M3;
        default: return -1;
    }
}
bool is_float(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

// The arguments of a call: the context, its device, then the function's own.
struct Args {
    PyObject *const *args;
    MsnhB200Ctx *ctx;
    c10::Device device;

    Args(PyObject *const *a, Py_ssize_t n, Py_ssize_t wanted) : args(a), device(c10::kCUDA, 0) {
        if (n != wanted) wrong("wrong number of arguments");
        ctx = static_cast<MsnhB200Ctx *>(PyLong_AsVoidPtr(a[0]));
        const long index = PyLong_AsLong(a[1]);
        if (PyErr_Occurred()) throw Refused();
        if (!ctx) wrong("the operators' context is closed");
        device = c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(index));
    }
    cudaStream_t stream() const { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }
    const at::Tensor &tensor(int i, const char *name) const {
        if (!THPVariable_Check(args[i])) wrong(std::string(name) + ": a tensor is wanted");
        const at::Tensor &t = THPVariable_Unpack(args[i]);
        if (t.requires_grad() && c10::GradMode::is_enabled()) wrong(std::string(name) + ": requires a gradient, and these operators have none (torch.no_grad() takes it as it is)");
        if (t.device() != device) wrong(std::string(name) + ": a tensor on " + t.device().str() + " in a call of " + device.str());
        return t;
    }
    // The call writes into t: torch learns of it as of its own writes in place, so what was saved of t for a backward pass counts as lost.
    static void writes(const at::Tensor &t) {
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
    // The tensors of a cache, which a call of its upkeep writes.
    void writes_cache(int i) const {
        if (!PyTuple_Check(args[i])) wrong("the cache: a tuple of tensors is wanted");
        for (Py_ssize_t k = 0; k < PyTuple_GET_SIZE(args[i]); ++k) {
            PyObject *one = PyTuple_GET_ITEM(args[i], k);
            if (!THPVariable_Check(one)) wrong("the cache: a tuple of tensors is wanted");
            writes(THPVariable_Unpack(one));
        }
    }
    const at::Tensor *maybe(int i, const char *name) const { return args[i] == Py_None ? nullptr : &tensor(i, name); }
    at::ScalarType dtype(int i, at::ScalarType otherwise) const {
        if (args[i] == Py_None) return otherwise;
        if (!THPDtype_Check(args[i])) wrong("a dtype is wanted");
        return reinterpret_cast<THPDtype *>(args[i])->scalar_type;
    }
    double number(int i) const {
        const double v = PyFloat_AsDouble(args[i]);
        if (PyErr_Occurred()) throw Refused();
        return v;
    }
    long long whole(int i) const {
        const long long v = PyLong_AsLongLong(args[i]);
        if (PyErr_Occurred()) throw Refused();
        return v;
    }
    template <typename T> T *pointer(int i) const {
        void *p = PyLong_AsVoidPtr(args[i]);
        if (PyErr_Occurred()) throw Refused();
        return static_cast<T *>(p);
    }
    // (torch's allocator without its dispatcher: 0.25 us less a tensor; what is allocated here is written whole, or is a workspace)
    at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type) const { return at::Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt)); }
};

template <typename F> PyObject *guarded(F f) noexcept {
    try {
        return f();
    } catch (const Refused &) {
    } catch (const std::bad_alloc &) {
        PyErr_NoMemory();
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown exception");
    }
    return nullptr;
}

void rows_of(const at::Tensor &t, int64_t rows, int64_t cols, at::ScalarType type, const char *name) {
    if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols || (t.stride(1) != 1 && cols > 1) || t.scalar_type() != type)
        wrong(std::string(name) + ": " + std::to_string(rows) + " rows of " + std::to_string(cols) + " values side by side, of type " + c10::toString(type));
}
void vector_of(const at::Tensor &t, int64_t n, at::ScalarType type, const char *name) {
    if (t.dim() != 1 || t.size(0) != n || t.scalar_type() != type || (t.stride(0) != 1 && n > 1))
        wrong(std::string(name) + ": " + std::to_string(n) + " values side by side, of type " + c10::toString(type));
}

PyObject *wrap(const at::Tensor &t) { return THPVariable_Wrap(t); }

// x, weight, eps, residual or None, out_dtype or None, residual_out or None, out or None
PyObject *rms_norm(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const Args a(args, n, 9);
        const at::Tensor &x = a.tensor(2, "x"), &weight = a.tensor(3, "weight");
        const auto type = x.scalar_type(), out_type = a.dtype(6, type);
        if (x.dim() != 2) wrong("x: rows of values");
        const int64_t rows = x.size(0), cols = x.size(1);
        if (!is_float(type) || (out_type != type && out_type != at::kFloat8_e4m3fn)) wrong(std::string("rms_norm: ") + c10::toString(type) + " to " + c10::toString(out_type));
        rows_of(x, rows, cols, type, "x");
        if (weight.scalar_type() != at::kFloat) vector_of(weight, cols, type, "weight");
        else vector_of(weight, cols, at::kFloat, "weight");
        const at::Tensor *residual = a.maybe(5, "residual"), *residual_out = a.maybe(7, "residual_out"), *out = a.maybe(8, "out");
        at::Tensor kept, y, scale;
        if (residual) rows_of(*residual, rows, cols, type, "residual");
        if (residual_out) {
            rows_of(*residual_out, rows, cols, type, "residual_out");
            kept = *residual_out;
        } else if (residual) {
            kept = a.empty({rows, cols}, type);
        }
        if (out) {
            rows_of(*out, rows, cols, out_type, "out");
            y = *out;
        } else {
            y = a.empty({rows, cols}, out_type);
        }
        if (out_type != type) scale = a.empty({rows}, at::kFloat);
        if (cols > INT32_MAX) wrong("x: rows that are too long");
        const MsnhB200RmsNorm call = {x.const_data_ptr(), residual ? residual->const_data_ptr() : nullptr, weight.const_data_ptr(),
                                      kept.defined() ? kept.mutable_data_ptr() : nullptr, y.mutable_data_ptr(),
                                      scale.defined() ? static_cast<float *>(scale.mutable_data_ptr()) : nullptr, rows, static_cast<int32_t>(cols), type_of(type),
                                      type_of(weight.scalar_type()), type_of(out_type), x.stride(0), residual ? residual->stride(0) : 0,
                                      kept.defined() ? kept.stride(0) : 0, y.stride(0), static_cast<float>(a.number(4))};
        check(a.ctx, msnh_b200_rms_norm(a.ctx, &call, a.stream()));
        if (out) a.writes(*out);
        if (residual_out) a.writes(*residual_out);
        if (!scale.defined() && !kept.defined()) return wrap(y);
        if (!scale.defined()) return Py_BuildValue("(NN)", wrap(y), wrap(kept));
        if (!kept.defined()) return Py_BuildValue("(NN)", wrap(y), wrap(scale));
        return Py_BuildValue("(NNN)", wrap(y), wrap(scale), wrap(kept));
    });
}

// x, address of the weights' struct, their packed tensor, bias or None, x_scale or None, out_dtype or None, out or None
PyObject *w4_linear(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const Args a(args, n, 9);
        const at::Tensor &x = a.tensor(2, "x");
        const MsnhB200W4 *weights = a.pointer<MsnhB200W4>(3);
        a.tensor(4, "the weights");
        const auto type = x.scalar_type();
        const at::Tensor *bias = a.maybe(5, "bias"), *x_scale = a.maybe(6, "x_scale"), *out = a.maybe(8, "out");
        const auto out_type = out ? out->scalar_type() : a.dtype(7, is_float(type) ? type : at::kHalf);
        if (x.dim() != 2) wrong("x: rows of values");
        const int64_t rows = x.size(0);
        rows_of(x, rows, weights->k, type, "x");
        if (type_of(type) < 0 || !is_float(out_type)) wrong(std::string("w4_linear: ") + c10::toString(type) + " to " + c10::toString(out_type));
        if (bias) vector_of(*bias, weights->n, at::kFloat, "bias");
        if (x_scale) vector_of(*x_scale, rows, at::kFloat, "x_scale");
        if (out) rows_of(*out, rows, weights->n, out_type, "out");
        if (rows > INT32_MAX) wrong("x: too many rows");
        const at::Tensor y = out ? *out : a.empty({rows, weights->n}, out_type);
        MsnhB200W4Linear call = {x.const_data_ptr(), y.mutable_data_ptr(), x_scale ? static_cast<const float *>(x_scale->const_data_ptr()) : nullptr,
                                 bias ? static_cast<const float *>(bias->const_data_ptr()) : nullptr, static_cast<int32_t>(rows), type_of(type), type_of(out_type),
                                 x.stride(0), y.stride(0), nullptr, 0};
        check(a.ctx, msnh_b200_w4_linear_workspace(a.ctx, weights, &call, &call.workspace_bytes));
        at::Tensor scratch;
        if (call.workspace_bytes) {
            scratch = a.empty({static_cast<int64_t>(call.workspace_bytes)}, at::kByte);
            call.workspace = scratch.mutable_data_ptr();
        }
        check(a.ctx, msnh_b200_w4_linear(a.ctx, weights, &call, a.stream()));
        if (out) a.writes(*out);
        return wrap(y);
    });
}

// x, positions, the table's turns, whether planes are interleaved, magnitude, out or None
PyObject *rotary(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const Args a(args, n, 8);
        const at::Tensor &x = a.tensor(2, "x"), &positions = a.tensor(3, "positions"), &turns = a.tensor(4, "the table");
        const auto type = x.scalar_type();
        if (x.dim() != 3 || !is_float(type) || (x.stride(2) != 1 && x.size(2) > 1)) wrong("x: [tokens, heads, head_dim] of a floating type, the values of a head side by side");
        const int64_t tokens = x.size(0), heads = x.size(1), dim = x.size(2);
        if (heads > INT32_MAX || dim > INT32_MAX) wrong("x: too many heads or values");
        if (positions.scalar_type() != at::kLong) vector_of(positions, tokens, at::kInt, "positions");
        else vector_of(positions, tokens, at::kLong, "positions");
        vector_of(turns, turns.numel(), at::kLong, "the table");
        const at::Tensor *given = a.maybe(7, "out");
        if (given && (given->sizes() != x.sizes() || given->scalar_type() != type || (given->stride(2) != 1 && dim > 1))) wrong("out: x's shape and type");
        const at::Tensor out = given ? *given : a.empty(x.sizes(), type);
        const int interleaved = PyObject_IsTrue(args[5]);
        const MsnhB200Rotary call = {x.const_data_ptr(), out.mutable_data_ptr(), positions.const_data_ptr(), static_cast<const int64_t *>(turns.const_data_ptr()), tokens,
                                     static_cast<int32_t>(heads), static_cast<int32_t>(dim), static_cast<int32_t>(std::min<int64_t>(2 * turns.numel(), INT32_MAX - 1)), type_of(type),
                                     interleaved, positions.scalar_type() == at::kLong, x.stride(0), x.stride(1), out.stride(0), out.stride(1), static_cast<float>(a.number(6))};
        check(a.ctx, msnh_b200_rotary(a.ctx, &call, a.stream()));
        if (given) a.writes(*given);
        return wrap(out);
    });
}

// logits, ids or None, how many of the likeliest
PyObject *token_scores(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const Args a(args, n, 5);
        const at::Tensor &logits = a.tensor(2, "logits");
        const auto type = logits.scalar_type();
        if (logits.dim() != 2 || !is_float(type) || (logits.stride(1) != 1 && logits.size(1) > 1)) wrong("logits: rows of floating values side by side");
        const int64_t rows = logits.size(0), cols = logits.size(1);
        if (cols > INT32_MAX) wrong("logits: rows that are too long");
        const at::Tensor *ids = a.maybe(3, "ids");
        if (ids) vector_of(*ids, rows, at::kLong, "ids");
        const long long top = a.whole(4);
        if (top > INT32_MAX || top < INT32_MIN) wrong("top: out of range");
        const at::Tensor entropy = a.empty({rows}, at::kFloat);
        at::Tensor logprob, top_logprobs, top_ids;
        if (ids) logprob = a.empty({rows}, at::kFloat);
        if (top > 0 && top <= MSNH_B200_SCORES_MAX_TOP) {
            top_logprobs = a.empty({rows, top}, at::kFloat);
            top_ids = a.empty({rows, top}, at::kLong);
        }
        const MsnhB200TokenScores call = {logits.const_data_ptr(), ids ? static_cast<const int64_t *>(ids->const_data_ptr()) : nullptr,
                                          ids ? static_cast<float *>(logprob.mutable_data_ptr()) : nullptr, static_cast<float *>(entropy.mutable_data_ptr()),
                                          top_logprobs.defined() ? static_cast<float *>(top_logprobs.mutable_data_ptr()) : nullptr,
                                          top_ids.defined() ? static_cast<int64_t *>(top_ids.mutable_data_ptr()) : nullptr, rows, logits.stride(0),
                                          static_cast<int32_t>(cols), type_of(type), static_cast<int32_t>(top)};
        check(a.ctx, msnh_b200_token_scores(a.ctx, &call, a.stream()));
        const auto or_none = [](const at::Tensor &t) -> PyObject * {
            if (t.defined()) return wrap(t);
            Py_RETURN_NONE;
        };
        return Py_BuildValue("(NNNN)", or_none(logprob), wrap(entropy), or_none(top_logprobs), or_none(top_ids));
    });
}

// The type that values beside a cache have: the cache's own, or any floating one beside 8-bit codes.
at::ScalarType fitting(at::ScalarType cache, at::ScalarType given) { return cache == at::kFloat8_e4m3fn && is_float(given) ? given : cache; }

// q, address of the cache's struct, its k_pages, seqs or None, scale or None, window, out or None, whether lse is wanted
PyObject *attn_decode(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const Args a(args, n, 10);
        const at::Tensor &q = a.tensor(2, "q"), &pages = a.tensor(4, "the cache");
        const MsnhB200KvCache *cache = a.pointer<MsnhB200KvCache>(3);
        const auto type = fitting(pages.scalar_type(), q.scalar_type());
        if (q.dim() != 3 || q.size(2) != cache->head_dim || q.scalar_type() != type || !is_float(type) || (q.stride(2) != 1 && q.size(2) > 1))
            wrong("q: [rows, n_heads, " + std::to_string(cache->head_dim) + "] of the cache's type " + c10::toString(pages.scalar_type()) + " (of a floating one over 8 bits)");
        const int64_t rows = q.size(0), heads = q.size(1);
        if (rows > INT32_MAX || heads > INT32_MAX) wrong("q: too many rows or heads");
        const at::Tensor *seqs = a.maybe(5, "seqs"), *given = a.maybe(8, "out");
        if (seqs) vector_of(*seqs, rows, at::kInt, "seqs");
        if (given && (given->sizes() != q.sizes() || given->scalar_type() != type || (given->stride(2) != 1 && q.size(2) > 1))) wrong("out: q's shape and type");
        const at::Tensor out = given ? *given : a.empty(q.sizes(), type);
        const int want_lse = PyObject_IsTrue(args[9]);
        const at::Tensor lse = want_lse ? a.empty({rows, heads}, at::kFloat) : at::Tensor();
        const long long window = a.whole(7);
        if (window > INT32_MAX || window < INT32_MIN) wrong("window: out of range");
        MsnhB200AttnDecode call = {q.const_data_ptr(), out.mutable_data_ptr(), want_lse ? static_cast<float *>(lse.mutable_data_ptr()) : nullptr,
                                   seqs ? static_cast<const int32_t *>(seqs->const_data_ptr()) : nullptr, static_cast<int32_t>(rows), static_cast<int32_t>(heads),
                                   q.stride(0), q.stride(1), out.stride(0), out.stride(1),
                                   args[6] == Py_None ? 1.f / std::sqrt(static_cast<float>(cache->head_dim)) : static_cast<float>(a.number(6)),
                                   static_cast<int32_t>(window), nullptr, 0, type_of(type)};
        check(a.ctx, msnh_b200_attn_decode_workspace(a.ctx, cache, &call, &call.workspace_bytes));
        at::Tensor scratch;
        if (call.workspace_bytes) {
            scratch = a.empty({static_cast<int64_t>(call.workspace_bytes)}, at::kByte);
            call.workspace = scratch.mutable_data_ptr();
        }
        check(a.ctx, msnh_b200_attn_decode(a.ctx, cache, &call, a.stream()));
        if (given) a.writes(*given);
        return want_lse ? Py_BuildValue("(NN)", wrap(out), wrap(lse)) : wrap(out);
    });
}

at::Tensor kv_scratch(const Args &a, const MsnhB200KvCache *cache, int64_t n) {
    if (n > INT32_MAX) wrong("too many sequences");
    size_t bytes = 0;
    check(a.ctx, msnh_b200_kv_workspace(a.ctx, cache, static_cast<int>(n), &bytes));
    return a.empty({static_cast<int64_t>(bytes)}, at::kByte);
}
const int32_t *ints(const at::Tensor &t) { return static_cast<const int32_t *>(t.const_data_ptr()); }

// address of the cache's struct, its k_pages, all its tensors, k, v, seqs or None, starts or None
PyObject *kv_append(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const Args a(args, n, 9);
        const MsnhB200KvCache *cache = a.pointer<MsnhB200KvCache>(2);
        const at::Tensor &pages = a.tensor(3, "the cache"), &k = a.tensor(5, "k"), &v = a.tensor(6, "v");
        if (k.dim() != 3 || v.sizes() != k.sizes() || k.size(1) != cache->n_kv_heads || k.size(2) != cache->head_dim || k.scalar_type() != fitting(pages.scalar_type(), k.scalar_type()) ||
            v.scalar_type() != k.scalar_type() || !is_float(k.scalar_type()))
            wrong("k, v: [tokens, " + std::to_string(cache->n_kv_heads) + ", " + std::to_string(cache->head_dim) + "] of the cache's type " + c10::toString(pages.scalar_type()) +
                  " (of a floating one for 8 bits)");
        if (v.strides() != k.strides() || (k.stride(2) != 1 && k.size(2) > 1)) wrong("k, v: the same strides, the values of a head side by side");
        const at::Tensor *seqs = a.maybe(7, "seqs"), *starts = a.maybe(8, "starts");
        const int64_t tokens = k.size(0), count = !starts ? tokens : starts->dim() == 1 && starts->size(0) ? starts->size(0) - 1 : -1;
        if (starts) vector_of(*starts, count + 1, at::kInt, "starts");
        if (count < 0) wrong("starts: one more than sequences");
        if (seqs) vector_of(*seqs, count, at::kInt, "seqs");
        if (tokens > INT32_MAX) wrong("k, v: too many tokens");
        const at::Tensor scratch = kv_scratch(a, cache, count);
        check(a.ctx, msnh_b200_kv_append_as(a.ctx, cache, seqs ? ints(*seqs) : nullptr, starts ? ints(*starts) : nullptr, static_cast<int>(count), k.const_data_ptr(),
                                            v.const_data_ptr(), type_of(k.scalar_type()), k.stride(0), k.stride(1), static_cast<int>(tokens), scratch.mutable_data_ptr(), scratch.numel(),
                                            a.stream()));
        a.writes_cache(4);
        Py_RETURN_NONE;
    });
}

// address of the cache's struct, its k_pages, starts, the number of rows, seqs or None, first or None, dtype or None, k_out or None, v_out or None
PyObject *kv_read(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const Args a(args, n, 11);
        const MsnhB200KvCache *cache = a.pointer<MsnhB200KvCache>(2);
        const at::Tensor &pages = a.tensor(3, "the cache"), &starts = a.tensor(4, "starts");
        const int64_t rows = a.whole(5), count = starts.dim() == 1 && starts.size(0) ? starts.size(0) - 1 : -1;
        if (count < 0) wrong("starts: one more than sequences");
        vector_of(starts, count + 1, at::kInt, "starts");
        if (rows < 0 || rows > INT32_MAX || count > INT32_MAX) wrong("kv_read: the number of tokens or sequences is out of range");
        const at::Tensor *seqs = a.maybe(6, "seqs"), *first = a.maybe(7, "first"), *k = a.maybe(9, "out"), *v = a.maybe(10, "out");
        if (seqs) vector_of(*seqs, count, at::kInt, "seqs");
        if (first) vector_of(*first, count, at::kInt, "first");
        if (!k != !v) wrong("out: keys and values");
        const auto type = a.dtype(8, k ? k->scalar_type() : is_float(pages.scalar_type()) ? pages.scalar_type() : at::kHalf);
        if (!is_float(type)) wrong(std::string("kv_read: a floating type is wanted, not ") + c10::toString(type));
        const std::vector<int64_t> shape = {rows, cache->n_kv_heads, cache->head_dim};
        if (k && (k->sizes() != shape || v->sizes() != shape || k->scalar_type() != type || v->scalar_type() != type || k->strides() != v->strides() ||
                  (k->stride(2) != 1 && cache->head_dim > 1)))
            wrong("out: keys and values [" + std::to_string(rows) + ", " + std::to_string(cache->n_kv_heads) + ", " + std::to_string(cache->head_dim) + "] of type " + c10::toString(type) +
                  " and the same strides, the values of a head side by side");
        const at::Tensor k_out = k ? *k : a.empty(shape, type), v_out = v ? *v : a.empty(shape, type);
        check(a.ctx, msnh_b200_kv_read(a.ctx, cache, seqs ? ints(*seqs) : nullptr, ints(starts), first ? ints(*first) : nullptr, static_cast<int>(count), k_out.mutable_data_ptr(),
                                       v_out.mutable_data_ptr(), type_of(type), k_out.stride(0), k_out.stride(1), static_cast<int>(rows), a.stream()));
        if (k) {
            a.writes(*k);
            a.writes(*v);
        }
        return Py_BuildValue("(NN)", wrap(k_out), wrap(v_out));
    });
}

void pair_of(const at::Tensor &src, const at::Tensor &dst) {
    vector_of(src, src.numel(), at::kInt, "src");
    vector_of(dst, src.numel(), at::kInt, "dst");
}

// address of the cache's struct, its k_pages, all its tensors, src, dst
PyObject *kv_fork(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const Args a(args, n, 7);
        const MsnhB200KvCache *cache = a.pointer<MsnhB200KvCache>(2);
        a.tensor(3, "the cache");
        const at::Tensor &src = a.tensor(5, "src"), &dst = a.tensor(6, "dst");
        pair_of(src, dst);
        const at::Tensor scratch = kv_scratch(a, cache, src.numel());
        check(a.ctx, msnh_b200_kv_fork(a.ctx, cache, ints(src), ints(dst), static_cast<int>(src.numel()), scratch.mutable_data_ptr(), scratch.numel(), a.stream()));
        a.writes_cache(4);
        Py_RETURN_NONE;
    });
}

// address of the cache's struct, its k_pages, all its tensors, seqs
PyObject *kv_free(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const Args a(args, n, 6);
        a.tensor(3, "the cache");
        const at::Tensor &seqs = a.tensor(5, "seqs");
        vector_of(seqs, seqs.numel(), at::kInt, "seqs");
        if (seqs.numel() > INT32_MAX) wrong("seqs: too many");
        check(a.ctx, msnh_b200_kv_free(a.ctx, a.pointer<MsnhB200KvCache>(2), ints(seqs), static_cast<int>(seqs.numel()), a.stream()));
        a.writes_cache(4);
        Py_RETURN_NONE;
    });
}

// address of the cache's struct, its page table, all its tensors, table_out, refs_out
PyObject *kv_compact(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const Args a(args, n, 7);
        const MsnhB200KvCache *cache = a.pointer<MsnhB200KvCache>(2);
        const at::Tensor &table = a.tensor(3, "the cache"), &table_out = a.tensor(5, "table_out"), &refs_out = a.tensor(6, "refs_out");
        if (table_out.sizes() != table.sizes() || table_out.strides() != table.strides() || table_out.scalar_type() != at::kInt)
            wrong("table_out: int32, the page table's shape and strides");
        vector_of(refs_out, cache->n_pages, at::kInt, "refs_out");
        const at::Tensor scratch = kv_scratch(a, cache, 0);
        check(a.ctx, msnh_b200_kv_compact(a.ctx, cache, static_cast<int32_t *>(table_out.mutable_data_ptr()), static_cast<int32_t *>(refs_out.mutable_data_ptr()),
                                          scratch.mutable_data_ptr(), scratch.numel(), a.stream()));
        a.writes_cache(4);
        a.writes(table_out);
        a.writes(refs_out);
        Py_RETURN_NONE;
    });
}

// address of the cache's struct, its k_pages, all its tensors, src, dst
PyObject *kv_copy_pages(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const Args a(args, n, 7);
        a.tensor(3, "the cache");
        const at::Tensor &src = a.tensor(5, "src"), &dst = a.tensor(6, "dst");
        pair_of(src, dst);
        if (src.numel() > INT32_MAX) wrong("src: too many pages");
        check(a.ctx, msnh_b200_kv_copy_pages(a.ctx, a.pointer<MsnhB200KvCache>(2), ints(src), ints(dst), static_cast<int>(src.numel()), a.stream()));
        a.writes_cache(4);
        Py_RETURN_NONE;
    });
}

template <PyObject *(*f)(PyObject *, PyObject *const *, Py_ssize_t)> PyMethodDef method(const char *name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr};
}
PyMethodDef kMethods[] = {method<rms_norm>("rms_norm"),   method<w4_linear>("w4_linear"),   method<attn_decode>("attn_decode"),
                          method<kv_append>("kv_append"), method<kv_fork>("kv_fork"),       method<kv_free>("kv_free"),
                          method<kv_compact>("kv_compact"), method<kv_copy_pages>("kv_copy_pages"),
                          method<rotary>("rotary"),       method<token_scores>("token_scores"), method<kv_read>("kv_read"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_tokens", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tokens(void) { return PyModule_Create(&kModule); }
