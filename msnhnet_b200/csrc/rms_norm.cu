// Root-mean-square norm of x + residual, output in x's type or in 8 bits with a scale for each row (msnh_b200_rms_norm).
//
// y = h * w / sqrt(mean(h^2) + eps). Every value is read once and h and y are written once, and those bytes bound it: 4099 bf16 rows of 5120
// values to 8 bits take 29 us, 5.0 TB/s; one row is a launch (4.5 us between calls). Rows whose parts are not 16-byte aligned cost twice
// the time (3000 fp16 rows of 6879 values to 8 bits 71 us), bound by their instructions.
#include "token_ops.h"
#include "token_types.cuh"

namespace msnh {
namespace {

struct RmsNormParams {
    const void *x, *residual, *weight;
    void *residual_out, *y;
    float *y_scale;
    long long rows, x_stride, residual_stride, residual_out_stride, y_stride;
    int cols;
    float eps;
};

// The largest of top, |a| and |b|, or NaN where one is: of the products with the weights, which the sum of squares knows nothing of.
__device__ __forceinline__ float max_or_nan(float top, float a, float b) {
    float y;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(top), "f"(a), "f"(b));
    return y;
}
// The same over a warp, of values that are not negative: their bits have the numbers' order, infinity and NaN above all of them.
__device__ __forceinline__ float warp_max_or_nan(float top) { return __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(top))); }

// Sum and, for 8 bits, maximum over a block; every thread gets both.
template <bool k8> __device__ __forceinline__ void block_sum_max(float &sum, float &top) {
    __shared__ float part[2][32];
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (k8) top = warp_max_or_nan(top);
    const int warps = blockDim.x / 32, lane = threadIdx.x % 32;
    if (lane == 0) { part[0][threadIdx.x / 32] = sum; part[1][threadIdx.x / 32] = top; }
    __syncthreads();
    sum = lane < warps ? part[0][lane] : 0.f;
    top = lane < warps ? part[1][lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (k8) top = warp_max_or_nan(top);
}

// The scale of a row's 8-bit codes; NaN, which leaves the codes 0, where a product with a weight is not finite or the sum of squares is not
// (the factor is 0 then); 0 for zeros, whose factor is infinite without an eps.
__device__ __forceinline__ float scale_of(float top, float factor) {
    return top == 0.f ? 0.f : top <= 3.4028235e38f && factor > 0.f ? top * factor / 448.f : __uint_as_float(0x7fffffffu);
}

// value / scale without the scale's own rounding: t * 448 / top, where t is the value before its row's common factor and top the
// largest |t|. (1 / top is infinite below 2^-127; the division is exact there, too.)
__device__ __forceinline__ float code_of(float t, float top, float inverse) { return top > 1e-30f ? t * inverse : t / top * 448.f; }

__device__ __forceinline__ void copy16(uint32_t to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

// Rows that a block (or a warp, kWarp) keeps in registers: one pass over memory, whose bytes bound it. A thread has kVecs vectors of 16 bytes
// of a row. With kStages it stays for every gridDim-th row and has the next kStages - 1 rows' vectors copied into shared memory meanwhile
// (its own, so it waits for nothing but its own copies); in registers they would cost half of the threads that keep the memory busy.
// 8-bit codes are h * w * (448 / max|h w|): the norm's factor cancels, so one reduction gives both the sum of squares and what the codes
// need.
template <typename T, typename W, bool k8, int kVecs, bool kWarp, int kStages>
__global__ void __launch_bounds__(kWarp ? 128 : kStages ? 512 : 1024) rms_norm_vectors_kernel(const __grid_constant__ RmsNormParams p) {
    constexpr int kVec = Vec16<T>::kVec, kParts = kVec * sizeof(W) / 16;
    extern __shared__ __align__(16) uint4 rows_ahead[];          // [kStages][kVecs][x, residual][thread]
    __shared__ float part[2][2][32];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = kWarp ? 1 : blockDim.x / 32;
    const int thread = kWarp ? lane : threadIdx.x, threads = kWarp ? 32 : blockDim.x, vectors = p.cols / kVec;
    const long long step = kWarp ? static_cast<long long>(gridDim.x) * (blockDim.x / 32) : gridDim.x;
    long long row = kWarp ? blockIdx.x * static_cast<long long>(blockDim.x / 32) + warp : blockIdx.x;
    const auto x_of = [&](long long at) { return reinterpret_cast<const uint4 *>(static_cast<const T *>(p.x) + at * p.x_stride); };
    const auto residual_of = [&](long long at) { return reinterpret_cast<const uint4 *>(static_cast<const T *>(p.residual) + at * p.residual_stride); };
    const auto weights_of = [&](int v, float (&c)[kVec]) {
        uint4 raw[kParts];
#pragma unroll
        for (int j = 0; j < kParts; ++j) raw[j] = __ldg(static_cast<const uint4 *>(p.weight) + v * kParts + j);
        const W *values = reinterpret_cast<const W *>(raw);
#pragma unroll
        for (int j = 0; j < kVec; ++j) c[j] = to_float(values[j]);
    };
    pdl_enter();
    const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(rows_ahead + threadIdx.x)), pitch = blockDim.x * 16;
    long long ahead = row;
    int filled = 0, stage = 0;
    const auto copy_next = [&] {
        if (ahead < p.rows) {
            const uint4 *x = x_of(ahead), *residual = residual_of(ahead);
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                const int v = thread + i * threads;
                const uint32_t to = mine + (filled * kVecs + i) * 2 * pitch;
                if (v < vectors) {
                    copy16(to, x + v);
                    if (p.residual) copy16(to + pitch, residual + v);
                }
            }
        }
        copy_commit();
        ahead += step;
        filled = filled == kStages - 1 ? 0 : filled + 1;
    };
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) copy_next();
    for (int turn = 0; row < p.rows; row += step, turn ^= 1) {
        if constexpr (kStages > 0) {
            copy_next();
            copy_wait<kStages - 1>();
        }
        float h[kVecs][kVec], sum = 0.f, top = 0.f;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int v = thread + i * threads;
#pragma unroll
            for (int j = 0; j < kVec; ++j) h[i][j] = 0.f;
            if (v >= vectors) continue;
            uint4 x, r = make_uint4(0, 0, 0, 0);
            if constexpr (kStages > 0) {
                x = rows_ahead[((stage * kVecs + i) * 2) * blockDim.x + threadIdx.x];
                if (p.residual) r = rows_ahead[((stage * kVecs + i) * 2 + 1) * blockDim.x + threadIdx.x];
            } else {
                x = x_of(row)[v];
                if (p.residual) r = residual_of(row)[v];
            }
            float a[kVec], b[kVec];
            Vec16<T>::unpack(x, a);
            Vec16<T>::unpack(r, b);
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                h[i][j] = a[j] + b[j];
                sum += h[i][j] * h[i][j];
            }
            if (p.residual_out) reinterpret_cast<uint4 *>(static_cast<T *>(p.residual_out) + row * p.residual_out_stride)[v] = Vec16<T>::pack(h[i]);
            if constexpr (k8) {                                  // (h times weight is all that is needed from here on)
                weights_of(v, b);
#pragma unroll
                for (int j = 0; j < kVec; ++j) h[i][j] *= b[j];
#pragma unroll
                for (int j = 0; j < kVec; j += 2) top = max_or_nan(top, h[i][j], h[i][j + 1]);
            }
        }
        stage = stage == kStages - 1 ? 0 : stage + 1;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if (k8) top = warp_max_or_nan(top);
        if (!kWarp && warps > 1) {
            // (two sets of places: the next row's are written while this one's may still be read)
            if (lane == 0) { part[turn][0][warp] = sum; part[turn][1][warp] = top; }
            __syncthreads();
            sum = lane < warps ? part[turn][0][lane] : 0.f;
            top = lane < warps ? part[turn][1][lane] : 0.f;
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
            if (k8) top = warp_max_or_nan(top);
        }
        const float factor = rsqrtf(sum / p.cols + p.eps);
        if constexpr (k8) {
            const float scale = scale_of(top, factor);
            if (thread == 0) p.y_scale[row] = scale;
            // (448 / top is infinite below 2^-119: both are taken times 2^64 there. No codes for a row without a scale.)
            if (!(top > 1e-30f)) {
                top *= 18446744073709551616.f;
#pragma unroll
                for (int i = 0; i < kVecs; ++i)
#pragma unroll
                    for (int j = 0; j < kVec; ++j) h[i][j] *= 18446744073709551616.f;
            }
            const float inverse = 448.f / top;
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                const int v = thread + i * threads;
                if (v >= vectors) continue;
                uint32_t codes[kVec / 4] = {};
                if (scale > 0.f)
#pragma unroll
                    for (int j = 0; j < kVec / 4; ++j) {
                        float c[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) c[k] = h[i][4 * j + k] * inverse;
                        codes[j] = to_e4m3x2(c[0], c[1]) | static_cast<uint32_t>(to_e4m3x2(c[2], c[3])) << 16;
                    }
                uint32_t *to = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(p.y) + row * p.y_stride + v * kVec);
                if constexpr (kVec == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(codes[0], codes[1]);
                else *to = codes[0];
            }
        } else {
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                const int v = thread + i * threads;
                if (v >= vectors) continue;
                float c[kVec];
                weights_of(v, c);
#pragma unroll
                for (int j = 0; j < kVec; ++j) c[j] = h[i][j] * factor * c[j];
                reinterpret_cast<uint4 *>(static_cast<T *>(p.y) + row * p.y_stride)[v] = Vec16<T>::pack(c);
            }
        }
    }
}

// Rows of any alignment in registers: values thread, thread + threads, ... (kEach of them), a value at a time. One pass over memory, but four
// to eight times the instructions of the vectors.
template <typename T, typename W, bool k8, int kEach>
__global__ void __launch_bounds__(1024) rms_norm_values_kernel(const __grid_constant__ RmsNormParams p) {
    pdl_enter();
    const long long row = blockIdx.x;
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
    const T *residual = p.residual ? static_cast<const T *>(p.residual) + row * p.residual_stride : nullptr;
    T *residual_out = p.residual_out ? static_cast<T *>(p.residual_out) + row * p.residual_out_stride : nullptr;
    const W *weight = static_cast<const W *>(p.weight);
    // (a place beyond the row reads its last value again: all reads are under way before the first is looked at)
    T a[kEach], b[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) a[j] = x[min(static_cast<int>(threadIdx.x + j * blockDim.x), p.cols - 1)];
    if (residual)
#pragma unroll
        for (int j = 0; j < kEach; ++j) b[j] = residual[min(static_cast<int>(threadIdx.x + j * blockDim.x), p.cols - 1)];
    float h[kEach], sum = 0.f, top = 0.f;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        h[j] = to_float(a[j]) + (residual ? to_float(b[j]) : 0.f);
        if (static_cast<int>(threadIdx.x + j * blockDim.x) >= p.cols) h[j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int i = threadIdx.x + j * blockDim.x;
        sum += h[j] * h[j];
        if (residual_out && i < p.cols) residual_out[i] = from_float<T>(h[j]);
        if (k8) {                                                // (h times weight is all that is needed from here on)
            h[j] *= i < p.cols ? to_float(weight[i]) : 0.f;
            if (j % 2) top = max_or_nan(top, h[j - 1], h[j]);
        }
    }
    block_sum_max<k8>(sum, top);
    const float r = rsqrtf(sum / p.cols + p.eps), scale = scale_of(top, r);
    if (k8 && threadIdx.x == 0) p.y_scale[row] = scale;
    // (448 / top is infinite below 2^-119: both are taken times 2^64 there. No codes for a row without a scale.)
    float lift = 1.f;
    if (!(top > 1e-30f)) lift = 18446744073709551616.f;
    const bool codes = scale > 0.f;
    const float inverse = 448.f / (top * lift);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int i = threadIdx.x + j * blockDim.x;
        if (i < p.cols) {
            if (k8) static_cast<uint8_t *>(p.y)[row * p.y_stride + i] = codes ? static_cast<uint8_t>(to_e4m3x2(h[j] * lift * inverse, 0.f)) : 0;
            else static_cast<T *>(p.y)[row * p.y_stride + i] = from_float<T>(h[j] * r * to_float(weight[i]));
        }
    }
}

// A block a row, two passes over it: the sum of squares and (8 bits) the largest |h * w|, then the outputs. Any row length,
// alignment and stride. (Places are unsigned: one behind a row of up to 2^31 - 1 values may pass 2^31.)
template <typename T, typename W, bool k8>
__global__ void rms_norm_rows_kernel(RmsNormParams p) {
    pdl_enter();
    const long long row = blockIdx.x;
    const uint32_t cols = p.cols;
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
    const T *residual = p.residual ? static_cast<const T *>(p.residual) + row * p.residual_stride : nullptr;
    T *residual_out = p.residual_out ? static_cast<T *>(p.residual_out) + row * p.residual_out_stride : nullptr;
    const W *weight = static_cast<const W *>(p.weight);
    float sum = 0.f, top = 0.f;
    for (uint32_t i = threadIdx.x; i < cols; i += blockDim.x) {
        const float h = to_float(x[i]) + (residual ? to_float(residual[i]) : 0.f);
        sum += h * h;
        if (k8) top = max_or_nan(top, h * to_float(weight[i]), 0.f);
    }
    block_sum_max<k8>(sum, top);
    const float r = rsqrtf(sum / p.cols + p.eps);
    const float scale = scale_of(top, r), inverse = 448.f / top;
    if (k8 && threadIdx.x == 0) p.y_scale[row] = scale;
    for (uint32_t i = threadIdx.x; i < cols; i += blockDim.x) {
        const float h = to_float(x[i]) + (residual ? to_float(residual[i]) : 0.f);
        const float w = to_float(weight[i]);
        if (residual_out) residual_out[i] = from_float<T>(h);
        if (k8) {
            const float code = scale > 0.f ? code_of(h * w, top, inverse) : 0.f;
            static_cast<uint8_t *>(p.y)[row * p.y_stride + i] = static_cast<uint8_t>(to_e4m3x2(code, 0.f));
        } else {
            static_cast<T *>(p.y)[row * p.y_stride + i] = from_float<T>(h * r * w);
        }
    }
}

template <typename T, typename W, bool k8, int kVecs, bool kWarp, int kStages>
cudaError_t launch_vectors(const MsnhB200Ctx *ctx, const RmsNormParams &p, int vectors, void *stream) {
    const auto kernel = rms_norm_vectors_kernel<T, W, k8, kVecs, kWarp, kStages>;
    const int threads = kWarp ? 128 : (vectors + kVecs * 32 - 1) / (kVecs * 32) * 32, rows = kWarp ? 4 : 1;
    const size_t smem = static_cast<size_t>(threads) * kVecs * 32 * kStages;
    if (smem > 47 * 1024) {                                      // (the kernel's own 256 bytes count to the 48 KB that need no attribute)
        // the attribute is a kernel's and a device's: set by the first call there
        static std::atomic<uint64_t> done{0};
        const uint64_t bit = 1ull << (ctx->device & 63);
        if (!(done.load(std::memory_order_acquire) & bit)) {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 512 * kVecs * 32 * kStages);
            if (e != cudaSuccess) return e;
            done.fetch_or(bit, std::memory_order_release);
        }
    }
    const long long all = (p.rows + rows - 1) / rows, blocks = kStages ? std::min<long long>(all, ctx->sm_count * static_cast<long long>(std::min<size_t>(1024 / threads, kStages ? (208 * 1024) / smem : 1))) : all;
    return launch_token_kernel(kernel, dim3(static_cast<unsigned>(blocks)), threads, smem, stream, ctx->pdl, p);
}

// A block a row, a vector a thread as far as that goes, so that a row's bytes are all asked for at once, except for many rows:
// - rows of up to 64 vectors: a warp a row, which needs no barrier (4100 fp16 rows of 256 and 512 values: 3.0 and 4.2 us against 4.7 and
//   4.8; at 128 vectors it loses, 8.3 against 7.4);
// - long rows to 8 bits, which leave a block more to compute than to write: blocks that stay and copy ahead (4100 bf16 rows of 5120 and
//   8192 values: 28.5 and 43.4 us, 5.1 TB/s, against 31.0 and 50.9; 600 of them 7.3 and 9.9 against 6.8 and 10.2; at 2048 values 4100 rows
//   lose, 14.4 against 12.9, and rows of x's own type at all lengths: 4100 fp32 rows of 5120 values 58 against 52 us, 4.9 TB/s).
template <typename T, typename W, bool k8>
cudaError_t launch(const MsnhB200Ctx *ctx, const RmsNormParams &p, bool aligned, void *stream) {
    const int vectors = p.cols / Vec16<T>::kVec;
    if (aligned && vectors <= 4096) {
        if (p.rows >= 4 * ctx->sm_count) {
            if (vectors <= 32) return launch_vectors<T, W, k8, 1, true, 3>(ctx, p, vectors, stream);
            if (vectors <= 64) return launch_vectors<T, W, k8, 2, true, 3>(ctx, p, vectors, stream);
            if constexpr (k8) {
                if (vectors > 512 && vectors <= 1024) return launch_vectors<T, W, k8, 2, false, 3>(ctx, p, vectors, stream);
                if (vectors > 1024 && vectors <= 2048) return launch_vectors<T, W, k8, 4, false, 2>(ctx, p, vectors, stream);
            }
        }
        return vectors <= 1024   ? launch_vectors<T, W, k8, 1, false, 0>(ctx, p, vectors, stream)
               : vectors <= 2048 ? launch_vectors<T, W, k8, 2, false, 0>(ctx, p, vectors, stream) : launch_vectors<T, W, k8, 4, false, 0>(ctx, p, vectors, stream);
    }
    // (eight values a thread: 600 fp16 rows of 1001 and 6879 values 3.5 and 15.1 us, in two passes 5.7 and 16.8; sixteen would have 12001
    // values in 39.0 us, two passes have them in 36.5)
    const dim3 rows(static_cast<unsigned>(p.rows));
    const auto threads_of = [&](int each) { return (p.cols + each * 32 - 1) / (each * 32) * 32; };
    if (p.cols <= 8192) return launch_token_kernel(rms_norm_values_kernel<T, W, k8, 8>, rows, threads_of(8), 0, stream, ctx->pdl, p);
    const int threads = 1024;
    return launch_token_kernel(rms_norm_rows_kernel<T, W, k8>, dim3(static_cast<unsigned>(p.rows)), threads, 0, stream, ctx->pdl, p);
}

template <typename T, typename W>
cudaError_t launch(const MsnhB200Ctx *ctx, const RmsNormParams &p, bool out8, void *stream) {
    // whole vectors of 16 bytes (of codes: as many values) everywhere
    constexpr int kVec = Vec16<T>::kVec;
    const auto fits = [](const void *at, long long stride, size_t size, size_t bytes) { return reinterpret_cast<uintptr_t>(at) % bytes == 0 && stride * size % bytes == 0; };
    const bool aligned = p.cols % kVec == 0 && fits(p.x, p.x_stride, sizeof(T), 16) && fits(p.residual, p.residual ? p.residual_stride : 0, sizeof(T), 16) &&
                         fits(p.residual_out, p.residual_out ? p.residual_out_stride : 0, sizeof(T), 16) && aligned16(p.weight) &&
                         fits(p.y, p.y_stride, out8 ? 1 : sizeof(T), out8 ? kVec : 16);
    return out8 ? launch<T, W, true>(ctx, p, aligned, stream) : launch<T, W, false>(ctx, p, aligned, stream);
}

template <typename T>
cudaError_t launch(const MsnhB200Ctx *ctx, const RmsNormParams &p, int weight_dtype, bool out8, void *stream) {
    return weight_dtype == MSNH_B200_F32 ? launch<T, float>(ctx, p, out8, stream) : launch<T, T>(ctx, p, out8, stream);
}

}  // namespace
}  // namespace msnh

using namespace msnh;

extern "C" int msnh_b200_rms_norm(MsnhB200Ctx *ctx, const MsnhB200RmsNorm *a, void *stream) try {
    if (!ctx || !a) return MSNH_B200_ERR_ARG;
    if (a->rows < 0 || a->rows > 0x7fffffff || a->cols < 1) return fail(ctx, MSNH_B200_ERR_ARG, "rms_norm: %lld rows of %d values", static_cast<long long>(a->rows), a->cols);
    if (!is_float_type(a->dtype)) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "rms_norm: type %d", a->dtype);
    if (a->weight_dtype != a->dtype && a->weight_dtype != MSNH_B200_F32) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "rms_norm: weight of type %d", a->weight_dtype);
    const bool out8 = a->out_dtype == MSNH_B200_E4M3;
    if (!out8 && a->out_dtype != a->dtype) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "rms_norm: output of type %d", a->out_dtype);
    if (a->rows == 0) return MSNH_B200_OK;
    if (!a->x || !a->weight || !a->y) return fail(ctx, MSNH_B200_ERR_ARG, "rms_norm: null x, weight or y");
    if (out8 != (a->y_scale != nullptr)) return fail(ctx, MSNH_B200_ERR_ARG, "rms_norm: y_scale goes with an output in 8 bits");
    if (!(a->eps >= 0.f)) return fail(ctx, MSNH_B200_ERR_ARG, "rms_norm: eps is negative");
    const int64_t least = a->rows > 1 ? a->cols : 0;
    if (a->y_stride < least || (a->residual_out && a->residual_out_stride < least) || a->x_stride < 0 || (a->residual && a->residual_stride < 0))
        return fail(ctx, MSNH_B200_ERR_ARG, "rms_norm: rows overlap");
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    const RmsNormParams p = {a->x, a->residual, a->weight, a->residual_out, a->y, a->y_scale, a->rows, a->x_stride, a->residual_stride,
                             a->residual_out_stride, a->y_stride, a->cols, a->eps};
    const cudaError_t e = a->dtype == MSNH_B200_F32 ? launch<float, float>(ctx, p, out8, stream)
                        : a->dtype == MSNH_B200_F16 ? launch<__half>(ctx, p, a->weight_dtype, out8, stream)
                                                    : launch<__nv_bfloat16>(ctx, p, a->weight_dtype, out8, stream);
    CUDA_TRY(ctx, e);
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }
