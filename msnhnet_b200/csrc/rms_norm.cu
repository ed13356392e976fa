// Root-mean-square norm of x + residual, output in x's type or in 8 bits with a scale for each row (msnh_b200_rms_norm).
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

// Sum and maximum over a block; every thread gets both. A NaN among the squares makes the sum NaN, so the maximum may drop it.
__device__ __forceinline__ void block_sum_max(float &sum, float &top) {
    __shared__ float part[2][32];
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        sum += __shfl_xor_sync(~0u, sum, o);
        top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    }
    const int warps = blockDim.x / 32, lane = threadIdx.x % 32;
    if (lane == 0) { part[0][threadIdx.x / 32] = sum; part[1][threadIdx.x / 32] = top; }
    __syncthreads();
    sum = lane < warps ? part[0][lane] : 0.f;
    top = lane < warps ? part[1][lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        sum += __shfl_xor_sync(~0u, sum, o);
        top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    }
}

// value / scale without the scale's own rounding: t * 448 / top, where t is the value before its row's common factor and top the
// largest |t|. (1 / top is infinite below 2^-127; the division is exact there, too.)
__device__ __forceinline__ float code_of(float t, float top, float inverse) { return top > 1e-30f ? t * inverse : t / top * 448.f; }

// A block a row, two passes over it: the sum of squares and (8 bits) the largest |h * w|, then the outputs. Any row length,
// alignment and stride.
template <typename T, typename W, bool k8>
__global__ void rms_norm_rows_kernel(RmsNormParams p) {
    const long long row = blockIdx.x;
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
    const T *residual = p.residual ? static_cast<const T *>(p.residual) + row * p.residual_stride : nullptr;
    T *residual_out = p.residual_out ? static_cast<T *>(p.residual_out) + row * p.residual_out_stride : nullptr;
    const W *weight = static_cast<const W *>(p.weight);
    float sum = 0.f, top = 0.f;
    for (int i = threadIdx.x; i < p.cols; i += blockDim.x) {
        const float h = to_float(x[i]) + (residual ? to_float(residual[i]) : 0.f);
        sum += h * h;
        if (k8) top = fmaxf(top, fabsf(h * to_float(weight[i])));
    }
    block_sum_max(sum, top);
    const float r = rsqrtf(sum / p.cols + p.eps);
    const float scale = top * r / 448.f, inverse = 448.f / top;
    if (k8 && threadIdx.x == 0) p.y_scale[row] = scale;
    for (int i = threadIdx.x; i < p.cols; i += blockDim.x) {
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

template <typename T, typename W>
cudaError_t launch(const RmsNormParams &p, bool out8, void *stream) {
    const int threads = p.cols <= 256 ? 64 : p.cols <= 2048 ? 256 : 1024;
    const dim3 grid(static_cast<unsigned>(p.rows));
    return out8 ? launch_token_kernel(rms_norm_rows_kernel<T, W, true>, grid, threads, 0, stream, false, p)
                : launch_token_kernel(rms_norm_rows_kernel<T, W, false>, grid, threads, 0, stream, false, p);
}

template <typename T>
cudaError_t launch(const RmsNormParams &p, int weight_dtype, bool out8, void *stream) {
    return weight_dtype == MSNH_B200_F32 ? launch<T, float>(p, out8, stream) : launch<T, T>(p, out8, stream);
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
    const cudaError_t e = a->dtype == MSNH_B200_F32 ? launch<float, float>(p, out8, stream)
                        : a->dtype == MSNH_B200_F16 ? launch<__half>(p, a->weight_dtype, out8, stream)
                                                    : launch<__nv_bfloat16>(p, a->weight_dtype, out8, stream);
    CUDA_TRY(ctx, e);
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }
