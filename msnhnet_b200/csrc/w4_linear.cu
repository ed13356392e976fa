// Products with 4-bit weights (msnh_b200_w4_pack, msnh_b200_w4_linear).
#include "token_ops.h"
#include "token_types.cuh"

namespace msnh {
namespace {

// Packed weights: codes in blocks of 16 rows by 64 values (512 bytes), the blocks of a 16-row tile one behind the other; then the
// scales [tile][group][16 rows] (fp16 or fp32), then the zero points in the same order, a byte each. Codes beyond n and k are 0.
// Inside a block, 16 bytes belong to a lane of the warp that reads it: lane l has rows l / 4 and l / 4 + 8, and in its word j the
// four values from 32 * (j / 2) + 8 * (l % 4) + 4 * (j % 2) on. That is the A operand of m16n8k16 with the 16 values of a k-step in an
// order that the B operand follows, so nothing is moved between lanes. Half-bytes of a word, from the lowest: value 0 of both rows,
// value 2 of both rows, value 1 of both, value 3 of both (pairs 16 bits apart are neighbours in k).
constexpr int kTileRows = 16, kBlockK = 64, kBlockBytes = 512;

struct W4Layout {
    int n, k, group, tiles, blocks, groups;
    size_t scale_size, scales_at, zeros_at, bytes;
    W4Layout(const MsnhB200W4 &w)
        : n(w.n), k(w.k), group(w.group), tiles((w.n + kTileRows - 1) / kTileRows), blocks((w.k + kBlockK - 1) / kBlockK),
          groups((w.k + w.group - 1) / w.group) {
        scale_size = w.scale_dtype == MSNH_B200_F16 ? 2 : 4;
        scales_at = static_cast<size_t>(tiles) * blocks * kBlockBytes;
        zeros_at = scales_at + static_cast<size_t>(tiles) * groups * kTileRows * scale_size;
        bytes = zeros_at + (w.has_zeros ? static_cast<size_t>(tiles) * groups * kTileRows : 0);
    }
};

__device__ __forceinline__ int code_at(const uint8_t *codes, long long stride, int n, int k, int row, int at) {
    if (row >= n || at >= k) return 0;
    return codes[row * stride + at / 2] >> (at % 2 * 4) & 15;
}

__global__ void w4_pack_codes_kernel(const uint8_t *codes, long long stride, int n, int k, int blocks, long long words, uint32_t *out) {
    for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < words; i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int j = static_cast<int>(i % 4), lane = static_cast<int>(i / 4 % 32);
        const long long block = i / 128;
        const int row = static_cast<int>(block / blocks) * kTileRows + lane / 4;
        const int at = static_cast<int>(block % blocks) * kBlockK + 32 * (j / 2) + 8 * (lane % 4) + 4 * (j % 2);
        uint32_t word = 0;
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int half = 0; half < 2; ++half)
                word |= static_cast<uint32_t>(code_at(codes, stride, n, k, row + 8 * half, at + v)) << (16 * (v % 2) + 8 * (v / 2) + 4 * half);
        out[i] = word;
    }
}

template <typename S, typename Out>
__global__ void w4_pack_scales_kernel(const S *scales, const uint8_t *zeros, int n, int groups, long long count, Out *scales_out, uint8_t *zeros_out) {
    for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < count; i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const long long tile_group = i / kTileRows;
        const long long row = tile_group / groups * kTileRows + i % kTileRows, group = tile_group % groups;
        const bool inside = row < n;
        scales_out[i] = inside ? static_cast<Out>(to_float(scales[row * groups + group])) : static_cast<Out>(0.f);
        if (zeros) zeros_out[i] = inside ? zeros[row * groups + group] : 0;
    }
}

struct W4Params {
    const uint8_t *packed;
    const void *x;
    void *y;
    const float *x_scale, *bias;
    long long x_stride, y_stride;
    size_t scales_at, zeros_at;
    int n, k, group, blocks, groups, rows, scale_size, has_zeros;
};

__device__ __forceinline__ float scale_at(const W4Params &p, size_t i) {
    return p.scale_size == 2 ? __half2float(reinterpret_cast<const __half *>(p.packed + p.scales_at)[i])
                             : reinterpret_cast<const float *>(p.packed + p.scales_at)[i];
}

// A warp an output value.
template <typename T, typename Out>
__global__ void w4_dot_kernel(W4Params p) {
    const long long i = (blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x) / 32;
    if (i >= static_cast<long long>(p.n) * p.rows) return;
    const int row = static_cast<int>(i / p.rows), m = static_cast<int>(i % p.rows), lane = threadIdx.x % 32;
    const int tile = row / kTileRows, in_tile = row % kTileRows;
    const T *x = static_cast<const T *>(p.x) + m * p.x_stride;
    float sum = 0.f;
    for (int at = lane; at < p.k; at += 32) {
        const int in_block = at % kBlockK, word = in_block / 32 * 2 + in_block / 4 % 2, v = at % 4;
        const size_t byte = (static_cast<size_t>(tile) * p.blocks + at / kBlockK) * kBlockBytes + (in_tile % 8 * 4 + in_block % 32 / 8) * 16 + word * 4 + v % 2 * 2 + v / 2;
        const int code = p.packed[byte] >> (in_tile / 8 * 4) & 15;
        const size_t g = (static_cast<size_t>(tile) * p.groups + at / p.group) * kTileRows + in_tile;
        const int zero = p.has_zeros ? p.packed[p.zeros_at + g] : 8;
        sum += (code - zero) * scale_at(p, g) * to_float(x[at]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) {
        const float y = sum * (p.x_scale ? p.x_scale[m] : 1.f) + (p.bias ? p.bias[row] : 0.f);
        static_cast<Out *>(p.y)[m * p.y_stride + row] = from_float<Out>(y);
    }
}

template <typename T, typename Out>
cudaError_t launch(const W4Params &p, void *stream) {
    const long long warps = static_cast<long long>(p.n) * p.rows;
    return launch_token_kernel(w4_dot_kernel<T, Out>, dim3(static_cast<unsigned>((warps + 7) / 8)), 256, 0, stream, false, p);
}

template <typename T>
cudaError_t launch(const W4Params &p, int out_dtype, void *stream) {
    return out_dtype == MSNH_B200_F32 ? launch<T, float>(p, stream) : out_dtype == MSNH_B200_F16 ? launch<T, __half>(p, stream) : launch<T, __nv_bfloat16>(p, stream);
}

int check_weights(MsnhB200Ctx *ctx, const MsnhB200W4 *w, const char *what) {
    if (w->n < 1 || w->k < 1 || w->n > (1 << 30) || w->k > (1 << 30)) return fail(ctx, MSNH_B200_ERR_ARG, "%s: %d x %d weights", what, w->n, w->k);
    if (w->group < 32 || w->group % 32) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "%s: groups of %d values (a multiple of 32 is wanted)", what, w->group);
    if (!is_float_type(w->scale_dtype)) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "%s: scales of type %d", what, w->scale_dtype);
    return MSNH_B200_OK;
}

template <typename S, typename Out>
cudaError_t launch_pack_scales(const W4Layout &l, const void *scales, const uint8_t *zeros, uint8_t *packed, void *stream) {
    const long long count = static_cast<long long>(l.tiles) * l.groups * kTileRows;
    const unsigned grid = static_cast<unsigned>(std::min<long long>((count + 255) / 256, 148 * 16));
    return launch_token_kernel(w4_pack_scales_kernel<S, Out>, dim3(grid), 256, 0, stream, false, static_cast<const S *>(scales), zeros, l.n, l.groups, count,
                               reinterpret_cast<Out *>(packed + l.scales_at), packed + l.zeros_at);
}

}  // namespace
}  // namespace msnh

using namespace msnh;

extern "C" {

int msnh_b200_w4_pack_bytes(MsnhB200Ctx *ctx, const MsnhB200W4 *w, size_t *bytes) try {
    if (!ctx || !w || !bytes) return MSNH_B200_ERR_ARG;
    if (const int rc = check_weights(ctx, w, "w4_pack_bytes")) return rc;
    *bytes = W4Layout(*w).bytes;
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

int msnh_b200_w4_pack(MsnhB200Ctx *ctx, const MsnhB200W4 *w, const uint8_t *codes, int64_t codes_stride, const void *scales, const uint8_t *zeros,
                      void *packed, void *stream) try {
    if (!ctx || !w) return MSNH_B200_ERR_ARG;
    if (const int rc = check_weights(ctx, w, "w4_pack")) return rc;
    if (!codes || !scales || !packed) return fail(ctx, MSNH_B200_ERR_ARG, "w4_pack: null codes, scales or packed");
    if ((w->has_zeros != 0) != (zeros != nullptr)) return fail(ctx, MSNH_B200_ERR_ARG, "w4_pack: has_zeros says whether there are zeros");
    if (!aligned16(packed)) return fail(ctx, MSNH_B200_ERR_ARG, "w4_pack: packed is not 16-byte aligned");
    if (codes_stride < 0) return fail(ctx, MSNH_B200_ERR_ARG, "w4_pack: codes_stride is negative");
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    const W4Layout l(*w);
    uint8_t *out = static_cast<uint8_t *>(packed);
    const long long words = static_cast<long long>(l.tiles) * l.blocks * (kBlockBytes / 4);
    const unsigned grid = static_cast<unsigned>(std::min<long long>((words + 255) / 256, 148 * 32));
    CUDA_TRY(ctx, launch_token_kernel(w4_pack_codes_kernel, dim3(grid), 256, 0, stream, false, codes, codes_stride, l.n, l.k, l.blocks, words, reinterpret_cast<uint32_t *>(out)));
    CUDA_TRY(ctx, w->scale_dtype == MSNH_B200_F16  ? (launch_pack_scales<__half, __half>(l, scales, zeros, out, stream))
                : w->scale_dtype == MSNH_B200_BF16 ? (launch_pack_scales<__nv_bfloat16, float>(l, scales, zeros, out, stream))
                                                   : (launch_pack_scales<float, float>(l, scales, zeros, out, stream)));
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

int msnh_b200_w4_linear_workspace(MsnhB200Ctx *ctx, const MsnhB200W4 *w, const MsnhB200W4Linear *a, size_t *bytes) try {
    if (!ctx || !w || !a || !bytes) return MSNH_B200_ERR_ARG;
    if (const int rc = check_weights(ctx, w, "w4_linear_workspace")) return rc;
    *bytes = 0;
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

int msnh_b200_w4_linear(MsnhB200Ctx *ctx, const MsnhB200W4 *w, const MsnhB200W4Linear *a, void *stream) try {
    if (!ctx || !w || !a) return MSNH_B200_ERR_ARG;
    if (const int rc = check_weights(ctx, w, "w4_linear")) return rc;
    if (a->rows < 0 || a->rows > MSNH_B200_W4_MAX_ROWS) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "w4_linear: %d rows (at most %d)", a->rows, MSNH_B200_W4_MAX_ROWS);
    if (!is_float_type(a->dtype) && a->dtype != MSNH_B200_E4M3) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "w4_linear: x of type %d", a->dtype);
    if (!is_float_type(a->out_dtype)) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "w4_linear: y of type %d", a->out_dtype);
    if (a->rows == 0) return MSNH_B200_OK;
    if (!a->x || !a->y || !w->packed) return fail(ctx, MSNH_B200_ERR_ARG, "w4_linear: null x, y or weights");
    if (!aligned16(w->packed)) return fail(ctx, MSNH_B200_ERR_ARG, "w4_linear: the packed weights are not 16-byte aligned");
    if (a->x_stride < 0 || a->y_stride < (a->rows > 1 ? w->n : 0)) return fail(ctx, MSNH_B200_ERR_ARG, "w4_linear: rows overlap");
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    const W4Layout l(*w);
    const W4Params p = {static_cast<const uint8_t *>(w->packed), a->x, a->y, a->x_scale, a->bias, a->x_stride, a->y_stride, l.scales_at, l.zeros_at,
                        l.n, l.k, l.group, l.blocks, l.groups, a->rows, static_cast<int>(l.scale_size), w->has_zeros};
    const cudaError_t e = a->dtype == MSNH_B200_F32  ? launch<float>(p, a->out_dtype, stream)
                        : a->dtype == MSNH_B200_F16  ? launch<__half>(p, a->out_dtype, stream)
                        : a->dtype == MSNH_B200_BF16 ? launch<__nv_bfloat16>(p, a->out_dtype, stream)
                                                     : launch<__nv_fp8_e4m3>(p, a->out_dtype, stream);
    CUDA_TRY(ctx, e);
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

}  // extern "C"
