// Rotary positions (msnh_b200_rotary): of every head of a token the first 2 * half values are turned in planes of two by the token's
// position times the plane's frequency; the values behind them are kept.
//
// The angle is position * frequency without the whole turns. Frequencies are given in turns, as 64-bit fractions, so the product modulo
// 2^64 is the exact fraction of a turn for any position: what is left of an angle's error is the frequency's own 2^-65 of a turn times the
// position, and the fraction's rounding to fp32, 2^-24 of an angle of up to half a turn.
//
// Every value is read and written once, and those bytes bound it. A block has some tokens' planes: it makes their sines and cosines once
// (into shared memory, while its first values are on their way) and turns all heads by them, two vectors of 16 bytes at a time. 4100 bf16 tokens of 40
// heads of 128 (84 MB) take 18.0 us with inputs that no cache holds (4.7 TB/s), 16.1 in a graph over three sets of them in turn; one token is bound by its
// launch (1.8 us in a graph, 3.7 between calls). With four pairs of vectors on their way and divisions instead of multiplications: 21.3 us, two blocks an SM.
#include "row_overlap.h"
#include "token_ops.h"
#include "token_types.cuh"

namespace msnh {
namespace {

constexpr int kThreads = 256;
constexpr int kTable = 1024;             // planes of a block's tokens at most
constexpr int kAhead = 2;                // vector pairs of a thread on their way together

struct RotaryParams {
    const uint8_t *x;
    uint8_t *y;
    const void *positions;
    const unsigned long long *turns;
    long long tokens, x_token, x_head, y_token, y_head;
    int heads, dim, half, wide_positions, tokens_of_block, heads_of_block;
    float magnitude;
    Divisor per_head, heads_in, kept;                            // items of a head, heads of a block, vectors of a head that are not turned (1: none)
};

// V values side by side (V = 1: of tensors without 16-byte alignment)
template <typename T, int V> __device__ __forceinline__ void copy_values(T *to, const T *from) {
    if constexpr (V == 1) *to = *from;
    else *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(from);
}

// An item is V planes of a head of a token: values i.. and half + i.. of it, or, interleaved, 2 V values side by side.
template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, 4) rotary_kernel(const __grid_constant__ RotaryParams p) {
    __shared__ __align__(16) float cosine[kTable], sine[kTable];
    pdl_enter();
    const long long first_token = static_cast<long long>(blockIdx.x) * p.tokens_of_block;
    const int tokens = static_cast<int>(min(static_cast<long long>(p.tokens_of_block), p.tokens - first_token));
    const int first_head = blockIdx.y * p.heads_of_block, heads = min(p.heads_of_block, p.heads - first_head);
    const T *x = reinterpret_cast<const T *>(p.x) + first_token * p.x_token + first_head * p.x_head;
    T *y = reinterpret_cast<T *>(p.y) + first_token * p.y_token + first_head * p.y_head;
    // (the last block's heads may be fewer: items are counted as if they were not, and left out)
    const int per_head = static_cast<int>(p.per_head.by), items = per_head * static_cast<int>(p.heads_in.by) * tokens;
    const int apart = kInterleaved ? V : p.half;
    bool made = false;
    for (int base = threadIdx.x; !made || base - static_cast<int>(threadIdx.x) < items; base += kThreads * kAhead) {
        struct alignas(16) { T v[2 * V]; } pair[kAhead];
        int plane[kAhead];                                       // of the table
        long long to[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int item = base + u * kThreads;
            const int row = p.per_head.quotient(item), token = p.heads_in.quotient(row), head = row - token * static_cast<int>(p.heads_in.by), i = (item - row * per_head) * V;
            plane[u] = item < items && head < heads ? token * p.half + i : -1;
            if (plane[u] < 0) continue;
            const int at = kInterleaved ? 2 * i : i;
            const T *from = x + token * p.x_token + head * p.x_head + at;
            to[u] = token * p.y_token + head * p.y_head + at;
            copy_values<T, V>(pair[u].v, from);
            copy_values<T, V>(pair[u].v + V, from + apart);
        }
        if (!made) {
            for (int i = threadIdx.x; i < tokens * p.half; i += kThreads) {
                const long long token = first_token + i / p.half;
                const long long position = p.wide_positions ? static_cast<const long long *>(p.positions)[token] : static_cast<const int *>(p.positions)[token];
                const unsigned long long turned = static_cast<unsigned long long>(position) * p.turns[i % p.half];
                float s, c;
                // (a signed number of half turns, from -1 to 1, in units of 2^-63: rounded once, so small angles keep 24 bits, too)
                sincospif(static_cast<float>(static_cast<long long>(turned)) * 1.0842021724855044e-19f, &s, &c);
                cosine[i] = c * p.magnitude;
                sine[i] = s * p.magnitude;
            }
            __syncthreads();
            made = true;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (plane[u] < 0) continue;
            float c[V], s[V];
            if constexpr (V == 1) {
                c[0] = cosine[plane[u]];
                s[0] = sine[plane[u]];
            } else {
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    *reinterpret_cast<float4 *>(c + j) = *reinterpret_cast<const float4 *>(cosine + plane[u] + j);
                    *reinterpret_cast<float4 *>(s + j) = *reinterpret_cast<const float4 *>(sine + plane[u] + j);
                }
            }
            T *v = pair[u].v;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                T &first = kInterleaved ? v[2 * j] : v[j], &second = kInterleaved ? v[2 * j + 1] : v[V + j];
                const float a = to_float(first), b = to_float(second);
                first = from_float<T>(fmaf(a, c[j], -b * s[j]));
                second = from_float<T>(fmaf(a, s[j], b * c[j]));
            }
            copy_values<T, V>(y + to[u], v);
            copy_values<T, V>(y + to[u] + apart, v + V);
        }
    }
    // what is not turned
    if (p.dim == 2 * p.half || (p.x == p.y && p.x_token == p.y_token && p.x_head == p.y_head)) return;
    const int kept = static_cast<int>(p.kept.by);
    for (int item = threadIdx.x; item < kept * static_cast<int>(p.heads_in.by) * tokens; item += kThreads) {
        const int row = p.kept.quotient(item), token = p.heads_in.quotient(row), head = row - token * static_cast<int>(p.heads_in.by), i = 2 * p.half + (item - row * kept) * V;
        if (head < heads) copy_values<T, V>(y + token * p.y_token + head * p.y_head + i, x + token * p.x_token + head * p.x_head + i);
    }
}

template <typename T>
cudaError_t launch(const MsnhB200Ctx *ctx, const MsnhB200Rotary &a, RotaryParams p, dim3 grid, void *stream) {
    constexpr int V = 16 / sizeof(T);
    bool wide = p.half % V == 0 && p.dim % V == 0 && aligned16(a.x) && aligned16(a.y);
    for (const long long stride : {p.x_token, p.x_head, p.y_token, p.y_head}) wide = wide && stride % V == 0;
    p.per_head = Divisor(p.half / (wide ? V : 1));
    p.heads_in = Divisor(p.heads_of_block);
    p.kept = Divisor(std::max(1, (p.dim - 2 * p.half) / (wide ? V : 1)));
    if (wide) return a.interleaved ? launch_token_kernel(rotary_kernel<T, V, true>, grid, kThreads, 0, stream, ctx->pdl, p)
                                   : launch_token_kernel(rotary_kernel<T, V, false>, grid, kThreads, 0, stream, ctx->pdl, p);
    return a.interleaved ? launch_token_kernel(rotary_kernel<T, 1, true>, grid, kThreads, 0, stream, ctx->pdl, p)
                         : launch_token_kernel(rotary_kernel<T, 1, false>, grid, kThreads, 0, stream, ctx->pdl, p);
}

}  // namespace
}  // namespace msnh

using namespace msnh;

extern "C" int msnh_b200_rotary(MsnhB200Ctx *ctx, const MsnhB200Rotary *a, void *stream) try {
    if (!ctx || !a) return MSNH_B200_ERR_ARG;
    if (!is_float_type(a->dtype)) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "rotary: values of type %d", a->dtype);
    if (a->tokens < 0 || a->heads < 0 || a->dim < 1 || a->rotary_dim < 2 || a->rotary_dim % 2 || a->rotary_dim > a->dim)
        return fail(ctx, MSNH_B200_ERR_ARG, "rotary: %d values in planes of two of heads of %d", a->rotary_dim, a->dim);
    if (a->rotary_dim > 2 * kTable || static_cast<long long>(a->heads) * a->dim >= 1 << 27)
        return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "rotary: more than %d turned values of a head, or 2^27 values of a token", 2 * kTable);
    if (a->tokens == 0 || a->heads == 0) return MSNH_B200_OK;
    if (!a->x || !a->y || !a->positions || !a->turns) return fail(ctx, MSNH_B200_ERR_ARG, "rotary: null x, y, positions or turns");
    if (a->x_token_stride < 0 || a->x_head_stride < 0) return fail(ctx, MSNH_B200_ERR_ARG, "rotary: a stride of x is negative");
    const int64_t size = dtype_size(a->dtype);
    const Rows from(a->tokens, a->heads, a->x_token_stride * size, a->x_head_stride * size, a->dim * size), to(a->tokens, a->heads, a->y_token_stride * size, a->y_head_stride * size, a->dim * size);
    if (rows_overlap(to)) return fail(ctx, MSNH_B200_ERR_ARG, "rotary: rows of y overlap");
    const bool in_place = a->x == a->y && from.n_step == to.n_step && from.m_step == to.m_step;
    if (!in_place && rows_meet(a->x, from, a->y, to)) return fail(ctx, MSNH_B200_ERR_ARG, "rotary: rows of x and y overlap, and y is not x");
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    RotaryParams p = {static_cast<const uint8_t *>(a->x), static_cast<uint8_t *>(a->y), a->positions, reinterpret_cast<const unsigned long long *>(a->turns), a->tokens,
                      a->x_token_stride, a->x_head_stride, a->y_token_stride, a->y_head_stride, a->heads, a->dim, a->rotary_dim / 2, a->wide_positions, 1, a->heads,
                      a->magnitude, Divisor(1), Divisor(1), Divisor(1)};
    // A block's tokens: as many as there are threads for their planes, up to eight, where that leaves every SM some blocks. Few tokens: their heads in
    // parts, as long as a part has an item for each thread.
    const long long most = std::max(1, std::min(8, kThreads / p.half));
    p.tokens_of_block = static_cast<int>(std::max<long long>(1, std::min<long long>(most, a->tokens / (4LL * ctx->sm_count))));
    const long long blocks = (a->tokens + p.tokens_of_block - 1) / p.tokens_of_block;
    if (blocks > 0x7fffffff) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "rotary: 2^31 tokens and more");
    const long long vectors = static_cast<long long>(p.heads) * p.half * dtype_size(a->dtype) / 16;
    const long long parts = std::max<long long>(1, std::min<long long>({vectors / kThreads, ctx->sm_count / blocks, a->heads}));
    p.heads_of_block = static_cast<int>((a->heads + parts - 1) / parts);
    const dim3 grid(static_cast<unsigned>(blocks), (a->heads + p.heads_of_block - 1) / p.heads_of_block);
    CUDA_TRY(ctx, a->dtype == MSNH_B200_F32 ? launch<float>(ctx, *a, p, grid, stream) : a->dtype == MSNH_B200_F16 ? launch<__half>(ctx, *a, p, grid, stream)
                                                                                                                 : launch<__nv_bfloat16>(ctx, *a, p, grid, stream));
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }
