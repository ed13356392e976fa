// Attention of one query token a row over a paged cache of 8-bit codes with a scale for each block of tokens and head (msnh_b200_attn_decode; the
// work's division and the rings are attn_decode.cuh's, the joining launch attn_decode.cu's).
//
// s_t = scale * log2(e) * ks_t * (q . K_t), out = sum_t 2^(s_t - m) vs_t V_t / sum_t 2^(s_t - m), with codes K_t, V_t and their scales ks_t, vs_t:
// the codes' bytes bound it. Codes become fp16, which holds all of them, on the way from shared memory to the tensor cores (two a conversion), so
// nothing is rounded but queries and weights: those of 16 bits are fp16 as they are or times a power of two for each head, fp32 ones two fp16
// parts.
//
// A weight and its value's scale, 2^(s_t - m) vs_t, are one factor, which has a running reference of its own: it goes to fp16 in two parts (22
// bits) relative to the largest factor, whatever the scales are. The sum of weights is fp32 and knows nothing of the scales. Both references
// are whole numbers, the largest exponent rounded up: what has been summed is then rescaled by powers of two, exactly, and seldom.
#include "attn_decode.cuh"

namespace msnh {
namespace attn {
namespace {

// two codes to two fp16 values
__device__ __forceinline__ uint32_t halves_low(uint32_t codes) {
    uint32_t r;
    asm("{ .reg .b16 low, high; mov.b32 {low, high}, %1; cvt.rn.f16x2.e4m3x2 %0, low; }" : "=r"(r) : "r"(codes));
    return r;
}
__device__ __forceinline__ uint32_t halves_high(uint32_t codes) {
    uint32_t r;
    asm("{ .reg .b16 low, high; mov.b32 {low, high}, %1; cvt.rn.f16x2.e4m3x2 %0, high; }" : "=r"(r) : "r"(codes));
    return r;
}
__device__ __forceinline__ float load_shared(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// Lane l holds, of a tile's scores, tokens l / 4 and l / 4 + 8 of heads 2 (l % 4) and + 1; of a block of 16 value columns the same two heads of
// columns 2 (l / 4) and + 1. A head's values are contracted in an order of the codes' own: a lane's four codes of a token lie side by side,
// two of them are the fragment's lower columns and two its upper ones, and so it is with the queries.
template <typename T, int kDim_, int kGroups_, int kStages_, int kWarps_, int kBlocks_> struct CodeHeads {
    using Type = T;
    using Cache = __nv_fp8_e4m3;
    static constexpr int kDim = kDim_, kStages = kStages_, kGroups = kGroups_, kWarps = kWarps_, kBlocks = kBlocks_;
    static constexpr int kParts = std::is_same<T, float>::value ? 2 : 1;       // fp16 parts of a query's value
    static constexpr float kLift = 14.f;                                       // factors are taken times 2^14: they are below 2, and fp16 goes to 2^16
    static constexpr int kScratch = 4;

    float acc[kGroups][kDim / 16][4], top[kGroups][2], best[kGroups][2], sum[kGroups][2], scale[kGroups][2];     // references: top of scores, best of factors
    uint32_t q[kParts][kGroups][kDim / 16][2];

    __device__ __forceinline__ void start(const AttnParams &p, int row, int head, int heads, int lane, float *) {
        const T *from = reinterpret_cast<const T *>(p.q) + row * p.q_row + head * p.q_head;
#pragma unroll
        for (int n = 0; n < kGroups; ++n) {
            const int r = n * 8 + lane / 4;
            float factor = 1.f, back = 1.f;
            if constexpr (!std::is_same<T, __half>::value) {
                // the head's largest magnitude to between 2^14 and 2^15
                uint32_t most = 0;
#pragma unroll
                for (int d = lane % 4 * 4; d < kDim; d += 16)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (r < heads && d + i < p.c.dim) most = max(most, __float_as_uint(to_float(from[r * p.q_head + d + i])) & 0x7fffffffu);
                most = max(most, __shfl_xor_sync(~0u, most, 1));
                most = max(most, __shfl_xor_sync(~0u, most, 2));
                if (most > 0 && most < 0x7f800000u) {
                    const int up = max(-113, min(126, 14 + 127 - static_cast<int>(most >> 23)));
                    factor = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
                    back = __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
                }
            }
#pragma unroll
            for (int s = 0; s < kDim / 16; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int d = s * 16 + lane % 4 * 4 + i * 2;
                    float a = 0.f, b = 0.f;
                    if (r < heads && d < p.c.dim) {
                        a = to_float(from[r * p.q_head + d]) * factor;
                        b = to_float(from[r * p.q_head + d + 1]) * factor;
                    }
#pragma unroll
                    for (int part = 0; part < kParts; ++part) {
                        q[part][n][s][i] = pack2<__half>(a, b);
                        float high_a, high_b;
                        unpack2<__half>(q[part][n][s][i], high_a, high_b);
                        a -= high_a;
                        b -= high_b;
                    }
                }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                scale[n][h] = p.scale * kLog2e * __shfl_sync(~0u, back, (lane % 4 * 2 + h) * 4);
                top[n][h] = best[n][h] = -INFINITY;
                sum[n][h] = 0.f;
            }
#pragma unroll
            for (int s = 0; s < kDim / 16; ++s) acc[n][s][0] = acc[n][s][1] = acc[n][s][2] = acc[n][s][3] = 0.f;
        }
    }
    static __device__ __forceinline__ float warp_max(float v) {                // over a head's tokens
#pragma unroll
        for (int o = 4; o < 32; o *= 2) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
        return v;
    }
    __device__ __forceinline__ void tile(uint32_t keys, uint32_t values, int mask, int lane, int, float *) {
        using R = Ring<Cache, kDim, kStages>;
        constexpr int kPitch = R::kPitch;
        const uint32_t scales = keys + 2 * R::kSide + lane / 4 * 4;
        float key_scale[2], factor[2], power[2];                               // of tokens l / 4 and + 8; a value's scale is factor * 2^power
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            key_scale[t] = load_shared(scales + t * 32);
            const float v = load_shared(scales + 64 + t * 32);
            const int exponent = max(static_cast<int>(__float_as_uint(v) >> 23 & 255), 1);
            power[t] = static_cast<float>(exponent - 127);
            factor[t] = exponent < 254 ? v * __uint_as_float(static_cast<uint32_t>(254 - exponent) << 23) : v * 1.17549435e-38f * 0.5f;
        }
        // whether all of the tile's values have one power: then the largest factor is the one of the largest score
        const float first_power = __shfl_sync(~0u, power[0], 0);
        const bool even = __all_sync(~0u, power[0] == first_power && power[1] == first_power) && mask == 0xffff;
        // two sums, of even and odd steps: a product waits for the one before the last
        float s[kGroups][2][4] = {};
        const uint32_t at_k = keys + lane % 16 * kPitch + lane / 16 * 16;
#pragma unroll
        for (int i = 0; i < kDim / 32; ++i) {
            uint32_t c[4];
            ldmatrix(c, at_k + i * 32);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t a[4] = {halves_low(c[2 * j]), halves_low(c[2 * j + 1]), halves_high(c[2 * j]), halves_high(c[2 * j + 1])};
#pragma unroll
                for (int n = 0; n < kGroups; ++n)
#pragma unroll
                    for (int part = 0; part < kParts; ++part) mma<__half>(s[n][j], a, q[part][n][2 * i + j][0], q[part][n][2 * i + j][1]);
            }
        }
        uint32_t high[kGroups][2], low[kGroups][2];
        bool grown = false;
        float keep[kGroups][2];
#pragma unroll
        for (int n = 0; n < kGroups; ++n) {
            float base[2], from[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[n][0][i] = (s[n][0][i] + s[n][1][i]) * (scale[n][i % 2] * key_scale[i / 2]);
                if (mask != 0xffff && !(mask >> (lane / 4 + i / 2 * 8) & 1)) s[n][0][i] = -INFINITY;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float most = warp_max(fmaxf(s[n][0][h], s[n][0][h + 2]));
                const float most_factor = even ? most + power[0] : warp_max(fmaxf(s[n][0][h] + power[0], s[n][0][h + 2] + power[1]));
                const float now = fmaxf(ceilf(most), top[n][h]), now_factor = fmaxf(ceilf(most_factor), best[n][h]);
                base[h] = now == -INFINITY ? 0.f : now;
                from[h] = now_factor == -INFINITY ? 0.f : now_factor - kLift;
                sum[n][h] *= now == top[n][h] ? 1.f : pow2(top[n][h] - now);
                keep[n][h] = now_factor == best[n][h] ? 1.f : pow2(best[n][h] - now_factor);
                grown |= now_factor != best[n][h];
                top[n][h] = now;
                best[n][h] = now_factor;
                sum[n][h] += pow2(s[n][0][h] - base[h]) + pow2(s[n][0][h + 2] - base[h]);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {                        // tokens l / 4 (+ 8): two heads of a token to two tokens of a head
                const float a = pow2(s[n][0][2 * t] - (from[0] - power[t])) * factor[t], b = pow2(s[n][0][2 * t + 1] - (from[1] - power[t])) * factor[t];
                const uint32_t pair = pack2<__half>(a, b);
                float high_a, high_b;
                unpack2<__half>(pair, high_a, high_b);
                high[n][t] = transposed(pair);
                low[n][t] = transposed(pack2<__half>(a - high_a, b - high_b));
            }
        }
        if (__any_sync(~0u, grown)) {
#pragma unroll
            for (int n = 0; n < kGroups; ++n)
#pragma unroll
                for (int i = 0; i < kDim / 16; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[n][i][c] *= keep[n][c % 2];
        }
        const uint32_t at_v = values + lane % 16 * kPitch + lane / 16 * 16;
#pragma unroll
        for (int i = 0; i < kDim / 32; ++i) {
            uint32_t c[4];
            ldmatrix_trans(c, at_v + i * 32);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                // two columns of two tokens each: the columns apart
                const uint32_t one = __byte_perm(c[2 * j], 0, 0x3120), two = __byte_perm(c[2 * j + 1], 0, 0x3120);
                const uint32_t a[4] = {halves_low(one), halves_high(one), halves_low(two), halves_high(two)};
#pragma unroll
                for (int n = 0; n < kGroups; ++n) {
                    mma<__half>(acc[n][2 * i + j], a, high[n][0], high[n][1]);
                    mma<__half>(acc[n][2 * i + j], a, low[n][0], low[n][1]);
                }
            }
        }
    }
    // done(head, maximum, sum) once for every head, which gives the factor of its values; then put(head, d, value)
    template <typename Done, typename Put> __device__ __forceinline__ void finish(int heads, int dim, int lane, Done done, Put put) {
#pragma unroll
        for (int n = 0; n < kGroups; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int o = 4; o < 32; o *= 2) sum[n][h] += __shfl_xor_sync(~0u, sum[n][h], o);
                const int head = n * 8 + lane % 4 * 2 + h;
                if (head >= heads) continue;
                const float f = done(head, top[n][h], sum[n][h], lane < 4);
                // (in two steps: the power by itself may be beyond fp32's range where its product with a value is not)
                const float apart = best[n][h] == -INFINITY ? 0.f : best[n][h] - kLift - top[n][h], half = pow2(0.5f * apart);
#pragma unroll
                for (int i = 0; i < kDim / 16; ++i)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int d = i * 16 + lane / 4 * 2 + r;
                        if (d < dim) put(head, d, acc[n][i][2 * r + h] * half * half * f);
                    }
            }
    }
};

template <typename T>
cudaError_t launch_type(const MsnhB200Ctx *ctx, const AttnParams &p, int blocks, void *stream) {
    constexpr int kMany = std::is_same<T, float>::value ? 1 : 2;               // (a pair has 8 heads of fp32 queries at most)
    const bool few = p.chunk <= 8;
    if (p.c.dim <= 32) return few ? launch<CodeHeads<T, 32, 1, 8, 4, 2>>(ctx, p, blocks, stream) : launch<CodeHeads<T, 32, kMany, 8, 4, 2>>(ctx, p, blocks, stream);
    if (p.c.dim <= 64) return few ? launch<CodeHeads<T, 64, 1, 8, 4, 2>>(ctx, p, blocks, stream) : launch<CodeHeads<T, 64, kMany, 8, 4, 2>>(ctx, p, blocks, stream);
    if (p.c.dim <= 96) return few ? launch<CodeHeads<T, 96, 1, 6, 4, 2>>(ctx, p, blocks, stream) : launch<CodeHeads<T, 96, kMany, 6, 4, 2>>(ctx, p, blocks, stream);
    if (p.c.dim <= 128) return few ? launch<CodeHeads<T, 128, 1, 5, 4, 2>>(ctx, p, blocks, stream) : launch<CodeHeads<T, 128, kMany, 5, 4, 2>>(ctx, p, blocks, stream);
    if (p.c.dim <= 192) return few ? launch<CodeHeads<T, 192, 1, 6, 4, 1>>(ctx, p, blocks, stream) : launch<CodeHeads<T, 192, kMany, 6, 4, 1>>(ctx, p, blocks, stream);
    return few ? launch<CodeHeads<T, 256, 1, 5, 4, 1>>(ctx, p, blocks, stream) : launch<CodeHeads<T, 256, kMany, 5, 4, 1>>(ctx, p, blocks, stream);
}

}  // namespace

BlockShape block_shape_codes(int dim) { return {4, dim <= 128 ? 2 : 1}; }

cudaError_t launch_codes(const MsnhB200Ctx *ctx, const AttnParams &p, int dtype, int blocks, void *stream) {
    return dtype == MSNH_B200_F32 ? launch_type<float>(ctx, p, blocks, stream) : dtype == MSNH_B200_F16 ? launch_type<__half>(ctx, p, blocks, stream)
                                                                                                      : launch_type<__nv_bfloat16>(ctx, p, blocks, stream);
}

}  // namespace attn
}  // namespace msnh
