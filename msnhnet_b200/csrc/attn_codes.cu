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
//
// Measured in graphs over three sets of inputs, both launches, 32 heads over 8 of 128: two fp16 rows of up to 131072 tokens (270 MB) 61.6 us, 4.4 TB/s; 48 bf16
// rows of up to 8192 (99 MB) 31.3; one of 37 in a short table 7.3 (from Python 62, 32 and 7.6). With the copies alone the first two take 58 and 29, with the
// arithmetic alone 45 and 27 (the joining launch, about 7, is in all of them): three warps a scheduler, each waiting five cycles for an instruction, hide most of
// one behind the other. Tiles of 16 tokens, as in 16 bits, had 83 and 49 us; two blocks an SM with three tiles
// on their way 67.2 and 39.4; rows asked for a tile earlier (to L2) 66.4. Lengths that are multiples of a share, so that the heads of a token are read at
// the same time, are 7 % faster: DRAM's share of it.
#include "attn_decode.cuh"

namespace msnh {
namespace attn {
namespace {

__device__ __forceinline__ float load_shared(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// A warp's ring of tiles of 32 tokens: the codes of keys and values in rows of kDim bytes, then a scale for each key and value. A row's 16-byte pieces
// are exchanged by its number, so that eight rows at one column lie in all the banks. What is not there is 0. Where eight tokens in a row lie in one page and are all seen (a run), a
// lane works out where that run's rows are, for eight tiles at a time; a tile then takes a few shuffles.
template <int kDim, int kStages> struct CodeRing {
    static constexpr int kTile = kCodeTile, kRuns = kTile / 8, kAhead = 32 / kRuns;
    static constexpr int kSide = kTile * kDim, kStage = 2 * kSide + 2 * kTile * 4, kBytes = kStages * kStage;
    static constexpr int kPieces = kDim / 16, kRows = 32 % kPieces == 0 ? 32 / kPieces : 0;

    // The piece of a row in which its column-th one lies.
    static __device__ __forceinline__ int piece_of(int row, int column) {
        return column ^ (kPieces % 8 == 0 ? row & 7 : kPieces % 4 == 0 ? row >> 1 & 3 : row >> 2 & 1);
    }

    const KvParams &c;
    int *masks;                              // [kStages] bit t: token t of the tile takes part
    uint32_t base;
    int lane;
    const uint8_t *k = nullptr, *v = nullptr;                    // of the key head
    const float *k_scales = nullptr, *v_scales = nullptr;
    const int *table = nullptr;              // of the sequence
    int first = 0, last = 0, origin = 0;     // tokens that are seen; token of the piece's first tile
    int next = -1;                           // a lane's page of one of the next runs, -1: no run
    int page = -1, place = 0;                // of one of this time's runs
    long long at_k = 0, at_v = 0;
    unsigned runs = 0;                       // lanes that have one

    __device__ __forceinline__ CodeRing(const KvParams &c_, int *masks_, uint32_t base_, int lane_) : c(c_), masks(masks_), base(base_), lane(lane_) {}

    __device__ __forceinline__ void start(int head, const int *table_, int first_, int last_, int first_tile) {
        k = c.k + head * c.k_head;
        v = c.v + head * c.v_head;
        k_scales = c.k_scales + static_cast<long long>(head) * c.blocks;
        v_scales = c.v_scales + static_cast<long long>(head) * c.blocks;
        table = table_;
        first = first_;
        last = last_;
        origin = (first / kTile + first_tile) * kTile;
    }
    __device__ __forceinline__ void look_ahead(int first_tile, int tiles) {
        next = -1;
        const int token = origin + first_tile * kTile + lane * 8;
        if (first_tile + lane / kRuns < tiles && c.page_size % 8 == 0 && token >= first && token <= last - 8 && c.k_token < 1 << 27 && c.v_token < 1 << 27) {
            next = table[token / c.page_size];
            if (next >= c.n_pages) next = -1;
        }
    }
    __device__ __forceinline__ void take_pages(int first_tile) {
        page = next;
        place = (origin + first_tile * kTile + lane * 8) % c.page_size;
        at_k = page * c.k_page + place * c.k_token;
        at_v = page * c.v_page + place * c.v_token;
        runs = __ballot_sync(~0u, page >= 0);
    }
    __device__ __forceinline__ int block_of(int token_place) const {
        return (c.block & (c.block - 1)) == 0 ? token_place >> (31 - __clz(c.block)) : token_place / c.block;
    }
    __device__ __forceinline__ void copy(int stage, int tile) const {
        const uint32_t to = base + stage * kStage, to_scales = to + 2 * kSide + lane * 4;
        const int from = tile % kAhead * kRuns;
        if ((runs >> from & ((1u << kRuns) - 1)) == (1u << kRuns) - 1) {
            // (rows of a run are less than 2^31 bytes apart, or it is none)
            const uint8_t *k_run[kRuns], *v_run[kRuns];
#pragma unroll
            for (int r = 0; r < kRuns; ++r) {
                k_run[r] = k + __shfl_sync(~0u, at_k, from + r);
                v_run[r] = v + __shfl_sync(~0u, at_v, from + r);
            }
            const int k_token = static_cast<int>(c.k_token), v_token = static_cast<int>(c.v_token);
            if constexpr (kRows > 0 && kRows <= 8) {             // a warp copies kRows whole rows at a time
                const int row0 = lane / kPieces, column = lane % kPieces;
                const int inside = min(column, c.dim / 16 - 1) * 16, bytes = column < c.dim / 16 ? 16 : 0;
                const int off_k = row0 * k_token + inside, off_v = row0 * v_token + inside;
                const uint32_t at = to + row0 * kDim;
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    constexpr int kStep = kRows > 0 ? kRows : 1;
                    const int more = i * kStep % 8, run = i * kStep / 8;
                    const uint32_t there = at + i * kStep * kDim + piece_of(row0 + more, column) * 16;
                    copy16(there, k_run[run] + (off_k + more * k_token), bytes);
                    copy16(there + kSide, v_run[run] + (off_v + more * v_token), bytes);
                }
            } else {
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    const int row = (lane + 32 * i) / kPieces, column = (lane + 32 * i) % kPieces;
                    constexpr int kRow = 8 * kPieces;            // pieces of a run
                    const int low = 32 * i / kRow, high = (32 * i + 31) / kRow;
                    const int inside = min(column, c.dim / 16 - 1) * 16;
                    const int bytes = column < c.dim / 16 ? 16 : 0;
                    const uint32_t at = to + row * kDim + piece_of(row, column) * 16;
                    copy16(at, (row / 8 == low ? k_run[low] : k_run[high]) + (row % 8 * k_token + inside), bytes);
                    copy16(at + kSide, (row / 8 == low ? v_run[low] : v_run[high]) + (row % 8 * v_token + inside), bytes);
                }
            }
            const int its_page = __shfl_sync(~0u, page, from + lane / 8), its_place = __shfl_sync(~0u, place, from + lane / 8) + lane % 8;
            const long long scale = static_cast<long long>(its_page) * (c.heads * c.blocks) + block_of(its_place);
            copy4(to_scales, k_scales + scale, 4);
            copy4(to_scales + kTile * 4, v_scales + scale, 4);
            if (lane == 0) masks[stage] = -1;
            return;
        }
        // any tile: a row's place from the lane that has its token
        const int token = origin + tile * kTile + lane;
        int its_page = -1;
        if (token >= first && token < last) its_page = table[token / c.page_size];
        const bool there = its_page >= 0 && its_page < c.n_pages;
        const int its_place = token % c.page_size;
        const long long row_k = there ? its_page * c.k_page + its_place * c.k_token : 0, row_v = there ? its_page * c.v_page + its_place * c.v_token : 0;
        const long long scale = there ? static_cast<long long>(its_page) * (c.heads * c.blocks) + block_of(its_place) : 0;
        copy4(to_scales, k_scales + scale, there ? 4 : 0);
        copy4(to_scales + kTile * 4, v_scales + scale, there ? 4 : 0);
        const unsigned mask = __ballot_sync(~0u, there);
        if (lane == 0) masks[stage] = static_cast<int>(mask);
#pragma unroll 1
        for (int i = 0; i < kPieces; ++i) {
            const int row = (lane + 32 * i) / kPieces, column = (lane + 32 * i) % kPieces;
            const long long from_k = __shfl_sync(~0u, row_k, row), from_v = __shfl_sync(~0u, row_v, row);
            const int inside = min(column, c.dim / 16 - 1) * 16;
            const int bytes = column < c.dim / 16 && (mask >> row & 1) ? 16 : 0;
            const uint32_t at = to + row * kDim + piece_of(row, column) * 16;
            copy16(at, k + from_k + inside, bytes);
            copy16(at + kSide, v + from_v + inside, bytes);
        }
    }
};

// A value's scale: factor * 2^power, the factor's magnitude from 1 to 2 (0 for 0).
struct Scale {
    float power, factor;
    __device__ __forceinline__ explicit Scale(float v) {
        const int exponent = max(static_cast<int>(__float_as_uint(v) >> 23 & 255), 1);
        power = static_cast<float>(exponent - 127);
        factor = exponent < 254 ? v * __uint_as_float(static_cast<uint32_t>(254 - exponent) << 23) : v * 1.17549435e-38f * 0.5f;
    }
    __device__ __forceinline__ float times(float more) const { return factor * pow2(power + more); }
};

// Lane l holds, of a tile's scores, tokens l / 4, + 8, + 16 and + 24 of heads 2 (l % 4) and + 1; of a block of 16 value columns the same two heads of
// columns 2 (l / 4) and + 1. A head's values are contracted in an order of the codes' own: a lane's four codes of a token lie side by side,
// two of them are the fragment's lower columns and two its upper ones, and so it is with the queries.
template <typename T, int kDim_, int kGroups_, int kStages_, int kWarps_, int kBlocks_> struct CodeHeads {
    using Type = T;
    using Ring = CodeRing<kDim_, kStages_>;
    // (let in early, the joining launch's blocks take the room of the next call's: 48 rows 47.5 us instead of 35.3, one call behind the other)
    static constexpr bool kEarly = false;
    static constexpr int kBegin = kCodeStart, kSmallest = kCodeSmallest;
    static constexpr int kDim = kDim_, kStages = kStages_, kGroups = kGroups_, kWarps = kWarps_, kBlocks = kBlocks_;
    static constexpr int kParts = std::is_same<T, float>::value ? 2 : 1;       // fp16 parts of a query's value
    static constexpr float kLift = 14.f;                                       // factors are taken times 2^14: they are below 2, and fp16 goes to 2^16
    static constexpr int kScratch = 4;

    float acc[kGroups][kDim / 16][4], top[kGroups][2], best[kGroups][2], sum[kGroups][2], scale[kGroups][2];     // references: top of scores, best of factors
    uint32_t q[kParts][kGroups][kDim / 16][2];

    __device__ __forceinline__ void start(const AttnParams &p, int row, int head, int heads, int lane, float *) {
        using Four = std::conditional_t<sizeof(T) == 4, uint4, uint2>;
        const T *from = reinterpret_cast<const T *>(p.q) + row * p.q_row + head * p.q_head;
#pragma unroll
        for (int n = 0; n < kGroups; ++n) {
            const int r = n * 8 + lane / 4;
            // values s * 16 + 4 (l % 4) and the three behind it: one load of four where
            // they are aligned, all of a head's loads under way before the first is
            // used. Two values a load, and read again for the largest magnitude: 48
            // bf16 rows 34.6 us instead of 31.8, four rows of heads of 256 23.5 for 20.2
            alignas(16) T v[kDim / 16][4];
            const T *mine = from + r * p.q_head + lane % 4 * 4;
            const int left = r < heads ? p.c.dim - lane % 4 * 4 : 0;
            if (p.wide_q) {
#pragma unroll
                for (int s = 0; s < kDim / 16; ++s) {
                    Four x{};
                    if (s * 16 < left) x = *reinterpret_cast<const Four *>(mine + s * 16);
                    *reinterpret_cast<Four *>(v[s]) = x;
                }
            } else {
#pragma unroll
                for (int s = 0; s < kDim / 16; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[s][i] = s * 16 < left ? mine[s * 16 + i] : T(0.f);
            }
            float factor = 1.f, back = 1.f;
            if constexpr (!std::is_same<T, __half>::value) {
                // the head's largest magnitude to between 2^14 and 2^15
                uint32_t most = 0;
#pragma unroll
                for (int s = 0; s < kDim / 16; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) most = max(most, __float_as_uint(to_float(v[s][i])) & 0x7fffffffu);
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
                    float a = to_float(v[s][2 * i]) * factor, b = to_float(v[s][2 * i + 1]) * factor;
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
        constexpr int kFour = Ring::kTile / 8;                                  // tokens of a lane
        const uint32_t scales = keys + 2 * Ring::kSide + lane / 4 * 4;
        float key_scale[kFour], value_scale[kFour];
#pragma unroll
        for (int t = 0; t < kFour; ++t) {
            key_scale[t] = load_shared(scales + t * 32);
            value_scale[t] = load_shared(scales + kFour * 32 + t * 32);
        }
        // Whether the tile's halves of 16 values have one scale each, and powers that are near one another (blocks of 16 tokens and more, mostly): then
        // a factor is a weight times one of two numbers.
        const float scale_low = __shfl_sync(~0u, value_scale[0], 0), scale_high = __shfl_sync(~0u, value_scale[kFour / 2], 0);
        bool even = mask == -1;
#pragma unroll
        for (int t = 0; t < kFour; ++t) even &= value_scale[t] == (t < kFour / 2 ? scale_low : scale_high);
        const Scale parts[2] = {Scale(scale_low), Scale(scale_high)};
        even = __all_sync(~0u, even) && fabsf(parts[0].power - parts[1].power) <= 4.f;
        float s[kGroups][kFour / 2][4] = {};
        const uint32_t at_k = keys + lane % 16 * kDim;
#pragma unroll
        for (int i = 0; i < kDim / 32; ++i)
#pragma unroll
            for (int u = 0; u < kFour / 2; ++u) {
                uint32_t c[4];
                ldmatrix(c, at_k + u * 16 * kDim + Ring::piece_of(lane % 16, 2 * i + lane / 16) * 16);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t a[4] = {halves_low(c[2 * j]), halves_low(c[2 * j + 1]), halves_high(c[2 * j]), halves_high(c[2 * j + 1])};
#pragma unroll
                    for (int n = 0; n < kGroups; ++n)
#pragma unroll
                        for (int part = 0; part < kParts; ++part) mma<__half>(s[n][u], a, q[part][n][2 * i + j][0], q[part][n][2 * i + j][1]);
                }
            }
        uint32_t high[kGroups][kFour], low[kGroups][kFour];
        bool grown = false;
        float keep[kGroups][2];
#pragma unroll
        for (int n = 0; n < kGroups; ++n) {
#pragma unroll
            for (int t = 0; t < kFour; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) s[n][t / 2][t % 2 * 2 + h] *= scale[n][h] * key_scale[t];
            if (mask != -1) {
#pragma unroll
                for (int t = 0; t < kFour; ++t)
                    if (!(mask >> (lane / 4 + t * 8) & 1)) s[n][t / 2][t % 2 * 2] = s[n][t / 2][t % 2 * 2 + 1] = -INFINITY;
            }
            float factors[kFour][2], now_best[2];
            bool near = even;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float most = s[n][0][h];
#pragma unroll
                for (int t = 1; t < kFour; ++t) most = fmaxf(most, s[n][t / 2][t % 2 * 2 + h]);
                const float here = ceilf(warp_max(most)), now = fmaxf(here, top[n][h]), base = now == -INFINITY ? 0.f : now;
                sum[n][h] *= now == top[n][h] ? 1.f : pow2(top[n][h] - now);
                now_best[h] = here + fmaxf(parts[0].power, parts[1].power);
                near &= now - here <= 64.f;                      // (not where a score is no number)
                top[n][h] = now;
                float more = 0.f;
#pragma unroll
                for (int t = 0; t < kFour; ++t) more += factors[t][h] = pow2(s[n][t / 2][t % 2 * 2 + h] - base);
                sum[n][h] += more;
            }
            if (__all_sync(~0u, near)) {
                // weights relative to the scores' reference become factors relative to their own: what is 0 of them here is 0 there, too, since the
                // references are less than 2^64 apart
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float now = fmaxf(now_best[h], best[n][h]), from = top[n][h] - now + kLift;
                    const float low_part = parts[0].times(from), high_part = parts[1].times(from);
#pragma unroll
                    for (int t = 0; t < kFour; ++t) factors[t][h] *= t < kFour / 2 ? low_part : high_part;
                    now_best[h] = now;
                }
            } else {
                float power[kFour], factor[kFour];
#pragma unroll
                for (int t = 0; t < kFour; ++t) {
                    const Scale v(value_scale[t]);
                    power[t] = v.power;
                    factor[t] = v.factor;
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float most = -INFINITY;
#pragma unroll
                    for (int t = 0; t < kFour; ++t) most = fmaxf(most, s[n][t / 2][t % 2 * 2 + h] + power[t]);
                    now_best[h] = fmaxf(ceilf(warp_max(most)), best[n][h]);
                    const float from = now_best[h] == -INFINITY ? 0.f : now_best[h] - kLift;
#pragma unroll
                    for (int t = 0; t < kFour; ++t) factors[t][h] = pow2(s[n][t / 2][t % 2 * 2 + h] - (from - power[t])) * factor[t];
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                keep[n][h] = now_best[h] == best[n][h] ? 1.f : pow2(best[n][h] - now_best[h]);
                grown |= now_best[h] != best[n][h];
                best[n][h] = now_best[h];
            }
#pragma unroll
            for (int t = 0; t < kFour; ++t) {                    // two heads of a token to two tokens of a head
                const uint32_t pair = pack2<__half>(factors[t][0], factors[t][1]);
                float high_a, high_b;
                unpack2<__half>(pair, high_a, high_b);
                high[n][t] = transposed(pair);
                low[n][t] = transposed(pack2<__half>(factors[t][0] - high_a, factors[t][1] - high_b));
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
        const uint32_t at_v = values + lane % 16 * kDim;
#pragma unroll
        for (int i = 0; i < kDim / 32; ++i)
#pragma unroll
            for (int u = 0; u < kFour / 2; ++u) {
                uint32_t c[4];
                ldmatrix_trans(c, at_v + u * 16 * kDim + Ring::piece_of(lane % 16, 2 * i + lane / 16) * 16);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    // two columns of two tokens each: the columns apart
                    const uint32_t one = __byte_perm(c[2 * j], 0, 0x3120), two = __byte_perm(c[2 * j + 1], 0, 0x3120);
                    const uint32_t a[4] = {halves_low(one), halves_high(one), halves_low(two), halves_high(two)};
#pragma unroll
                    for (int n = 0; n < kGroups; ++n) {
                        mma<__half>(acc[n][2 * i + j], a, high[n][2 * u], high[n][2 * u + 1]);
                        mma<__half>(acc[n][2 * i + j], a, low[n][2 * u], low[n][2 * u + 1]);
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
    constexpr int kMany = std::is_same<T, float>::value ? 1 : 2;               // (a pair has 8 heads of fp32 queries at most, see most_heads_codes)
    const bool few = p.chunk <= 8;
    if (p.c.dim <= 32) return few ? launch<CodeHeads<T, 32, 1, 7, 4, 3>>(ctx, p, blocks, stream) : launch<CodeHeads<T, 32, kMany, 7, 4, 3>>(ctx, p, blocks, stream);
    if (p.c.dim <= 64) return few ? launch<CodeHeads<T, 64, 1, 4, 4, 3>>(ctx, p, blocks, stream) : launch<CodeHeads<T, 64, kMany, 4, 4, 3>>(ctx, p, blocks, stream);
    if (p.c.dim <= 96) return few ? launch<CodeHeads<T, 96, 1, 2, 4, 3>>(ctx, p, blocks, stream) : launch<CodeHeads<T, 96, kMany, 2, 4, 3>>(ctx, p, blocks, stream);
    if (p.c.dim <= 128) return few ? launch<CodeHeads<T, 128, 1, 2, 4, 3>>(ctx, p, blocks, stream) : launch<CodeHeads<T, 128, kMany, 3, 4, 2>>(ctx, p, blocks, stream);
    if (p.c.dim <= 192) return few ? launch<CodeHeads<T, 192, 1, 4, 4, 1>>(ctx, p, blocks, stream) : launch<CodeHeads<T, 192, kMany, 4, 4, 1>>(ctx, p, blocks, stream);
    return launch<CodeHeads<T, 256, 1, 3, 4, 1>>(ctx, p, blocks, stream);
}

}  // namespace

// Three blocks an SM where a pair's values have registers for it: two rows of 65536 tokens, heads of 96 and 16 of them a key head 82.6 us instead of 91.1 with two,
// heads of 128 118 instead of 84.3, which is why those have two; four blocks were slower throughout (heads of 64, 4 a key head: 104 us instead of 71).
BlockShape block_shape_codes(int dim, int chunk) { return {4, dim <= 96 || (dim <= 128 && chunk <= 8) ? 3 : dim <= 128 ? 2 : 1}; }
// fp32 queries are two parts, and heads of more than 192 values have no registers for 16 of them (294 us for two rows of 65536 tokens, 16 heads a key head; in
// two pairs, which read the cache twice, 216).
int most_heads_codes(int dtype, int dim) { return dtype == MSNH_B200_F32 || dim > 192 ? 8 : 16; }

cudaError_t launch_codes(const MsnhB200Ctx *ctx, const AttnParams &p, int dtype, int blocks, void *stream) {
    return dtype == MSNH_B200_F32 ? launch_type<float>(ctx, p, blocks, stream) : dtype == MSNH_B200_F16 ? launch_type<__half>(ctx, p, blocks, stream)
                                                                                                      : launch_type<__nv_bfloat16>(ctx, p, blocks, stream);
}

}  // namespace attn
}  // namespace msnh
