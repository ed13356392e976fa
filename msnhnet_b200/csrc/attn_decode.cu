// Attention of one query token a row over a paged cache (msnh_b200_attn_decode).
//
// out = sum_t p_t v_t / sum_t p_t, p_t = 2^(s_t - m), s_t = scale * log2(e) * q . k_t, m the running maximum: one pass over keys and
// values. Every key and value is read once for all query heads that share it, so the bytes of the cache bound it: 4 * dim operations for
// 2 * dim values a query head and token, far below what either the tensor cores or the CUDA cores do meanwhile.
//
// Work: the 16-token tiles of all (row, key head) pairs are laid end to end, each pair's after kStart more for what a pair costs by
// itself, and every warp of the grid takes an equal share, whatever the sequences' lengths. A pair that lies in one share is finished by
// its warp; one that is cut leaves its parts (sum, maximum, unnormalised values, fp32) in the workspace, and a second launch joins them
// in the order of the tokens. Where no sequence can have more than kWholeTiles tiles, warps take whole pairs and nothing is joined.
//
// A warp copies its tiles through a ring of its own with cp.async (rows of 16-byte pieces, gathered page by page), running on into the
// tiles of its next pair while it works on this one's, and keeps running maximum, sum and values of the query heads in registers. Warps
// wait for nobody. 16-bit caches: m16n8k16. fp32 caches: CUDA cores (tf32 would lose 13 bits of the products).
//
// Measured, both launches: two sequences of up to 131072 fp16 tokens with 8 key heads of 128 (538 MB) 105 to 110 us, 4.9 to 5.1 TB/s; 48 of up to 8192
// bf16 tokens (197 MB) 46 us, 4.3 TB/s, of which the launches, the first tiles and the join are 12; nine of up to 1500 fp32 tokens 14.4 us.
// Blocks in equal parts of a sequence instead of shares by warp had 115, 140 and 35 us; two to eight times as many blocks, taken up as SMs
// come free, 114 to 144 us for the first: a warp's start costs 3.5 us.
#include "kv_cache.h"
#include "token_types.cuh"

namespace msnh {
namespace {

constexpr int kTile = 16;                    // tokens of a tile
constexpr int kMaxRows = 256;                // rows of a launch: what they see is kept in shared memory
// Tiles that a pair's start counts for, and tiles of a share, where there are as many. fp16, 32 heads over 8, with kStart 1, 3 and 6: one row
// of 500 tokens 9.7, 10.8 and 13.1 us, 16 of them 17.2, 16.5 and 18.0, one of 65536 beside 63 of 100 76.7, 75.2 and 75.7, one of 4000 14.2,
// 14.8 and 16.1; 16 of 4000 and more tokens are the same within 1 %.
constexpr int kStart = 3, kLeast = 2;
// Where the table's rows (or the window) hold at most so many tiles no sequence is cut, which saves the join: tables of 128 tokens with one
// row of 37 or 120 tokens 6.6 and 10.3 us, 64 of 120 14.0 (with kWholeTiles 2: 9.1, 10.1, 17.2). With 32, tables of 512 tokens: one, 16, 64
// and 128 rows of 500 tokens 28.1, 29.8, 36.7 and 50.6 us, cut 10.8, 16.5, 34.2 and 59.5: many pairs would do without the cuts. Lengths are
// not known on the host: in tables of 4096 tokens one row of 37, 120 and 500 tokens takes 12.1, 13.2 and 13.7 us.
constexpr int kWholeTiles = 8;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnParams {
    KvParams c;
    const uint8_t *q;
    uint8_t *out;
    float *lse;
    const int *seqs;
    long long q_row, q_head, out_row, out_head;
    int rows, n_heads, each, chunk, chunks, window;      // each: query heads of a key head; chunk: how many of them a pair has
    int first_row;                                       // of this launch
    int whole;
    float scale;
    int *prefix;                                         // workspace: the line's tiles before each row (rows + 1), then the parts
    float2 *part_ml;                                     // [slot][chunk] maximum and sum
    float *part;                                         // [slot][chunk][dim]
};

struct Row { int seq, first, last; };
__device__ __forceinline__ Row row_of(const AttnParams &p, int row) {
    Row r;
    r.seq = p.seqs ? p.seqs[row] : row;
    r.last = r.seq >= 0 && r.seq < p.c.n_seqs ? max(0, min(p.c.lengths[r.seq], p.c.max_pages * p.c.page_size)) : 0;
    r.first = p.window > 0 ? max(0, r.last - p.window) : 0;
    return r;
}
__device__ __forceinline__ int tiles_of(const Row &r) { return r.last > r.first ? (r.last - 1) / kTile - r.first / kTile + 1 : 0; }

// The share of a warp, in tiles of the line. (A launch's line has less than 2^30 tiles: code for longer ones is a microsecond of reading
// instructions alone.)
__device__ __forceinline__ int share_of(int line, int workers) {
    return max((line + workers - 1) / workers, kStart + kLeast);
}

// 16 bytes to shared memory, of which the first `bytes` are copied (16 or none) and the others are 0
__device__ __forceinline__ void copy16(uint32_t to, const void *from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
// 2^x to 2 units in the last place; below 2^-126 it is 0
__device__ __forceinline__ float pow2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

// A warp's ring: kStages tiles of keys and values. Rows are 16 bytes longer than kDim values: eight rows at one column then lie in all
// the banks. Pieces of tokens that are not there, and keys' columns beyond dim, are filled with zeros: a weight of 0 meets a 0.
template <typename T, int kDim, int kStages> struct Ring {
    static constexpr int kPitch = kDim * sizeof(T) + 16;
    static constexpr int kSide = kTile * kPitch, kStage = 2 * kSide, kBytes = kStages * kStage;
    static constexpr int kPieces = kDim * sizeof(T) / 16, kValues = 16 / sizeof(T);

    const KvParams &c;
    const T *k, *v;                          // of the key head
    const int *table;                        // of the sequence
    int *masks;                              // [kStages] bit t: token t of the tile takes part
    uint32_t base;
    int first, last, lane;                   // tokens that are seen; lane of the warp

    // The page of a run of eight tokens that are all seen, in a cache whose pages are multiples of eight; -1 otherwise.
    __device__ __forceinline__ int page_of(int token) const {
        if (c.page_size % 8 || token < first || token + 8 > last) return -1;
        const int page = table[token / c.page_size];
        return page < c.n_pages ? page : -1;
    }
    // A tile of two such runs.
    __device__ __forceinline__ void issue(int stage, int token, int page_low, int page_high) const {
        const uint32_t to = base + stage * kStage;
        if (lane == 0) masks[stage] = 0xffff;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const long long page = half ? page_high : page_low, place = (token + 8 * half) % c.page_size;
            const T *from_k = k + page * c.k_page + place * c.k_token, *from_v = v + page * c.v_page + place * c.v_token;
            if (32 % kPieces == 0) {                             // a warp copies whole rows at a time
                const int row = lane / kPieces, column = lane % kPieces;
                const bool inside = column < c.dim / kValues;
                if (inside) { from_k += row * c.k_token + column * kValues; from_v += row * c.v_token + column * kValues; }
                const uint32_t at = to + (8 * half + row) * kPitch + column * 16;
                const int bytes = inside ? 16 : 0;
#pragma unroll
                for (int i = 0; i < kPieces / 4; ++i) {
                    copy16(at + i * (32 / kPieces * kPitch), from_k, bytes);
                    copy16(at + i * (32 / kPieces * kPitch) + kSide, from_v, bytes);
                    from_k += 32 / kPieces * c.k_token;
                    from_v += 32 / kPieces * c.v_token;
                }
            } else {
#pragma unroll
                for (int i = 0; i < kPieces / 4; ++i) {
                    const int piece = lane + 32 * i, row = piece / kPieces, column = piece % kPieces;
                    const uint32_t at = to + (8 * half + row) * kPitch + column * 16;
                    const bool inside = column < c.dim / kValues;
                    copy16(at, inside ? from_k + row * c.k_token + column * kValues : from_k, inside ? 16 : 0);
                    copy16(at + kSide, inside ? from_v + row * c.v_token + column * kValues : from_v, inside ? 16 : 0);
                }
            }
        }
    }
    // Any tile: a row's place from the lane that has its token.
    __device__ __forceinline__ void issue_any(int stage, int token) const {
        const int mine = token + lane;
        int page = -1;
        if (lane < kTile && mine >= first && mine < last) page = table[mine / c.page_size];
        const bool there = page >= 0 && page < c.n_pages;
        const long long place = mine % c.page_size;
        const long long at_k = there ? page * c.k_page + place * c.k_token : 0, at_v = there ? page * c.v_page + place * c.v_token : 0;
        const unsigned mask = __ballot_sync(~0u, there);
        if (lane == 0) masks[stage] = static_cast<int>(mask);
        const uint32_t to = base + stage * kStage;
#pragma unroll 1
        for (int i = 0; i < kTile * kPieces / 32; ++i) {
            const int piece = lane + 32 * i, row = piece / kPieces, column = piece % kPieces;
            const long long from_k = __shfl_sync(~0u, at_k, row), from_v = __shfl_sync(~0u, at_v, row);
            const bool inside = column < c.dim / kValues;
            const int bytes = inside && (mask >> row & 1) ? 16 : 0, more = inside ? column * kValues : 0;
            copy16(to + row * kPitch + column * 16, k + from_k + more, bytes);
            copy16(to + kSide + row * kPitch + column * 16, v + from_v + more, bytes);
        }
    }
};

__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename T> __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of 16-bit values (lane l: row l / 4, columns 2 (l % 4) and + 1), transposed
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    T v[2] = {from_float<T>(a), from_float<T>(b)};
    uint32_t r;
    memcpy(&r, v, 4);
    return r;
}
// the same, rounded toward 0
template <typename T> __device__ __forceinline__ uint32_t pack2_down(float a, float b) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <typename T> __device__ __forceinline__ void unpack2(uint32_t r, float &a, float &b) {
    T v[2];
    memcpy(v, &r, 4);
    a = to_float(v[0]);
    b = to_float(v[1]);
}

// Running softmax of up to 8 * kGroups query heads over a warp's tiles, on the tensor cores (16-bit caches). The tokens are the 16 rows
// of the scores' product and the values' columns those of the second one, so the query heads are the 8 columns: a key head serves 1 to 8
// query heads in most nets, and as rows of m16n8k16 they would leave half of it empty. Lane l holds, of a tile's scores, tokens l / 4
// and l / 4 + 8 of heads 2 (l % 4) and + 1; of a block of 16 value columns the same two heads of columns l / 4 and l / 4 + 8.
template <typename T, int kDim_, int kGroups_, int kStages_, int kBlocks_> struct TensorHeads {
    using Type = T;
    static constexpr int kDim = kDim_, kStages = kStages_, kGroups = kGroups_, kWarps = 4, kBlocks = kBlocks_;
    // fp16 weights are taken times 2^14, so that a weight of 2^-29 of the largest is still a normal number (sum and values carry the
    // same factor); what a weight loses when it is rounded to the cache's type goes into a second product. Both parts are above 0 where the
    // weight is (2^-38 of the largest at least), so that an infinite value stays one: times parts of both signs, or 0, it would be NaN.
    static constexpr float kLift = std::is_same<T, __half>::value ? 14.f : 0.f;
    static constexpr float kLeast = std::is_same<T, __half>::value ? 5.9604644775390625e-8f : 1.17549435e-38f;      // smallest fp16, smallest normal bf16
    static constexpr int kScratch = 4;

    float acc[kGroups][kDim / 16][4], top[kGroups][2], sum[kGroups][2], scale;
    uint32_t q[kGroups][kDim / 16][2];

    __device__ __forceinline__ void start(const AttnParams &p, int row, int head, int heads, int lane, float *) {
        const T *from = reinterpret_cast<const T *>(p.q) + row * p.q_row + head * p.q_head;
#pragma unroll
        for (int n = 0; n < kGroups; ++n) {
            const int r = n * 8 + lane / 4;
#pragma unroll
            for (int s = 0; s < kDim / 16; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int d = s * 16 + lane % 4 * 2 + i * 8;
                    T v[2] = {from_float<T>(0.f), from_float<T>(0.f)};
                    if (r < heads && d < p.c.dim) { v[0] = from[r * p.q_head + d]; v[1] = from[r * p.q_head + d + 1]; }
                    memcpy(&q[n][s][i], v, 4);
                }
#pragma unroll
            for (int s = 0; s < kDim / 16; ++s) acc[n][s][0] = acc[n][s][1] = acc[n][s][2] = acc[n][s][3] = 0.f;
            top[n][0] = top[n][1] = -INFINITY;
            sum[n][0] = sum[n][1] = 0.f;
        }
        scale = p.scale * kLog2e;
    }
    __device__ __forceinline__ void tile(uint32_t keys, uint32_t values, int mask, int lane, int, float *) {
        constexpr int kPitch = Ring<T, kDim, kStages>::kPitch;
        // two sums, of even and odd steps: a product waits for the one before the last
        float s[kGroups][2][4] = {};
        const uint32_t at_k = keys + lane % 16 * kPitch + lane / 16 * 16;
#pragma unroll
        for (int i = 0; i < kDim / 16; ++i) {
            uint32_t a[4];
            ldmatrix(a, at_k + i * 32);
#pragma unroll
            for (int n = 0; n < kGroups; ++n) mma<T>(s[n][i % 2], a, q[n][i][0], q[n][i][1]);
        }
        uint32_t high[kGroups][2], low[kGroups][2];
        bool grown = false;
        float keep[kGroups][2];
#pragma unroll
        for (int n = 0; n < kGroups; ++n) {
            float base[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[n][0][i] = (s[n][0][i] + s[n][1][i]) * scale;
                if (mask != 0xffff && !(mask >> (lane / 4 + i / 2 * 8) & 1)) s[n][0][i] = -INFINITY;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float best = fmaxf(s[n][0][h], s[n][0][h + 2]);
#pragma unroll
                for (int o = 4; o < 32; o *= 2) best = fmaxf(best, __shfl_xor_sync(~0u, best, o));
                best = fmaxf(best, top[n][h]);
                base[h] = best == -INFINITY ? 0.f : best - kLift;
                keep[n][h] = best == top[n][h] ? 1.f : pow2(top[n][h] - best);
                grown |= best != top[n][h];
                top[n][h] = best;
            }
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pow2(s[n][0][i] - base[i % 2]);
#pragma unroll
            for (int h = 0; h < 2; ++h) sum[n][h] = sum[n][h] * keep[n][h] + (w[h] + w[h + 2]);
#pragma unroll
            for (int t = 0; t < 2; ++t) {                        // tokens l / 4 (+ 8): two heads of a token to two tokens of a head
                const uint32_t pair = pack2_down<T>(w[2 * t], w[2 * t + 1]);
                float a, b;
                unpack2<T>(pair, a, b);
                high[n][t] = transposed(pair);
                low[n][t] = transposed(pack2<T>(a > 0.f ? fmaxf(w[2 * t] - a, kLeast) : w[2 * t] - a, b > 0.f ? fmaxf(w[2 * t + 1] - b, kLeast) : w[2 * t + 1] - b));
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
        const uint32_t at_v = values + (lane / 16 * 8 + lane % 8) * kPitch + lane / 8 % 2 * 16;
#pragma unroll
        for (int i = 0; i < kDim / 16; ++i) {
            uint32_t a[4];
            ldmatrix_trans(a, at_v + i * 32);
#pragma unroll
            for (int n = 0; n < kGroups; ++n) {
                mma<T>(acc[n][i], a, high[n][0], high[n][1]);
                mma<T>(acc[n][i], a, low[n][0], low[n][1]);
            }
        }
    }
    // done(head, maximum without the lift, sum) once for every head, which gives the factor of its values; then put(head, d, value)
    template <typename Done, typename Put> __device__ __forceinline__ void finish(int heads, int dim, int lane, Done done, Put put) {
#pragma unroll
        for (int n = 0; n < kGroups; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int o = 4; o < 32; o *= 2) sum[n][h] += __shfl_xor_sync(~0u, sum[n][h], o);
                const int head = n * 8 + lane % 4 * 2 + h;
                if (head >= heads) continue;
                const float f = done(head, top[n][h] - kLift, sum[n][h], lane < 4);
#pragma unroll
                for (int i = 0; i < kDim / 16; ++i)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int d = i * 16 + r * 8 + lane / 4;
                        if (d < dim) put(head, d, acc[n][i][2 * r + h] * f);
                    }
            }
    }
};

// The same on the CUDA cores (fp32 caches), for up to kHeads query heads. Scores: two lanes a token, half of its values each; values:
// kDim / 32 columns a lane.
template <int kDim_, int kHeads_, int kStages_, int kWarps_> struct PlainHeads {
    using Type = float;
    static constexpr int kDim = kDim_, kStages = kStages_, kWarps = kWarps_, kHeads = kHeads_, kBlocks = 1;
    static constexpr int kColumns = kDim / 32, kVec = kColumns % 4 == 0 ? 4 : kColumns % 2 == 0 ? 2 : 1;

    float acc[kHeads][kColumns], top[kHeads], sum[kHeads];

    // scratch of a warp: the queries [kHeads][kDim], then a tile's weights [kHeads][16]
    static constexpr int kScratch = kHeads * (kDim + kTile);
    __device__ __forceinline__ void start(const AttnParams &p, int row, int head, int heads, int lane, float *scratch) {
        const float *from = reinterpret_cast<const float *>(p.q) + row * p.q_row + head * p.q_head;
        const float scale = p.scale * kLog2e;
        for (int i = lane; i < kHeads * kDim; i += 32) {
            const int r = i / kDim, d = i % kDim;
            scratch[i] = r < heads && d < p.c.dim ? from[r * p.q_head + d] * scale : 0.f;
        }
        __syncwarp();
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            top[h] = -INFINITY;
            sum[h] = 0.f;
#pragma unroll
            for (int i = 0; i < kColumns; ++i) acc[h][i] = 0.f;
        }
    }
    static __device__ __forceinline__ float4 load4(uint32_t at) {
        float4 v;
        asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
        return v;
    }
    __device__ __forceinline__ void tile(uint32_t keys, uint32_t values, int mask, int lane, int, float *scratch) {
        constexpr int kPitch = Ring<float, kDim, kStages>::kPitch;
        float *weights = scratch + kHeads * kDim;
        const float4 *q = reinterpret_cast<const float4 *>(scratch) + lane / 16 * (kDim / 8);
        float s[kHeads] = {};
        const uint32_t at_k = keys + lane % 16 * kPitch + lane / 16 * (kDim * 2);
#pragma unroll 4
        for (int i = 0; i < kDim / 8; ++i) {
            const float4 k = load4(at_k + i * 16);
#pragma unroll
            for (int h = 0; h < kHeads; ++h) {
                const float4 w = q[h * (kDim / 4) + i];
                s[h] = fmaf(w.x, k.x, fmaf(w.y, k.y, fmaf(w.z, k.z, fmaf(w.w, k.w, s[h]))));
            }
        }
        bool grown = false;
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            s[h] += __shfl_xor_sync(~0u, s[h], 16);
            if (!(mask >> (lane % 16) & 1)) s[h] = -INFINITY;
            float best = s[h];
#pragma unroll
            for (int o = 8; o; o >>= 1) best = fmaxf(best, __shfl_xor_sync(~0u, best, o));
            best = fmaxf(best, top[h]);
            const float base = best == -INFINITY ? 0.f : best;
            const float keep = best == top[h] ? 1.f : pow2(top[h] - base), weight = pow2(s[h] - base);
            grown |= keep != 1.f;
            sum[h] = sum[h] * keep + (lane < 16 ? weight : 0.f);
            top[h] = best;
            if (lane < 16) weights[h * kTile + lane] = weight;
            if (grown) {
#pragma unroll
                for (int i = 0; i < kColumns; ++i) acc[h][i] *= keep;
            }
        }
        __syncwarp();
#pragma unroll
        for (int four = 0; four < kTile; four += 4) {
            float4 w[kHeads];
#pragma unroll
            for (int h = 0; h < kHeads; ++h) w[h] = *reinterpret_cast<const float4 *>(weights + h * kTile + four);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                float v[kColumns];
#pragma unroll
                for (int i = 0; i < kColumns / kVec; ++i) {
                    const uint32_t at = values + (four + t) * kPitch + (i * 32 + lane) * kVec * 4;
                    if constexpr (kVec == 4) {
                        const float4 x = load4(at);
                        v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
                    } else if constexpr (kVec == 2) {
                        asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v[2 * i]), "=f"(v[2 * i + 1]) : "r"(at) : "memory");
                    } else {
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[i]) : "r"(at) : "memory");
                    }
                }
#pragma unroll
                for (int h = 0; h < kHeads; ++h) {
                    const float x = t == 0 ? w[h].x : t == 1 ? w[h].y : t == 2 ? w[h].z : w[h].w;
#pragma unroll
                    for (int i = 0; i < kColumns; ++i) acc[h][i] = fmaf(x, v[i], acc[h][i]);
                }
            }
        }
    }
    template <typename Done, typename Put> __device__ __forceinline__ void finish(int heads, int dim, int lane, Done done, Put put) {
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
#pragma unroll
            for (int o = 8; o; o >>= 1) sum[h] += __shfl_xor_sync(~0u, sum[h], o);
            const float whole = __shfl_sync(~0u, sum[h], 0);      // (the lanes from 16 on have no weights)
            if (h >= heads) continue;
            const float f = done(h, top[h], whole, lane == 0);
#pragma unroll
            for (int i = 0; i < kColumns / kVec; ++i)
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    const int d = (i * 32 + lane) * kVec + j;
                    if (d < dim) put(h, d, acc[h][i * kVec + j] * f);
                }
        }
    }
};

// What a block keeps beside its rings.
template <typename Heads> struct Side {
    int prefix[kMaxRows + 1];                                    // the line's tiles before each row
    int seq[kMaxRows], first[kMaxRows], last[kMaxRows];
    int warp_sum[Heads::kWarps];
    __align__(16) float scratch[Heads::kWarps][Heads::kScratch];
    int masks[Heads::kWarps][Heads::kStages];
};

// A warp's walk along its share: pieces of pairs, one after the other.
template <typename Heads> struct Walk {
    const AttnParams &p;
    const Side<Heads> &side;
    int left;                                                    // of the share
    int row, pair, pairs, at, length;                            // where it stands: row (of the launch), pair, tile of the line within it
    int worker;

    __device__ __forceinline__ int length_of(int r) const { return p.whole ? 1 : (side.last[r] - 1) / kTile - side.first[r] / kTile + 1 + kStart; }
    // tiles [begin, end) of the row's tiles; slot of the workspace or -1
    struct Piece { int row, pair, begin, end, slot; };
    __device__ __forceinline__ bool next(Piece &piece) {
        while (left > 0) {
            const int to = min(length, at + left);
            piece.row = row;
            piece.pair = pair;
            if (p.whole) {
                piece.begin = 0;
                piece.end = (side.last[row] - 1) / kTile - side.first[row] / kTile + 1;
                piece.slot = -1;
            } else {
                piece.begin = max(0, at - kStart);
                piece.end = to - kStart;
                piece.slot = piece.begin == 0 && to == length ? -1 : 2 * worker + (piece.begin == 0);
            }
            left -= to - at;
            at = 0;
            if (++pair == pairs) {
                pair = 0;
                do ++row; while (row < p.rows && side.prefix[row + 1] == side.prefix[row]);
                if (row < p.rows) length = length_of(row); else left = 0;
            }
            if (piece.end > piece.begin) return true;
        }
        return false;
    }
};

template <typename Heads>
__global__ void __launch_bounds__(Heads::kWarps * 32, Heads::kBlocks) attn_decode_kernel(const __grid_constant__ AttnParams p) {
    using T = typename Heads::Type;
    using R = Ring<T, Heads::kDim, Heads::kStages>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Side<Heads> side;
    constexpr int kWarps = Heads::kWarps, kThreads = kWarps * 32, kStages = Heads::kStages;
    pdl_enter();
    const int pairs = p.c.heads * p.chunks, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int line = 0;
    for (int base = 0; base < p.rows; base += kThreads) {
        const int i = base + threadIdx.x;
        Row r = {0, 0, 0};
        if (i < p.rows) {
            r = row_of(p, p.first_row + i);
            side.seq[i] = r.seq;
            side.first[i] = r.first;
            side.last[i] = r.last;
        }
        const int tiles = tiles_of(r);
        const int mine = tiles == 0 ? 0 : (p.whole ? 1 : tiles + kStart) * pairs;
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int below = __shfl_up_sync(~0u, sum, o);
            if (lane >= o) sum += below;
        }
        if (lane == 31) side.warp_sum[warp] = sum;
        __syncthreads();
        int before = line;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += side.warp_sum[w];
            line += side.warp_sum[w];
        }
        if (i < p.rows) side.prefix[i] = before + sum - mine;
        __syncthreads();
    }
    if (threadIdx.x == 0) side.prefix[p.rows] = line;
    __syncthreads();
    if (!p.whole && blockIdx.x == 0)
        for (int i = threadIdx.x; i <= p.rows; i += kThreads) p.prefix[i] = side.prefix[i];
    for (int i = blockIdx.x; i < p.rows; i += gridDim.x)
        if (side.prefix[i + 1] == side.prefix[i]) {              // a row without a token
            for (int d = threadIdx.x; d < p.n_heads * p.c.dim; d += kThreads)
                reinterpret_cast<T *>(p.out)[(p.first_row + i) * p.out_row + d / p.c.dim * p.out_head + d % p.c.dim] = from_float<T>(0.f);
            if (p.lse)
                for (int d = threadIdx.x; d < p.n_heads; d += kThreads) p.lse[(p.first_row + i) * static_cast<long long>(p.n_heads) + d] = -INFINITY;
        }
    // the share; neighbours in the line are in different blocks, so that a short line is spread over the SMs
    const int workers = gridDim.x * kWarps, worker = warp * gridDim.x + blockIdx.x;
    const int share = p.whole ? (line + workers - 1) / workers : share_of(line, workers), unit = worker * share;
    if (unit >= line) return;
    int low = 0;                                                 // the last row that begins at or before the share
    for (int step = kMaxRows / 32; step; step = step == kMaxRows / 32 ? 1 : 0) {
        const int r = low + lane * step;
        const unsigned before = __ballot_sync(~0u, r < p.rows && side.prefix[r] <= unit && (step > 1 || lane < kMaxRows / 32));
        low += (31 - __clz(before)) * step;
    }
    Walk<Heads> ahead = {p, side, min(share, line - unit), low, 0, pairs, 0, 0, worker};
    ahead.length = ahead.length_of(low);
    ahead.pair = (unit - side.prefix[low]) / ahead.length;
    ahead.at = unit - side.prefix[low] - ahead.pair * ahead.length;
    Walk<Heads> walk = ahead;

    // the copies' side: the piece they are at, its next tile, and a lane's page of one of the next 32 tiles
    typename Walk<Heads>::Piece from;
    R ring = {p.c, nullptr, nullptr, nullptr, side.masks[warp], static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * R::kBytes, 0, 0, lane};
    int tile = 0, tiles = 0, origin = 0, low_page = -1, high_page = -1, next_low = -1, next_high = -1, filled = 0, queued = 0;
    const auto pages_from = [&](int first_tile) {
        next_low = next_high = -1;
        if (first_tile + lane < tiles) {
            const int token = origin + (first_tile + lane) * kTile;
            next_low = ring.page_of(token);
            next_high = ring.page_of(token + 8);
        }
    };
    const auto advance = [&] {                                   // to the next piece; its pages are on their way when this returns
        if (!ahead.next(from)) { tiles = 0; return; }
        const int kv = from.pair / p.chunks;
        ring.k = reinterpret_cast<const T *>(p.c.k) + kv * p.c.k_head;
        ring.v = reinterpret_cast<const T *>(p.c.v) + kv * p.c.v_head;
        ring.table = p.c.table + side.seq[from.row] * p.c.table_stride;
        ring.first = side.first[from.row];
        ring.last = side.last[from.row];
        origin = (ring.first / kTile + from.begin) * kTile;
        tile = 0;
        tiles = from.end - from.begin;
        pages_from(0);
    };
    const auto copy_next = [&] {
        if (tile >= tiles) return;
        if (tile % 32 == 0) {
            low_page = next_low;
            high_page = next_high;
            if (tile + 32 < tiles) pages_from(tile + 32);
        }
        const int a = __shfl_sync(~0u, low_page, tile % 32), b = __shfl_sync(~0u, high_page, tile % 32);
        if ((a | b) >= 0) ring.issue(filled, origin + tile * kTile, a, b);
        else ring.issue_any(filled, origin + tile * kTile);
        copy_commit();
        filled = filled == kStages - 1 ? 0 : filled + 1;
        ++queued;
        if (++tile == tiles) advance();
    };
    advance();
    typename Walk<Heads>::Piece piece;
    int stage = 0;
    bool more = walk.next(piece);
    while (more) {
        const int kv = piece.pair / p.chunks, chunk = piece.pair % p.chunks, head = kv * p.each + chunk * p.chunk, heads = min(p.chunk, p.each - chunk * p.chunk);
        const int row = p.first_row + piece.row;
        Heads h;
        h.start(p, row, head, heads, lane, side.scratch[warp]);
        for (int left = piece.end - piece.begin; left > 0;) {
            // kStages - 1 tiles on their way before the first of them is waited for (the one of the last turn has been read by then)
            if (queued == kStages - 1) copy_wait<kStages - 2>();
            else if (tile >= tiles) copy_wait<0>();
            __syncwarp();
            const bool ready = queued == kStages - 1 || tile >= tiles;
            copy_next();
            if (!ready) continue;
            const uint32_t keys = ring.base + stage * R::kStage;
            h.tile(keys, keys + R::kSide, ring.masks[stage], lane, p.c.dim, side.scratch[warp]);
            stage = stage == kStages - 1 ? 0 : stage + 1;
            --queued;
            --left;
        }
        if (piece.slot >= 0) {
            const long long at = static_cast<long long>(piece.slot) * p.chunk;
            h.finish(heads, p.c.dim, lane,
                     [&](int i, float top, float sum, bool writes) { if (writes) p.part_ml[at + i] = make_float2(top, sum); return 1.f; },
                     [&](int i, int d, float v) { p.part[(at + i) * p.c.dim + d] = v; });
        } else {
            T *out = reinterpret_cast<T *>(p.out) + row * p.out_row + head * p.out_head;
            h.finish(heads, p.c.dim, lane,
                     [&](int i, float top, float sum, bool writes) {
                         if (p.lse && writes) p.lse[row * static_cast<long long>(p.n_heads) + head + i] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
                         return sum == 0.f ? 0.f : 1.f / sum;     // (a sum of 0: no token was left; the output is 0)
                     },
                     [&](int i, int d, float v) { out[i * p.out_head + d] = from_float<T>(v); });
        }
        more = walk.next(piece);
    }
}

constexpr int kJoinFew = 128, kJoinMany = 1024;                // threads of a joining block

// A block a (row, query head): the parts of a pair that was cut, in the order of the tokens. Each warp has every fourth or 32nd part,
// a lane four columns of up to two blocks of 128.
template <typename T, int kJoinThreads>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const __grid_constant__ AttnParams p, int workers) {
    constexpr int kWarps = kJoinThreads / 32;
    __shared__ float4 values[kWarps][64];
    __shared__ float2 state[kWarps];
    pdl_enter();
    const int row = blockIdx.x, head = blockIdx.y, kv = head / p.each, chunk = head % p.each / p.chunk, in_chunk = head % p.each % p.chunk;
    const int pairs = p.c.heads * p.chunks, dim = p.c.dim;
    const int before = p.prefix[row], after = p.prefix[row + 1], line = p.prefix[p.rows], length = (after - before) / pairs;
    if (length == 0) return;
    const int share = share_of(line, workers), unit = before + (kv * p.chunks + chunk) * length;
    const int first = (unit + kStart) / share, last = (unit + length - 1) / share;
    if (first == last) return;                                   // (finished by its warp)
    const int parts = last - first + 1, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    float top = -INFINITY, sum = 0.f;
    float4 acc[2] = {};
#pragma unroll 4
    for (int i = warp; i < parts; i += kWarps) {
        const long long at = static_cast<long long>(2 * (first + i) + (i == 0)) * p.chunk + in_chunk;
        const float2 one = p.part_ml[at];
        const float *from = p.part + at * dim;
        float4 v[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) v[c] = c * 128 + lane * 4 < dim ? *reinterpret_cast<const float4 *>(from + c * 128 + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float best = fmaxf(top, one.x), base = best == -INFINITY ? 0.f : best, keep = pow2(top - base), f = pow2(one.x - base);
        sum = sum * keep + one.y * f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            acc[c].x = acc[c].x * keep + v[c].x * f;
            acc[c].y = acc[c].y * keep + v[c].y * f;
            acc[c].z = acc[c].z * keep + v[c].z * f;
            acc[c].w = acc[c].w * keep + v[c].w * f;
        }
        top = best;
    }
    if (lane == 0) state[warp] = make_float2(top, sum);
#pragma unroll
    for (int c = 0; c < 2; ++c) values[warp][c * 32 + lane] = acc[c];
    __syncthreads();
    top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, state[w].x);
    const float base = top == -INFINITY ? 0.f : top;
    float factor[kWarps];
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) { factor[w] = pow2(state[w].x - base); sum += state[w].y * factor[w]; }
    const long long out_row = p.first_row + row;
    for (int d = threadIdx.x; d < dim; d += kJoinThreads) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += reinterpret_cast<const float *>(values[w])[d] * factor[w];
        reinterpret_cast<T *>(p.out)[out_row * p.out_row + head * p.out_head + d] = from_float<T>(sum == 0.f ? 0.f : v / sum);
    }
    if (p.lse && threadIdx.x == 0) p.lse[out_row * p.n_heads + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// How a call is cut up: query heads of a pair, warps, slots of the workspace.
struct AttnPlan {
    int each, chunk, chunks, rows, blocks, workers, whole;       // rows: of a launch
    long long tiles;                                             // of a row at most
    size_t ml_at, part_at, bytes;
};

struct BlockShape { int warps, of_sm; };
BlockShape block_shape(int dtype, int dim) {
    return dtype == MSNH_B200_F32 ? BlockShape{dim <= 128 ? 4 : 2, 1} : BlockShape{4, dim <= 128 ? 2 : 1};
}

AttnPlan plan_of(const MsnhB200Ctx *ctx, const MsnhB200KvCache &c, const MsnhB200AttnDecode &a) {
    AttnPlan l = {};
    l.each = a.n_heads / c.n_kv_heads;
    l.chunk = std::min(l.each, c.dtype == MSNH_B200_F32 ? 8 : 16);
    l.chunks = (l.each + l.chunk - 1) / l.chunk;
    const BlockShape shape = block_shape(c.dtype, c.head_dim);
    const long long blocks = static_cast<long long>(ctx->sm_count) * shape.of_sm;
    const long long most_tokens = static_cast<long long>(c.max_pages) * c.page_size, seen = a.window > 0 ? std::min<long long>(most_tokens, a.window) : most_tokens;
    const long long tiles = (seen + kTile - 1) / kTile + (a.window > 0);        // (a window may start inside a tile)
    l.tiles = tiles;
    l.whole = tiles <= kWholeTiles;
    const long long row_tiles = (tiles + kStart) * c.n_kv_heads * l.chunks;
    l.rows = static_cast<int>(std::min<long long>(std::min(a.rows, kMaxRows), ((1LL << 30) - 1) / row_tiles));
    if (l.rows == 0) return l;                                   // (a row alone is too long)
    const long long pairs = static_cast<long long>(l.rows) * c.n_kv_heads * l.chunks;
    l.blocks = static_cast<int>(std::min(l.whole ? pairs : pairs * tiles, blocks));
    l.workers = l.blocks * shape.warps;
    if (!l.whole) {
        l.ml_at = (static_cast<size_t>(l.rows + 1) * 4 + 15) / 16 * 16;
        l.part_at = (l.ml_at + static_cast<size_t>(l.workers) * 2 * l.chunk * sizeof(float2) + 15) / 16 * 16;
        l.bytes = l.part_at + static_cast<size_t>(l.workers) * 2 * l.chunk * c.head_dim * 4;
    }
    return l;
}

template <typename Heads>
cudaError_t launch(const MsnhB200Ctx *ctx, const AttnParams &p, int blocks, void *stream) {
    // the attribute is a kernel's and a device's: set by the first call there
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (!(done.load(std::memory_order_acquire) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(attn_decode_kernel<Heads>, cudaFuncAttributeMaxDynamicSharedMemorySize, Heads::kWarps * Ring<typename Heads::Type, Heads::kDim, Heads::kStages>::kBytes);
        if (e != cudaSuccess) return e;
        done.fetch_or(bit, std::memory_order_release);
    }
    return launch_token_kernel(attn_decode_kernel<Heads>, dim3(blocks), Heads::kWarps * 32, Heads::kWarps * Ring<typename Heads::Type, Heads::kDim, Heads::kStages>::kBytes, stream, ctx->pdl, p);
}

// Ring depths and blocks of an SM: as far as the shared memory goes.
template <typename T>
cudaError_t launch16(const MsnhB200Ctx *ctx, const AttnParams &p, int blocks, void *stream) {
    const bool few = p.chunk <= 8;
    if (p.c.dim <= 32) return few ? launch<TensorHeads<T, 32, 1, 8, 2>>(ctx, p, blocks, stream) : launch<TensorHeads<T, 32, 2, 8, 2>>(ctx, p, blocks, stream);
    if (p.c.dim <= 64) return few ? launch<TensorHeads<T, 64, 1, 5, 2>>(ctx, p, blocks, stream) : launch<TensorHeads<T, 64, 2, 5, 2>>(ctx, p, blocks, stream);
    if (p.c.dim <= 96) return few ? launch<TensorHeads<T, 96, 1, 4, 2>>(ctx, p, blocks, stream) : launch<TensorHeads<T, 96, 2, 4, 2>>(ctx, p, blocks, stream);
    if (p.c.dim <= 128) return few ? launch<TensorHeads<T, 128, 1, 3, 2>>(ctx, p, blocks, stream) : launch<TensorHeads<T, 128, 2, 3, 2>>(ctx, p, blocks, stream);
    if (p.c.dim <= 192) return few ? launch<TensorHeads<T, 192, 1, 4, 1>>(ctx, p, blocks, stream) : launch<TensorHeads<T, 192, 2, 4, 1>>(ctx, p, blocks, stream);
    return few ? launch<TensorHeads<T, 256, 1, 3, 1>>(ctx, p, blocks, stream) : launch<TensorHeads<T, 256, 2, 3, 1>>(ctx, p, blocks, stream);
}
template <int kHeads>
cudaError_t launch32(const MsnhB200Ctx *ctx, const AttnParams &p, int blocks, void *stream) {
    if (p.c.dim <= 32) return launch<PlainHeads<32, kHeads, 8, 4>>(ctx, p, blocks, stream);
    if (p.c.dim <= 64) return launch<PlainHeads<64, kHeads, 5, 4>>(ctx, p, blocks, stream);
    if (p.c.dim <= 96) return launch<PlainHeads<96, kHeads, 4, 4>>(ctx, p, blocks, stream);
    if (p.c.dim <= 128) return launch<PlainHeads<128, kHeads, 3, 4>>(ctx, p, blocks, stream);
    if (p.c.dim <= 192) return launch<PlainHeads<192, kHeads, 3, 2>>(ctx, p, blocks, stream);
    return launch<PlainHeads<256, kHeads, 3, 2>>(ctx, p, blocks, stream);
}

// The parts of a pair in a full table: as many as there are shares of its tiles, or as it has warps to itself. Parts that few warps take turns
// at cost more than starting 32 warps does from kManyParts on: with 74 and 148 parts a pair 101 against 97 us (2 rows of 60000 fp16 tokens)
// and 47.5 against 34.8 (one of 30000), with 51 as much either way (one of 4000: 15.6 and 14.8), with 9 and 7 the other way round (16 rows
// of 4000: 56 against 72; one of 500: 10.9 against 13.6). It is an estimate, since the host does not know the lengths. A pair can have more
// parts: beside 63 rows of 100 tokens one of 65536 has some 147, which few warps join in no more time (75 against 92 us); and fewer: of one
// row of 37 or 500 tokens in a table of 4096 few warps would be through in 9.4 and 10.9 us instead of 12.1 and 13.7.
constexpr int kManyParts = 32;
template <typename T>
cudaError_t launch_join(const MsnhB200Ctx *ctx, const AttnParams &p, int workers, long long tiles, void *stream) {
    const dim3 grid(p.rows, p.n_heads);
    const long long parts = std::min<long long>(workers / (static_cast<long long>(p.rows) * p.c.heads * p.chunks), (tiles + kStart) / (kStart + kLeast));
    return parts < kManyParts ? launch_token_kernel(attn_join_kernel<T, kJoinFew>, grid, kJoinFew, 0, stream, ctx->pdl, p, workers)
                              : launch_token_kernel(attn_join_kernel<T, kJoinMany>, grid, kJoinMany, 0, stream, ctx->pdl, p, workers);
}

int check_attn(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, const MsnhB200AttnDecode *a, const char *what) {
    if (const int rc = check_cache(ctx, c, false, what)) return rc;
    if (a->rows < 0 || a->n_heads < 1 || a->n_heads > 65535 || a->n_heads % c->n_kv_heads) return fail(ctx, MSNH_B200_ERR_ARG, "%s: %d rows, %d heads over %d kv heads", what, a->rows, a->n_heads, c->n_kv_heads);
    if (a->window < 0) return fail(ctx, MSNH_B200_ERR_ARG, "%s: a window of %d", what, a->window);
    if (c->head_dim > 256 || c->head_dim * dtype_size(c->dtype) % 16) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "%s: heads of %d values (a multiple of 16 bytes and at most 256 values are wanted)", what, c->head_dim);
    if (!kv_rows_multiple_of(*c, 16)) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "%s: the cache's rows are not 16-byte aligned", what);
    if (!a->seqs && a->rows > c->n_seqs) return fail(ctx, MSNH_B200_ERR_ARG, "%s: %d rows of %d sequences", what, a->rows, c->n_seqs);
    if (a->rows && plan_of(ctx, *c, *a).rows == 0) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "%s: a row of 2^34 and more tokens times heads", what);
    return MSNH_B200_OK;
}

}  // namespace
}  // namespace msnh

using namespace msnh;

extern "C" {

int msnh_b200_attn_decode_workspace(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, const MsnhB200AttnDecode *a, size_t *bytes) try {
    if (!ctx || !c || !a || !bytes) return MSNH_B200_ERR_ARG;
    if (const int rc = check_attn(ctx, c, a, "attn_decode_workspace")) return rc;
    *bytes = a->rows ? plan_of(ctx, *c, *a).bytes : 0;
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

int msnh_b200_attn_decode(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, const MsnhB200AttnDecode *a, void *stream) try {
    if (!ctx || !c || !a) return MSNH_B200_ERR_ARG;
    if (const int rc = check_attn(ctx, c, a, "attn_decode")) return rc;
    if (a->rows == 0) return MSNH_B200_OK;
    if (!a->q || !a->out) return fail(ctx, MSNH_B200_ERR_ARG, "attn_decode: null q or out");
    if (a->q_row_stride < 0 || a->q_head_stride < 0 || (a->n_heads > 1 && a->out_head_stride < c->head_dim) || (a->rows > 1 && a->out_row_stride < c->head_dim))
        return fail(ctx, MSNH_B200_ERR_ARG, "attn_decode: a stride of q is negative, or rows of out overlap");
    const AttnPlan l = plan_of(ctx, *c, *a);
    if (l.bytes && (!a->workspace || a->workspace_bytes < l.bytes || !aligned16(a->workspace)))
        return fail(ctx, MSNH_B200_ERR_ARG, "attn_decode: %zu bytes of workspace, 16-byte aligned, are wanted", l.bytes);
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    uint8_t *work = static_cast<uint8_t *>(a->workspace);
    AttnParams p = {kv_params(*c), static_cast<const uint8_t *>(a->q), static_cast<uint8_t *>(a->out), a->lse, a->seqs, a->q_row_stride, a->q_head_stride,
                    a->out_row_stride, a->out_head_stride, 0, a->n_heads, l.each, l.chunk, l.chunks, a->window, 0, l.whole, a->scale,
                    reinterpret_cast<int *>(work), reinterpret_cast<float2 *>(work + l.ml_at), reinterpret_cast<float *>(work + l.part_at)};
    for (int row = 0; row < a->rows; row += l.rows) {
        p.first_row = row;
        p.rows = std::min(l.rows, a->rows - row);
        cudaError_t e;
        if (c->dtype == MSNH_B200_F32)
            e = l.chunk == 1 ? launch32<1>(ctx, p, l.blocks, stream) : l.chunk <= 4 ? launch32<4>(ctx, p, l.blocks, stream)
                                                                                           : launch32<8>(ctx, p, l.blocks, stream);
        else
            e = c->dtype == MSNH_B200_F16 ? launch16<__half>(ctx, p, l.blocks, stream) : launch16<__nv_bfloat16>(ctx, p, l.blocks, stream);
        CUDA_TRY(ctx, e);
        if (l.whole) continue;
        e = c->dtype == MSNH_B200_F32 ? launch_join<float>(ctx, p, l.workers, l.tiles, stream) : c->dtype == MSNH_B200_F16 ? launch_join<__half>(ctx, p, l.workers, l.tiles, stream)
                                                                                                                 : launch_join<__nv_bfloat16>(ctx, p, l.workers, l.tiles, stream);
        CUDA_TRY(ctx, e);
    }
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

}  // extern "C"
