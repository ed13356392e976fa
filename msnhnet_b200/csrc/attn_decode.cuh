// What the kernels of attention over a paged cache share (attn_decode.cu: 16 and 32 bits, attn_codes.cu: 8 bits): the line of tiles, a warp's
// ring of tiles, its walk along its share, and the kernel around a type `Heads` that keeps the running softmax of a pair's query heads.
#pragma once
#include "kv_cache.h"
#include "token_types.cuh"

namespace msnh {
namespace attn {

constexpr int kMaxRows = 256;                // rows of a launch: what they see is kept in shared memory
// Tiles that a pair's start counts for, and the smallest share, a start and two tiles, where there are as many. fp16, 32 heads over 8, with kStart 1, 3 and
// 6: one row of 500 tokens 9.7, 10.8 and 13.1 us, 16 of them 17.2, 16.5 and 18.0, one of 65536 beside 63 of 100 76.7, 75.2 and 75.7, one of 4000 14.2,
// 14.8 and 16.1; 16 of 4000 and more tokens are the same within 1 %.
constexpr int kStart = 3, kSmallest = 5;
// The same of 8-bit codes, whose tiles are of 32 tokens. With a start of 1, 2, 3 and 5: 48 rows of up to 8192 tokens 37.9, 31.7, 31.7 and 31.7 us, five of up to
// 20000 25.2, 23.0, 23.2 and 26.5, 16 of up to 1000 15.2, 16.9, 17.6 and 18.4, one of 500 12.0, 12.1, 12.7 and 15.4, one of 65536 beside 63 of 100 65.8, 66.6, 62.5
// and 63.5. With one tile at least and a start of 2: 31.7, 23.1, 15.1, 11.2 and 65.2; four of up to 1418 with heads of 256 14.4 and not 16.0.
constexpr int kCodeStart = 2, kCodeSmallest = 3;
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
    int whole, start, smallest;                          // start: tiles that a pair's start counts for; smallest: share of a warp
    float scale;
    int *prefix;                                         // workspace: the line's tiles before each row (rows + 1), then the parts
    float2 *part_ml;                                     // [slot][chunk] maximum and sum
    float *part;                                         // [slot][chunk][dim]
    int wide_q;                                          // four values of a query, from every fourth one on, are aligned (8-bit caches)
};

struct Row { int seq, first, last; };
__device__ __forceinline__ Row row_of(const AttnParams &p, int row) {
    Row r;
    r.seq = p.seqs ? p.seqs[row] : row;
    r.last = r.seq >= 0 && r.seq < p.c.n_seqs ? max(0, min(p.c.lengths[r.seq], p.c.max_pages * p.c.page_size)) : 0;
    r.first = p.window > 0 ? max(0, r.last - p.window) : 0;
    return r;
}
template <int kTile> __device__ __forceinline__ int tiles_of(const Row &r) { return r.last > r.first ? (r.last - 1) / kTile - r.first / kTile + 1 : 0; }

// The share of a warp, in tiles of the line. (A launch's line has less than 2^30 tiles: code for longer ones is a microsecond of reading
// instructions alone.)
__device__ __forceinline__ int share_of(int line, int workers, int smallest) {
    return max((line + workers - 1) / workers, smallest);
}

// 16 bytes to shared memory, of which the first `bytes` are copied (16 or none) and the others are 0
__device__ __forceinline__ void copy16(uint32_t to, const void *from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void *from, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
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
    static constexpr int kTile = 16, kAhead = 32;                // tokens of a tile; tiles whose pages are looked up together
    static constexpr int kPitch = kDim * sizeof(T) + 16;
    static constexpr int kSide = kTile * kPitch, kStage = 2 * kSide, kBytes = kStages * kStage;
    static constexpr int kPieces = kDim * sizeof(T) / 16, kValues = 16 / sizeof(T);

    const KvParams &c;
    int *masks;                              // [kStages] bit t: token t of the tile takes part
    uint32_t base;
    int lane;
    const T *k = nullptr, *v = nullptr;      // of the key head
    const int *table = nullptr;              // of the sequence
    int first = 0, last = 0, origin = 0;     // tokens that are seen; token of the piece's first tile
    int low_page = -1, high_page = -1, next_low = -1, next_high = -1;         // a lane's pages of one of 32 tiles, and of one of the 32 behind them

    __device__ __forceinline__ Ring(const KvParams &c_, int *masks_, uint32_t base_, int lane_) : c(c_), masks(masks_), base(base_), lane(lane_) {}

    __device__ __forceinline__ void start(int head, const int *table_, int first_, int last_, int first_tile) {
        k = reinterpret_cast<const T *>(c.k) + head * c.k_head;
        v = reinterpret_cast<const T *>(c.v) + head * c.v_head;
        table = table_;
        first = first_;
        last = last_;
        origin = (first / kTile + first_tile) * kTile;
    }
    // Asks for the pages of the tiles from first_tile on.
    __device__ __forceinline__ void look_ahead(int first_tile, int tiles) {
        next_low = next_high = -1;
        if (first_tile + lane < tiles) {
            const int token = origin + (first_tile + lane) * kTile;
            next_low = page_of(token);
            next_high = page_of(token + 8);
        }
    }
    // What has been asked for is of the tiles from here on.
    __device__ __forceinline__ void take_pages(int) {
        low_page = next_low;
        high_page = next_high;
    }
    __device__ __forceinline__ void copy(int stage, int tile) const {
        const int a = __shfl_sync(~0u, low_page, tile % 32), b = __shfl_sync(~0u, high_page, tile % 32);
        if ((a | b) >= 0) issue(stage, origin + tile * kTile, a, b);
        else issue_any(stage, origin + tile * kTile);
    }

    // The page of a run of eight tokens that are all seen, in a cache whose pages are multiples of eight; -1 otherwise. (Tokens go to
    // 2^31 - 1: sums behind the last one would pass it.)
    __device__ __forceinline__ int page_of(int token) const {
        if (c.page_size % 8 || token < first || token > last - 8) return -1;
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
    static constexpr int kTile = Heads::Ring::kTile, kBegin = Heads::kBegin;
    const AttnParams &p;
    const Side<Heads> &side;
    int left;                                                    // of the share
    int row, pair, pairs, at, length;                            // where it stands: row (of the launch), pair, tile of the line within it
    int worker;

    __device__ __forceinline__ int length_of(int r) const { return p.whole ? 1 : (side.last[r] - 1) / kTile - side.first[r] / kTile + 1 + kBegin; }
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
                piece.begin = max(0, at - kBegin);
                piece.end = to - kBegin;
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
    using R = typename Heads::Ring;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Side<Heads> side;
    constexpr int kWarps = Heads::kWarps, kThreads = kWarps * 32, kStages = Heads::kStages;
    const bool early = Heads::kEarly || p.whole;                 // (nothing is joined after whole pairs)
    pdl_wait();
    if (early) pdl_launch_dependents();
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
        const int tiles = tiles_of<R::kTile>(r);
        const int mine = tiles == 0 ? 0 : (p.whole ? 1 : tiles + Heads::kBegin) * pairs;
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
    const int share = p.whole ? (line + workers - 1) / workers : share_of(line, workers, Heads::kSmallest), unit = worker * share;
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

    // the copies' side: the piece they are at, and its next tile
    typename Walk<Heads>::Piece from;
    R ring(p.c, side.masks[warp], static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * R::kBytes, lane);
    int tile = 0, tiles = 0, filled = 0, queued = 0;
    const auto advance = [&] {                                   // to the next piece; its pages are on their way when this returns
        if (!ahead.next(from)) { tiles = 0; return; }
        ring.start(from.pair / p.chunks, p.c.table + side.seq[from.row] * p.c.table_stride, side.first[from.row], side.last[from.row], from.begin);
        tile = 0;
        tiles = from.end - from.begin;
        ring.look_ahead(0, tiles);
    };
    const auto copy_next = [&] {
        if (tile >= tiles) return;
        if (tile % R::kAhead == 0) {
            ring.take_pages(tile);
            if (tile + R::kAhead < tiles) ring.look_ahead(tile + R::kAhead, tiles);
        }
        ring.copy(filled, tile);
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
    if (!early) pdl_launch_dependents();
}

template <typename Heads>
inline cudaError_t launch(const MsnhB200Ctx *ctx, const AttnParams &p, int blocks, void *stream) {
    // the attribute is a kernel's and a device's: set by the first call there
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (!(done.load(std::memory_order_acquire) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(attn_decode_kernel<Heads>, cudaFuncAttributeMaxDynamicSharedMemorySize, Heads::kWarps * Heads::Ring::kBytes);
        if (e != cudaSuccess) return e;
        done.fetch_or(bit, std::memory_order_release);
    }
    return launch_token_kernel(attn_decode_kernel<Heads>, dim3(blocks), Heads::kWarps * 32, Heads::kWarps * Heads::Ring::kBytes, stream, ctx->pdl, p);
}

struct BlockShape { int warps, of_sm; };
// Caches of 8-bit codes (attn_codes.cu): tokens of a tile; dtype: of queries and output.
constexpr int kCodeTile = 32;
BlockShape block_shape_codes(int dim, int chunk);         // chunk: query heads of a pair
int most_heads_codes(int dtype, int dim);                // of a pair
cudaError_t launch_codes(const MsnhB200Ctx *ctx, const AttnParams &p, int dtype, int blocks, void *stream);

}  // namespace attn
}  // namespace msnh
