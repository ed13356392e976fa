// Upkeep of a paged cache of keys and values: append, fork, free, compact, copy, read (msnh_b200_kv_*).
//
// Append, fork and compact are two launches: one block decides (which pages, in what order: the lowest free ones first, by a scan
// over the page counts, so the result does not depend on timing) and writes its decisions into the workspace, then a grid moves the
// rows. Every launch may be scheduled while the one before it runs, and waits for it (pdl_enter).
//
// The moves are bound by their bytes, read and written once: of the 28.1 us of a compaction of 6000 pages of 16 tokens, 8 heads, 128 fp16
// values (107 MB) they take 17 (6.3 TB/s). The rest is the deciding block: a few reads that wait for one another and two scans; it is
// one block because every page's place depends on all counts before it. A step of a beam search of 256 sequences (fork, append, free: five
// launches, 15.9 MB) takes 20 us, 4 a launch.
//
// In a cache of 8-bit codes append quantises: a block of tokens and head has one scale, a power of two, so that a scale can grow under older codes
// without a second rounding (a shift of their exponents; only codes below 2^-6 lose bits). Read is the way back, for any cache. Both are bound by their
// bytes, read and written once: prompts of 26200 bf16 tokens, 8 heads of 128 (161 MB) are written in 42 us (31 the codes' launch by itself, 5.2 TB/s; the deciding block
// is most of the rest) and read in 31.5 (5.1 TB/s).
#include "kv_cache.h"
#include "row_overlap.h"
#include "token_types.cuh"

namespace msnh {
namespace {

constexpr int kDecide = 1024;          // threads of the deciding block

// Exclusive sum over a block of kDecide threads; *total receives the whole sum. Ends with a barrier.
__device__ __forceinline__ int block_scan(int value, int *total) {
    __shared__ int warp_sum[32];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int sum = value;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int below = __shfl_up_sync(~0u, sum, o);
        if (lane >= o) sum += below;
    }
    __syncthreads();                                             // (the last call's sums have been read)
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kDecide / 32; ++w) {
        if (w < warp) before += warp_sum[w];
        all += warp_sum[w];
    }
    *total = all;
    return before + sum - value;
}

// Page counts of kEach pages from `first` on (1, a count that is none's business, beyond the last).
constexpr int kEach = 8;
__device__ __forceinline__ void load_refs(const KvParams &c, int first, int (&refs)[kEach]) {
    if (first + kEach <= c.n_pages && reinterpret_cast<uintptr_t>(c.refs) % 16 == 0) {
#pragma unroll
        for (int i = 0; i < kEach / 4; ++i) {
            const int4 v = reinterpret_cast<const int4 *>(c.refs + first)[i];
            refs[4 * i] = v.x; refs[4 * i + 1] = v.y; refs[4 * i + 2] = v.z; refs[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i) refs[i] = first + i < c.n_pages ? c.refs[first + i] : 1;
    }
}

// The `need` lowest free pages, in order, into list; returns how many there are of them (at most need). For the whole block.
__device__ int lowest_free(const KvParams &c, int need, int *list) {
    int found = 0;
    for (long long base = 0; base < c.n_pages && found < need; base += kDecide * kEach) {
        const int first = static_cast<int>(min(base + threadIdx.x * kEach, static_cast<long long>(c.n_pages)));
        int refs[kEach], mine = 0;
        load_refs(c, first, refs);
#pragma unroll
        for (int i = 0; i < kEach; ++i) mine += refs[i] == 0;
        int total, rank = found + block_scan(mine, &total);
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (refs[i] == 0) {
                if (rank < need) list[rank] = first + i;
                ++rank;
            }
        found += total;
    }
    __syncthreads();
    return min(found, need);
}

// What append decides for a sequence of the call.
struct AppendWork { int first, need, had, start, block; };       // first of its pages in the list; start: the length before, -1: refused;
                                                                 // block: the blocks of scales that sequences before it write to (codes only)

// What an append's kernels divide by.
struct AppendDivisors { Divisor heads, block, page; };

__global__ void kv_append_decide_kernel(KvParams c, const int *seqs, const int *starts, int n, int n_tokens, AppendWork *work, int *list, AppendDivisors by) {
    pdl_enter();
    int all = 0, all_blocks = 0;
    bool down = false;                                           // starts that are not in order: then no token's sequence is certain
    for (int base = 0; base < n; base += kDecide) {
        const int i = base + threadIdx.x;
        AppendWork w = {0, 0, 0, -1, 0};
        int blocks = 0;
        if (i < n) {
            const int s = seqs ? seqs[i] : i;
            const long long from = starts ? starts[i] : i, to = starts ? starts[i + 1] : i + 1;
            down |= to < from;
            if (s >= 0 && s < c.n_seqs && from >= 0 && to >= from && to <= n_tokens) {
                const int len = max(c.lengths[s], 0);
                if (len + to - from <= static_cast<long long>(c.max_pages) * c.page_size) {
                    const int after = static_cast<int>(len + to - from);
                    const auto pages_of = [&](int tokens) {
                        const int whole = by.page.quotient(tokens);
                        return whole + (whole * c.page_size < tokens);
                    };
                    const int had = pages_of(len);
                    w = {0, pages_of(after) - had, had, len, 0};
                    if (c.block && after > len) blocks = by.block.quotient(after - 1) - by.block.quotient(len) + 1;
                }
            }
        }
        int total;
        w.first = all + block_scan(w.need, &total);
        all += total;
        if (c.block && starts) {
            w.block = all_blocks + block_scan(blocks, &total);
            all_blocks += total;
        }
        if (i < n) work[i] = w;
    }
    const int found = lowest_free(c, all, list);
    if (starts) down = __syncthreads_or(down);
    for (int i = threadIdx.x; i < n; i += kDecide) {
        AppendWork w = work[i];
        if (w.start >= 0 && (down || (w.need > 0 && w.first + w.need > found))) work[i].start = w.start = -1;
        if (w.start < 0) { atomicAdd(c.refused, 1); continue; }
        const int s = seqs ? seqs[i] : i;
        c.lengths[s] = w.start + (starts ? starts[i + 1] - starts[i] : 1);
    }
    __syncthreads();
    // pages to their sequences: page r of the list belongs to the last sequence whose first is not above r
    for (int r = threadIdx.x; r < found; r += kDecide) {
        int low = 0, high = n - 1;
        while (low < high) {
            const int mid = (low + high + 1) / 2;
            if (work[mid].first <= r) low = mid; else high = mid - 1;
        }
        const AppendWork w = work[low];
        if (w.start < 0 || r >= w.first + w.need) continue;
        const int s = seqs ? seqs[low] : low;
        c.table[s * c.table_stride + w.had + r - w.first] = list[r];
        c.refs[list[r]] = 1;
    }
}

template <typename Unit>
__global__ void kv_append_write_kernel(KvParams c, const int *seqs, const int *starts, int n, int n_tokens, const AppendWork *work, const Unit *k_new,
                                       const Unit *v_new, long long token_stride, long long head_stride, int units) {
    pdl_enter();
    const int per_token = c.heads * units;
    const long long total = static_cast<long long>(n_tokens) * per_token;
    for (long long u = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; u < total; u += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int token = static_cast<int>(u / per_token), rest = static_cast<int>(u % per_token);
        const int head = rest / units, unit = rest % units;
        int i = token;
        if (starts) {                                            // the last sequence that starts at or before this token
            int low = 0, high = n - 1;
            while (low < high) {
                const int mid = (low + high + 1) / 2;
                if (starts[mid] <= token) low = mid; else high = mid - 1;
            }
            i = low;
            if (token < starts[i] || token >= starts[i + 1]) continue;
        }
        const int before = work[i].start;
        if (before < 0) continue;
        const int at = before + (starts ? token - starts[i] : 0);
        const int page = c.table[(seqs ? seqs[i] : i) * c.table_stride + at / c.page_size];
        if (page < 0 || page >= c.n_pages) continue;
        const int place = at % c.page_size;
        reinterpret_cast<Unit *>(c.k)[page * c.k_page + place * c.k_token + head * c.k_head + unit] = k_new[token * token_stride + head * head_stride + unit];
        reinterpret_cast<Unit *>(c.v)[page * c.v_page + place * c.v_token + head * c.v_head + unit] = v_new[token * token_stride + head * head_stride + unit];
    }
}

// The last of n sequences whose number at(i) is not above x, for a whole warp: at(0), at(1), ... do not fall. Always one of them.
template <typename At> __device__ __forceinline__ int last_not_above(int n, int x, int lane, At at) {
    int low = 0, range = n;
    while (range > 1) {
        const int step = (range + 31) / 32, probe = low + lane * step;
        const unsigned below = __ballot_sync(~0u, lane * step < range && at(probe) <= x);
        const int which = below ? 31 - __clz(below) : 0;
        low += which * step;
        range = min(step, range - which * step);
    }
    return low;
}

// (four values or eight: what 16 bytes of the new ones hold)
template <int kVec> __device__ __forceinline__ void store_codes(uint8_t *to, const float (&x)[kVec]) {
    uint32_t words[kVec / 4];
#pragma unroll
    for (int i = 0; i < kVec / 4; ++i) words[i] = to_e4m3x2(x[4 * i], x[4 * i + 1]) | static_cast<uint32_t>(to_e4m3x2(x[4 * i + 2], x[4 * i + 3])) << 16;
    if constexpr (kVec == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(words[0], words[1]);
    else *reinterpret_cast<uint32_t *>(to) = words[0];
}
// kVec values side by side, 16 bytes of them
template <typename T, int kVec> struct Piece {
    alignas(16) T v[kVec];
    __device__ __forceinline__ void load(const T *from) {
        *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(from);
    }
    // The larger one of `before` and the magnitudes' bits; 16-bit values in two halves, which last() joins.
    __device__ __forceinline__ uint32_t top(uint32_t before) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < kVec; ++i) before = max(before, __float_as_uint(v[i]) & 0x7fffffffu);
        } else {
#pragma unroll
            for (int i = 0; i < kVec / 2; ++i) before = __vmaxu2(before, reinterpret_cast<const uint32_t *>(v)[i] & 0x7fff7fffu);
        }
        return before;
    }
    // The largest magnitude as an fp32 number's bits.
    static __device__ __forceinline__ uint32_t last(uint32_t top) {
        if constexpr (sizeof(T) == 4) return top;
        const uint16_t bits = static_cast<uint16_t>(max(top & 0xffffu, top >> 16));
        return __float_as_uint(to_float(reinterpret_cast<const T &>(bits)));
    }
    // The same of what is finite.
    __device__ __forceinline__ uint32_t finite_top(uint32_t before) const {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const uint32_t bits = __float_as_uint(to_float(v[i])) & 0x7fffffffu;
            if (bits < 0x7f800000u) before = max(before, bits);
        }
        return before;
    }
    template <typename Code> __device__ __forceinline__ void store(uint8_t *to, Code code) const {
        float x[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) x[i] = code(to_float(v[i]));
        store_codes<kVec>(to, x);
    }
};
template <int kVec> struct Codes {
    alignas(8) __nv_fp8_e4m3 v[kVec];
    __device__ __forceinline__ void load(const uint8_t *from) {
        if constexpr (kVec == 8) *reinterpret_cast<uint2 *>(v) = *reinterpret_cast<const uint2 *>(from);
        else *reinterpret_cast<uint32_t *>(v) = *reinterpret_cast<const uint32_t *>(from);
    }
    template <typename Code> __device__ __forceinline__ void store(uint8_t *to, Code code) const {
        float x[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) x[i] = code(to_float(v[i]));
        store_codes<kVec>(to, x);
    }
};

// The smallest power of two by which a magnitude (its bits) is at most 448 = 1.75 * 2^8, from 2^-126 on; 0 for 0.
__device__ __forceinline__ float scale_of(uint32_t top) {
    if (top == 0) return 0.f;
    const int exponent = static_cast<int>((top + 0x1fffffu) >> 23) - 8;      // (biased; mantissas above 1.75 carry)
    return __uint_as_float(static_cast<uint32_t>(max(exponent, 1)) << 23);
}
// A block's scale from the one it has (the caller's own may be negative: it is as good as its magnitude) and the least one that its new values take.
__device__ __forceinline__ float larger_scale(float had, float least) { return fabsf(had) >= least ? had : least; }
// Whether x / scale is x times the scale's reciprocal, exactly.
__device__ __forceinline__ bool is_power(float scale) {
    const uint32_t bits = __float_as_uint(scale);
    return (bits & 0x807fffffu) == 0 && bits >= 0x00800000u && bits <= 0x7e800000u;
}

// A lane's walk over the pieces of some rows, 32 pieces a step. kWhole: a step is whole rows.
template <bool kWhole> struct RowWalk {
    int vecs, right, column;
    long long step, wrap;                                        // between pieces; more where the step passes a row's end
    __device__ __forceinline__ RowWalk(int vecs_, int lane, int per_vec, long long row_step) : vecs(vecs_), right(32 % vecs_), column(lane % vecs_) {
        step = 32 / vecs * row_step + right * per_vec;
        wrap = row_step - static_cast<long long>(vecs) * per_vec;
    }
    template <typename P> __device__ __forceinline__ void next(P *&at) {
        at += step;
        if constexpr (!kWhole) {
            column += right;
            if (column >= vecs) { column -= vecs; at += wrap; }
        }
    }
};

// The call's tokens in one block of scales: where they go, and where they come from.
struct BlockOfScales {
    bool there;
    int page, place, older, count;                               // place of the first new token, older tokens of the block before it, new ones
    long long first;                                             // row of the first new one
};
// For whole warps: every lane has the answer.
__device__ __forceinline__ BlockOfScales block_of_scales(const KvParams &c, const int *seqs, const int *starts, int n, const AppendWork *work, int unit, int lane,
                                                         const AppendDivisors &by) {
    BlockOfScales b = {false, 0, 0, 0, 0, 0};
    const int i = starts ? last_not_above(n, unit, lane, [&](int at) { return work[at].block; }) : unit;
    const int before = work[i].start, row = starts ? starts[i] : i, count = starts ? starts[i + 1] - row : 1;
    if (before < 0 || count <= 0) return b;
    const long long begin = (by.block.quotient(before) + static_cast<long long>(starts ? unit - work[i].block : 0)) * c.block;
    const long long last = min(begin + c.block, before + static_cast<long long>(count));
    if (last <= begin) return b;                                 // (the bound on blocks is not reached)
    const int from = static_cast<int>(max(begin, static_cast<long long>(before))), nth = by.page.quotient(from);
    b.page = c.table[(seqs ? seqs[i] : i) * c.table_stride + nth];
    b.there = b.page >= 0 && b.page < c.n_pages;
    b.place = from - nth * c.page_size;
    b.older = from - static_cast<int>(begin);
    b.count = static_cast<int>(last) - from;
    b.first = static_cast<long long>(row) + from - before;
    return b;
}

// Threads of an appending block, and tokens whose pieces a thread keeps between the maximum and the codes. The prompts above: 42.0 us, with blocks of 256 threads 46.0,
// of 64 43.5; with a warp for a block of one head, eight pieces a lane, 48.0. What is looked up of the next block waits for nothing: 46 instead of 59.
constexpr int kColumns = 128;
constexpr int kHeld = 16;

// A block of threads for one block of scales of some heads, keys and values: a thread has a 16-byte column of a head and goes down the tokens, all of
// its reads on their way together. The head's largest magnitude, from its columns' threads; the scale; the block's older codes by the new
// scale where that has grown; the new codes. kWarp: a head's columns are threads of one warp, a power of two of them.
template <typename T, bool kWarp>
__global__ void __launch_bounds__(kColumns, 512 / kColumns) kv_append_codes_kernel(KvParams c, const int *seqs, const int *starts, int n, const AppendWork *work, const T *k_new, const T *v_new,
                                                                 long long token_stride, long long head_stride, int items, Divisor groups, int heads_of_block, AppendDivisors by) {
    constexpr int kVec = 16 / sizeof(T);
    using Column = Piece<T, kVec>;
    __shared__ uint32_t tops[kColumns];
    pdl_enter();
    const int lane = threadIdx.x % 32, vecs = c.dim / kVec, mine = threadIdx.x / vecs, column = threadIdx.x - mine * vecs;
    BlockOfScales next = block_of_scales(c, seqs, starts, n, work, groups.quotient(blockIdx.x), lane, by);
    // (counted without a sign: items go up to 2^31 - 2, and what is behind the last one has to be behind it still)
    for (uint32_t turn = blockIdx.x; turn < static_cast<uint32_t>(items); turn += gridDim.x) {
        const BlockOfScales b = next;
        const int item = static_cast<int>(turn);
        const int unit = groups.quotient(item), both = (item - unit * static_cast<int>(groups.by)) * heads_of_block + mine;      // a head of the keys, then of the values
        const bool active = mine < heads_of_block && both < 2 * c.heads, values = both >= c.heads;
        const int head = values ? both - c.heads : both;
        const long long token_step = values ? c.v_token : c.k_token;
        uint8_t *codes = (values ? c.v + b.page * c.v_page + head * c.v_head + b.place * c.v_token : c.k + b.page * c.k_page + head * c.k_head + b.place * c.k_token) + column * kVec;
        float *scale_at = (values ? c.v_scales : c.k_scales) + (static_cast<long long>(b.page) * c.heads + head) * c.blocks + by.block.quotient(b.place);
        const T *source = (values ? v_new : k_new) + b.first * token_stride + head * head_stride + column * kVec;
        const int count = active && b.there ? b.count : 0;

        Column held[kHeld];
        const float had = active && b.there && b.older ? *scale_at : 0.f;
#pragma unroll
        for (int t = 0; t < kHeld; ++t)
            if (t < count) held[t].load(source + t * token_stride);
        // (where the next one is, is looked up while these are on their way)
        if (turn + gridDim.x < static_cast<uint32_t>(items)) next = block_of_scales(c, seqs, starts, n, work, groups.quotient(static_cast<int>(turn + gridDim.x)), lane, by);
        if (!b.there) continue;
        uint32_t top = 0;
#pragma unroll
        for (int t = 0; t < kHeld; ++t)
            if (t < count) top = held[t].top(top);
#pragma unroll 4
        for (int t = kHeld; t < count; ++t) {
            Column p;
            p.load(source + t * token_stride);
            top = p.top(top);
        }
        top = Column::last(top);
        const auto over_head = [&](uint32_t top) {               // the head's largest one
            if constexpr (kWarp) {
                for (int o = vecs / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
                return top;
            } else {
                __syncthreads();                                 // (what was there has been read)
                if (column == 0) tops[mine] = 0;
                __syncthreads();
                atomicMax(&tops[mine], top);
                __syncthreads();
                return tops[mine];
            }
        };
        top = over_head(top);
        const bool odd = top >= 0x7f800000u;                     // a NaN or infinity: once more without them
        if (__syncthreads_or(odd)) {
            uint32_t finite = 0;
            for (int t = 0; t < count; ++t) {
                Column p;
                p.load(source + t * token_stride);
                finite = p.finite_top(finite);
            }
            finite = over_head(finite);
            if (odd) top = finite;
        }
        const float scale = larger_scale(had, scale_of(top));
        const bool power = is_power(scale);
        const float inverse = power ? 1.f / scale : 0.f;
        if (active && b.older && scale != had) {
            const auto again = [&](float x) { return power ? x * had * inverse : x * had / scale; };
            constexpr int kTurn = 8;                             // of them on their way together
            for (int first = -b.older; first < 0; first += kTurn) {
                Codes<kVec> p[kTurn];
#pragma unroll
                for (int t = 0; t < kTurn; ++t)
                    if (first + t < 0) p[t].load(codes + (first + t) * token_step);
#pragma unroll
                for (int t = 0; t < kTurn; ++t)
                    if (first + t < 0) p[t].store(codes + (first + t) * token_step, again);
            }
        }
        if (power && !odd) {
            const auto code = [&](float x) { return x * inverse; };
#pragma unroll
            for (int t = 0; t < kHeld; ++t)
                if (t < count) held[t].store(codes + t * token_step, code);
#pragma unroll 4
            for (int t = kHeld; t < count; ++t) {
                Column p;
                p.load(source + t * token_stride);
                p.store(codes + t * token_step, code);
            }
        } else {
            const auto code = [&](float x) {
                if (!isfinite(x)) return __uint_as_float(0x7fffffffu);
                return scale == 0.f ? 0.f * x : x / scale;
            };
            for (int t = 0; t < count; ++t) {
                Column p;
                p.load(source + t * token_stride);
                p.store(codes + t * token_step, code);
            }
        }
        if (active && column == 0) *scale_at = scale;
    }
}

// The same for rows of any alignment and length, a value at a time: a warp for a head.
template <typename T>
__global__ void __launch_bounds__(256) kv_append_values_kernel(KvParams c, const int *seqs, const int *starts, int n, const AppendWork *work, const T *k_new, const T *v_new,
                                                               long long token_stride, long long head_stride, int total, AppendDivisors by) {
    pdl_enter();
    const int lane = threadIdx.x % 32;
    for (long long w = (blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x) / 32; w < total; w += static_cast<long long>(gridDim.x) * blockDim.x / 32) {
        const int pair = by.heads.quotient(static_cast<int>(w)), head = static_cast<int>(w) - pair * c.heads;
        const bool values = pair % 2;
        const BlockOfScales b = block_of_scales(c, seqs, starts, n, work, pair / 2, lane, by);
        if (!b.there) continue;
        const long long token_step = values ? c.v_token : c.k_token;
        uint8_t *codes = values ? c.v + b.page * c.v_page + head * c.v_head + b.place * c.v_token : c.k + b.page * c.k_page + head * c.k_head + b.place * c.k_token;
        float *scale_at = (values ? c.v_scales : c.k_scales) + (static_cast<long long>(b.page) * c.heads + head) * c.blocks + by.block.quotient(b.place);
        const float had = b.older ? *scale_at : 0.f;
        const T *source = (values ? v_new : k_new) + b.first * token_stride + head * head_stride;
        uint32_t top = 0;
        for (int t = 0; t < b.count; ++t)
            for (int d = lane; d < c.dim; d += 32) {
                const uint32_t bits = __float_as_uint(to_float(source[t * token_stride + d])) & 0x7fffffffu;
                if (bits < 0x7f800000u) top = max(top, bits);
            }
        const float scale = larger_scale(had, scale_of(__reduce_max_sync(~0u, top)));
        for (int t = -b.older; t < b.count; ++t)
            for (int d = lane; d < c.dim; d += 32) {
                uint8_t &code = codes[t * token_step + d];
                float x;
                if (t < 0) {
                    if (scale == had) continue;
                    __nv_fp8_e4m3 old;
                    old.__x = code;
                    x = to_float(old) * had / scale;
                } else {
                    x = to_float(source[t * token_stride + d]);
                    x = !isfinite(x) ? __uint_as_float(0x7fffffffu) : scale == 0.f ? 0.f * x : x / scale;
                }
                code = static_cast<uint8_t>(to_e4m3x2(x, 0.f));
            }
        if (lane == 0) *scale_at = scale;
    }
}

// kVec values side by side, and what they are as another type, times a scale
template <typename In, int kVec> struct Values {
    alignas(16) In v[kVec];
    __device__ __forceinline__ void load(const In *from) {
        if constexpr (kVec == 1) {
            v[0] = from[0];
        } else if constexpr (sizeof(v) == 8) {
            *reinterpret_cast<uint2 *>(v) = *reinterpret_cast<const uint2 *>(from);
        } else {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(v)) / 16; ++i) reinterpret_cast<uint4 *>(v)[i] = reinterpret_cast<const uint4 *>(from)[i];
        }
    }
    template <typename Out> __device__ __forceinline__ void store(Out *to, float scale) const {
        alignas(16) Out out[kVec];
        if constexpr (sizeof(In) == 1 && kVec > 1) {
#pragma unroll
            for (int i = 0; i < kVec / 4; ++i) {
                float x[4];
                to_floats(reinterpret_cast<const uint32_t *>(v)[i], x);
#pragma unroll
                for (int j = 0; j < 4; ++j) out[4 * i + j] = from_float<Out>(x[j] * scale);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kVec; ++i) out[i] = from_float<Out>(sizeof(In) == 1 ? to_float(v[i]) * scale : to_float(v[i]));
        }
        if constexpr (kVec == 1) {
            to[0] = out[0];
        } else {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(out)) / 16; ++i) reinterpret_cast<uint4 *>(to)[i] = reinterpret_cast<const uint4 *>(out)[i];
        }
    }
};

// A warp a row of the output: keys and values of all heads of one token, kTurn pieces of each on their way together.
template <typename In, typename Out, int kVec, bool kWhole>
__global__ void __launch_bounds__(256) kv_read_kernel(KvParams c, const int *seqs, const int *starts, const int *firsts, int n, Out *k_out, Out *v_out, long long token_stride,
                                                      long long head_stride, int n_rows, Divisor by_page, Divisor by_block) {
    constexpr bool kCodes = sizeof(In) == 1;
    constexpr int kTurn = kVec > 1 && sizeof(In) <= 2 ? 4 : 2;
    pdl_enter();
    const int lane = threadIdx.x % 32, vecs = c.dim / kVec, total = c.heads * vecs, head_step = 32 / vecs, head0 = lane / vecs;
    for (long long row = (blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x) / 32; row < n_rows; row += static_cast<long long>(gridDim.x) * blockDim.x / 32) {
        int page = -1;
        long long at = 0;
        if (n > 0) {
            const int r = static_cast<int>(row), i = last_not_above(n, r, lane, [&](int at) { return starts[at]; });
            const int s = seqs ? seqs[i] : i;
            if (r >= starts[i] && r < starts[i + 1] && s >= 0 && s < c.n_seqs) {
                at = static_cast<long long>(r) - starts[i] + (firsts ? firsts[i] : 0);
                if (at >= 0 && at < min(static_cast<long long>(c.lengths[s]), static_cast<long long>(c.max_pages) * c.page_size)) {
                    const int nth = by_page.quotient(static_cast<int>(at));
                    page = c.table[s * c.table_stride + nth];
                    at -= static_cast<long long>(nth) * c.page_size;
                }
            }
        }
        const bool there = page >= 0 && page < c.n_pages;
        RowWalk<kWhole> walk_k(vecs, lane, kVec, c.k_head), walk_v(vecs, lane, kVec, c.v_head), walk_out(vecs, lane, kVec, head_stride);
        const int place = there ? static_cast<int>(at) : 0;
        const In *k = reinterpret_cast<const In *>(c.k) + (there ? page * c.k_page + place * c.k_token : 0) + head0 * c.k_head + walk_k.column * kVec;
        const In *v = reinterpret_cast<const In *>(c.v) + (there ? page * c.v_page + place * c.v_token : 0) + head0 * c.v_head + walk_v.column * kVec;
        long long to = row * token_stride + head0 * head_stride + walk_out.column * kVec;
        const long long scales = kCodes && there ? static_cast<long long>(page) * c.heads * c.blocks + by_block.quotient(place) : 0;
        int head = head0;
        for (int u = lane; u < total; u += 32 * kTurn) {
            Values<In, kVec> a[kTurn], b[kTurn];
            float scale_a[kTurn], scale_b[kTurn];
#pragma unroll
            for (int j = 0; j < kTurn; ++j) {
                scale_a[j] = scale_b[j] = 0.f;
                if (there && u + 32 * j < total) {
                    a[j].load(k);
                    b[j].load(v);
                    if (kCodes) {
                        scale_a[j] = c.k_scales[scales + head * c.blocks];
                        scale_b[j] = c.v_scales[scales + head * c.blocks];
                    }
                }
                head += head_step + (!kWhole && walk_k.column + walk_k.right >= vecs);
                walk_k.next(k);
                walk_v.next(v);
            }
#pragma unroll
            for (int j = 0; j < kTurn; ++j) {
                if (u + 32 * j < total) {
                    if (there) {
                        a[j].store(k_out + to, scale_a[j]);
                        b[j].store(v_out + to, scale_b[j]);
                    } else {
#pragma unroll
                        for (int i = 0; i < kVec; ++i) k_out[to + i] = v_out[to + i] = from_float<Out>(0.f);
                    }
                }
                const Out *next = k_out + to;
                walk_out.next(next);
                to = next - k_out;
            }
        }
    }
}

// The scales of the first `blocks` blocks of page src to page dst, by threads first, first + step, ...
__device__ __forceinline__ void copy_scales(const KvParams &c, int src, int dst, int blocks, int first, int step) {
    const long long from = static_cast<long long>(src) * c.heads * c.blocks, to = static_cast<long long>(dst) * c.heads * c.blocks;
    for (int i = first; i < c.heads * blocks; i += step) {
        const int at = i / blocks * c.blocks + i % blocks;
        c.k_scales[to + at] = c.k_scales[from + at];
        c.v_scales[to + at] = c.v_scales[from + at];
    }
}

// Of the first `rows` tokens of page src the units from `first` on, `step` apart, below `total`, keys and values, to page dst. Four units a
// turn, so that their reads are under way together.
template <typename Unit>
__device__ __forceinline__ void copy_units(const KvParams &c, int src, int dst, int units, int first, int step, int total) {
    const Unit *k = reinterpret_cast<const Unit *>(c.k) + src * c.k_page, *v = reinterpret_cast<const Unit *>(c.v) + src * c.v_page;
    Unit *k_to = reinterpret_cast<Unit *>(c.k) + dst * c.k_page, *v_to = reinterpret_cast<Unit *>(c.v) + dst * c.v_page;
    const int per_token = c.heads * units;
    const bool flat = c.k_token == per_token && c.v_token == per_token && c.k_head == units && c.v_head == units;     // tokens one behind the other
    for (int base = first; base < total; base += 4 * step) {
        long long at_k[4], at_v[4];
        Unit a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int u = base + i * step;
            if (u >= total) break;
            if (flat) {
                at_k[i] = at_v[i] = u;
            } else {
                const int place = u / per_token, head = u % per_token / units, unit = u % units;
                at_k[i] = place * c.k_token + head * c.k_head + unit;
                at_v[i] = place * c.v_token + head * c.v_head + unit;
            }
            a[i] = k[at_k[i]];
            b[i] = v[at_v[i]];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (base + i * step >= total) break;
            k_to[at_k[i]] = a[i];
            v_to[at_v[i]] = b[i];
        }
    }
}

constexpr int kPiece = 1024;           // units of a page that a block of 256 threads moves at a time

struct ForkWork { int from, to, rows, full; };                   // the copied page and its rows (to < 0: none); full < 0: refused

__global__ void kv_fork_decide_kernel(KvParams c, const int *src, const int *dst, int n, ForkWork *work, int *list) {
    pdl_enter();
    int all = 0;
    for (int base = 0; base < n; base += kDecide) {
        const int i = base + threadIdx.x;
        ForkWork w = {0, -1, 0, -1};
        bool wants = false;
        if (i < n) {
            const int a = src[i], b = dst[i];
            if (a >= 0 && a < c.n_seqs && b >= 0 && b < c.n_seqs && a != b && c.lengths[b] == 0) {
                const int len = max(0, min(c.lengths[a], c.max_pages * c.page_size));
                w.full = len / c.page_size;
                w.rows = len % c.page_size;
                if (w.rows) {
                    w.from = c.table[a * c.table_stride + w.full];
                    wants = w.from >= 0 && w.from < c.n_pages;
                }
            }
        }
        int total;
        const int rank = all + block_scan(wants, &total);
        if (wants) w.to = rank;                                  // its place in the list for now
        if (i < n) work[i] = w;
        all += total;
    }
    const int found = lowest_free(c, all, list);
    for (int i = threadIdx.x; i < n; i += kDecide) {
        ForkWork w = work[i];
        if (w.full >= 0 && w.to >= found) w.full = -1;
        if (w.full < 0) {
            work[i].full = -1;
            atomicAdd(c.refused, 1);
            continue;
        }
        const int b = dst[i];
        if (w.to >= 0) {
            w.to = list[w.to];
            work[i].to = w.to;
            c.refs[w.to] = 1;
        }
        if (w.rows) c.table[b * c.table_stride + w.full] = w.to >= 0 ? w.to : w.from;     // (a hole stays a hole)
        c.lengths[b] = w.full * c.page_size + w.rows;
    }
}

template <typename Unit>
__global__ void kv_fork_copy_kernel(KvParams c, const int *src, const int *dst, const ForkWork *work, int units) {
    pdl_enter();
    const ForkWork w = work[blockIdx.x];
    if (w.full < 0) return;
    const long long a = src[blockIdx.x] * c.table_stride, b = dst[blockIdx.x] * c.table_stride;
    const int first = blockIdx.y * blockDim.x + threadIdx.x, step = gridDim.y * blockDim.x;
    for (int j = first; j < w.full; j += step) {
        const int page = c.table[a + j];
        c.table[b + j] = page;
        if (page >= 0 && page < c.n_pages) atomicAdd(&c.refs[page], 1);
    }
    if (w.to >= 0) {
        copy_units<Unit>(c, w.from, w.to, units, first, step, w.rows * c.heads * units);
        if (c.block) copy_scales(c, w.from, w.to, (w.rows + c.block - 1) / c.block, first, step);
    }
}

__global__ void kv_free_kernel(KvParams c, const int *seqs) {
    __shared__ int length;
    pdl_enter();
    const int s = seqs[blockIdx.x];
    if (s < 0 || s >= c.n_seqs) {
        if (threadIdx.x == 0) atomicAdd(c.refused, 1);
        return;
    }
    if (threadIdx.x == 0) length = atomicExch(&c.lengths[s], 0);
    __syncthreads();
    const int pages = static_cast<int>(min((static_cast<long long>(length) + c.page_size - 1) / c.page_size, static_cast<long long>(c.max_pages)));
    for (int j = threadIdx.x; j < pages; j += blockDim.x) {
        const int page = c.table[s * c.table_stride + j];
        if (page >= 0 && page < c.n_pages) atomicSub(&c.refs[page], 1);
    }
}

// A compaction's decisions: [0] the number of moves, then n_pages each (up to 8, so that 16-byte stores fit): where a page's contents go,
// the moves' destinations, their sources.
struct CompactWork {
    int *moves, *where, *to, *from;
    __host__ __device__ static long long pitch(int n_pages) { return (n_pages + 7LL) / 8 * 8; }
    __host__ __device__ static size_t bytes(int n_pages) { return (4 + 3 * static_cast<size_t>(pitch(n_pages))) * 4; }
    __device__ CompactWork(int *work, int n_pages) : moves(work), where(work + 4), to(where + pitch(n_pages)), from(to + pitch(n_pages)) {}
};

__global__ void kv_compact_decide_kernel(KvParams c, int *refs_out, int *work) {
    pdl_enter();
    const CompactWork w(work, c.n_pages);
    int live = 0;
    for (long long base = 0; base < c.n_pages; base += kDecide * kEach) {
        const int first = static_cast<int>(min(base + threadIdx.x * kEach, static_cast<long long>(c.n_pages)));
        int refs[kEach];
        load_refs(c, first, refs);
#pragma unroll
        for (int i = 0; i < kEach; ++i) live += refs[i] != 0 && first + i < c.n_pages;
    }
    int n_live;
    block_scan(live, &n_live);
    int holes = 0, movers = 0;
    for (long long base = 0; base < c.n_pages; base += kDecide * kEach) {
        const int first = static_cast<int>(min(base + threadIdx.x * kEach, static_cast<long long>(c.n_pages)));
        int refs[kEach], mine = 0;                               // holes in the low half, movers in the high one (at most 8192 of each)
        load_refs(c, first, refs);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int page = first + i;
            if (page < n_live) mine += refs[i] == 0;
            else if (page < c.n_pages) mine += (refs[i] != 0) << 16;
        }
        int total;
        const int rank = block_scan(mine, &total);
        int hole = holes + (rank & 0xffff), mover = movers + (rank >> 16);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int page = first + i;
            if (page >= c.n_pages) break;
            if (page < n_live && refs[i] == 0) w.to[hole++] = page;
            if (page >= n_live && refs[i] != 0) w.from[mover++] = page;
            if (refs_out != c.refs) refs_out[page] = refs[i];
        }
        if (first < c.n_pages)
#pragma unroll
            for (int i = 0; i < kEach; i += 4) *reinterpret_cast<int4 *>(w.where + first + i) = make_int4(first + i, first + i + 1, first + i + 2, first + i + 3);
        holes += total & 0xffff;
        movers += total >> 16;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < movers; i += kDecide) w.where[w.from[i]] = w.to[i];
    if (threadIdx.x == 0) *w.moves = movers;
}

template <typename Unit>
__global__ void kv_compact_move_kernel(KvParams c, int *work, int *table_out, int *refs_out, int units) {
    pdl_enter();
    const CompactWork w(work, c.n_pages);
    const int moves = *w.moves;
    const long long entries = static_cast<long long>(c.n_seqs) * c.max_pages;
    for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < entries; i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const long long s = i / c.max_pages, j = i % c.max_pages;
        const int page = c.table[s * c.table_stride + j];
        const bool held = j * c.page_size < c.lengths[s] && page >= 0 && page < c.n_pages;
        table_out[s * c.table_stride + j] = held ? w.where[page] : page;
    }
    // pieces of pages, so that the blocks end together
    const int total = c.page_size * c.heads * units, pieces = (total + kPiece - 1) / kPiece;
    for (long long i = blockIdx.x; i < static_cast<long long>(moves) * pieces; i += gridDim.x) {
        const int move = static_cast<int>(i / pieces), first = static_cast<int>(i - static_cast<long long>(move) * pieces) * kPiece;
        const int from = w.from[move], to = w.to[move];
        if (first == 0 && threadIdx.x == 0) {
            refs_out[to] = c.refs[from];
            refs_out[from] = 0;
        }
        if (first == 0 && c.block) copy_scales(c, from, to, c.blocks, threadIdx.x, blockDim.x);
        copy_units<Unit>(c, from, to, units, first + threadIdx.x, blockDim.x, min(total, first + kPiece));
    }
}

template <typename Unit>
__global__ void kv_copy_pages_kernel(KvParams c, const int *src, const int *dst, int n, int units) {
    pdl_enter();
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const int a = src[i], b = dst[i];
        if (a < 0 || a >= c.n_pages || b < 0 || b >= c.n_pages || a == b) {
            if (a != b && threadIdx.x == 0) atomicAdd(c.refused, 1);
            continue;
        }
        copy_units<Unit>(c, a, b, units, threadIdx.x, blockDim.x, c.page_size * c.heads * units);
        if (c.block) copy_scales(c, a, b, c.blocks, threadIdx.x, blockDim.x);
    }
}

// The cache with strides in units of `bytes` and the units of a row.
KvParams in_units(KvParams p, size_t size, size_t bytes, int *units) {
    const long long per = static_cast<long long>(bytes / size);
    for (long long *stride : {&p.k_page, &p.k_token, &p.k_head, &p.v_page, &p.v_token, &p.v_head}) *stride /= per;
    *units = p.dim / static_cast<int>(per);
    return p;
}

size_t workspace_bytes_of(const MsnhB200KvCache &c, int n) {
    return std::max(static_cast<size_t>(n) * sizeof(AppendWork) + static_cast<size_t>(c.n_pages) * 4, CompactWork::bytes(c.n_pages));
}

int check_workspace(MsnhB200Ctx *ctx, const MsnhB200KvCache &c, int n, const void *workspace, size_t bytes, const char *what) {
    const size_t wanted = workspace_bytes_of(c, n);
    if (!workspace || bytes < wanted) return fail(ctx, MSNH_B200_ERR_ARG, "%s: %zu bytes of workspace are wanted, %zu given", what, wanted, workspace ? bytes : size_t(0));
    if (!aligned16(workspace)) return fail(ctx, MSNH_B200_ERR_ARG, "%s: the workspace is not 16-byte aligned", what);
    return MSNH_B200_OK;
}

int blocks_for(const MsnhB200Ctx *ctx, long long items, int per_block) {
    return static_cast<int>(std::max<long long>(1, std::min<long long>((items + per_block - 1) / per_block, ctx->sm_count * 8LL)));
}

}  // namespace
}  // namespace msnh

using namespace msnh;

extern "C" {

int msnh_b200_kv_workspace(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, int n, size_t *bytes) try {
    if (!ctx || !c || !bytes) return MSNH_B200_ERR_ARG;
    if (n < 0 || c->n_pages < 1) return fail(ctx, MSNH_B200_ERR_ARG, "kv_workspace: %d sequences, %d pages", n, c->n_pages);
    *bytes = workspace_bytes_of(*c, n);
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

int msnh_b200_kv_append(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, const int32_t *seqs, const int32_t *starts, int n, const void *k_new, const void *v_new,
                        int64_t new_token_stride, int64_t new_head_stride, int n_tokens, void *workspace, size_t workspace_bytes, void *stream) {
    return msnh_b200_kv_append_as(ctx, c, seqs, starts, n, k_new, v_new, c ? c->dtype : 0, new_token_stride, new_head_stride, n_tokens, workspace, workspace_bytes, stream);
}

int msnh_b200_kv_append_as(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, const int32_t *seqs, const int32_t *starts, int n, const void *k_new, const void *v_new, int new_dtype,
                           int64_t new_token_stride, int64_t new_head_stride, int n_tokens, void *workspace, size_t workspace_bytes, void *stream) try {
    if (!ctx || !c) return MSNH_B200_ERR_ARG;
    if (const int rc = check_cache(ctx, c, true, "kv_append")) return rc;
    const bool codes = c->dtype == MSNH_B200_E4M3;
    if (codes ? !is_float_type(new_dtype) : new_dtype != c->dtype) return fail(ctx, MSNH_B200_ERR_ARG, "kv_append: values of type %d for a cache of type %d", new_dtype, c->dtype);
    if (n < 0 || n_tokens < 0) return fail(ctx, MSNH_B200_ERR_ARG, "kv_append: %d sequences, %d tokens", n, n_tokens);
    if (!starts && n_tokens != n) return fail(ctx, MSNH_B200_ERR_ARG, "kv_append: %d tokens for %d sequences without starts", n_tokens, n);
    if (!seqs && n > c->n_seqs) return fail(ctx, MSNH_B200_ERR_ARG, "kv_append: %d sequences of %d", n, c->n_seqs);
    if (n == 0) return MSNH_B200_OK;
    if (n_tokens > 0 && (!k_new || !v_new)) return fail(ctx, MSNH_B200_ERR_ARG, "kv_append: null k_new or v_new");
    if (new_token_stride < 0 || new_head_stride < 0) return fail(ctx, MSNH_B200_ERR_ARG, "kv_append: a stride is negative");
    if (const int rc = check_workspace(ctx, *c, n, workspace, workspace_bytes, "kv_append")) return rc;
    // blocks of scales that n_tokens tokens of n sequences lie in, at most
    const long long most_blocks = codes ? starts ? n_tokens / c->scale_block + 2LL * std::min(n, n_tokens) : n : 0;
    if (most_blocks > 0x7fffffff / 2 / c->n_kv_heads) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "kv_append: 2^31 scales and more");
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    AppendWork *work = static_cast<AppendWork *>(workspace);
    int *list = reinterpret_cast<int *>(work + n);
    const KvParams p = kv_params(*c);
    const AppendDivisors by = {Divisor(c->n_kv_heads), Divisor(codes ? c->scale_block : 1), Divisor(c->page_size)};
    CUDA_TRY(ctx, launch_token_kernel(kv_append_decide_kernel, dim3(1), kDecide, 0, stream, ctx->pdl, p, seqs, starts, n, n_tokens, work, list, by));
    if (n_tokens == 0) return MSNH_B200_OK;
    const size_t size = dtype_size(new_dtype);
    const bool aligned = aligned16(k_new) && aligned16(v_new) && new_token_stride * size % 16 == 0 && new_head_stride * size % 16 == 0;
    if (codes) {
        // a block has as many heads as its threads are columns of
        const int vecs = static_cast<int>(c->head_dim * size / 16);
        const bool wide = aligned && kv_rows_multiple_of(*c, 16 / size) && vecs >= 1 && vecs <= kColumns, warps = wide && vecs <= 32 && (vecs & (vecs - 1)) == 0;
        const int total = static_cast<int>(most_blocks * c->n_kv_heads * 2), heads_of_block = wide ? std::min(kColumns / vecs, 2 * c->n_kv_heads) : 1;
        const int groups = (2 * c->n_kv_heads + heads_of_block - 1) / heads_of_block, items = static_cast<int>(most_blocks * groups);
        const auto by_type = [&](auto type) {
            using T = decltype(type);
            const T *k = static_cast<const T *>(k_new), *v = static_cast<const T *>(v_new);
            if (!wide) return launch_token_kernel(kv_append_values_kernel<T>, dim3(blocks_for(ctx, total, 8)), 256, 0, stream, ctx->pdl, p, seqs, starts, n, work, k, v, new_token_stride,
                                                  new_head_stride, total, by);
            return launch_token_kernel(warps ? kv_append_codes_kernel<T, true> : kv_append_codes_kernel<T, false>, dim3(blocks_for(ctx, items, 1)), kColumns, 0, stream, ctx->pdl, p, seqs,
                                       starts, n, work, k, v, new_token_stride, new_head_stride, items, Divisor(groups), heads_of_block, by);
        };
        CUDA_TRY(ctx, new_dtype == MSNH_B200_F32 ? by_type(float()) : new_dtype == MSNH_B200_F16 ? by_type(__half()) : by_type(__nv_bfloat16()));
        return MSNH_B200_OK;
    }
    const bool wide = aligned && kv_rows_multiple_of(*c, 16);
    int units;
    const KvParams q = in_units(p, size, wide ? 16 : size, &units);
    const long long per = wide ? static_cast<long long>(16 / size) : 1;
    const dim3 grid(blocks_for(ctx, static_cast<long long>(n_tokens) * c->n_kv_heads * units, 256));
    const auto write = [&](auto unit) {
        using Unit = decltype(unit);
        return launch_token_kernel(kv_append_write_kernel<Unit>, grid, 256, 0, stream, ctx->pdl, q, seqs, starts, n, n_tokens, work, static_cast<const Unit *>(k_new),
                                   static_cast<const Unit *>(v_new), new_token_stride / per, new_head_stride / per, units);
    };
    CUDA_TRY(ctx, wide ? write(uint4()) : size == 4 ? write(uint32_t()) : write(uint16_t()));
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

int msnh_b200_kv_read(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, const int32_t *seqs, const int32_t *starts, const int32_t *first, int n, void *k_out, void *v_out, int out_dtype,
                      int64_t out_token_stride, int64_t out_head_stride, int n_rows, void *stream) try {
    if (!ctx || !c) return MSNH_B200_ERR_ARG;
    if (const int rc = check_cache(ctx, c, false, "kv_read")) return rc;
    if (!is_float_type(out_dtype)) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "kv_read: values of type %d", out_dtype);
    if (n < 0 || n_rows < 0) return fail(ctx, MSNH_B200_ERR_ARG, "kv_read: %d sequences, %d rows", n, n_rows);
    if (!seqs && n > c->n_seqs) return fail(ctx, MSNH_B200_ERR_ARG, "kv_read: %d sequences of %d", n, c->n_seqs);
    if (n_rows == 0) return MSNH_B200_OK;
    if (!k_out || !v_out || (n && !starts)) return fail(ctx, MSNH_B200_ERR_ARG, "kv_read: null k_out, v_out or starts");
    const int64_t out_size = static_cast<int64_t>(dtype_size(out_dtype));
    const Rows rows(n_rows, c->n_kv_heads, out_token_stride * out_size, out_head_stride * out_size, c->head_dim * out_size);
    if (rows_overlap(rows) || rows_meet(k_out, rows, v_out, rows)) return fail(ctx, MSNH_B200_ERR_ARG, "kv_read: rows of the output overlap");
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    const KvParams p = kv_params(*c);
    const size_t size = dtype_size(out_dtype);
    constexpr int kVec = 8;
    const bool wide = c->head_dim % kVec == 0 && aligned16(k_out) && aligned16(v_out) && out_token_stride * size % 16 == 0 && out_head_stride * size % 16 == 0 &&
                      kv_rows_multiple_of(*c, c->dtype == MSNH_B200_E4M3 ? 8 : 16);
    const dim3 grid(blocks_for(ctx, n_rows, 8));
    const auto read = [&](auto in, auto out) {
        using In = decltype(in);
        using Out = decltype(out);
        return launch_token_kernel(!wide ? kv_read_kernel<In, Out, 1, false> : 32 % (c->head_dim / kVec) == 0 ? kv_read_kernel<In, Out, kVec, true> : kv_read_kernel<In, Out, kVec, false>, grid,
                                   256, 0, stream, ctx->pdl, p, seqs, starts, first, n, static_cast<Out *>(k_out), static_cast<Out *>(v_out), out_token_stride, out_head_stride, n_rows,
                                   Divisor(c->page_size), Divisor(p.block ? p.block : 1));
    };
    const auto from = [&](auto in) { return out_dtype == MSNH_B200_F32 ? read(in, float()) : out_dtype == MSNH_B200_F16 ? read(in, __half()) : read(in, __nv_bfloat16()); };
    CUDA_TRY(ctx, c->dtype == MSNH_B200_F32 ? from(float()) : c->dtype == MSNH_B200_F16 ? from(__half()) : c->dtype == MSNH_B200_BF16 ? from(__nv_bfloat16()) : from(__nv_fp8_e4m3()));
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

int msnh_b200_kv_fork(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, const int32_t *src, const int32_t *dst, int n, void *workspace, size_t workspace_bytes,
                      void *stream) try {
    if (!ctx || !c) return MSNH_B200_ERR_ARG;
    if (const int rc = check_cache(ctx, c, true, "kv_fork")) return rc;
    if (n < 0) return fail(ctx, MSNH_B200_ERR_ARG, "kv_fork: %d sequences", n);
    if (n == 0) return MSNH_B200_OK;
    if (!src || !dst) return fail(ctx, MSNH_B200_ERR_ARG, "kv_fork: null src or dst");
    if (const int rc = check_workspace(ctx, *c, n, workspace, workspace_bytes, "kv_fork")) return rc;
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    ForkWork *work = static_cast<ForkWork *>(workspace);
    int *list = reinterpret_cast<int *>(work + n);
    const KvParams p = kv_params(*c);
    CUDA_TRY(ctx, launch_token_kernel(kv_fork_decide_kernel, dim3(1), kDecide, 0, stream, ctx->pdl, p, src, dst, n, work, list));
    const size_t size = dtype_size(c->dtype);
    const bool wide = kv_rows_multiple_of(*c, 16);
    int units;
    const KvParams q = in_units(p, size, wide ? 16 : size, &units);
    const dim3 grid(n, std::max(1, std::min(8, 2 * ctx->sm_count / n)));
    const auto copy = [&](auto unit) { return launch_token_kernel(kv_fork_copy_kernel<decltype(unit)>, grid, 256, 0, stream, ctx->pdl, q, src, dst, work, units); };
    CUDA_TRY(ctx, wide ? copy(uint4()) : size == 4 ? copy(uint32_t()) : size == 2 ? copy(uint16_t()) : copy(uint8_t()));
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

int msnh_b200_kv_free(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, const int32_t *seqs, int n, void *stream) try {
    if (!ctx || !c) return MSNH_B200_ERR_ARG;
    if (const int rc = check_cache(ctx, c, true, "kv_free")) return rc;
    if (n < 0) return fail(ctx, MSNH_B200_ERR_ARG, "kv_free: %d sequences", n);
    if (n == 0) return MSNH_B200_OK;
    if (!seqs) return fail(ctx, MSNH_B200_ERR_ARG, "kv_free: null seqs");
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    CUDA_TRY(ctx, launch_token_kernel(kv_free_kernel, dim3(n), 128, 0, stream, ctx->pdl, kv_params(*c), seqs));
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

int msnh_b200_kv_compact(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, int32_t *table_out, int32_t *refs_out, void *workspace, size_t workspace_bytes,
                         void *stream) try {
    if (!ctx || !c) return MSNH_B200_ERR_ARG;
    if (const int rc = check_cache(ctx, c, true, "kv_compact")) return rc;
    if (!table_out || !refs_out) return fail(ctx, MSNH_B200_ERR_ARG, "kv_compact: null table_out or refs_out");
    if (const int rc = check_workspace(ctx, *c, 0, workspace, workspace_bytes, "kv_compact")) return rc;
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    int *work = static_cast<int *>(workspace);
    const KvParams p = kv_params(*c);
    CUDA_TRY(ctx, launch_token_kernel(kv_compact_decide_kernel, dim3(1), kDecide, 0, stream, ctx->pdl, p, refs_out, work));
    const size_t size = dtype_size(c->dtype);
    const bool wide = kv_rows_multiple_of(*c, 16);
    int units;
    const KvParams q = in_units(p, size, wide ? 16 : size, &units);
    const dim3 grid(blocks_for(ctx, std::max<long long>(c->n_pages, static_cast<long long>(c->n_seqs) * c->max_pages / 256), 1));
    const auto move = [&](auto unit) { return launch_token_kernel(kv_compact_move_kernel<decltype(unit)>, grid, 256, 0, stream, ctx->pdl, q, work, table_out, refs_out, units); };
    CUDA_TRY(ctx, wide ? move(uint4()) : size == 4 ? move(uint32_t()) : size == 2 ? move(uint16_t()) : move(uint8_t()));
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

int msnh_b200_kv_copy_pages(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, const int32_t *src, const int32_t *dst, int n, void *stream) try {
    if (!ctx || !c) return MSNH_B200_ERR_ARG;
    if (const int rc = check_cache(ctx, c, true, "kv_copy_pages")) return rc;
    if (n < 0) return fail(ctx, MSNH_B200_ERR_ARG, "kv_copy_pages: %d pages", n);
    if (n == 0) return MSNH_B200_OK;
    if (!src || !dst) return fail(ctx, MSNH_B200_ERR_ARG, "kv_copy_pages: null src or dst");
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    const size_t size = dtype_size(c->dtype);
    const bool wide = kv_rows_multiple_of(*c, 16);
    int units;
    const KvParams q = in_units(kv_params(*c), size, wide ? 16 : size, &units);
    const dim3 grid(blocks_for(ctx, n, 1));
    const auto copy = [&](auto unit) { return launch_token_kernel(kv_copy_pages_kernel<decltype(unit)>, grid, 256, 0, stream, ctx->pdl, q, src, dst, n, units); };
    CUDA_TRY(ctx, wide ? copy(uint4()) : size == 4 ? copy(uint32_t()) : size == 2 ? copy(uint16_t()) : copy(uint8_t()));
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

}  // extern "C"
