// Scores of tokens from rows of logits: log probability of a given one, entropy, the likeliest ones (msnh_b200_token_scores).
//
// p = e^(z - m) / s, s = sum e^(z - m), m the running maximum: log p = z - m - log s, entropy = log s + sum e^(z - m) (m - z) / s, in
// which nothing cancels. One pass: every logit is read once, and those bytes bound it where there are many rows.
//
// Each thread keeps both sums, relative to its warp's maximum, and its own maximum. The `top` best logits of a row are among the chunks of the threads whose
// maxima are at least the top-th best of those: only these threads' chunks are looked at again, a warp for each. What orders logits then is a
// 64-bit key, the number's bits in the numbers' order above the lowest index first, so all keys differ. Sorted lists of 32 lie across a warp's lanes;
// two of them are joined by five steps of a bitonic merge.
//
// A row is one block's or, where there are fewer rows than SMs, one cluster's: its blocks hand their sums and lists to the first one
// through distributed shared memory, so that there is one launch and no workspace.
//
// Measured: 2000 rows of 50000 bf16 logits (200 MB) with the best 8 in 51 us, 3.9 TB/s; instructions bound it (eleven a logit, one of them 2^x at 16
// a cycle and SM, which alone would take 22 us).
#include <cooperative_groups.h>
#include "token_ops.h"
#include "token_types.cuh"

namespace msnh {
namespace {

namespace cg = cooperative_groups;
using Key = unsigned long long;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFar = 1000.f;           // distances are bounded by it where they are factors, so that 0 times infinity does not come up: e^-1000 is 0

struct ScoreParams {
    const uint8_t *logits;
    const long long *ids;
    float *logprob, *entropy, *top_logprobs;
    long long *top_ids;
    long long rows, stride;
    int cols, top;
};

// Bits of a float in the numbers' order (-0 counts as 0); above 0 for every number and infinity.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t bits = __float_as_uint(v + 0.f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ Key key_of(float v, uint32_t index) { return static_cast<Key>(ordered(v)) << 32 | static_cast<uint32_t>(~index); }
__device__ __forceinline__ uint32_t index_of(Key key) { return ~static_cast<uint32_t>(key); }

__device__ __forceinline__ float pow2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Sums of some logits: the largest, sum e^(z - top), sum e^(z - top) (top - z).
struct Sums {
    float top, sum, more;
    // to a maximum that is not smaller
    __device__ __forceinline__ void lift(float best) {
        if (best == top) return;
        const float d = best - top, f = pow2(d * -kLog2e);
        more = f * fmaf(sum, fminf(d, kFar), more);              // (NaN where the distance is)
        sum *= f;
        top = best;
    }
    // (a sum that is NaN stays one, and so does a maximum of infinity)
    __device__ __forceinline__ void join(Sums o) {
        const float best = fmaxf(top, o.top);
        lift(best);
        o.lift(best);
        sum += o.sum;
        more += o.more;
    }
    __device__ __forceinline__ void join_warp() {
#pragma unroll
        for (int o = 16; o; o >>= 1) join(Sums{__shfl_xor_sync(~0u, top, o), __shfl_xor_sync(~0u, sum, o), __shfl_xor_sync(~0u, more, o)});
    }
};

// Two fp32 numbers in a register pair, and their arithmetic in one instruction.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair_of(float a, float b) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void parts_of(Pair p, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ Pair add(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair multiply_add(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Two values of T side by side, or one of fp32: the larger one (NaN where one is), place by place.
template <typename T> struct Lanes;
template <> struct Lanes<float> {
    using Word = float;
    static __device__ __forceinline__ Word of(uint32_t w) { return __uint_as_float(w); }
    static __device__ __forceinline__ Word larger(Word a, Word b) { return max_or_nan(a, b); }
    static __device__ __forceinline__ float first(Word a) { return a; }
    static __device__ __forceinline__ float second(Word a) { return a; }
};
template <> struct Lanes<__half> {
    using Word = __half2;
    static __device__ __forceinline__ Word of(uint32_t w) { return reinterpret_cast<const Word &>(w); }
    static __device__ __forceinline__ Word larger(Word a, Word b) { return __hmax2_nan(a, b); }
    static __device__ __forceinline__ float first(Word a) { return __low2float(a); }
    static __device__ __forceinline__ float second(Word a) { return __high2float(a); }
};
template <> struct Lanes<__nv_bfloat16> {
    using Word = __nv_bfloat162;
    static __device__ __forceinline__ Word of(uint32_t w) { return reinterpret_cast<const Word &>(w); }
    static __device__ __forceinline__ Word larger(Word a, Word b) { return __hmax2_nan(a, b); }
    static __device__ __forceinline__ float first(Word a) { return __low2float(a); }
    static __device__ __forceinline__ float second(Word a) { return __high2float(a); }
};
// The largest of the warp's numbers, NaN where one is.
__device__ __forceinline__ float warp_max_or_nan(float v) {
    float y;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(v));
    return y;
}

// Across a warp's lanes: the larger keys of a pair at distance `o` to the lower lanes.
template <typename K> __device__ __forceinline__ K exchange(K mine, int o, bool larger) {
    const K other = __shfl_xor_sync(~0u, mine, o);
    return larger ? max(mine, other) : min(mine, other);
}
// 32 keys, lane 0 the largest
template <typename K> __device__ __forceinline__ K sort_warp(K key, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
        for (int o = size / 2; o; o /= 2) key = exchange(key, o, ((lane & o) == 0) == ((lane & size) == 0 || size == 32));
    return key;
}
// The 32 largest of two sorted lists (the other one's key of lane 31 - l is given to lane l), sorted.
template <typename K> __device__ __forceinline__ K merge_warp(K key, K other_reversed, int lane) {
    key = max(key, other_reversed);
#pragma unroll
    for (int o = 16; o; o /= 2) key = exchange(key, o, (lane & o) == 0);
    return key;
}
// The lists of a block's warps joined in warp 0; list[] has 32 keys of every warp. Begins and ends with a barrier.
template <int kWarps, typename K> __device__ __forceinline__ K merge_block(K key, K (*list)[32], int warp, int lane) {
    list[warp][lane] = key;
    __syncthreads();
#pragma unroll
    for (int n = kWarps / 2; n; n /= 2) {
        if (warp < n) {
            key = merge_warp(key, list[warp + n][31 - lane], lane);
            list[warp][lane] = key;
        }
        __syncthreads();
    }
    return key;
}

// A row's 16-byte chunks: chunk c has logits c * kVec - shift and on, so that whole chunks are aligned.
template <typename T> struct Row {
    static constexpr int kVec = 16 / sizeof(T);
    const T *at;
    int cols, shift, chunks;
    __device__ __forceinline__ Row(const T *from, int cols_) : at(from), cols(cols_) {
        shift = static_cast<int>(reinterpret_cast<uintptr_t>(from) % 16 / sizeof(T));
        chunks = static_cast<int>((static_cast<long long>(cols) + shift + kVec - 1) / kVec);
    }
    __device__ __forceinline__ int first_of(int chunk) const { return chunk * kVec - shift; }
    __device__ __forceinline__ int whole_chunks() const { return static_cast<int>((static_cast<long long>(cols) + shift) / kVec); }      // the ones before it are whole, or the first one
    // whether all of the chunk's values are the row's
    __device__ __forceinline__ bool whole(int chunk) const { return (chunk > 0 || shift == 0) && first_of(chunk) <= cols - kVec; }
    __device__ __forceinline__ uint4 load_whole(int chunk) const { return *reinterpret_cast<const uint4 *>(at + first_of(chunk)); }
    // places that are not the row's hold `none`, and so does the chunk -1
    __device__ __forceinline__ uint4 load(int chunk, float none) const {
        if (chunk >= 0 && whole(chunk)) return load_whole(chunk);
        const int first = chunk < 0 ? cols : first_of(chunk);
        uint4 raw;
#pragma unroll
        for (int i = 0; i < kVec; ++i) reinterpret_cast<T *>(&raw)[i] = first + i >= 0 && first + i < cols ? at[first + i] : from_float<T>(none);
        return raw;
    }
};

// Some chunks' logits to the sums, whatever their distances from the maximum.
template <typename T, int kCount> __device__ __forceinline__ void add_far(const uint4 (&raw)[kCount], Sums &to) {
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
        float v[16 / sizeof(T)];
        Vec16<T>::unpack(raw[u], v);
#pragma unroll
        for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) {
            const float d = fminf(to.top - v[i], kFar), e = pow2(d * -kLog2e);
            to.sum += e;
            to.more = fmaf(e, d, to.more);
        }
    }
}
// The same for a maximum of up to kLarge: 2^t with t = z log2(e) - m log2(e) in one operation. What the second term is off by, rounded, is the same
// factor for all of them, and taken back behind them. False, and nothing added, where a logit is so far away that t is infinite.
constexpr float kLarge = 65536.f;
template <typename T, int kCount> __device__ __forceinline__ bool add_near(const uint4 (&raw)[kCount], Sums &to) {
    constexpr int kVec = 16 / sizeof(T);
    const float reference = to.top * kLog2e, off = fmaf(to.top, kLog2e, -reference);
    const Pair scale = pair_of(kLog2e, kLog2e), minus = pair_of(-reference, -reference);
    Pair sum = 0, more = 0;
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
        float v[kVec];
        Vec16<T>::unpack(raw[u], v);
#pragma unroll
        for (int i = 0; i < kVec; i += 2) {
            const Pair t = multiply_add(pair_of(v[i], v[i + 1]), scale, minus);
            float a, b;
            parts_of(t, a, b);
            const Pair e = pair_of(pow2(a), pow2(b));
            sum = add(sum, e);
            more = multiply_add(e, t, more);
        }
    }
    float a, b, c, d;
    parts_of(sum, a, b);
    parts_of(more, c, d);
    c += d;
    if (__any_sync(~0u, c != c)) return false;                   // (0 times infinity)
    const float back = pow2(-off), all = a + b;
    to.sum = fmaf(all, back, to.sum);
    to.more = fmaf(fmaf(off, all, -c) * kLn2, back, to.more);
    return true;
}

// What a warp's lanes know of their logits: sums relative to one reference, and each lane's own maximum.
template <typename T, int kCount> __device__ __forceinline__ void take(const uint4 (&raw)[kCount], Sums &sums, float &lane_top) {
    using L = Lanes<T>;
    typename L::Word top;
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
        const auto here = L::larger(L::larger(L::of(raw[u].x), L::of(raw[u].y)), L::larger(L::of(raw[u].z), L::of(raw[u].w)));
        top = u == 0 ? here : L::larger(top, here);
    }
    const float here = max_or_nan(L::first(top), L::second(top)), all = warp_max_or_nan(here);
    lane_top = fmaxf(lane_top, here);
    if (!(all <= sums.top)) sums.lift(all);
    if (sums.top == -INFINITY) return;                           // (nothing but -infinity so far)
    if (!(fabsf(sums.top) <= kLarge) || !add_near<T>(raw, sums)) add_far<T>(raw, sums);
}

template <int kWarps> struct ScoreShared {
    Key list[kWarps][32];
    Key keys[32];                        // the block's best logits
    uint32_t tops[kWarps][32];           // threads' maxima
    uint32_t least;
    int count, threads[kWarps * 32];     // the threads whose chunks are looked at again
    Sums sums[kWarps], all;
};

template <typename T, int kThreads, int kCluster>
__global__ void __launch_bounds__(kThreads, kThreads == 128 ? 7 : kThreads == 32 ? 28 : 1) token_scores_kernel(const __grid_constant__ ScoreParams p) {
    constexpr int kVec = 16 / sizeof(T), kWarps = kThreads / 32, kAhead = kCluster > 1 ? 2 : 4;
    __shared__ ScoreShared<kWarps> shared;
    pdl_enter();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, part = kCluster > 1 ? blockIdx.x % kCluster : 0;
    for (long long r = blockIdx.x / kCluster; r < p.rows; r += gridDim.x / kCluster) {
        const Row<T> row(reinterpret_cast<const T *>(p.logits) + r * p.stride, p.cols);
        const int per_part = (row.chunks + kCluster - 1) / kCluster, begin = min(part * per_part, row.chunks), end = min(begin + per_part, row.chunks);
        Sums mine = {-INFINITY, 0.f, 0.f};
        float thread_top = -INFINITY;
        // groups of kAhead chunks a thread, the next one on its way while this one is added up; chunks one by one where not all of a warp's are whole
        const int whole_begin = max(begin, row.shift ? 1 : 0), whole_end = min(end, row.whole_chunks());
        const auto whole = [&](int c) { return c - lane >= whole_begin && c - lane + kThreads * (kAhead - 1) + 31 < whole_end; };
        uint4 next[kAhead];
        const auto fetch = [&](int c) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) next[u] = row.load_whole(c + u * kThreads);
        };
        int c = begin + threadIdx.x;
        bool ready = whole(c);
        if (ready) fetch(c);
        for (; c - lane < end; c += kThreads * kAhead) {
            const bool now = ready;
            uint4 raw[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) raw[u] = next[u];
            ready = whole(c + kThreads * kAhead);
            if (ready) fetch(c + kThreads * kAhead);
            if (now) {
                take<T>(raw, mine, thread_top);
            } else {
#pragma unroll 1
                for (int at = c; at - lane < min(end, c - lane + kThreads * kAhead); at += kThreads) {
                    const uint4 one[1] = {row.load(at < end ? at : -1, -INFINITY)};
                    take<T>(one, mine, thread_top);
                }
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            mine.sum += __shfl_xor_sync(~0u, mine.sum, o);
            mine.more += __shfl_xor_sync(~0u, mine.more, o);
        }
        if (lane == 0) shared.sums[warp] = mine;
        if (p.top > 0) {
            // the top-th best of the threads' maxima, and the threads that have it or a better one (a thread without a chunk has 0, below all)
            const uint32_t its_top = begin + static_cast<int>(threadIdx.x) < end ? ordered(thread_top) : 0;
            const uint32_t merged = merge_block<kWarps>(sort_warp(its_top, lane), shared.tops, warp, lane);
            if (warp == 0 && lane == p.top - 1) shared.least = merged;
            if (threadIdx.x == 0) shared.count = 0;
            __syncthreads();
            const uint32_t least = shared.least;
            const unsigned chosen = __ballot_sync(~0u, its_top && its_top >= least);
            int place = 0;
            if (lane == 0 && chosen) place = atomicAdd(&shared.count, __popc(chosen));
            place = __shfl_sync(~0u, place, 0) + __popc(chosen & ((1u << lane) - 1));
            if (chosen >> lane & 1) shared.threads[place] = threadIdx.x;
            __syncthreads();
            // (their order depends on timing; the keys of what they hold do not)
            Key found = 0;
            const float least_value = least ? unordered(least) : -INFINITY;
            // (so many lanes for a thread as it has chunks, up to all of them)
            const int each = (end - begin + kThreads - 1) / kThreads, bits = each >= 32 ? 5 : each > 1 ? 32 - __clz(each - 1) : 0, width = 1 << bits;
            const int at_once = 32 >> bits, count = shared.count;
            for (int j = warp * at_once; j < count; j += kWarps * at_once) {
                const int its = j + (lane >> bits), first = its < count ? begin + shared.threads[its] : end;
                for (int base = 0; base < each; base += width) {
                    const int c = min(first + (base + (lane & (width - 1))) * kThreads, end);
                    float v[kVec];
                    if (c < end) Vec16<T>::unpack(row.load(c, __uint_as_float(0x7fffffffu)), v);
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        // (what is not of the row is NaN here, and so not above anything; neither is a NaN of the row, whose ids are -1 anyway)
                        const bool above_least = c < end && v[i] >= least_value;
                        if (!__any_sync(~0u, above_least)) continue;
                        const Key candidate = above_least ? key_of(v[i], row.first_of(c) + i) : 0;
                        const Key last = __shfl_sync(~0u, found, p.top - 1);
                        unsigned who = __ballot_sync(~0u, candidate > last);
                        while (who) {
                            const Key next = __shfl_sync(~0u, candidate, __ffs(who) - 1);
                            who &= who - 1;
                            const int place = __popc(__ballot_sync(~0u, found > next));
                            const Key above = __shfl_up_sync(~0u, found, 1);
                            found = lane < place ? found : lane == place ? next : above;
                        }
                    }
                }
            }
            found = merge_block<kWarps>(found, shared.list, warp, lane);
            if (warp == 0) shared.keys[lane] = found;
        }
        __syncthreads();
        if (warp == 0) {
            Sums all = lane < kWarps ? shared.sums[lane] : Sums{-INFINITY, 0.f, 0.f};
            all.join_warp();
            if (lane == 0) shared.all = all;
        }
        if constexpr (kCluster > 1) cg::this_cluster().sync();
        Key best = 0;
        if (p.top > 0 && part == 0) {
            best = shared.keys[lane];
            if constexpr (kCluster > 1) {                        // a list of another block for each warp
                static_assert(kWarps >= kCluster, "a warp for each block of a cluster");
                if (warp > 0) best = warp < kCluster ? cg::this_cluster().map_shared_rank(&shared, warp)->keys[lane] : 0;
                best = merge_block<kWarps>(best, shared.list, warp, lane);
            }
        }
        if (part == 0 && warp == 0) {
            __syncwarp();
            Sums all = shared.all;
            if constexpr (kCluster > 1) {
                all = lane < kCluster ? cg::this_cluster().map_shared_rank(&shared, lane)->all : Sums{-INFINITY, 0.f, 0.f};
                all.join_warp();
            }
            const float nan = __uint_as_float(0x7fffffffu);
            // (a NaN has sums that are NaN, a maximum of +infinity ones of 0 or NaN. A good row's sum is 1 or more and its second one 0 or more, but for
            // their roundings: the maximum's own term may come out as 1 - 2^-24, and where one token has all of the probability there is little else)
            const bool good = all.top > -INFINITY && all.top < INFINITY && all.sum > 0.f;
            const float sum = fmaxf(all.sum, 1.f), log_sum = good ? logf(sum) : nan;
            if (lane == 0) {
                if (p.entropy) p.entropy[r] = good ? log_sum + fmaxf(all.more, 0.f) / sum : nan;
                if (p.logprob) {
                    const long long id = p.ids[r];
                    p.logprob[r] = good && id >= 0 && id < p.cols ? to_float(row.at[id]) - all.top - log_sum : nan;
                }
            }
            if (lane < p.top) {
                p.top_ids[r * p.top + lane] = good ? static_cast<long long>(index_of(best)) : -1;
                p.top_logprobs[r * p.top + lane] = good ? unordered(static_cast<uint32_t>(best >> 32)) - all.top - log_sum : nan;
            }
        }
        if constexpr (kCluster > 1) cg::this_cluster().sync();
        else __syncthreads();                                    // (shared memory is the next row's)
    }
}

template <typename T, int kThreads, int kCluster>
cudaError_t launch(const MsnhB200Ctx *ctx, const ScoreParams &p, void *stream) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(std::min<long long>(p.rows, 1 << 24)) * kCluster);
    config.blockDim = kThreads;
    config.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    if (kCluster > 1) {
        attr[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[config.numAttrs].val.clusterDim.x = kCluster;
        attr[config.numAttrs].val.clusterDim.y = attr[config.numAttrs].val.clusterDim.z = 1;
        ++config.numAttrs;
    }
    if (ctx->pdl) {
        attr[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[config.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++config.numAttrs;
    }
    config.attrs = attr;
    return cudaLaunchKernelEx(&config, token_scores_kernel<T, kThreads, kCluster>, p);
}

// Blocks of a row: as many as leave every SM two, each with 4096 logits at least, of 256 threads (clusters of 512 find less room: 16 rows of 50000 bf16 logits took
// 17.4 us and not 9.8; now 8.0, three of 128000 fp16 ones 8.3, 120 of 128000 16.2 with the best 8 and 12.7 without them). A row that is one block's has 128 threads, since what follows the pass over
// the logits grows with the warps, and seven such blocks an SM have registers for the next chunks (2000 rows of 50000: 51 us; a microsecond more with eight, 18 more
// with nine). Narrow rows are one warp's each, without other warps' lists to join, where there are more than the SMs hold at 128 threads a row, and always where a
// warp has a row in one chunk a lane: 4000 bf16 rows of 1000 with the best 5 8.5 us instead of 20.9, 1200 of 4000 9.4 instead of 12.9, 20000 of 500 32.0 instead of 95.6. A
// warp looks at more chunks again the more logits are wanted, hence the bounds (1200 rows of 8000 with the best 8 would take 16.3 instead of 14.7, of 1000
// fp32 ones with the best 32 16.0 instead of 11.6).
template <typename T>
cudaError_t launch_by_size(const MsnhB200Ctx *ctx, const ScoreParams &p, void *stream) {
    const long long parts = std::min<long long>(2LL * ctx->sm_count / p.rows, p.cols / 4096);
    if (parts >= 8) return launch<T, 256, 8>(ctx, p, stream);
    if (parts >= 4) return launch<T, 256, 4>(ctx, p, stream);
    if (parts >= 2) return launch<T, 256, 2>(ctx, p, stream);
    const long long warps = 7LL * ctx->sm_count;
    const int narrow = p.rows < warps ? 0 : (p.top > 8 ? 512 : 4096) * (p.rows < 3 * warps ? 1 : 2);
    if (p.cols <= std::max<int>(narrow, 32 * 16 / sizeof(T))) return launch<T, 32, 1>(ctx, p, stream);
    return launch<T, 128, 1>(ctx, p, stream);
}

}  // namespace
}  // namespace msnh

using namespace msnh;

extern "C" int msnh_b200_token_scores(MsnhB200Ctx *ctx, const MsnhB200TokenScores *a, void *stream) try {
    if (!ctx || !a) return MSNH_B200_ERR_ARG;
    if (!is_float_type(a->dtype)) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "token_scores: logits of type %d", a->dtype);
    if (a->rows < 0 || a->cols < 1 || a->top < 0 || a->top > a->cols) return fail(ctx, MSNH_B200_ERR_ARG, "token_scores: the %d best of rows of %d logits", a->top, a->cols);
    if (a->top > MSNH_B200_SCORES_MAX_TOP) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "token_scores: the %d best (at most %d are given)", a->top, MSNH_B200_SCORES_MAX_TOP);
    if (a->cols > 1 << 30) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "token_scores: rows of %d logits (at most 2^30 are taken)", a->cols);
    if (a->rows == 0) return MSNH_B200_OK;
    if (!a->logits || (a->logprob && !a->ids) || (a->top && (!a->top_logprobs || !a->top_ids))) return fail(ctx, MSNH_B200_ERR_ARG, "token_scores: null logits, ids, top_logprobs or top_ids");
    if (a->logits_stride < 0) return fail(ctx, MSNH_B200_ERR_ARG, "token_scores: a stride is negative");
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    const ScoreParams p = {static_cast<const uint8_t *>(a->logits), reinterpret_cast<const long long *>(a->ids), a->logprob, a->entropy, a->top_logprobs,
                           reinterpret_cast<long long *>(a->top_ids), a->rows, a->logits_stride, a->cols, a->top};
    CUDA_TRY(ctx, a->dtype == MSNH_B200_F32 ? launch_by_size<float>(ctx, p, stream) : a->dtype == MSNH_B200_F16 ? launch_by_size<__half>(ctx, p, stream)
                                                                                                              : launch_by_size<__nv_bfloat16>(ctx, p, stream));
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }
