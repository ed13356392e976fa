// Upkeep of a paged cache of keys and values: append, fork, free, compact, copy (msnh_b200_kv_*).
//
// Append, fork and compact are two launches: one block decides (which pages, in what order: the lowest free ones first, by a scan
// over the page counts, so the result does not depend on timing) and writes its decisions into the workspace, then a grid moves the
// rows. Every launch may be scheduled while the one before it runs, and waits for it (pdl_enter).
//
// The moves are bound by their bytes, read and written once: of the 28.1 us of a compaction of 6000 pages of 16 tokens, 8 heads, 128 fp16
// values (107 MB) they take 17 (6.3 TB/s). The rest is the deciding block: a few reads that wait for one another and two scans; it is
// one block because every page's place depends on all counts before it. A step of a beam search of 256 sequences (fork, append, free: five
// launches, 15.9 MB) takes 20 us, 4 a launch.
#include "kv_cache.h"
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
struct AppendWork { int first, need, had, start; };              // first of its pages in the list; start: the length before, -1: refused

__global__ void kv_append_decide_kernel(KvParams c, const int *seqs, const int *starts, int n, int n_tokens, AppendWork *work, int *list) {
    pdl_enter();
    int all = 0;
    bool down = false;                                           // starts that are not in order: then no token's sequence is certain
    for (int base = 0; base < n; base += kDecide) {
        const int i = base + threadIdx.x;
        AppendWork w = {0, 0, 0, -1};
        if (i < n) {
            const int s = seqs ? seqs[i] : i;
            const long long from = starts ? starts[i] : i, to = starts ? starts[i + 1] : i + 1;
            down |= to < from;
            if (s >= 0 && s < c.n_seqs && from >= 0 && to >= from && to <= n_tokens) {
                const long long len = max(c.lengths[s], 0), had = (len + c.page_size - 1) / c.page_size;
                const long long want = (len + to - from + c.page_size - 1) / c.page_size;
                if (want <= c.max_pages) w = {0, static_cast<int>(want - had), static_cast<int>(had), static_cast<int>(len)};
            }
        }
        int total;
        w.first = all + block_scan(w.need, &total);
        if (i < n) work[i] = w;
        all += total;
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
    if (w.to >= 0) copy_units<Unit>(c, w.from, w.to, units, first, step, w.rows * c.heads * units);
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
                        int64_t new_token_stride, int64_t new_head_stride, int n_tokens, void *workspace, size_t workspace_bytes, void *stream) try {
    if (!ctx || !c) return MSNH_B200_ERR_ARG;
    if (const int rc = check_cache(ctx, c, true, "kv_append")) return rc;
    if (n < 0 || n_tokens < 0) return fail(ctx, MSNH_B200_ERR_ARG, "kv_append: %d sequences, %d tokens", n, n_tokens);
    if (!starts && n_tokens != n) return fail(ctx, MSNH_B200_ERR_ARG, "kv_append: %d tokens for %d sequences without starts", n_tokens, n);
    if (!seqs && n > c->n_seqs) return fail(ctx, MSNH_B200_ERR_ARG, "kv_append: %d sequences of %d", n, c->n_seqs);
    if (n == 0) return MSNH_B200_OK;
    if (n_tokens > 0 && (!k_new || !v_new)) return fail(ctx, MSNH_B200_ERR_ARG, "kv_append: null k_new or v_new");
    if (new_token_stride < 0 || new_head_stride < 0) return fail(ctx, MSNH_B200_ERR_ARG, "kv_append: a stride is negative");
    if (const int rc = check_workspace(ctx, *c, n, workspace, workspace_bytes, "kv_append")) return rc;
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    AppendWork *work = static_cast<AppendWork *>(workspace);
    int *list = reinterpret_cast<int *>(work + n);
    const KvParams p = kv_params(*c);
    CUDA_TRY(ctx, launch_token_kernel(kv_append_decide_kernel, dim3(1), kDecide, 0, stream, ctx->pdl, p, seqs, starts, n, n_tokens, work, list));
    if (n_tokens == 0) return MSNH_B200_OK;
    const size_t size = dtype_size(c->dtype);
    const bool wide = kv_rows_multiple_of(*c, 16) && aligned16(k_new) && aligned16(v_new) && new_token_stride * size % 16 == 0 && new_head_stride * size % 16 == 0;
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
    CUDA_TRY(ctx, wide ? copy(uint4()) : size == 4 ? copy(uint32_t()) : copy(uint16_t()));
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
    CUDA_TRY(ctx, wide ? move(uint4()) : size == 4 ? move(uint32_t()) : move(uint16_t()));
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
    CUDA_TRY(ctx, wide ? copy(uint4()) : size == 4 ? copy(uint32_t()) : copy(uint16_t()));
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

}  // extern "C"
