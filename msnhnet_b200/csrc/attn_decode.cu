// Attention of one query token a row over a paged cache (msnh_b200_attn_decode).
#include "kv_cache.h"
#include "token_types.cuh"

namespace msnh {
namespace {

struct AttnParams {
    KvParams c;
    const void *q;
    void *out;
    float *lse;
    const int *seqs;
    long long q_row, q_head, out_row, out_head;
    int rows, n_heads, window;
    float scale;
};

constexpr int kThreads = 128;

// The tokens [first, last) that a row attends to; none for a sequence number that is none.
__device__ __forceinline__ void tokens_of(const AttnParams &p, int row, int *s, int *first, int *last) {
    *s = p.seqs ? p.seqs[row] : row;
    *last = *s >= 0 && *s < p.c.n_seqs ? max(0, min(p.c.lengths[*s], p.c.max_pages * p.c.page_size)) : 0;
    *first = p.window > 0 ? max(0, *last - p.window) : 0;
}

// A block a (row, head): tiles of 128 tokens, a score a thread, then a value column a thread.
template <typename T>
__global__ void attn_decode_rows_kernel(AttnParams p) {
    __shared__ float q[256], prob[kThreads], part[4];
    const int row = blockIdx.x, head = blockIdx.y, kv = head / (p.n_heads / p.c.heads), dim = p.c.dim, tid = threadIdx.x;
    int s, first, last;
    tokens_of(p, row, &s, &first, &last);
    const T *query = static_cast<const T *>(p.q) + row * p.q_row + head * p.q_head;
    for (int d = tid; d < dim; d += kThreads) q[d] = to_float(query[d]) * p.scale;
    __syncthreads();
    float top = -INFINITY, sum = 0.f, acc[2] = {0.f, 0.f};
    for (int base = first; base < last; base += kThreads) {
        const int t = base + tid;
        float score = -INFINITY;
        if (t < last) {
            const int page = p.c.table[s * p.c.table_stride + t / p.c.page_size];
            if (page >= 0 && page < p.c.n_pages) {
                const T *k = reinterpret_cast<const T *>(p.c.k) + page * p.c.k_page + t % p.c.page_size * p.c.k_token + kv * p.c.k_head;
                score = 0.f;
                for (int d = 0; d < dim; ++d) score += q[d] * to_float(k[d]);
            }
        }
        float best = score;
#pragma unroll
        for (int o = 16; o; o >>= 1) best = fmaxf(best, __shfl_xor_sync(~0u, best, o));
        if (tid % 32 == 0) part[tid / 32] = best;
        __syncthreads();
        best = fmaxf(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])), top);
        const float base_of = best == -INFINITY ? 0.f : best, keep = expf(top - base_of);
        prob[tid] = expf(score - base_of);
        __syncthreads();
        top = best;
        sum *= keep; acc[0] *= keep; acc[1] *= keep;
        for (int i = 0; i < kThreads && base + i < last; ++i) {
            sum += prob[i];
            if (prob[i] == 0.f) continue;
            const int u = base + i;
            const T *v = reinterpret_cast<const T *>(p.c.v) + p.c.table[s * p.c.table_stride + u / p.c.page_size] * p.c.v_page +
                         u % p.c.page_size * p.c.v_token + kv * p.c.v_head;
            if (tid < dim) acc[0] += prob[i] * to_float(v[tid]);
            if (tid + kThreads < dim) acc[1] += prob[i] * to_float(v[tid + kThreads]);
        }
        __syncthreads();
    }
    T *out = static_cast<T *>(p.out) + row * p.out_row + head * p.out_head;
    for (int i = 0; i < 2; ++i)
        if (tid + i * kThreads < dim) out[tid + i * kThreads] = from_float<T>(sum == 0.f ? 0.f : acc[i] / sum);
    if (p.lse && tid == 0) p.lse[row * static_cast<long long>(p.n_heads) + head] = sum == 0.f ? -INFINITY : top + logf(sum);
}

int check_attn(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, const MsnhB200AttnDecode *a, const char *what) {
    if (const int rc = check_cache(ctx, c, false, what)) return rc;
    if (a->rows < 0 || a->n_heads < 1 || a->n_heads > 65535 || a->n_heads % c->n_kv_heads) return fail(ctx, MSNH_B200_ERR_ARG, "%s: %d rows, %d heads over %d kv heads", what, a->rows, a->n_heads, c->n_kv_heads);
    if (a->window < 0) return fail(ctx, MSNH_B200_ERR_ARG, "%s: a window of %d", what, a->window);
    if (c->head_dim > 256 || c->head_dim * dtype_size(c->dtype) % 16) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "%s: heads of %d values (a multiple of 16 bytes and at most 256 values are wanted)", what, c->head_dim);
    if (!kv_rows_multiple_of(*c, 16)) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "%s: the cache's rows are not 16-byte aligned", what);
    if (!a->seqs && a->rows > c->n_seqs) return fail(ctx, MSNH_B200_ERR_ARG, "%s: %d rows of %d sequences", what, a->rows, c->n_seqs);
    return MSNH_B200_OK;
}

}  // namespace
}  // namespace msnh

using namespace msnh;

extern "C" {

int msnh_b200_attn_decode_workspace(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, const MsnhB200AttnDecode *a, size_t *bytes) try {
    if (!ctx || !c || !a || !bytes) return MSNH_B200_ERR_ARG;
    if (const int rc = check_attn(ctx, c, a, "attn_decode_workspace")) return rc;
    *bytes = 0;
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

int msnh_b200_attn_decode(MsnhB200Ctx *ctx, const MsnhB200KvCache *c, const MsnhB200AttnDecode *a, void *stream) try {
    if (!ctx || !c || !a) return MSNH_B200_ERR_ARG;
    if (const int rc = check_attn(ctx, c, a, "attn_decode")) return rc;
    if (a->rows == 0) return MSNH_B200_OK;
    if (!a->q || !a->out) return fail(ctx, MSNH_B200_ERR_ARG, "attn_decode: null q or out");
    if (a->q_row_stride < 0 || a->q_head_stride < 0 || (a->n_heads > 1 && a->out_head_stride < c->head_dim) || (a->rows > 1 && a->out_row_stride < c->head_dim))
        return fail(ctx, MSNH_B200_ERR_ARG, "attn_decode: a stride of q is negative, or rows of out overlap");
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    const AttnParams p = {kv_params(*c), a->q, a->out, a->lse, a->seqs, a->q_row_stride, a->q_head_stride, a->out_row_stride, a->out_head_stride,
                          a->rows, a->n_heads, a->window, a->scale};
    const dim3 grid(a->rows, a->n_heads);
    const cudaError_t e = c->dtype == MSNH_B200_F32   ? launch_token_kernel(attn_decode_rows_kernel<float>, grid, kThreads, 0, stream, false, p)
                          : c->dtype == MSNH_B200_F16 ? launch_token_kernel(attn_decode_rows_kernel<__half>, grid, kThreads, 0, stream, false, p)
                                                      : launch_token_kernel(attn_decode_rows_kernel<__nv_bfloat16>, grid, kThreads, 0, stream, false, p);
    CUDA_TRY(ctx, e);
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

}  // extern "C"
