// Attention of one new token a request over a paged key-value cache (reef_ops_paged_attention).
#include <cmath>

#include "ops_common.h"

namespace {
using namespace reef_ops;

constexpr int kThreads = 256;

struct Args {
    reef_paged_attention_desc d;
    const void *query, *key_cache, *value_cache;
    const int32_t *table, *lengths;
    void* out;
    float* lse;
};

// One workgroup a query head: 256 scores at a time, a token a thread, then the sum over them, an element a thread.
template <class Q, class C>
__global__ void __launch_bounds__(kThreads) paged_attention(Args a) {
    const reef_paged_attention_desc& d = a.d;
    const int r = blockIdx.x / d.heads, h = blockIdx.x % d.heads, kvh = h / (d.heads / d.cache.kv_heads), D = d.cache.head_dim;
    const PagedView view{d.cache.blocks, d.cache.block_size, d.max_blocks, d.cache.block_stride, d.cache.slot_stride};
    const int32_t n = held_length(a.lengths[r], d.max_blocks, d.cache.block_size);
    const int32_t first = d.window && n > d.window ? n - d.window : 0;
    __shared__ float q[256], p[kThreads], red[kThreads];
    __shared__ int64_t rows[kThreads];
    const Q* query = (const Q*)a.query + r * d.query_stride + h * d.query_head_stride;
    const C* keys = (const C*)a.key_cache + kvh * d.cache.head_stride;
    const C* values = (const C*)a.value_cache + kvh * d.cache.head_stride;
    const int tid = threadIdx.x;
    if (tid < D) q[tid] = (float)query[tid] * d.scale;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int64_t t0 = first; t0 < n; t0 += kThreads) {
        __syncthreads();
        const int64_t t = t0 + tid;
        float s = -INFINITY;
        rows[tid] = -1;
        if (t < n) {
            const int64_t row = paged_row(view, a.table[(int64_t)r * d.table_stride + t / view.block_size], (int32_t)(t % view.block_size));
            rows[tid] = row;
            if (row >= 0) {
                s = 0.0f;
                for (int i = 0; i < D; ++i) s = fmaf(q[i], (float)keys[row + i], s);
            }
        }
        red[tid] = s;
        __syncthreads();
        float top = m;
        for (int i = 0; i < kThreads; ++i) top = fmaxf(top, red[i]);
        const float base = top == -INFINITY ? 0.0f : top;
        p[tid] = rows[tid] >= 0 ? expf(s - base) : 0.0f;
        __syncthreads();
        const float f = expf(m - base);
        l *= f;
        o *= f;
        for (int i = 0; i < kThreads; ++i) l += p[i];
        if (tid < D)
            for (int i = 0; i < kThreads; ++i)
                if (rows[i] >= 0) o = fmaf(p[i], (float)values[rows[i] + tid], o);
        m = top;
    }
    Q* out = (Q*)a.out + r * d.out_stride + h * d.out_head_stride;
    if (tid < D) out[tid] = (Q)(l == 0.0f ? 0.0f : o / l);
    if (tid == 0 && a.lse) a.lse[(int64_t)r * d.heads + h] = l == 0.0f ? -INFINITY : m + logf(l);
}

int check(const char* what, const reef_paged_attention_desc* d) {
    if (!d) return refuse(what, "null argument");
    if (int rc = check_layout(what, d->cache)) return rc;
    if (d->type != d->cache.type && d->type != REEF_TYPE_F32) return refuse(what, "queries of type %d over a cache of type %d", d->type, d->cache.type);
    if (d->requests < 0 || d->heads < 1 || d->heads % d->cache.kv_heads) return refuse(what, "%d requests, %d heads over %d", d->requests, d->heads, d->cache.kv_heads);
    if ((int64_t)d->requests * d->heads >= 1ll << 24) return refuse(what, "%d requests of %d heads are too many", d->requests, d->heads);
    if (d->max_blocks < 1 || d->table_stride < d->max_blocks || (int64_t)d->max_blocks * d->cache.block_size >= 1ll << 31)
        return refuse(what, "bad table: rows of %d entries, %d apart, blocks of %d tokens", d->max_blocks, d->table_stride, d->cache.block_size);
    if (d->longest < 0 || d->window < 0) return refuse(what, "negative length or window");
    if (!std::isfinite(d->scale)) return refuse(what, "scale is not a finite number");
    const int bytes = type_bytes(d->type);
    if (!stride16(d->requests, d->query_stride, bytes) || !stride16(d->requests, d->out_stride, bytes) || !stride16(d->heads, d->query_head_stride, bytes) ||
        !stride16(d->heads, d->out_head_stride, bytes))
        return refuse(what, "strides of query or out are not multiples of 16 bytes");
    return 0;
}

}  // namespace

extern "C" int64_t reef_ops_paged_attention_workspace(const reef_paged_attention_desc* d) {
    if (check("reef_ops_paged_attention_workspace", d)) return -1;
    return 0;
}

extern "C" int reef_ops_paged_attention(const reef_paged_attention_desc* d, const void* query, const void* key_cache, const void* value_cache,
                                        const int32_t* table, const int32_t* lengths, void* out, float* lse, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
    const char* what = "reef_ops_paged_attention";
    if (int rc = check(what, d)) return rc;
    if (!d->requests) return 0;
    if (!rows16(query) || !rows16(key_cache) || !rows16(value_cache) || !rows16(out) || !words(table) || !words(lengths) || !aligned(lse, 4))
        return refuse(what, "null or unaligned argument");
    const Args a{*d, query, key_cache, value_cache, table, lengths, out, lse};
    const dim3 grid((unsigned)(d->requests * d->heads)), block(kThreads);
    switch (d->type * 4 + d->cache.type) {
        case REEF_TYPE_F32 * 4 + REEF_TYPE_F32: return launch(what, paged_attention<float, float>, grid, block, a, stream);
        case REEF_TYPE_F32 * 4 + REEF_TYPE_F16: return launch(what, paged_attention<float, _Float16>, grid, block, a, stream);
        case REEF_TYPE_F32 * 4 + REEF_TYPE_BF16: return launch(what, paged_attention<float, __bf16>, grid, block, a, stream);
        case REEF_TYPE_F16 * 4 + REEF_TYPE_F16: return launch(what, paged_attention<_Float16, _Float16>, grid, block, a, stream);
        default: return launch(what, paged_attention<__bf16, __bf16>, grid, block, a, stream);
    }
}
