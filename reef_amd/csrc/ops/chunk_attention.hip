// Attention of the new tokens of all requests over a paged key-value cache (reef_ops_chunk_attention).
#include <algorithm>
#include <cmath>

#include "ops_common.h"

namespace {
using namespace reef_ops;

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Args {
    reef_chunk_attention_desc d;
    const void *query, *key_cache, *value_cache;
    const int32_t *table, *starts, *cached, *lengths;
    void* out;
    float* lse;
    Divider block;
};

__device__ inline int32_t start_of(const Args& a, int32_t i) { return max(0, min(a.starts[i], a.d.tokens)); }

// A wavefront for each row and head, a token of the cache after the other.
template <class Q, class C>
__global__ void __launch_bounds__(kThreads) chunk_attention(Args a) {
    const reef_chunk_attention_desc& d = a.d;
    const int lane = threadIdx.x & 63, D = d.cache.head_dim;
    const int64_t id = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (id >= (int64_t)d.tokens * d.heads) return;
    const int32_t row = (int32_t)(id / d.heads), h = (int32_t)(id - (int64_t)row * d.heads);
    int32_t lo = 0, hi = d.requests;         // the last request that starts at or in front of the row
    while (hi - lo > 1) {
        const int32_t mid = (lo + hi) / 2;
        if (start_of(a, mid) <= row) lo = mid;
        else hi = mid;
    }
    const int32_t first = start_of(a, lo);
    if (row < first || row >= start_of(a, lo + 1)) return;
    const int32_t n = held_length(a.lengths[lo], d.max_blocks, d.cache.block_size);
    const int64_t place = (int64_t)held_length(a.cached[lo], d.max_blocks, d.cache.block_size) + (row - first);
    int32_t begin = 0, end = 0;
    if (place < n) {
        end = (int32_t)place + 1;
        begin = d.window ? max(0, end - d.window) : 0;
    }
    const PagedView view{d.cache.blocks, d.cache.block_stride, d.cache.slot_stride};
    const int32_t* table = a.table + (int64_t)lo * d.table_stride;
    const int kvh = h / (d.heads / d.cache.kv_heads), at = lane * 4;
    float q[4] = {0, 0, 0, 0}, o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.0f;
    if (at < D)
        for (int e = 0; e < 4; ++e) q[e] = (float)((const Q*)a.query)[row * d.query_stride + h * d.query_head_stride + at + e] * (d.scale * kLog2e);
    for (int32_t t = begin; t < end; ++t) {
        const uint32_t entry = divided((uint32_t)t, a.block);
        const int64_t from = paged_row(view, table[entry], (int32_t)(t - entry * a.block.by));
        if (from < 0) continue;
        const int64_t base = from + kvh * d.cache.head_stride + at;
        float s = 0.0f, v[4] = {0, 0, 0, 0};
        if (at < D)
            for (int e = 0; e < 4; ++e) {
                s = fmaf(q[e], (float)((const C*)a.key_cache)[base + e], s);
                v[e] = (float)((const C*)a.value_cache)[base + e];
            }
        for (int x = 32; x; x >>= 1) s += __shfl_xor(s, x);
        const float top = fmaxf(m, s), of = top == -INFINITY ? 0.0f : top, f = __builtin_amdgcn_exp2f(m - of), p = __builtin_amdgcn_exp2f(s - of);
        m = top;
        l = l * f + p;
        for (int e = 0; e < 4; ++e) o[e] = fmaf(o[e], f, p * v[e]);
    }
    if (at < D)
        for (int e = 0; e < 4; ++e) ((Q*)a.out)[row * d.out_stride + h * d.out_head_stride + at + e] = (Q)(l == 0.0f ? 0.0f : o[e] / l);
    if (lane == 0 && a.lse) a.lse[id] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

int check(const char* what, const reef_chunk_attention_desc* d) {
    if (!d) return refuse(what, "null argument");
    if (int rc = check_layout(what, d->cache)) return rc;
    if (d->type != d->cache.type && d->type != REEF_TYPE_F32) return refuse(what, "queries of type %d over a cache of type %d", d->type, d->cache.type);
    if (d->requests < 0 || d->heads < 1 || d->heads % d->cache.kv_heads || d->tokens < 0)
        return refuse(what, "%d requests, %d tokens, %d heads over %d", d->requests, d->tokens, d->heads, d->cache.kv_heads);
    if ((int64_t)d->requests * d->heads >= 1ll << 24 || (int64_t)d->tokens * d->heads >= 1ll << 28)
        return refuse(what, "%d requests with %d tokens of %d heads are too many", d->requests, d->tokens, d->heads);
    if (d->max_blocks < 1 || d->table_stride < d->max_blocks || (int64_t)d->max_blocks * d->cache.block_size >= 1ll << 31)
        return refuse(what, "bad table: rows of %d entries, %d apart, blocks of %d tokens", d->max_blocks, d->table_stride, d->cache.block_size);
    if (d->longest < 0 || d->window < 0) return refuse(what, "negative length or window");
    if (!std::isfinite(d->scale * kLog2e)) return refuse(what, "scale %g is not a finite number, or not one as a power of two", (double)d->scale);
    const int bytes = type_bytes(d->type);
    if (!stride16(d->tokens, d->query_stride, bytes) || !stride16(d->tokens, d->out_stride, bytes) || !stride16(d->heads, d->query_head_stride, bytes) ||
        !stride16(d->heads, d->out_head_stride, bytes))
        return refuse(what, "strides of query or out are not multiples of 16 bytes");
    if (rows_overlap(d->tokens, d->out_stride, d->heads, d->out_head_stride, d->cache.head_dim)) return refuse(what, "strides let rows of out overlap");
    return 0;
}

template <class Q, class C>
int run(const char* what, const Args& a, void* stream) {
    return launch(what, chunk_attention<Q, C>, dim3((unsigned)(((int64_t)a.d.tokens * a.d.heads + 3) / 4)), dim3(kThreads), a, stream);
}

}  // namespace

extern "C" int64_t reef_ops_chunk_attention_workspace(const reef_chunk_attention_desc* d) {
    if (check("reef_ops_chunk_attention_workspace", d)) return -1;
    return 0;
}

extern "C" int reef_ops_chunk_attention(const reef_chunk_attention_desc* d, const void* query, const void* key_cache, const void* value_cache,
                                        const int32_t* table, const int32_t* starts, const int32_t* cached, const int32_t* lengths, void* out, float* lse,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "reef_ops_chunk_attention";
    if (int rc = check(what, d)) return rc;
    if (!d->requests || !d->tokens) return 0;
    if (!rows16(query) || !rows16(key_cache) || !rows16(value_cache) || !rows16(out) || !words(table) || !words(starts) || !words(cached) || !words(lengths) ||
        !aligned(lse, 4))
        return refuse(what, "null or unaligned argument");
    const Args a{*d, query, key_cache, value_cache, table, starts, cached, lengths, out, lse, divider((uint32_t)d->cache.block_size)};
    switch (d->type * 4 + d->cache.type) {
        case REEF_TYPE_F32 * 4 + REEF_TYPE_F32: return run<float, float>(what, a, stream);
        case REEF_TYPE_F32 * 4 + REEF_TYPE_F16: return run<float, _Float16>(what, a, stream);
        case REEF_TYPE_F32 * 4 + REEF_TYPE_BF16: return run<float, __bf16>(what, a, stream);
        case REEF_TYPE_F16 * 4 + REEF_TYPE_F16: return run<_Float16, _Float16>(what, a, stream);
        default: return run<__bf16, __bf16>(what, a, stream);
    }
}
