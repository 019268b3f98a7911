// New keys and values into a paged cache (reef_ops_cache_append), and the places of tokens in it.
#include "ops_common.h"

namespace {
using namespace reef_ops;

constexpr int kThreads = 256;

struct Args {
    reef_cache_append_desc d;
    const void *key, *value;
    const int32_t* slots;
    void *key_cache, *value_cache;
    int32_t tokens_a_group;
};

// Eight values of a row, in the cache's type.  From 32 bits to 16 they are rounded once, to nearest even.
template <class From, class To>
__device__ inline void move8(const From* from, To* to) {
    if constexpr (sizeof(From) == sizeof(To)) {
        const u32x4* s = (const u32x4*)from;
        u32x4* t = (u32x4*)to;
        for (int i = 0; i < (int)sizeof(From) / 2; ++i) t[i] = s[i];
    } else {
        const f32x4 a = ((const f32x4*)from)[0], b = ((const f32x4*)from)[1];
        typedef To To8 __attribute__((ext_vector_type(8)));
        const To8 v = {(To)a[0], (To)a[1], (To)a[2], (To)a[3], (To)b[0], (To)b[1], (To)b[2], (To)b[3]};
        *(To8*)to = v;
    }
}

template <class From, class To>
__global__ void __launch_bounds__(kThreads) cache_append(Args a) {
    const reef_cache_append_desc& d = a.d;
    const int pieces = d.cache.head_dim / 8, row = 2 * d.cache.kv_heads * pieces;
    const int64_t t0 = (int64_t)blockIdx.x * a.tokens_a_group;
    const int n = (int)min((int64_t)a.tokens_a_group, d.tokens - t0) * row;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int t = i / row, in = i - t * row;
        const int h2 = in / pieces, p = in - h2 * pieces, h = h2 >= d.cache.kv_heads ? h2 - d.cache.kv_heads : h2;
        const bool is_value = h2 >= d.cache.kv_heads;
        const int32_t slot = a.slots[t0 + t];
        if (slot < 0) continue;
        const int32_t block = slot / d.cache.block_size;
        if (block >= d.cache.blocks) continue;
        const int64_t from = is_value ? (t0 + t) * d.value_stride + h * d.value_head_stride : (t0 + t) * d.key_stride + h * d.key_head_stride;
        const int64_t to = block * d.cache.block_stride + (slot - block * d.cache.block_size) * d.cache.slot_stride + h * d.cache.head_stride;
        move8((const From*)(is_value ? a.value : a.key) + from + p * 8, (To*)(is_value ? a.value_cache : a.key_cache) + to + p * 8);
    }
}

}  // namespace

extern "C" int reef_ops_cache_append(const reef_cache_append_desc* d, const void* key, const void* value, const int32_t* slots,
                                     void* key_cache, void* value_cache, void* stream) {
    const char* what = "reef_ops_cache_append";
    if (!d) return refuse(what, "null argument");
    if (int rc = check_layout(what, d->cache)) return rc;
    if (d->type != d->cache.type && d->type != REEF_TYPE_F32) return refuse(what, "rows of type %d into a cache of type %d", d->type, d->cache.type);
    if (d->tokens < 0) return refuse(what, "negative size");
    const int bytes = type_bytes(d->type), heads = d->cache.kv_heads;
    if (!stride16(d->tokens, d->key_stride, bytes) || !stride16(d->tokens, d->value_stride, bytes) || !stride16(heads, d->key_head_stride, bytes) ||
        !stride16(heads, d->value_head_stride, bytes))
        return refuse(what, "strides of the rows are not multiples of 16 bytes");
    if (!d->tokens) return 0;
    if (!rows16(key) || !rows16(value) || !rows16(key_cache) || !rows16(value_cache) || !words(slots)) return refuse(what, "null or unaligned argument");
    const int64_t row = 2ll * heads * (d->cache.head_dim / 8);
    if (row >= 1 << 24) return refuse(what, "too many heads");
    const int per = row >= 512 ? 1 : (int)(512 / row);
    const Args a{*d, key, value, slots, key_cache, value_cache, per};
    const dim3 grid((unsigned)(((int64_t)d->tokens + per - 1) / per)), block(kThreads);
    switch (d->type * 4 + d->cache.type) {
        case REEF_TYPE_F32 * 4 + REEF_TYPE_F32: return launch(what, cache_append<float, float>, grid, block, a, stream);
        case REEF_TYPE_F32 * 4 + REEF_TYPE_F16: return launch(what, cache_append<float, _Float16>, grid, block, a, stream);
        case REEF_TYPE_F32 * 4 + REEF_TYPE_BF16: return launch(what, cache_append<float, __bf16>, grid, block, a, stream);
        default: return launch(what, cache_append<uint16_t, uint16_t>, grid, block, a, stream);
    }
}

extern "C" int reef_ops_paged_row(const reef_cache_layout* c, const int32_t* table_row, int max_blocks, int64_t token, int64_t* offset) {
    if (!c || !table_row || !offset || c->block_size < 1 || token < 0 || token >= 1ll << 31) return 0;
    const Divider by = divider((uint32_t)c->block_size);
    const uint32_t t = (uint32_t)token, entry = divided(t, by);
    if ((int64_t)entry >= max_blocks) return 0;
    const PagedView v{c->blocks, c->block_stride, c->slot_stride};
    const int64_t at = paged_row(v, table_row[entry], (int32_t)(t - entry * by.by));
    if (at < 0) return 0;
    *offset = at;
    return 1;
}
