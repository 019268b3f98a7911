// Beam search: the choice over beams and vocabulary (reef_ops_beam_select), and tables and half-filled
// blocks of a paged cache that follow it (reef_ops_beam_reorder).
#include "ops_common.h"

namespace {
using namespace reef_ops;

constexpr int kThreads = 256;
constexpr int kMaxBeams = 128, kMaxSelect = 128;

struct SelectArgs {
    reef_beam_select_desc d;
    const void* logits;
    const float* scores;
    const uint8_t* ended;
    float* best;
    int32_t *parents, *tokens;
};

// A candidate: its score, its place beam * vocab + token.  Whether one goes before another.
struct Offer {
    double score;
    int32_t beam, token;
};
__device__ inline bool before(const Offer& a, const Offer& b) {
    return a.score != b.score ? a.score > b.score : a.beam != b.beam ? a.beam < b.beam : a.token < b.token;
}
// Anything that is not a finite number counts as -infinity.
__device__ inline double offered(double s) { return s < INFINITY && s > -INFINITY ? s : -INFINITY; }

template <class T>
__global__ void __launch_bounds__(kThreads) beam_select(SelectArgs a) {
    const reef_beam_select_desc& d = a.d;
    const int tid = threadIdx.x;
    __shared__ double red[kThreads];
    __shared__ double lse[kMaxBeams];
    __shared__ Offer top[kThreads];
    const int64_t row0 = (int64_t)blockIdx.x * d.beams;
    for (int b = 0; b < d.beams; ++b) {
        const T* x = (const T*)a.logits + (row0 + b) * d.logits_stride;
        float m = -INFINITY;
        for (int v = tid; v < d.vocab; v += kThreads) m = fmaxf(m, (float)x[v]);
        red[tid] = m;
        __syncthreads();
        double top_m = -INFINITY;
        for (int i = 0; i < kThreads; ++i) top_m = fmax(top_m, red[i]);
        double s = 0.0;
        for (int v = tid; v < d.vocab; v += kThreads) s += exp((double)(float)x[v] - top_m);
        __syncthreads();
        red[tid] = s;
        __syncthreads();
        if (tid == 0) {
            double all = 0.0;
            for (int i = 0; i < kThreads; ++i) all += red[i];
            lse[b] = top_m + log(all);
        }
        __syncthreads();
    }
    Offer last = {INFINITY, -1, 0};
    for (int k = 0; k < d.select; ++k) {
        Offer mine = {-INFINITY, d.beams, 0};
        for (int b = 0; b < d.beams; ++b) {
            const T* x = (const T*)a.logits + (row0 + b) * d.logits_stride;
            const double score = offered((double)a.scores[row0 + b]);
            const bool over = a.ended && a.ended[row0 + b];
            for (int v = tid; v < d.vocab; v += kThreads) {
                const Offer o = {over ? (v == d.end_token ? score : -INFINITY) : offered(score + ((double)(float)x[v] - lse[b])), b, v};
                if (before(last, o) && before(o, mine)) mine = o;
            }
        }
        top[tid] = mine;
        __syncthreads();
        for (int i = 0; i < kThreads; ++i)
            if (before(top[i], mine)) mine = top[i];
        last = mine;
        if (tid == 0) {
            const int64_t at = (int64_t)blockIdx.x * d.select + k;
            a.best[at] = (float)mine.score;
            a.parents[at] = (int32_t)(row0 + mine.beam);
            a.tokens[at] = mine.token;
        }
        __syncthreads();
    }
}

int check_select(const char* what, const reef_beam_select_desc* d) {
    if (!d) return refuse(what, "null argument");
    if (!type_bytes(d->type)) return refuse(what, "unknown type %d", d->type);
    if (d->requests < 0 || d->beams < 1 || d->beams > kMaxBeams || d->vocab < 1 || d->vocab >= 1 << 24 || (int64_t)d->requests * d->beams >= 1 << 24)
        return refuse(what, "bad sizes: %d requests, %d beams (up to %d), %d tokens", d->requests, d->beams, kMaxBeams, d->vocab);
    if (d->select < 1 || d->select > kMaxSelect || d->select > (int64_t)d->beams * d->vocab)
        return refuse(what, "%d of %d beams of %d tokens cannot be selected (up to %d)", d->select, d->beams, d->vocab, kMaxSelect);
    if ((int64_t)d->requests * d->beams > 1 && d->logits_stride < d->vocab) return refuse(what, "rows of logits overlap");
    return 0;
}

struct ReorderArgs {
    reef_beam_reorder_desc d;
    const int32_t *parents, *lengths, *table, *spare;
    int32_t *table_out, *lengths_out;
    void *key_cache, *value_cache;
};

// A workgroup: one row's table, or the tokens of its last block in one layer of one pool.
__global__ void __launch_bounds__(kThreads) beam_reorder(ReorderArgs a) {
    const reef_beam_reorder_desc& d = a.d;
    const int64_t i = blockIdx.x;
    const int32_t p = a.parents[i], bs = d.cache.block_size;
    if ((uint32_t)p >= (uint32_t)d.table_rows) return;
    const int32_t n = held_length(a.lengths[p], d.max_blocks, bs), full = n / bs, rest = n % bs;
    const int32_t* from_row = a.table + (int64_t)p * d.table_stride;
    const bool moved = rest && p != i;
    int32_t source = -1, target = -1;
    if (moved) {
        source = from_row[full];
        target = a.spare[i];
        if ((uint32_t)source >= (uint32_t)d.cache.blocks || (uint32_t)target >= (uint32_t)d.cache.blocks) source = target = -1;
    }
    if (blockIdx.y == 0) {
        int32_t* to_row = a.table_out + i * d.out_stride;
        for (int j = threadIdx.x; j < full; j += kThreads) to_row[j] = from_row[j];
        if (threadIdx.x == 0) {
            if (rest) to_row[full] = moved ? target : from_row[full];
            a.lengths_out[i] = n;
        }
        return;
    }
    if (target < 0) return;
    const int part = blockIdx.y - 1, bytes = d.cache.type == REEF_TYPE_F32 ? 4 : 2;
    unsigned char* pool = (unsigned char*)(part & 1 ? a.value_cache : a.key_cache) + (int64_t)(part >> 1) * d.layer_stride * bytes;
    const int pieces = d.cache.head_dim * bytes / 16;
    const int64_t all = (int64_t)rest * d.cache.kv_heads * pieces;
    for (int64_t k = threadIdx.x; k < all; k += kThreads) {
        const int64_t th = k / pieces;
        const int piece = (int)(k - th * pieces), h = (int)(th % d.cache.kv_heads), t = (int)(th / d.cache.kv_heads);
        const int64_t in = (int64_t)t * d.cache.slot_stride + (int64_t)h * d.cache.head_stride;
        const u32x4 v = *(const u32x4*)(pool + (source * d.cache.block_stride + in) * bytes + piece * 16);
        *(u32x4*)(pool + (target * d.cache.block_stride + in) * bytes + piece * 16) = v;
    }
}

}  // namespace

extern "C" int64_t reef_ops_beam_select_workspace(const reef_beam_select_desc* d) {
    if (check_select("reef_ops_beam_select_workspace", d)) return -1;
    return 0;
}

extern "C" int reef_ops_beam_select(const reef_beam_select_desc* d, const void* logits, const float* scores, const uint8_t* ended, float* best,
                                    int32_t* parents, int32_t* tokens, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "reef_ops_beam_select";
    if (int rc = check_select(what, d)) return rc;
    if (!d->requests) return 0;
    if (!logits || !aligned(logits, type_bytes(d->type)) || !words(scores) || !words(best) || !words(parents) || !words(tokens))
        return refuse(what, "null or unaligned argument");
    const SelectArgs a{*d, logits, scores, ended, best, parents, tokens};
    const dim3 grid((unsigned)d->requests), block(kThreads);
    switch (d->type) {
        case REEF_TYPE_F32: return launch(what, beam_select<float>, grid, block, a, stream);
        case REEF_TYPE_F16: return launch(what, beam_select<_Float16>, grid, block, a, stream);
        default: return launch(what, beam_select<__bf16>, grid, block, a, stream);
    }
}

extern "C" int reef_ops_beam_reorder(const reef_beam_reorder_desc* d, const int32_t* parents, const int32_t* lengths, const int32_t* table,
                                     const int32_t* spare, int32_t* table_out, int32_t* lengths_out, void* key_cache, void* value_cache, void* stream) {
    const char* what = "reef_ops_beam_reorder";
    if (!d) return refuse(what, "null argument");
    if (d->layers < 1 || d->layers > 30000) return refuse(what, "%d layers", d->layers);
    if (int rc = check_layout(what, d->cache, d->layers, d->layer_stride)) return rc;
    if (d->rows < 0 || d->table_rows < 1) return refuse(what, "bad rows: %d of %d", d->rows, d->table_rows);
    if (d->max_blocks < 1 || d->table_stride < d->max_blocks || d->out_stride < d->max_blocks || (int64_t)d->max_blocks * d->cache.block_size >= 1ll << 31)
        return refuse(what, "bad table: rows of %d entries, %d and %d apart", d->max_blocks, d->table_stride, d->out_stride);
    if (!d->rows) return 0;
    if (!words(parents) || !words(lengths) || !words(table) || !words(spare) || !words(table_out) || !words(lengths_out) || !rows16(key_cache) ||
        !rows16(value_cache))
        return refuse(what, "null or unaligned argument");
    const int32_t *t0 = table, *t1 = t0 + ((int64_t)d->table_rows - 1) * d->table_stride + d->max_blocks;
    const int32_t *o0 = table_out, *o1 = o0 + ((int64_t)d->rows - 1) * d->out_stride + d->max_blocks;
    if (t0 < o1 && o0 < t1) return refuse(what, "table and table_out overlap");
    const ReorderArgs a{*d, parents, lengths, table, spare, table_out, lengths_out, key_cache, value_cache};
    return launch(what, beam_reorder, dim3((unsigned)d->rows, 1 + 2 * d->layers), dim3(kThreads), a, stream);
}
