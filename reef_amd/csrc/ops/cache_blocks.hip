// Blocks of a paged cache: which are in use and which are free (reef_ops_block_sweep), requests that continue a part of another one
// (reef_ops_cache_fork), blocks in use moved to the front of the pool (reef_ops_cache_compact).
#include <algorithm>

#include "ops_common.h"

namespace {
using namespace reef_ops;

constexpr int kThreads = 256, kWaves = kThreads / 64;

// ---- which blocks the rows of a table use ---------------------------------------------------------
struct Table {
    int32_t rows, blocks, block_size, max_blocks, stride;
    const int32_t *entries, *lengths;
};
__device__ inline int32_t used_entries(const Table& t, int64_t row) {
    const int32_t n = held_length(t.lengths[row], t.max_blocks, t.block_size);
    return n / t.block_size + (n % t.block_size != 0);
}

struct Use {
    Table t;
    int32_t* uses;          // [blocks]: of a sweep how many entries name the block, of a compaction 1 where one does
    int32_t* segments;      // [segments]: blocks in use of each; behind them the entries that name no block
    int32_t n_segments;
    int32_t *free_list, *counts;     // of a sweep
    int32_t *source, *target;        // of a compaction: [moves]
};
constexpr int32_t kSegment = 4096;

__global__ void __launch_bounds__(kThreads) clear(Use a) {
    const int64_t n = (int64_t)a.t.blocks + a.n_segments + 1;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads)
        if (i < a.t.blocks) a.uses[i] = 0;
        else a.segments[i - a.t.blocks] = 0;
}

// A row a wavefront; gridDim.y of them go through a row in turn, 256 entries each, which are on their way together.  (4000 rows, 290000 entries in use: 11 us,
// nearly all of it the additions.)
constexpr int32_t kRun = 256;
template <bool kCount>
__global__ void __launch_bounds__(kThreads) name_blocks(Use a) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
    if (row >= a.t.rows) return;
    const int32_t n = used_entries(a.t, row);
    const int32_t* entries = a.t.entries + row * a.t.stride;
    for (int64_t j0 = (int64_t)blockIdx.y * kRun; j0 < n; j0 += (int64_t)gridDim.y * kRun) {
        int32_t b[kRun / 64];
#pragma unroll
        for (int u = 0; u < kRun / 64; ++u) b[u] = entries[min((int64_t)n - 1, j0 + u * 64 + lane)];
#pragma unroll
        for (int u = 0; u < kRun / 64; ++u) {
            if (j0 + u * 64 + lane >= n) continue;
            const bool inside = (uint32_t)b[u] < (uint32_t)a.t.blocks;
            if constexpr (kCount) {
                if (inside) atomicAdd(a.uses + b[u], 1);
                else atomicAdd(a.segments + a.n_segments, 1);
            } else if (inside) {
                a.uses[b[u]] = 1;            // (whoever comes last: all write the same)
            }
        }
    }
}

// Exclusive prefix sums of one value a wavefront; *all: the sum.
__device__ inline int32_t over_waves(int32_t mine, int32_t* counts, int32_t* all) {
    const int wave = threadIdx.x >> 6, waves = (int)blockDim.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) counts[wave] = mine;
    __syncthreads();
    int32_t at = 0;
    *all = 0;
    for (int w = 0; w < waves; ++w) {
        if (w < wave) at += counts[w];
        *all += counts[w];
    }
    return at;
}

// A segment a workgroup, four blocks a thread: whether each is in use.  (300001 blocks: 4 us, and 4.3 to place them, most of it the launch.)
constexpr int kWide = kSegment / 4, kWideWaves = kWide / 64;
__device__ inline uint32_t in_use(const Use& a, int64_t b) {
    uint32_t who = 0;
    if (b + 4 <= a.t.blocks && aligned(a.uses, 16)) {
        const int4 n = *(const int4*)(a.uses + b);
        who = (n.x != 0) | (n.y != 0) << 1 | (n.z != 0) << 2 | (n.w != 0) << 3;
    } else {
        for (int k = 0; k < 4; ++k) who |= b + k < a.t.blocks && a.uses[b + k] != 0 ? 1u << k : 0;
    }
    return who;
}
__device__ inline int32_t sum_of(int32_t v) {
    for (int x = 32; x; x >>= 1) v += __shfl_xor(v, x);
    return v;
}
__global__ void __launch_bounds__(kWide) count_segments(Use a) {
    __shared__ int32_t counts[kWideWaves];
    int32_t all;
    over_waves(sum_of(__popc(in_use(a, (int64_t)blockIdx.x * kSegment + threadIdx.x * 4))), counts, &all);
    if (threadIdx.x == 0) a.segments[blockIdx.x] = all;
}

// What becomes of block b: `before` blocks in front of it are in use, `used` in all.
template <bool kSweep>
__device__ inline void place_block(const Use& a, int32_t b, bool in_use, int32_t before, int32_t used) {
    if constexpr (kSweep) {
        if (!in_use) a.free_list[b - before] = b;
    } else {
        // The k-th block in use from the end goes to the k-th free one from the front.
        if (in_use && b >= used) {
            const int32_t k = used - 1 - before;
            a.source[k] = b;
            a.uses[b] = k;
        } else if (!in_use && b < used) {
            a.target[b - before] = b;
        }
        if (b == used) a.counts[1] = used - before;
    }
}
template <bool kSweep>
__device__ inline void place_counts(const Use& a, int32_t used, int32_t outside) {
    if constexpr (kSweep) {
        a.counts[0] = a.t.blocks - used;
        a.counts[1] = used;
        a.counts[2] = outside;
    } else {
        a.counts[0] = used;
        if (used == a.t.blocks) a.counts[1] = 0;
    }
}

template <bool kSweep>
__global__ void __launch_bounds__(kWide) place_blocks(Use a) {
    __shared__ int32_t counts[kWideWaves];
    const int lane = threadIdx.x & 63;
    const int64_t b = (int64_t)blockIdx.x * kSegment + threadIdx.x * 4;
    const uint32_t who = in_use(a, b);
    int32_t before = 0, used = 0;            // blocks in use of the segments in front, and of all
    for (int32_t s = threadIdx.x; s < a.n_segments; s += kWide) {
        const int32_t n = a.segments[s];
        used += n;
        if (s < (int32_t)blockIdx.x) before += n;
    }
    int32_t sum;
    over_waves(sum_of(used), counts, &sum);
    used = sum;
    over_waves(sum_of(before), counts, &sum);
    before = sum;
    if (blockIdx.x == 0 && threadIdx.x == 0) place_counts<kSweep>(a, used, a.segments[a.n_segments]);
    const int32_t mine = __popc(who);
    int32_t at = mine;
    for (int x = 1; x < 64; x <<= 1) {
        const int32_t o = __shfl_up(at, x);
        if (lane >= x) at += o;
    }
    before += over_waves(__shfl(at, 63), counts, &sum) + at - mine;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (b + k < a.t.blocks) place_block<kSweep>(a, (int32_t)(b + k), who >> k & 1, before, used);
        before += who >> k & 1;
    }
}

// All of it by one workgroup, the uses held near: 4.6 us for 8 rows of 64 entries, 8.8 for 64 of 512, 11.8 for 256 of 128, where the four launches take 11.4 to 11.7.
constexpr int kAlone = 1024;
constexpr int32_t kNear = 8192, kNearEntries = 1 << 15, kNearRows = 192;
template <bool kSweep>
__global__ void __launch_bounds__(kAlone) place_near(Use a) {
    __shared__ int32_t uses[kNear];
    __shared__ int32_t counts[kAlone / 64], outside;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < a.t.blocks; i += kAlone) uses[i] = 0;
    if (tid == 0) outside = 0;
    __syncthreads();
    for (int64_t row = wave; row < a.t.rows; row += kAlone / 64) {
        const int32_t n = used_entries(a.t, row);
        for (int32_t j = lane; j < n; j += 64) {
            const int32_t b = a.t.entries[row * a.t.stride + j];
            atomicAdd((uint32_t)b < (uint32_t)a.t.blocks ? &uses[b] : &outside, 1);
        }
    }
    __syncthreads();
    constexpr int kMine = kNear / kAlone;
    int32_t mine = 0, used;
    uint64_t who[kMine];
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
        const int32_t b = wave * (kMine * 64) + k * 64 + lane;
        who[k] = __builtin_amdgcn_ballot_w64(b < a.t.blocks && uses[b] != 0);
        mine += (int32_t)__popcll(who[k]);
    }
    int32_t before = over_waves(mine, counts, &used);
    if (tid == 0) place_counts<kSweep>(a, used, outside);
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
        const int32_t b = wave * (kMine * 64) + k * 64 + lane;
        if (b < a.t.blocks) {
            if constexpr (kSweep) a.uses[b] = uses[b];
            place_block<kSweep>(a, b, who[k] >> lane & 1, before + (int32_t)__popcll(who[k] & ((1ull << lane) - 1)), used);
        }
        before += (int32_t)__popcll(who[k]);
    }
}

int32_t segments_of(int32_t blocks) { return (int32_t)(((int64_t)blocks + kSegment - 1) / kSegment); }
bool near(const Table& t) { return t.blocks <= kNear && t.rows <= kNearRows && (int64_t)t.rows * t.max_blocks <= kNearEntries; }

// Workgroups of four rows, and how many of them go through a row.
dim3 rows_grid(const Table& t) {
    const int64_t x = std::max<int64_t>(1, ((int64_t)t.rows + kWaves - 1) / kWaves);
    return dim3((unsigned)x, (unsigned)std::min<int64_t>(((int64_t)t.max_blocks + kRun - 1) / kRun, std::max<int64_t>(1, 4096 / x)));
}

template <bool kSweep>
int place(const char* what, const Use& a, void* stream) {
    if (near(a.t)) return launch(what, place_near<kSweep>, dim3(1), dim3(kAlone), a, stream);
    const unsigned clears = (unsigned)std::min<int64_t>(((int64_t)a.t.blocks + a.n_segments + kThreads) / kThreads, 2048);
    if (int rc = launch(what, clear, dim3(clears), dim3(kThreads), a, stream)) return rc;
    if (int rc = launch(what, name_blocks<kSweep>, rows_grid(a.t), dim3(kThreads), a, stream)) return rc;
    if (int rc = launch(what, count_segments, dim3((unsigned)a.n_segments), dim3(kWide), a, stream)) return rc;
    return launch(what, place_blocks<kSweep>, dim3((unsigned)a.n_segments), dim3(kWide), a, stream);
}

int check_table(const char* what, int32_t rows, int32_t blocks, int32_t block_size, int32_t max_blocks, int32_t stride) {
    if (rows < 0 || rows >= 1 << 24) return refuse(what, "%d rows", rows);
    if (blocks < 1 || block_size < 1 || (int64_t)blocks * block_size >= 1ll << 31) return refuse(what, "bad pool: %d blocks of %d tokens", blocks, block_size);
    if (max_blocks < 1 || stride < max_blocks || (int64_t)max_blocks * block_size >= 1ll << 31)
        return refuse(what, "bad table: rows of %d entries, %d apart, blocks of %d tokens", max_blocks, stride, block_size);
    return 0;
}
int64_t table_bytes(int64_t rows, int32_t max_blocks, int32_t stride) { return rows ? 4 * ((rows - 1) * stride + max_blocks) : 0; }

// ---- copies of blocks -------------------------------------------------------------------------------
// A block of one layer of one pool as 16-byte pieces, the inner of heads and tokens next to each other.
struct Pieces {
    uint32_t row;           // pieces of a head of a token
    uint32_t heads;
    bool tokens_inside;
    int64_t slot_bytes, head_bytes;
};
Pieces pieces_of(const reef_cache_layout& c) {
    const int bytes = type_bytes(c.type);
    return {(uint32_t)(c.head_dim * bytes / 16), (uint32_t)c.kv_heads, c.head_stride > c.slot_stride && c.kv_heads > 1 && c.block_size > 1, c.slot_stride * bytes,
            c.head_stride * bytes};
}
// Pieces [k0, k0 + 4 threads) of the first `tokens` tokens, four a thread in flight.
__device__ inline void copy_pieces(const Pieces& p, const unsigned char* from, unsigned char* to, uint32_t tokens, uint32_t k0) {
    const uint32_t inner = p.tokens_inside ? tokens : p.heads, total = tokens * p.heads * p.row;
    const int64_t inner_bytes = p.tokens_inside ? p.slot_bytes : p.head_bytes, outer_bytes = p.tokens_inside ? p.head_bytes : p.slot_bytes;
    int64_t at[4];
    u32x4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const uint32_t k = min(k0 + u * kThreads + threadIdx.x, total - 1), r = k / p.row, o = r / inner;
        at[u] = o * outer_bytes + (r - o * inner) * inner_bytes + (k - r * p.row) * 16;
        v[u] = *(const u32x4*)(from + at[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (k0 + u * kThreads + threadIdx.x < total) *(u32x4*)(to + at[u]) = v[u];
}

constexpr int32_t kMostForks = 1 << 15;      // (each looks at those in front of it)
struct ForkArgs {
    reef_cache_fork_desc d;
    const int32_t *parents, *children, *tokens, *free_list;
    int32_t *table, *lengths, *counts;
    void *key_cache, *value_cache;
    Pieces pieces;
    int32_t each;           // caches (a layer of a pool) a workgroup
};

// The tokens of fork j, or -1: refused for its rows.
__device__ inline int32_t fork_tokens(const ForkArgs& a, int64_t j) {
    const int32_t p = a.parents[j], c = a.children[j], n = a.tokens[j];
    if ((uint32_t)p >= (uint32_t)a.d.table_rows || (uint32_t)c >= (uint32_t)a.d.table_rows || p == c) return -1;
    return max(0, min(n, held_length(a.lengths[p], a.d.max_blocks, a.d.cache.block_size)));
}

// A workgroup: one fork's row, or its half-filled block in some caches.  Each counts for itself the blocks that the forks in front take (no launch
// ahead, no memory for sums); lengths that are read are parents', those written children's.  (224 forks, 24 layers, 114 MB copied: 58 us, 3.9 TB/s both ways; three: 5.7.)
__global__ void __launch_bounds__(kThreads) cache_fork(ForkArgs a) {
    const reef_cache_fork_desc& d = a.d;
    const int64_t i = blockIdx.x;
    const int32_t bs = d.cache.block_size;
    const bool last = i + 1 >= d.forks && blockIdx.y == 0;    // counts for all
    __shared__ int32_t counts[kWaves];
    int32_t n = -1, parent = 0;
    if (i < d.forks) {
        n = fork_tokens(a, i);
        parent = a.parents[i];
    }
    const int32_t full = n < 0 ? 0 : n / bs, rest = n < 0 ? 0 : n % bs;
    if (!last && blockIdx.y && !rest) return;
    int32_t before = 0, bad = 0;
    if (rest || last) {
        for (int64_t j0 = 0; j0 < i; j0 += kThreads) {
            const int64_t j = j0 + threadIdx.x;
            const int32_t m = j < i ? fork_tokens(a, j) : 0;
            before += (int32_t)__popcll(__builtin_amdgcn_ballot_w64(m > 0 && m % bs != 0));
            bad += (int32_t)__popcll(__builtin_amdgcn_ballot_w64(m < 0));
        }
        int32_t sum;
        over_waves(before, counts, &sum);
        before = sum;
        over_waves(bad, counts, &sum);
        bad = sum;
    }
    if (last && threadIdx.x == 0) {
        const int32_t need = before + (rest != 0), refused = bad + (i < d.forks && n < 0);
        a.counts[0] = min(need, d.free_blocks);
        a.counts[1] = refused + max(0, need - d.free_blocks);
    }
    if (n < 0 || (rest && before >= d.free_blocks)) return;
    int32_t* const from_row = a.table + (int64_t)parent * d.table_stride;
    int32_t source = -1, target = -1;
    if (rest) {
        source = from_row[full];
        target = a.free_list[before];
        if ((uint32_t)source >= (uint32_t)d.cache.blocks || (uint32_t)target >= (uint32_t)d.cache.blocks) source = target = -1;
    }
    if (blockIdx.y == 0) {
        const int32_t child = a.children[i];
        int32_t* const to_row = a.table + (int64_t)child * d.table_stride;
        for (int32_t j = threadIdx.x; j < full; j += kThreads) to_row[j] = from_row[j];
        if (threadIdx.x == 0) {
            if (rest) to_row[full] = target;
            a.lengths[child] = n;
        }
        return;
    }
    if (target < 0) return;
    const int bytes = d.cache.type == REEF_TYPE_F32 ? 4 : 2, end = min(2 * d.layers, (int)blockIdx.y * a.each);
    const uint32_t total = (uint32_t)rest * a.pieces.heads * a.pieces.row;
    for (int part = ((int)blockIdx.y - 1) * a.each; part < end; ++part) {
        unsigned char* pool = (unsigned char*)(part & 1 ? a.value_cache : a.key_cache) + (int64_t)(part >> 1) * d.layer_stride * bytes;
        for (uint32_t k0 = 0; k0 < total; k0 += 4 * kThreads)
            copy_pieces(a.pieces, pool + source * d.cache.block_stride * bytes, pool + target * d.cache.block_stride * bytes, rest, k0);
    }
}

struct MoveArgs {
    reef_cache_compact_desc d;
    Use use;
    int32_t* table_out;
    void *key_cache, *value_cache;
    Pieces pieces;
    int32_t row_groups, row_turns;       // workgroups of the table: of four rows each, and how many go through a row
    int32_t chunks;                      // of 4 kThreads pieces a block
};

// The first workgroups write the table, the others copy: pieces of blocks in turn, of layers, of pools.  (468 MB moved: 189 us, 4.95 TB/s both ways.)
__global__ void __launch_bounds__(kThreads) move_blocks(MoveArgs a) {
    const reef_cache_compact_desc& d = a.d;
    const int32_t used = a.use.counts[0], moves = a.use.counts[1];
    const int32_t table_groups = a.row_groups * a.row_turns;
    if ((int32_t)blockIdx.x < table_groups) {
        const int lane = threadIdx.x & 63;
        const int32_t turn = (int32_t)blockIdx.x / a.row_groups;
        const int64_t row = (int64_t)(blockIdx.x - turn * a.row_groups) * kWaves + (threadIdx.x >> 6);
        if (row >= d.rows) return;
        const int32_t n = used_entries(a.use.t, row);
        for (int64_t j0 = (int64_t)turn * kRun; j0 < n; j0 += (int64_t)a.row_turns * kRun) {
            const int32_t end = (int32_t)min((int64_t)n, j0 + kRun);
            for (int32_t j = (int32_t)j0 + lane; j < end; j += 64) {
                int32_t b = a.use.t.entries[row * d.table_stride + j];
                if ((uint32_t)b < (uint32_t)d.cache.blocks && b >= used) b = a.use.target[a.use.uses[b]];
                a.table_out[row * d.out_stride + j] = b;
            }
        }
        return;
    }
    const int bytes = d.cache.type == REEF_TYPE_F32 ? 4 : 2;
    const int64_t caches = 2ll * d.layers, all = (int64_t)moves * caches * a.chunks;
    for (int64_t w = blockIdx.x - table_groups; w < all; w += gridDim.x - table_groups) {
        const int64_t u = w / a.chunks;
        const int32_t chunk = (int32_t)(w - u * a.chunks), part = (int32_t)(u % caches), k = (int32_t)(u / caches);
        unsigned char* pool = (unsigned char*)(part & 1 ? a.value_cache : a.key_cache) + (int64_t)(part >> 1) * d.layer_stride * bytes;
        copy_pieces(a.pieces, pool + a.use.source[k] * d.cache.block_stride * bytes, pool + a.use.target[k] * d.cache.block_stride * bytes,
                    (uint32_t)d.cache.block_size, (uint32_t)chunk * 4 * kThreads);
    }
}

int check_caches(const char* what, const reef_cache_layout& c, int32_t layers, int64_t layer_stride) {
    if (layers < 1 || layers > 30000) return refuse(what, "%d layers", layers);
    if (int rc = check_layout(what, c, layers, layer_stride)) return rc;
    if ((int64_t)c.block_size * c.kv_heads * c.head_dim >= 1 << 30) return refuse(what, "blocks of %d tokens are too large", c.block_size);
    return 0;
}

int check_sweep(const char* what, const reef_block_sweep_desc* d) {
    if (!d) return refuse(what, "null argument");
    return check_table(what, d->rows, d->blocks, d->block_size, d->max_blocks, d->table_stride);
}
Table table_of(const reef_block_sweep_desc& d, const int32_t* table, const int32_t* lengths) {
    return {d.rows, d.blocks, d.block_size, d.max_blocks, d.table_stride, table, lengths};
}
int64_t sweep_bytes(const reef_block_sweep_desc& d) { return near(table_of(d, nullptr, nullptr)) ? 0 : 4 * ((int64_t)segments_of(d.blocks) + 1); }

int check_compact(const char* what, const reef_cache_compact_desc* d) {
    if (!d) return refuse(what, "null argument");
    if (int rc = check_caches(what, d->cache, d->layers, d->layer_stride)) return rc;
    if (int rc = check_table(what, d->rows, d->cache.blocks, d->cache.block_size, d->max_blocks, d->table_stride)) return rc;
    if (d->out_stride < d->max_blocks) return refuse(what, "rows of the new table are %d apart, for %d entries", d->out_stride, d->max_blocks);
    return 0;
}
Table table_of(const reef_cache_compact_desc& d, const int32_t* table, const int32_t* lengths) {
    return {d.rows, d.cache.blocks, d.cache.block_size, d.max_blocks, d.table_stride, table, lengths};
}
// Places of moves, both ends; numbers of blocks, on 16 bytes; sums of segments.
int64_t most_moves(int32_t blocks) { return ((int64_t)blocks / 2 + 2) / 2 * 2; }
int64_t compact_bytes(const reef_cache_compact_desc& d) { return 4 * (2 * most_moves(d.cache.blocks) + d.cache.blocks + segments_of(d.cache.blocks) + 1); }

}  // namespace

extern "C" int64_t reef_ops_block_sweep_workspace(const reef_block_sweep_desc* d) {
    if (check_sweep("reef_ops_block_sweep_workspace", d)) return -1;
    return sweep_bytes(*d);
}

extern "C" int reef_ops_block_sweep(const reef_block_sweep_desc* d, const int32_t* table, const int32_t* lengths, int32_t* uses, int32_t* free_list,
                                    int32_t* counts, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "reef_ops_block_sweep";
    if (int rc = check_sweep(what, d)) return rc;
    if ((d->rows && (!words(table) || !words(lengths))) || !words(uses) || !words(free_list) || !words(counts)) return refuse(what, "null or unaligned argument");
    const int64_t need = sweep_bytes(*d);
    if (need && (!rows16(workspace) || workspace_bytes < need))
        return refuse(what, "a workspace of %lld bytes on 16 is needed, %lld are given", (long long)need, (long long)workspace_bytes);
    const Span out[] = {{uses, 4ll * d->blocks}, {free_list, 4ll * d->blocks}, {counts, 12}, {workspace, need}};
    const Span in[] = {{table, table_bytes(d->rows, d->max_blocks, d->table_stride)}, {lengths, 4ll * d->rows}};
    if (overlap(out, in)) return refuse(what, "an output overlaps an input");
    return place<true>(what, {table_of(*d, table, lengths), uses, (int32_t*)workspace, segments_of(d->blocks), free_list, counts, nullptr, nullptr}, stream);
}

extern "C" int reef_ops_cache_fork(const reef_cache_fork_desc* d, const int32_t* parents, const int32_t* children, const int32_t* tokens, const int32_t* free_list,
                                   int32_t* table, int32_t* lengths, int32_t* counts, void* key_cache, void* value_cache, void* stream) {
    const char* what = "reef_ops_cache_fork";
    if (!d) return refuse(what, "null argument");
    if (int rc = check_caches(what, d->cache, d->layers, d->layer_stride)) return rc;
    if (int rc = check_table(what, d->table_rows, d->cache.blocks, d->cache.block_size, d->max_blocks, d->table_stride)) return rc;
    if (d->forks < 0 || d->forks > d->table_rows || d->forks > kMostForks || d->free_blocks < 0) return refuse(what, "%d forks in a table of %d rows, %d free blocks", d->forks, d->table_rows, d->free_blocks);
    if (!words(counts) || (d->forks && (!words(parents) || !words(children) || !words(tokens) || !words(table) || !words(lengths) || !rows16(key_cache) || !rows16(value_cache))) ||
        (d->forks && d->free_blocks && !words(free_list)))
        return refuse(what, "null or unaligned argument");
    const int64_t n = d->forks;
    const Span out[] = {{table, n ? table_bytes(d->table_rows, d->max_blocks, d->table_stride) : 0}, {lengths, n ? 4ll * d->table_rows : 0}, {counts, 8}};
    const Span in[] = {{parents, 4 * n}, {children, 4 * n}, {tokens, 4 * n}, {free_list, n ? 4ll * d->free_blocks : 0}};
    if (overlap(out, in)) return refuse(what, "an output overlaps an input");
    // Many forks take several caches a workgroup, as each counts what is in front of it.
    const int each = d->forks <= 1024 ? 1 : 8;
    const ForkArgs a{*d, parents, children, tokens, free_list, table, lengths, counts, key_cache, value_cache, pieces_of(d->cache), each};
    return launch(what, cache_fork, dim3((unsigned)std::max(1, d->forks), n ? 1 + (2 * d->layers + each - 1) / each : 1), dim3(kThreads), a, stream);
}

extern "C" int64_t reef_ops_cache_compact_workspace(const reef_cache_compact_desc* d) {
    if (check_compact("reef_ops_cache_compact_workspace", d)) return -1;
    return compact_bytes(*d);
}

extern "C" int reef_ops_cache_compact(const reef_cache_compact_desc* d, const int32_t* table, const int32_t* lengths, int32_t* table_out, int32_t* counts,
                                      void* key_cache, void* value_cache, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "reef_ops_cache_compact";
    if (int rc = check_compact(what, d)) return rc;
    if ((d->rows && (!words(table) || !words(lengths) || !words(table_out) || !rows16(key_cache) || !rows16(value_cache))) || !words(counts))
        return refuse(what, "null or unaligned argument");
    const int64_t need = compact_bytes(*d);
    if (!rows16(workspace) || workspace_bytes < need)
        return refuse(what, "a workspace of %lld bytes on 16 is needed, %lld are given", (long long)need, (long long)workspace_bytes);
    const Span out[] = {{table_out, table_bytes(d->rows, d->max_blocks, d->out_stride)}, {counts, 8}, {workspace, need}};
    const Span in[] = {{table, table_bytes(d->rows, d->max_blocks, d->table_stride)}, {lengths, 4ll * d->rows}};
    if (overlap(out, in)) return refuse(what, "an output overlaps an input");
    const int64_t half = most_moves(d->cache.blocks);
    int32_t* const w = (int32_t*)workspace;
    const Use use{table_of(*d, table, lengths), w + 2 * half, w + 2 * half + d->cache.blocks, segments_of(d->cache.blocks), nullptr, counts, w, w + half};
    if (int rc = place<false>(what, use, stream)) return rc;
    if (!d->rows) return 0;
    const Pieces p = pieces_of(d->cache);
    const dim3 rows = rows_grid(use.t);
    const int64_t pieces = (int64_t)d->cache.block_size * p.heads * p.row, chunks = (pieces + 4 * kThreads - 1) / (4 * kThreads);
    const int64_t most = (int64_t)d->cache.blocks / 2 * 2 * d->layers * chunks;
    const MoveArgs a{*d, use, table_out, key_cache, value_cache, p, (int32_t)rows.x, (int32_t)rows.y, (int32_t)chunks};
    return launch(what, move_blocks, dim3((unsigned)(rows.x * rows.y + std::max<int64_t>(1, std::min<int64_t>(most, 4096)))), dim3(kThreads), a, stream);
}
