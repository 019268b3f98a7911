// Block tables and slot maps from the lengths of the requests (reef_ops_block_plan).
#include "ops_common.h"

namespace {
using namespace reef_ops;

constexpr int kThreads = 256;
constexpr int kMine = 4;                     // requests a thread and round
constexpr int kRound = kThreads * kMine;
constexpr int kWaves = kThreads / 64;

struct Args {
    reef_block_plan_desc d;
    const int32_t *cached, *added, *free_list;
    int32_t *table, *lengths, *starts, *slots, *counts;
};

// Exclusive prefix sums over the workgroup, and the sum of all in *total.
__device__ inline int64_t scan(int64_t v, int64_t* sums, int64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t s = v;
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t o = __shfl_up((long long)s, d);
        if (lane >= d) s += o;
    }
    __syncthreads();                         // (the sums of the scan before are read)
    if (lane == 63) sums[wave] = s;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += sums[w];
        all += sums[w];
    }
    *total = all;
    return before + s - v;
}

__device__ inline int32_t up(int64_t n, int32_t d) { return (int32_t)((n + d - 1) / d); }

// Two prefix sums over the requests (new tokens, new blocks) decide everything, and each place of the outputs is a function
// of them.  Sums are 64-bit: 2^31 requests of 2^31 tokens fit.
__global__ void __launch_bounds__(kThreads) block_plan(Args a) {
    const reef_block_plan_desc& d = a.d;
    const int32_t bs = d.block_size;
    __shared__ int64_t sums[kWaves];
    __shared__ int32_t ends[kRound], first[kRound], taken[kRound], have_[kRound];   // of the round's requests
    __shared__ int32_t used, refused;
    if (threadIdx.x == 0) used = refused = 0;
    int64_t tokens = 0, blocks = 0;          // of the rounds before
    for (int64_t base = 0; base < d.requests; base += kRound) {
        int32_t c[kMine];
        int64_t n[kMine], t_end[kMine], mine = 0, total;
        for (int k = 0; k < kMine; ++k) {
            const int64_t i = base + threadIdx.x * kMine + k;
            c[k] = i < d.requests ? max(a.cached[i], 0) : 0;
            n[k] = i < d.requests ? max(a.added[i], 0) : 0;
            mine += n[k];
        }
        int64_t at = tokens + scan(mine, sums, &total);
        const int64_t token0 = tokens;
        tokens += total;
        int32_t need[kMine];
        mine = 0;
        for (int k = 0; k < kMine; ++k) {
            at += n[k];
            t_end[k] = at;
            const bool fits = c[k] + n[k] <= (int64_t)d.max_blocks * bs && at <= d.max_tokens;
            need[k] = fits ? up(c[k] + n[k], bs) - up(c[k], bs) : -1;
            mine += max(need[k], 0);
        }
        int64_t b_at = blocks + scan(mine, sums, &total);
        blocks += total;
        for (int k = 0; k < kMine; ++k) {
            const int r = threadIdx.x * kMine + k;
            const int64_t i = base + r;
            b_at += max(need[k], 0);
            const bool granted = need[k] >= 0 && (need[k] == 0 || b_at <= d.free_blocks);
            ends[r] = (int32_t)min(t_end[k], (int64_t)d.max_tokens);
            // where the request's first token would lie if its cached ones were counted too; none: refused
            first[r] = granted ? c[k] : -1;
            have_[r] = up(c[k], bs);
            taken[r] = granted ? (int32_t)(b_at - need[k]) : 0;
            if (i < d.requests) {
                a.lengths[i] = granted ? (int32_t)(c[k] + n[k]) : c[k];
                a.starts[i] = (int32_t)min(t_end[k] - n[k], (int64_t)d.max_tokens);
                if (!granted) atomicAdd(&refused, 1);
                if (granted) {
                    atomicMax(&used, (int32_t)min(b_at, (int64_t)INT32_MAX));
                    for (int j = 0; j < need[k]; ++j) a.table[i * d.table_stride + have_[r] + j] = a.free_list[b_at - need[k] + j];
                }
            }
        }
        __syncthreads();
        // the slots of the round's tokens
        const int32_t lo = (int32_t)min(token0, (int64_t)d.max_tokens), hi = (int32_t)min(tokens, (int64_t)d.max_tokens);
        for (int64_t t = lo + threadIdx.x; t < hi; t += kThreads) {
            int r = 0;                       // the first request that ends behind t
            for (int step = kRound / 2; step; step >>= 1)
                if (ends[r + step - 1] <= t) r += step;
            int32_t slot = -1;
            if (first[r] >= 0) {
                const int32_t start = r ? ends[r - 1] : lo;
                const int32_t p = first[r] + (int32_t)(t - start), j = p / bs;
                const int32_t block = j >= have_[r] ? a.free_list[taken[r] + j - have_[r]] : a.table[(base + r) * d.table_stride + j];
                if ((uint32_t)block < (uint32_t)d.blocks) slot = block * bs + p % bs;
            }
            a.slots[t] = slot;
        }
        __syncthreads();
    }
    const int32_t end = (int32_t)min(tokens, (int64_t)d.max_tokens);
    for (int64_t t = end + threadIdx.x; t < d.max_tokens; t += kThreads) a.slots[t] = -1;
    __syncthreads();
    if (threadIdx.x == 0) {
        a.starts[d.requests] = end;
        a.counts[0] = used;
        a.counts[1] = end;
        a.counts[2] = refused;
    }
}

}  // namespace

extern "C" int reef_ops_block_plan(const reef_block_plan_desc* d, const int32_t* cached, const int32_t* added, const int32_t* free_list,
                                   int32_t* table, int32_t* lengths, int32_t* starts, int32_t* slots, int32_t* counts, void* stream) {
    const char* what = "reef_ops_block_plan";
    if (!d) return refuse(what, "null argument");
    if (d->requests < 0 || d->free_blocks < 0 || d->max_tokens < 0) return refuse(what, "negative size");
    if (d->blocks < 1 || d->block_size < 1 || (int64_t)d->blocks * d->block_size >= (1ll << 31))
        return refuse(what, "bad pool: %d blocks of %d tokens", d->blocks, d->block_size);
    if (d->max_blocks < 1 || d->table_stride < d->max_blocks || (int64_t)d->max_blocks * d->block_size >= (1ll << 31))
        return refuse(what, "bad table: rows of %d entries, %d apart, blocks of %d tokens", d->max_blocks, d->table_stride, d->block_size);
    if (d->requests && (!words(cached) || !words(added) || !words(table) || !words(lengths))) return refuse(what, "null or unaligned argument");
    if (!words(starts) || !words(counts) || (d->free_blocks && !words(free_list)) || (d->max_tokens && !words(slots)))
        return refuse(what, "null or unaligned argument");
    return launch(what, block_plan, dim3(1), dim3(kThreads), Args{*d, cached, added, free_list, table, lengths, starts, slots, counts}, stream);
}
