// Block tables and slot maps from the lengths of the requests (reef_ops_block_plan).
#include <algorithm>

#include "ops_common.h"

namespace {
using namespace reef_ops;

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kMostGroups = 512;

struct Args {
    reef_block_plan_desc d;
    const int32_t *cached, *added, *free_list;
    int32_t *table, *lengths, *starts, *slots, *counts;
};

// Sums saturate at 2^32 - 1, which is more than any size that they are compared with (saturating addition is associative).
__device__ inline uint32_t plus(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

// Exclusive prefix sums over the workgroup, and the sum of all in *total.
__device__ inline uint32_t scan(uint32_t v, uint32_t* sums, uint32_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = v;
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(s, d);
        if (lane >= d) s = plus(s, o);
    }
    uint32_t before = __shfl_up(s, 1);
    if (lane == 0) before = 0;
    __syncthreads();                         // (the sums of the scan before are read)
    if (lane == 63) sums[wave] = s;
    __syncthreads();
    uint32_t all = 0, waves = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) waves = plus(waves, sums[w]);
        all = plus(all, sums[w]);
    }
    *total = all;
    return plus(waves, before);
}

__device__ inline uint32_t up(uint32_t n, uint32_t d) { return n / d + (n % d != 0); }

// Two prefix sums over the requests (new tokens, new blocks) decide everything, and each place of the outputs is a function
// of them.  Every workgroup makes all sums for itself (a round takes 2 us, less than a launch for them alone) and writes its share of slots and table rows; none waits for another.  A slot's block comes from the free list itself where
// it is new, so the table is only read where no workgroup writes it.
// kMine: requests a thread and round.
template <int kMine>
__global__ void __launch_bounds__(kThreads) block_plan(Args a) {
    constexpr int kRound = kThreads * kMine;
    const reef_block_plan_desc& d = a.d;
    const uint32_t bs = d.block_size, room = (uint32_t)d.max_blocks * bs, max_tokens = d.max_tokens;
    __shared__ uint32_t sums[kWaves];
    __shared__ uint32_t ends[kRound], first[kRound], taken[kRound], have_[kRound], need_[kRound];   // of the round's requests
    constexpr uint32_t kRefused = 0xFFFFFFFFu;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const bool chief = blockIdx.x == 0;      // writes what is one word a request
    uint32_t used = 0, refused = 0;          // of this thread's requests
    uint32_t tokens = 0, blocks = 0;         // of the rounds before
    for (int64_t base = 0; base < d.requests; base += kRound) {
        uint32_t c[kMine], n[kMine], end[kMine], need[kMine], mine = 0, total;
        bool fits[kMine];
        for (int k = 0; k < kMine; ++k) {
            const int64_t i = base + threadIdx.x * kMine + k;
            c[k] = i < d.requests ? max(a.cached[i], 0) : 0;
            n[k] = i < d.requests ? max(a.added[i], 0) : 0;
            mine = plus(mine, n[k]);
        }
        uint32_t at = plus(tokens, scan(mine, sums, &total));
        const uint32_t lo = min(tokens, max_tokens);
        tokens = plus(tokens, total);
        mine = 0;
        for (int k = 0; k < kMine; ++k) {
            const uint32_t start = at;
            at = plus(at, n[k]);
            end[k] = min(at, max_tokens);
            fits[k] = c[k] + n[k] <= room && at <= max_tokens;
            need[k] = fits[k] ? up(c[k] + n[k], bs) - up(c[k], bs) : 0;
            mine = plus(mine, need[k]);
            const int64_t i = base + threadIdx.x * kMine + k;
            if (chief && i < d.requests) a.starts[i] = (int32_t)min(start, max_tokens);
        }
        uint32_t b_at = plus(blocks, scan(mine, sums, &total));
        blocks = plus(blocks, total);
        for (int k = 0; k < kMine; ++k) {
            const int r = threadIdx.x * kMine + k;
            const int64_t i = base + r;
            b_at = plus(b_at, need[k]);
            const bool granted = fits[k] && (need[k] == 0 || b_at <= (uint32_t)d.free_blocks);
            ends[r] = end[k];
            first[r] = granted ? c[k] : kRefused;
            have_[r] = up(c[k], bs);
            taken[r] = b_at - need[k];
            need_[r] = granted ? need[k] : 0;
            if (chief && i < d.requests) {
                a.lengths[i] = (int32_t)(granted ? c[k] + n[k] : c[k]);
                if (granted) used = b_at;    // (the sums only grow)
                else ++refused;
            }
        }
        __syncthreads();
        const int count = (int)min((int64_t)kRound, d.requests - base);
        for (int r = blockIdx.x * kWaves + wave; r < count; r += gridDim.x * kWaves) {
            int32_t* to = a.table + (base + r) * d.table_stride + have_[r];
            for (uint32_t j = lane; j < need_[r]; j += 64) to[j] = a.free_list[taken[r] + j];
        }
        // The slots of the round's tokens.  Where requests bring four and more, four in a row a thread: one search, and their blocks are
        // mostly one (2000 prompts, 0.8 M tokens: 13 against 33 us, four requests a thread and 256 threads).  In decode steps each has a block of its own, and four loads in a row
        // would wait for each other (four requests: 7.0 against 4.9 us).
        const uint32_t hi = min(tokens, max_tokens), per = (hi - lo) / 4 >= (uint32_t)count ? 4 : 1;
        for (uint64_t t0 = lo / per * per + (uint64_t)per * (blockIdx.x * kThreads + threadIdx.x); t0 < hi; t0 += (uint64_t)per * gridDim.x * kThreads) {
            int r = -1;
            uint32_t page = 0, slot_of = 0;
            bool known = false;
            for (uint32_t k = 0; k < per; ++k) {
                const uint32_t t = (uint32_t)t0 + k;
                if (t < lo || t >= hi) continue;
                if (r < 0 || ends[r] <= t) {
                    r = 0;                   // the first request that ends behind t
                    for (int step = kRound / 2; step; step >>= 1)
                        if (ends[r + step - 1] <= t) r += step;
                    known = false;
                }
                int32_t slot = -1;
                if (first[r] != kRefused) {
                    const uint32_t p = first[r] + t - (r ? ends[r - 1] : lo), j = p / bs;
                    if (!known || j != page) {
                        page = j;
                        known = true;
                        slot_of = (uint32_t)(j >= have_[r] ? a.free_list[taken[r] + j - have_[r]] : a.table[(base + r) * d.table_stride + j]);
                    }
                    if (slot_of < (uint32_t)d.blocks) slot = (int32_t)(slot_of * bs + p % bs);
                }
                a.slots[t] = slot;
            }
        }
        __syncthreads();
    }
    const uint32_t end = min(tokens, max_tokens);
    for (uint64_t t = (uint64_t)end + blockIdx.x * kThreads + threadIdx.x; t < max_tokens; t += (uint64_t)gridDim.x * kThreads) a.slots[t] = -1;
    if (!chief) return;
    for (int x = 32; x; x >>= 1) {
        used = max(used, __shfl_xor(used, x));
        refused += __shfl_xor(refused, x);
    }
    if (lane == 0) {
        ends[wave] = used;
        first[wave] = refused;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWaves; ++w) {
            used = max(used, ends[w]);
            refused += first[w];
        }
        a.starts[d.requests] = (int32_t)end;
        a.counts[0] = (int32_t)min(used, (uint32_t)INT32_MAX);
        a.counts[1] = (int32_t)end;
        a.counts[2] = (int32_t)refused;
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
    const int64_t n = d->requests;
    const Span out[] = {{table, n ? 4 * ((n - 1) * d->table_stride + d->max_blocks) : 0}, {lengths, 4 * n}, {starts, 4 * (n + 1)}, {slots, 4ll * d->max_tokens}, {counts, 12}};
    const Span in[] = {{cached, 4 * n}, {added, 4 * n}, {free_list, 4ll * d->free_blocks}};
    if (overlap(out, in)) return refuse(what, "an output overlaps an input");
    // a workgroup for about 1024 slots or 16 table rows
    const int64_t want = std::max((d->max_tokens + 1023ll) / 1024, (std::min(d->requests, 1024) + 15ll) / 16);
    const dim3 grid((unsigned)std::min<int64_t>(std::max<int64_t>(want, 1), kMostGroups));
    const Args a{*d, cached, added, free_list, table, lengths, starts, slots, counts};
    // Up to 1024 requests go through in one round of two a thread, more in rounds of four: 2000 prompts 10.5 against 12.8 us, 4000
    // decode steps 10.5 against 13.8, but four requests 5.3 against 4.6.
    if (d->requests <= 2 * kThreads) return launch(what, block_plan<2>, grid, dim3(kThreads), a, stream);
    return launch(what, block_plan<4>, grid, dim3(kThreads), a, stream);
}
