// Attention of the new tokens of all requests over a paged key-value cache (reef_ops_chunk_attention).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ops_common.h"

namespace {
using namespace reef_ops;

constexpr int kRows = 32;                    // query rows of a wavefront: heads of one token next to each other, token after token
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int32_t kLeast = 256, kLeastFew = 512;   // cached tokens a share at least, of tiles of 32 rows for each wavefront and of 32 in all
constexpr int32_t kLooked = 640, kLookedFew = 2048;  // up to so many tokens no cutting is looked at; where a pair takes more than one product, two thirds
// (four pieces of 100 over 500, 12 heads of 64, f32: 47 us whole, 31 cut; over 300, 16 heads over 4 of 128: 70 whole, 79 cut; bf16, eight pieces of 60 over 400,
// 32 heads over 8 of 128: 27 whole, 33 cut)
constexpr float kJoin = 420.0f;              // tokens whose time it takes to write and read a share's sums, over the products per token
constexpr int kCus = 256;
constexpr float kSlack = 8.0f;               // powers of two by which weights may pass their reference

struct Args {
    reef_chunk_attention_desc d;
    const void *query, *key_cache, *value_cache;
    const int32_t *table, *starts, *cached, *lengths;
    void* out;
    float* lse;
    int2* info;             // [request], where there are many: first item, first slot
    int32_t* list;          // numbers of all (kListHead), then the request of each item
    float* parts;           // [slot (a share of a tile that is cut)][cache head][row of the tile][head_dim], sums that are not divided yet
    float2* stats;          // [slot][cache head][row of the tile]: power of two that they are to be multiplied by, sum of the weights
    float scale;            // |scale| log2 e, or log2 e where it is 0
    uint32_t flip;          // of the queries' sign where scale is negative
    int32_t zero;           // scale is 0
    int32_t group;
    int32_t tile_rows;      // of a workgroup
    int32_t at_once;        // workgroups that run at once
    int32_t looked;         // tokens up to which no cutting is looked at
    float join;             // tokens whose time a share's sums take
    int32_t budget;         // workgroups that tiles are cut for, beside one each; 0: they are not cut
    int32_t most_items, most_slots;
    int32_t* used;          // slots that there are; behind it (int4 aligned) what each belongs to
    int4* jobs;             // [slot]: request, tile, share, shares
    Divider block, by_group;
};

// A request: the rows of its new tokens, and how they are worked on.
struct Request {
    int32_t first, added, cached, n;         // first row, rows; tokens in front of them and in all
    int32_t tiles;
};
// An item: a tile of rows over a share of the tokens that they see.
struct Item {
    Request r;
    int32_t request, tile, share, shares, slot;   // tile < 0: there is no such item; slot of the tile's first share where there are several
    int32_t slots;                           // of all
};

__device__ inline int32_t start_of(const Args& a, int32_t i) { return max(0, min(a.starts[i], a.d.tokens)); }
__device__ inline Request request_of(const Args& a, int32_t i) {
    Request r;
    r.first = start_of(a, i);
    r.added = max(0, start_of(a, i + 1) - r.first);
    r.cached = held_length(a.cached[i], a.d.max_blocks, a.d.cache.block_size);
    r.n = held_length(a.lengths[i], a.d.max_blocks, a.d.cache.block_size);
    r.tiles = (r.added * a.group + a.tile_rows - 1) / a.tile_rows;
    return r;
}
// The cached tokens [.x, .y) that some row of a tile sees.  (Places may pass 2^31, not 2^32.)
__device__ inline uint2 span_of(const Args& a, const Request& r, int32_t tile) {
    const uint32_t last = (uint32_t)min((tile + 1) * a.tile_rows, r.added * a.group) - 1;
    const uint32_t p0 = (uint32_t)r.cached + divided((uint32_t)(tile * a.tile_rows), a.by_group), p1 = (uint32_t)r.cached + divided(last, a.by_group);
    if (p0 >= (uint32_t)r.n) return make_uint2(0, 0);
    return make_uint2(a.d.window && p0 + 1 > (uint32_t)a.d.window ? p0 + 1 - a.d.window : 0, min((uint32_t)r.n, p1 + 1));
}
// A request's tiles in four parts, as those of a prompt see more and more: what the tiles of each see at most, and all of them together
// (spans grow with the tile, by steps that do not).  No products are contracted here and below: what a launch lists the next one has to find again.
constexpr int kParts = 4;
struct Sizes {
    float most[kParts], top, all;
};
__device__ inline int32_t part_of(const Request& r, int q) { return r.tiles * q / kParts; }
__device__ inline Sizes size_up(const Args& a, const Request& r) {
#pragma clang fp contract(off)
    Sizes s{};
    if (!r.tiles) return s;
    const uint2 x = span_of(a, r, 0);
    float before = (float)(x.y - x.x);
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
        const int32_t from = part_of(r, q), to = part_of(r, q + 1);
        if (from == to) continue;
        const uint2 y = span_of(a, r, to - 1);
        const float v = (float)(y.y - y.x);
        s.most[q] = fmaxf(before, v);
        s.top = fmaxf(s.top, s.most[q]);
        s.all += (float)(to - from) * (before + v) * 0.5f;
        before = v;
    }
    return s;
}
// How long shares are.  Let w be the tokens of all tiles over the workgroups that run at once, and c the tokens whose time it takes to write and
// read a share's sums.  Shares of T tokens take about w (1 + c / T), and 0.7 T until the last are done, least at T = (1.4 w c)^(1/2); a request whose
// longest tile is done sooner is not cut, nor are its tiles of up to 1.3 T.  (One prompt of 2000 tokens, 32 heads over 8 of 128, bf16: 76 us, cut all the
// same 90; of 2348, 10 heads over 5 of 64, f32: cut 99 us, else 160.)  T is half of w at least (two prompts of 2048, 16 heads over 4 of 128, f32: 290 us, 335
// without that; the one of 2348 would take 91).
// Where there are fewer workgroups than the budget, and tiles of a request are much alike (not as a prompt's, of which long ones and short ones make up for
// each other), they are cut into the number n that takes the least rounds, ceil(n N / at once) (1 / n + c / tokens).
// Where all that makes more items than there are workgroups for, or shares than there are slots, shares are made longer, up to four times; then (lengths that were not expected) none is cut.
struct Cut {
    float whole, tokens, alike;              // tiles of up to `whole` tokens are not cut, others into shares of `tokens`; alike: of tiles much alike; 0: as others
};
__host__ __device__ inline Cut cut_for(float w, float join, bool few) {
    Cut c;
    if (few) {
        c.tokens = 1.02f * w;
        c.whole = kLookedFew + 1.3f * w;
    } else {
        c.tokens = fmaxf((float)kLeast, fmaxf(0.51f * w, sqrtf(1.4f * w * join)));
        c.whole = w + w * join / c.tokens;
    }
    c.alike = 0.0f;
    return c;
}
__device__ inline Cut cut_of(const Args& a, float all, float tiles) {
    const float at_once = (float)a.at_once, groups = tiles * (float)a.d.cache.kv_heads;
    Cut c = cut_for(all * (float)a.d.cache.kv_heads / at_once, a.join, a.tile_rows == kRows);
    if (groups < (float)a.budget) {
        const float join = a.join * tiles / all;
        float best = ceilf(groups / at_once), n = 1.0f;
        for (float k = 2.0f; k * groups <= (float)a.budget && k <= 64.0f; k += 1.0f) {
            const float rounds = ceilf(k * groups / at_once) * (__builtin_amdgcn_rcpf(k) + join);
            if (rounds < 0.95f * best) {
                best = rounds;
                n = k;
            }
        }
        if (n > 1.0f) c.alike = all * 1.02f / (tiles * n);
    }
    return c;
}
// Into how many shares the tiles of each part are cut.
struct Shares {
    int32_t n[kParts];
    bool first;             // shares that are longer than half a round come first, so that none of them begins when the others are nearly done
};
__device__ inline Shares shares_of(const Args& a, const Cut& c, const Sizes& s, int32_t tiles) {
#pragma clang fp contract(off)
    const bool few = a.tile_rows == kRows, alike = c.alike > 0.0f && s.top * (float)tiles < 1.5f * s.all;
    const float least = (float)(few ? kLeastFew : kLeast), looked = (float)a.looked;
    const float each = fmaxf(least, alike ? c.alike : c.tokens), whole = fmaxf(1.5f * least, 1.3f * (alike ? c.alike : c.tokens));
    const bool cut = s.top > fmaxf(looked, alike ? c.alike : c.whole);
    Shares x;
    x.first = false;
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
        x.n[q] = !cut || s.most[q] <= whole ? 1 : (int32_t)ceilf(s.most[q] / each);
        x.first |= s.most[q] > 0.5f * c.tokens * (float)x.n[q];
    }
    return x;
}
__device__ inline Shares not_cut() {
    Shares x;
#pragma unroll
    for (int q = 0; q < kParts; ++q) x.n[q] = 1;
    x.first = true;
    return x;
}
__device__ inline void cut_less(Cut& c) {
    c.whole *= 1.5f;
    c.tokens *= 1.5f;
    c.alike *= 1.5f;
}
constexpr int kTries = 5;

// Items and slots are counted up to 2^32 - 1: more there are only where starts do not ascend, and then nothing may run over.
__device__ inline uint32_t plus(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
__device__ inline uint32_t product(int32_t tiles, int32_t shares) { return (uint32_t)min((uint64_t)(uint32_t)tiles * (uint32_t)shares, (uint64_t)UINT32_MAX); }
__device__ inline uint32_t items_of(const Request& r, const Shares& x) {
    uint32_t n = 0;
#pragma unroll
    for (int q = 0; q < kParts; ++q) n = plus(n, product(part_of(r, q + 1) - part_of(r, q), x.n[q]));
    return n;
}
// Those of tiles that are cut, which have a slot each.
__device__ inline uint32_t slots_of(const Request& r, const Shares& x) {
    uint32_t n = 0;
#pragma unroll
    for (int q = 0; q < kParts; ++q) n = plus(n, x.n[q] > 1 ? product(part_of(r, q + 1) - part_of(r, q), x.n[q]) : 0);
    return n;
}
// Prefix sums over the wavefront without the lane's own value; *all: with all of them.
template <int CONTROL, int ROWS>
__device__ inline uint32_t moved(uint32_t x) { return __builtin_amdgcn_update_dpp(0, x, CONTROL, ROWS, 0xF, true); }
__device__ inline uint32_t before_me(uint32_t v, uint32_t* all) {
    constexpr int kUp = 0x110, kLast15 = 0x142, kLast31 = 0x143;     // rows of 16 by lanes; the last lane of a row, of a half, to the next
    const uint32_t mine = v;
    v = plus(v, moved<kUp | 1, 0xF>(v));
    v = plus(v, moved<kUp | 2, 0xF>(v));
    v = plus(v, moved<kUp | 4, 0xF>(v));
    v = plus(v, moved<kUp | 8, 0xF>(v));
    v = plus(v, moved<kLast15, 0xA>(v));
    v = plus(v, moved<kLast31, 0xC>(v));
    *all = __builtin_amdgcn_readlane(v, 63);
    return v == UINT32_MAX ? v : v - mine;
}
__device__ inline float sum_of(float v) {
    for (int x = 32; x; x >>= 1) v += __shfl_xor(v, x);
    return v;
}

// Up to kFewRequests requests each wavefront finds its item by itself, a request a lane; more are listed by a launch ahead.
constexpr int32_t kFewRequests = 64, kListHead = 6;           // (items, slots, the cut, whether there is one)
__device__ inline Item find_item(const Args& a, int32_t id) {
    Item it;
    it.tile = -1;
    int32_t local;
    Shares shares = not_cut();
    if (a.list) {
        if (id >= a.list[0]) return it;
        it.request = a.list[kListHead + id];
        const int2 info = a.info[it.request];
        it.r = request_of(a, it.request);
        local = id - info.x;
        if (a.list[5]) shares = shares_of(a, {__int_as_float(a.list[2]), __int_as_float(a.list[3]), __int_as_float(a.list[4])}, size_up(a, it.r), it.r.tiles);
        it.slot = info.y;
        it.slots = a.list[1];
    } else if (a.d.requests == 1) {
        it.request = 0;
        it.r = request_of(a, 0);
        uint32_t items = (uint32_t)it.r.tiles, slots = 0;
        if (a.budget) {
            const Sizes sizes = size_up(a, it.r);
            Cut cut = cut_of(a, sizes.all, (float)it.r.tiles);
            for (int tries = 1;; ++tries) {
                shares = shares_of(a, cut, sizes, it.r.tiles);
                items = items_of(it.r, shares);
                slots = slots_of(it.r, shares);
                if (items <= (uint32_t)a.most_items && slots <= (uint32_t)a.most_slots) break;
                if (tries == kTries) {
                    shares = not_cut();
                    items = (uint32_t)it.r.tiles;
                    slots = 0;
                    break;
                }
                cut_less(cut);
            }
        }
        if ((uint32_t)id >= items) return it;
        it.slot = 0;
        it.slots = (int32_t)slots;
        local = id;
    } else {
        const int lane = threadIdx.x & 63;
        Request r{};
        if (lane < a.d.requests) r = request_of(a, lane);
        uint32_t firsts, others = 0, all_slots = 0, slot = 0, mine = (uint32_t)r.tiles, at;
        if (a.budget) {
            const Sizes sizes = size_up(a, r);
            Cut cut = cut_of(a, sum_of(sizes.all), sum_of((float)r.tiles));
            for (int tries = 1;; ++tries) {
                shares = shares_of(a, cut, sizes, r.tiles);
                mine = items_of(r, shares);
                at = before_me(shares.first ? mine : 0, &firsts);
                const uint32_t x = before_me(shares.first ? 0 : mine, &others);
                at = shares.first ? at : plus(firsts, x);
                slot = before_me(slots_of(r, shares), &all_slots);
                if (plus(firsts, others) <= (uint32_t)a.most_items && all_slots <= (uint32_t)a.most_slots) break;
                if (tries == kTries) {
                    shares = not_cut();
                    mine = (uint32_t)r.tiles;
                    at = before_me(mine, &firsts);
                    all_slots = 0;
                    break;
                }
                cut_less(cut);
            }
        } else {
            at = before_me(mine, &firsts);
        }
        const uint64_t who = __builtin_amdgcn_ballot_w64((uint32_t)id >= at && (uint32_t)id - at < mine);
        if (!who) return it;
        const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(who));
        it.request = l;
        it.r.first = __builtin_amdgcn_readlane(r.first, l);
        it.r.added = __builtin_amdgcn_readlane(r.added, l);
        it.r.cached = __builtin_amdgcn_readlane(r.cached, l);
        it.r.n = __builtin_amdgcn_readlane(r.n, l);
        it.r.tiles = __builtin_amdgcn_readlane(r.tiles, l);
#pragma unroll
        for (int q = 0; q < kParts; ++q) shares.n[q] = __builtin_amdgcn_readlane(shares.n[q], l);
        it.slot = __builtin_amdgcn_readlane((int32_t)slot, l);
        it.slots = (int32_t)all_slots;
        local = id - (int32_t)__builtin_amdgcn_readlane(at, l);
    }
    // the last tiles, which see most, first
    int32_t before = 0, from = 0, to = 0, slots_before = 0, slots_from = 0;
    it.shares = 1;
#pragma unroll
    for (int q = kParts - 1; q >= 0; --q) {
        const int32_t f = part_of(it.r, q), t = part_of(it.r, q + 1), n = (t - f) * shares.n[q];
        if (local >= before && local - before < n) {
            from = before;
            to = t;
            it.shares = shares.n[q];
            slots_from = slots_before;
        }
        before += n;
        if (shares.n[q] > 1) slots_before += n;
    }
    const int32_t k = (local - from) / it.shares;
    it.share = local - from - k * it.shares;
    it.tile = to - 1 - k;
    it.slot = __builtin_amdgcn_readfirstlane(it.slot + slots_from + k * it.shares);
    it.shares = __builtin_amdgcn_readfirstlane(it.shares);
    it.share = __builtin_amdgcn_readfirstlane(it.share);
    it.tile = __builtin_amdgcn_readfirstlane(it.tile);
    return it;
}

constexpr int kListThreads = 1024;
__global__ void __launch_bounds__(kListThreads) list_items(Args a) {
    constexpr int kListWaves = kListThreads / 64;
    __shared__ float2 sums[kListWaves];
    __shared__ uint3 counts[kListWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t R = a.d.requests, per = (R + kListThreads - 1) / kListThreads, lo = min(R, tid * per), hi = min(R, lo + per);
    Cut cut{};
    if (a.budget) {
        float sum = 0.0f, tiles = 0.0f;
        for (int32_t i = lo; i < hi; ++i) {
            const Request r = request_of(a, i);
            sum += size_up(a, r).all;
            tiles += (float)r.tiles;
        }
        sum = sum_of(sum);
        tiles = sum_of(tiles);
        if (lane == 0) sums[wave] = make_float2(sum, tiles);
        __syncthreads();
        sum = tiles = 0.0f;
        for (int w = 0; w < kListWaves; ++w) {
            sum += sums[w].x;
            tiles += sums[w].y;
        }
        cut = cut_of(a, sum, tiles);
    }
    bool is_cut = a.budget != 0;
    auto shares_and_items = [&](int32_t i, uint32_t* mine, uint32_t* slots) {
        const Request r = request_of(a, i);
        const Shares x = is_cut ? shares_of(a, cut, size_up(a, r), r.tiles) : not_cut();
        *mine = items_of(r, x);
        *slots = slots_of(r, x);
        return x;
    };
    uint32_t all, all_slots, item, later, slot;            // later: where the next request that does not come first has its items
    for (int tries = 1;; ++tries) {
        uint32_t items = 0, others = 0, slots = 0, of_wave, others_of_wave, slots_of_wave, mine, its_slots;
        for (int32_t i = lo; i < hi; ++i) {
            const Shares x = shares_and_items(i, &mine, &its_slots);
            if (x.first) items = plus(items, mine);
            else others = plus(others, mine);
            slots = plus(slots, its_slots);
        }
        item = before_me(items, &of_wave);
        later = before_me(others, &others_of_wave);
        slot = before_me(slots, &slots_of_wave);
        __syncthreads();
        if (lane == 0) counts[wave] = make_uint3(of_wave, others_of_wave, slots_of_wave);
        __syncthreads();
        uint32_t firsts = 0;
        all = all_slots = 0;
        for (int w = 0; w < kListWaves; ++w) {
            if (w < wave) {
                item = plus(item, counts[w].x);
                later = plus(later, counts[w].y);
                slot = plus(slot, counts[w].z);
            }
            firsts = plus(firsts, counts[w].x);
            all = plus(all, plus(counts[w].x, counts[w].y));
            all_slots = plus(all_slots, counts[w].z);
        }
        later = plus(later, firsts);
        if (!is_cut || (all <= (uint32_t)a.most_items && all_slots <= (uint32_t)a.most_slots)) break;
        if (tries == kTries) is_cut = false;
        else cut_less(cut);
    }
    for (int32_t i = lo; i < hi; ++i) {
        uint32_t mine, its_slots;
        const Shares x = shares_and_items(i, &mine, &its_slots);
        uint32_t& at = x.first ? item : later;
        a.info[i] = make_int2((int32_t)min(at, 1u << 30), (int32_t)slot);
        for (uint32_t k = at; k < min(plus(at, mine), (uint32_t)a.most_items); ++k) a.list[kListHead + k] = i;
        at = plus(at, mine);
        slot += its_slots;
    }
    if (tid == 0) {
        a.list[0] = (int32_t)min(all, (uint32_t)a.most_items);
        a.list[1] = (int32_t)all_slots;
        a.list[2] = __float_as_int(cut.whole);
        a.list[3] = __float_as_int(cut.tokens);
        a.list[4] = __float_as_int(cut.alike);
        a.list[5] = is_cut;
    }
}

typedef float f32x16 __attribute__((ext_vector_type(16)));
__device__ inline f32x16 product(u32x4 a, u32x4 b, f32x16 c, _Float16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ inline f32x16 product(u32x4 a, u32x4 b, f32x16 c, __bf16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Two values as N terms of a 16-bit type, whose sums they are but for what the last rounds off.  The first of several is cut, so that it is
// finite where the value is.
template <int N>
__device__ inline void terms(float a, float b, uint32_t (&t)[N], __bf16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    if constexpr (N > 1) {
        t[0] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
        a -= __uint_as_float(__float_as_uint(a) & 0xFFFF0000u);
        b -= __uint_as_float(__float_as_uint(b) & 0xFFFF0000u);
    }
    if constexpr (N == 3) {
        const bf16x2 x = {(__bf16)a, (__bf16)b};
        t[1] = __builtin_bit_cast(uint32_t, x);
        a -= __uint_as_float(t[1] << 16);
        b -= __uint_as_float(t[1] & 0xFFFF0000u);
    }
    const bf16x2 last = {(__bf16)a, (__bf16)b};
    t[N - 1] = __builtin_bit_cast(uint32_t, last);
}
template <int N>
__device__ inline void terms(float a, float b, uint32_t (&t)[N], _Float16) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const f16x2 x = {(_Float16)a, (_Float16)b};
        t[i] = __builtin_bit_cast(uint32_t, x);
        a -= (float)x[0];
        b -= (float)x[1];
    }
}

// Which bits of a word hold finite values.
__device__ inline uint32_t keep_of(uint32_t w, float) { return (w & 0x7F800000u) == 0x7F800000u ? 0 : ~0u; }
__device__ inline uint32_t keep_of(uint32_t w, __bf16) { return ((w & 0x7F80u) == 0x7F80u ? 0 : 0xFFFFu) | ((w & 0x7F800000u) == 0x7F800000u ? 0 : 0xFFFF0000u); }
__device__ inline uint32_t keep_of(uint32_t w, _Float16) { return ((w & 0x7C00u) == 0x7C00u ? 0 : 0xFFFFu) | ((w & 0x7C000000u) == 0x7C000000u ? 0 : 0xFFFF0000u); }

// A value of both halves of the wavefront, joined: lanes l and l + 32 have the same row.
__device__ inline float other_max(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ inline float other_sum(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
// A value that is to be made where it is used, not ahead of a loop and held in registers, of which there are none left.
__device__ inline uint32_t again(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

template <class Q>
__device__ inline void put4(Q* to, float a, float b, float c, float d) {
    typedef Q Q4 __attribute__((ext_vector_type(4)));
    const Q4 x = {(Q)a, (Q)b, (Q)c, (Q)d};
    *(Q4*)to = x;
}

// How heads of up to DP values lie in LDS: rows of kPitch bytes, their 16-byte pieces exchanged by the row's number, so that neither 16 rows' same
// piece nor four rows' same 64 bytes meet in a bank.
template <int DP>
struct Near {
    static constexpr int kPieces = DP <= 64 ? 8 : DP <= 128 ? 16 : 32, kPitch = kPieces * 16;
    static __device__ inline uint32_t turn(uint32_t row) {
        return kPieces == 8 ? (row >> 1 & 1) << 2 | (row >> 2 & 3) : (row & 3) << 2 | (row >> 2 & 3);
    }
    static __device__ inline uint32_t at(uint32_t row, uint32_t piece) { return row * kPitch + ((piece ^ turn(row)) << 4); }
};

// How a kernel is laid out, by its types and head size.  kTile: tokens of a tile of keys and values; kWaves of 32 rows each share them.
template <class Q, class C, int DP>
struct Shape {
    static constexpr bool kHalf = __is_same(C, _Float16);
    static constexpr int kTermsC = sizeof(C) == 4 ? 3 : 1, kTermsQ = sizeof(Q) == 2 ? 1 : kHalf ? 2 : 3;
    static constexpr int kTermsFew = sizeof(Q) == 2 ? 2 : kTermsQ;           // of weights in tiles of 32 rows in all; in others kTermsQ
    static constexpr bool kPair = DP <= 64;
    static constexpr int kWaves = DP <= 128 && !kPair ? 8 : 4, kTile = kTermsQ == 1 && DP <= 128 ? 64 : 32;
    // Tiles of 32 rows in all: registers of what a wavefront holds (keys, values, queries, output, weights), and so how many wavefronts; 0: too many for any.
    static constexpr int kFewV = DP <= 64 ? 2 : DP <= 128 ? 4 : 8;            // values of a row of V a lane
    static constexpr int kFewHeld = DP * (int)sizeof(C) / 8 + 16 * kFewV * (int)sizeof(C) / 4 + kTermsQ * DP / 4 + kFewV * 16 + 16 + 8 * kTermsFew;
    // (Four wavefronts of heads of 192 and 256 hold 30 to 120 registers more than there are, in scratch, and are faster than the other tiles all the same: 64 single tokens over
    // 4000, 32 heads over 8, bf16 292 us against 399 for 192 and 401 against 466 for 256, 32-bit queries over bf16 647 against 677; but 725 against 677 over fp16 for 256.)
    static constexpr int kFewWaves = kFewHeld <= 220 ? 8 : kFewHeld <= 440 ? 4 : 0;
};

// A tile of query rows over a share of the tokens they see, one cache head: each wavefront has 32 rows, all of them the keys and values that
// the workgroup brings to LDS.
//
// Both products are 32x32x16 MFMAs:  S^T[token][row] = K Q^T, then O^T[dim][row] = V^T P^T.  A product does not care in which order its k
// runs: S^T leaves lane (row, half h) the tokens 8 j + 4 h + {0..3} of 32, so these are its k, and V^T's operand comes transposed out of LDS four tokens a
// read.  So weights stay in the lane that made them, and a row's reference, sum and rescaling are one value a lane.
//
// Scores are made a tile ahead: the products of the next tile's keys run beside the exponentials of this one's scores, and those of this
// one's values beside the next one's maximum, so that the matrix cores have work while the lanes have theirs.
//
// Weights are 2^(s c - R): R is a whole number near the largest s c so far (within kSlack above), so that one rounding makes the exponent, and rescaling
// by 2^(R - R') is exact and rare.  For fp16, whose weights want room below, they are 2^kGrow times larger.
//
// 32-bit queries over 16-bit caches are two terms of fp16 or three of bf16 each, and so are their weights; 32-bit caches are three terms of bf16 on
// both sides, six products (the others are below 2^-22).  Weights of 16-bit types are two terms in tiles of 32 rows in all, which memory or latency
// bounds (64 single tokens over 4000, 32 heads over 8 of 128, bf16: 199 us with one term, 204 with two).  In larger tiles they are rounded to the type once, half a
// step of each at most, and their sum is of those that are not rounded: the output is off by no more than the mean |value| times that half step, as much as its
// own rounding where it is of values' size.  Products bound these, and a second term would double those with the values: 600 -> 771 us for the prompt
// below, 2225 -> 2948 for the three pieces, 164 -> 205 for two prompts of 2797 (heads of 80, fp16).
//
// One prompt of 8191 tokens, 32 heads over 8 of 128, bf16: 616 us, 0.89 PFLOP/s; three pieces of 509 over 40000, 64 heads over 8, fp16: 2.30 ms, 0.88.  When
// the former took 646 us, it took 588 without loads, 541 without stores to LDS too, 503 without exponentials too, and 463 with its products alone
// (1.19 PFLOP/s, what a large matrix product reaches here).  Heads of up to 64 leave room for two workgroups of four wavefronts a CU, which do not wait
// for each other (four prompts of 2048, 12 heads of 64, bf16: 89 -> 79 us; two pieces of 300 over 20000: 91 -> 99); for heads of 80 and 128 eight wavefronts
// that share what they read are faster (98 against 104 us, 616 against 688).
template <class Q, class C, int DP, bool FEW>
__global__ void __launch_bounds__((FEW ? Shape<Q, C, DP>::kFewWaves : Shape<Q, C, DP>::kWaves) * 64, (!FEW && Shape<Q, C, DP>::kPair ? 2 : 1)) chunk_attention(Args a) {
    using E = std::conditional_t<sizeof(C) == 4, __bf16, C>;                  // what is multiplied
    using Sh = Shape<Q, C, DP>;
    constexpr bool kHalf = Sh::kHalf;
    constexpr int kTermsC = Sh::kTermsC, kTermsQ = Sh::kTermsQ, kTermsP = FEW ? Sh::kTermsFew : kTermsQ;
    constexpr int kTile = Sh::kTile, kSub = kTile / 32, kWaves = FEW ? Sh::kFewWaves : Sh::kWaves, kThreads = kWaves * 64;
    constexpr float kGrow = kHalf ? 6.0f : 0.0f;                              // 2^(6 + 8 + 1/2) < 65504
    constexpr int kSteps = DP / 16, kSlabs = DP / 32, kTileRows = FEW ? kRows : kWaves * kRows;
    using N = Near<DP>;
    constexpr int kPlane = kTile * N::kPitch, kBuffer = kTermsC * kPlane;
    constexpr int kRowPieces = DP * (int)sizeof(C) / 16, kAllPieces = kTile * kRowPieces;    // 16-byte pieces of a row in memory, of a tile
    constexpr int kMine = (kAllPieces + kThreads - 1) / kThreads;             // of a thread
    constexpr int kValues = kTermsC == 3 && DP > 128 ? 1 : 2;                 // buffers of values: there is no room for two of three terms of these
    constexpr bool kEven = kAllPieces % kThreads == 0;
    constexpr int kFewV = Sh::kFewV;
    constexpr int kKeysNear = 2 * kBuffer, kNear = FEW ? kWaves * kFewV * 16 * 64 * 4 : kKeysNear + kValues * kBuffer;
    __shared__ __align__(16) unsigned char near[kNear];
    unsigned char* const k_near = near;
    unsigned char* const v_near = near + kKeysNear;
    __shared__ int64_t offsets[kWaves][2][kTile];
    __shared__ uint32_t odd_first, odd_end;  // of the tiles whose values were cleaned

    const reef_chunk_attention_desc& d = a.d;
    const int32_t id = (int32_t)(blockIdx.x / (uint32_t)d.cache.kv_heads), kvh = (int32_t)(blockIdx.x - (uint32_t)id * (uint32_t)d.cache.kv_heads);
    const Item it = find_item(a, id);
    if (a.budget && kvh == 0 && threadIdx.x == 0) {
        if (it.tile >= 0 && it.shares > 1) a.jobs[it.slot + it.share] = make_int4(it.request, it.tile, it.share, it.shares);
        if (id == 0) *a.used = it.tile < 0 ? 0 : it.slots;   // (without a first item there are none)
    }
    if (it.tile < 0) return;
    const Request& r = it.r;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 31, h = lane >> 5;
    const int D = d.cache.head_dim;

    // this lane's row; up to 32 of them are those of all wavefronts
    const uint32_t rows = (uint32_t)(r.added * a.group);
    const uint32_t in_tile = (uint32_t)((FEW ? 0 : wave * kRows) + n), row = (uint32_t)it.tile * kTileRows + in_tile;
    const bool valid = row < rows;
    const uint32_t token = divided(row, a.by_group);
    const int32_t head = kvh * a.group + (int32_t)(row - token * a.by_group.by);
    const int64_t out_row = (int64_t)r.first + token;
    const uint32_t place = (uint32_t)r.cached + token;
    const uint32_t hi = valid && place < (uint32_t)r.n ? place + 1 : 0, lo = d.window && hi > (uint32_t)d.window ? hi - d.window : 0;
    // what all rows of the wavefront see, and what some do (its rows' places ascend)
    const uint32_t row0 = __builtin_amdgcn_readfirstlane(row), row_end = min(row0 + kRows, rows);
    const uint32_t place0 = (uint32_t)r.cached + divided(row0, a.by_group), place1 = row0 < rows ? (uint32_t)r.cached + divided(row_end - 1, a.by_group) : place0;
    const bool sees_any = row0 < rows && place0 < (uint32_t)r.n, see_all = sees_any && place1 < (uint32_t)r.n;
    const uint32_t some_hi = sees_any ? min(place1 + 1, (uint32_t)r.n) : 0;
    const uint32_t all_hi = see_all ? place0 + 1 : 0, all_lo = d.window && place1 + 1 > (uint32_t)d.window ? place1 + 1 - d.window : 0;

    const uint2 span = span_of(a, r, it.tile);
    uint32_t begin = span.x, end = span.y;
    if (it.shares > 1) {
        const uint32_t count = (end - begin + kTile - 1) / kTile;
        const uint32_t x = (uint32_t)((uint64_t)count * it.share / it.shares), y = (uint32_t)((uint64_t)count * (it.share + 1) / it.shares);
        end = min(end, begin + y * kTile);
        begin = min(end, begin + x * kTile);
    }
    const PagedView view{d.cache.blocks, d.cache.block_stride, d.cache.slot_stride};
    const C* keys = (const C*)a.key_cache + kvh * d.cache.head_stride;
    const C* values = (const C*)a.value_cache + kvh * d.cache.head_stride;
    const int32_t* table = a.table + (int64_t)it.request * d.table_stride;

    // the table's entry of one token of a tile a lane; -1: no token
    auto entry_of = [&](uint32_t t0) __attribute__((always_inline)) -> int32_t {
        const uint32_t t = t0 + lane;
        return lane < kTile && t < end ? table[divided(t, a.block)] : -1;
    };
    // its place, for all lanes to read; which of the tile's tokens there are
    auto find = [&](uint32_t t0, int32_t entry, int slot) __attribute__((always_inline)) -> uint64_t {
        int64_t at = -1;
        if (lane < kTile) {
            const uint32_t t = t0 + lane;
            at = paged_row(view, entry, (int32_t)(t - divided(t, a.block) * a.block.by));
            offsets[wave][slot][lane] = at < 0 ? 0 : at;
        }
        return __builtin_amdgcn_ballot_w64(at >= 0);
    };
    constexpr uint64_t kAll = kTile == 64 ? ~0ull : 0xFFFFFFFFull;
    u32x4 k_on_way[kMine], v_on_way[kMine];
    auto load = [&](const C* pool, u32x4 (&on_way)[kMine], int slot) __attribute__((always_inline)) {
        const uint32_t tid = again(threadIdx.x);
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const uint32_t x = i * kThreads + tid, at = x / kRowPieces, piece = x - at * kRowPieces;
            if (!kEven && x >= kAllPieces) continue;
            on_way[i] = *(const u32x4*)(pool + offsets[wave][slot][at] + (piece * 16 < D * (uint32_t)sizeof(C) ? piece * (16 / (uint32_t)sizeof(C)) : 0));
        }
    };
    // Into LDS: zeros where there is no token, or no such dimension.  Where not all rows see all of a tile, infinities and NaN among its values must not
    // be multiplied by weights of 0: they become 0 as well, and are looked for again at the end.
    auto store = [&](unsigned char* to, u32x4 (&on_way)[kMine], uint64_t there, bool clean, uint32_t number) __attribute__((always_inline)) {
        const uint32_t tid = again(threadIdx.x);
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const uint32_t x = i * kThreads + tid, at = x / kRowPieces, piece = x - at * kRowPieces;
            if (!kEven && x >= kAllPieces) continue;
            u32x4 w = on_way[i];
            const bool inside = (there >> at & 1) && piece * 16 < D * (uint32_t)sizeof(C);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = inside ? w[j] : 0;
            if (clean) {
                bool found = false;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t keep = keep_of(w[j], C());
                    found |= keep != ~0u;
                    w[j] &= keep;
                }
                if (found) {
                    atomicMin(&odd_first, number);
                    atomicMax(&odd_end, number + 1);
                }
            }
            if constexpr (kTermsC == 1) {
                *(u32x4*)(to + N::at(at, piece)) = w;
            } else {
                const uint32_t place = N::at(at, piece >> 1) + (piece & 1) * 8;
                uint32_t t[2][3];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float x0 = __uint_as_float(w[2 * j]), x1 = __uint_as_float(w[2 * j + 1]);
                    terms(x0, x1, t[j], __bf16());
                    // an infinity is its first term alone, and so is a NaN, which must not be cut to one
                    const bool odd0 = !(fabsf(x0) < INFINITY), odd1 = !(fabsf(x1) < INFINITY);
                    if (odd0 | odd1) {
                        const uint32_t keep = (odd0 ? 0 : 0xFFFFu) | (odd1 ? 0 : 0xFFFF0000u);
                        t[j][1] &= keep;
                        t[j][2] &= keep;
                        if (x0 != x0) t[j][0] |= 0x7FFFu;
                        if (x1 != x1) t[j][0] |= 0x7FFF0000u;
                    }
                }
#pragma unroll
                for (int x = 0; x < 3; ++x) *(u32x2*)(to + x * kPlane + place) = u32x2{t[0][x], t[1][x]};
            }
        }
    };

    int32_t entry = begin < end ? entry_of(begin) : -1;        // (asked for ahead of the queries: keys and values wait for them)

    // the queries: this lane's row, the pieces that its half of the keys has
    float scale = a.scale, shrink = 1.0f;    // scores: products * shrink * scale
    u32x4 q[kTermsQ][kSteps];
    {
        const Q* from = (const Q*)a.query + out_row * d.query_stride + head * d.query_head_stride;
        constexpr int kWords = (int)sizeof(Q) * 2;             // of eight values
        uint32_t raw[kSteps][kWords];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int at = s * 16 + h * 8;
#pragma unroll
            for (int w = 0; w < kWords; w += 4) {
                u32x4 x = {0, 0, 0, 0};
                if (valid && at < D && !a.zero) x = *(const u32x4*)(from + at + w * 4 / (int)sizeof(Q));
#pragma unroll
                for (int i = 0; i < 4; ++i) raw[s][w + i] = x[i] ^ a.flip;
            }
        }
        if constexpr (kTermsQ == 1) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) q[0][s] = {raw[s][0], raw[s][1], raw[s][2], raw[s][3]};
        } else {
            // Terms of fp16 need room below: a row is scaled by a power of two to 2^13; bf16 has it but for values below 2^-133, so rows below 2^-100 are
            // brought there.
            float grow = 1.0f, top = 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
#pragma unroll
                for (int w = 0; w < kWords; ++w) top = fmaxf(top, fabsf(__uint_as_float(raw[s][w])));
            top = other_max(top);
            if (top > 0.0f && top < INFINITY) {
                const int power = (int)(__float_as_uint(top) >> 23) - 127, by = kHalf ? min(126, 13 - power) : max(0, -100 - power);
                grow = __uint_as_float((uint32_t)(127 + by) << 23);
                const float back = __uint_as_float((uint32_t)(127 - by) << 23);
                // One factor where it is one: large queries and a large scale may pass 32 bits together where a product is 0.
                if (back > 1.0f && scale > 1.0f) shrink = back;
                else scale *= back;
            }
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t t[kTermsQ];
                    terms(__uint_as_float(raw[s][2 * w]) * grow, __uint_as_float(raw[s][2 * w + 1]) * grow, t, E());
#pragma unroll
                    for (int x = 0; x < kTermsQ; ++x) q[x][s][w] = t[x];
                }
        }
        if (scale == 0.0f) scale = 0x1p-149f;                  // (weights of what is not seen are 2^(-infinity scale))
    }

    float R = -INFINITY, l = 0.0f;
    f32x16 o[FEW ? kFewV : kSlabs];
#pragma unroll
    for (int m = 0; m < (int)(sizeof(o) / sizeof(o[0])); ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[m][i] = 0.0f;

    // where this lane reads: keys' row n; values' rows 4 (lane / 32) + (lane % 16) / 4, four dimensions from 16 (lane / 16 % 2) + 4 (lane % 4) on
    const int t16 = lane & 15;
    // (pieces are exchanged by bits, so those of other slabs, and of 8 rows below, are at places with other bits)
    const uint32_t k_at = N::at(n, h), v_at = N::at(4 * h + (t16 >> 2), 2 * (lane >> 4 & 1) + ((t16 & 3) >> 1)) + (t16 & 1) * 8;

    // Scores of a tile, as products.
    auto multiply_keys = [&](f32x16 (&s)[kSub], const unsigned char* k_tile) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[u][i] = 0.0f;
#pragma unroll
        for (int c = 0; c < kSteps; ++c)
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                const unsigned char* const from = k_tile + (k_at ^ c * 32) + u * 32 * N::kPitch;
                if constexpr (kTermsC == 1) {
                    const u32x4 k = *(const u32x4*)from;
#pragma unroll
                    for (int x = kTermsQ - 1; x >= 0; --x) s[u] = product(k, q[x][c], s[u], E());
                } else {
                    u32x4 k[3];
#pragma unroll
                    for (int x = 0; x < 3; ++x) k[x] = *(const u32x4*)(from + x * kPlane);
#pragma unroll
                    for (int both = 2; both >= 0; --both)
#pragma unroll
                        for (int x = both; x >= 0; --x) s[u] = product(k[x], q[both - x][c], s[u], E());
                }
            }
    };
    // Which of the tokens of 32 that this lane has of a row it sees, a bit each.  (Nothing of it is to be made ahead of the loop, and held in registers.)
    auto sees = [&](uint32_t t0, uint32_t there) __attribute__((always_inline)) {
        uint32_t from = t0 + 4 * h - lo, many = hi - lo, in = there >> (4 * h), yes = 0;
        asm volatile("" : "+v"(from), "+v"(many), "+v"(in));
#pragma unroll
        for (int i = 0; i < 16; ++i) yes |= from + (8 * (i >> 2) + (i & 3)) < many ? 1u << i : 0u;
        if (there != ~0u) {
            // bits 0..3, 8..11, 16..19 and 24..27 of `in`
            const uint32_t x = in & 0x0F0F0F0Fu, y = x | x >> 4;
            yes &= (y & 0xFFu) | (y >> 8 & 0xFF00u);
        }
        return yes;
    };
    auto hide = [&](auto& s, uint32_t t0, uint64_t there) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < (int)(sizeof(s) / sizeof(s[0])); ++u) {
            const uint32_t yes = sees(t0 + u * 32, (uint32_t)(there >> (u * 32)));
#pragma unroll
            for (int i = 0; i < 16; ++i) s[u][i] = yes >> i & 1 ? s[u][i] : -INFINITY;
        }
    };
    // Products as scores but for `scale`: once a tile.
    auto shrunk = [&](auto& s) __attribute__((always_inline)) {
        if constexpr (kHalf && kTermsQ > 1) {
#pragma unroll
            for (int u = 0; u < (int)(sizeof(s) / sizeof(s[0])); ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[u][i] *= shrink;
        }
    };
    auto largest = [&](auto& s) __attribute__((always_inline)) {
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < (int)(sizeof(s) / sizeof(s[0])); ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
        return other_max(top) * scale;
    };
    auto refer = [&](float top, auto slabs) __attribute__((always_inline)) {
        const bool passes = top > R + kSlack;
        if (__builtin_amdgcn_ballot_w64(passes)) {
            const float next = passes ? rintf(top) : R;
            const float f = passes ? __builtin_amdgcn_exp2f(R - next) : 1.0f;
            R = next;
            l *= f;
#pragma unroll
            for (int m = 0; m < decltype(slabs)::value; ++m)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[m][i] *= f;
        }
    };
    // From 2^20 on a score's product and its difference from the reference are not exact together: it is rounded first there.
    float times = scale, plus = kGrow;
    auto approach = [&](auto& s) __attribute__((always_inline)) {
        const float base = R == -INFINITY ? 0.0f : R;
        times = scale;
        plus = kGrow - base;
        if (__builtin_amdgcn_ballot_w64(fabsf(base) >= 0x1p20f)) {
#pragma unroll
            for (int u = 0; u < (int)(sizeof(s) / sizeof(s[0])); ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
#pragma clang fp contract(off)
                    const float x = s[u][i] * scale;
                    s[u][i] = x - base;
                }
            times = 1.0f;
            plus = kGrow;
        }
    };
    // Weights of a tile, as operands.
    u32x4 p[kTile / 16][kTermsP];
    auto weigh = [&](auto& s) __attribute__((always_inline)) {
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < 2 * (int)(sizeof(s) / sizeof(s[0])); ++c)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int i = (c & 1) * 8 + 2 * w;
                const float x = __builtin_amdgcn_exp2f(fmaf(s[c >> 1][i], times, plus)), y = __builtin_amdgcn_exp2f(fmaf(s[c >> 1][i + 1], times, plus));
                sum[w] += x + y;
                uint32_t t[kTermsP];
                terms(x, y, t, E());
#pragma unroll
                for (int k = 0; k < kTermsP; ++k) p[c][k][w] = t[k];
            }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    };
    auto values_of = [&](const unsigned char* v_tile, int c, int m, u32x4 (&v)[kTermsC]) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < kTermsC; ++x) {
            typedef short s4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s4 near_s4;
            const unsigned char* const from = v_tile + x * kPlane + c * 16 * N::kPitch;
            const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((near_s4*)(from + (v_at ^ m * 64))));
            const u32x2 z = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((near_s4*)(from + 8 * N::kPitch + (v_at ^ (m * 64 + 32)))));
            v[x] = {y[0], y[1], z[0], z[1]};
        }
    };
    auto multiply_by = [&](u32x4 (&v)[kTermsC], int c, int m) __attribute__((always_inline)) {
        if constexpr (kTermsC == 1) {
#pragma unroll
            for (int x = kTermsP - 1; x >= 0; --x) o[m] = product(v[0], p[c][x], o[m], E());
        } else {
#pragma unroll
            for (int both = 2; both >= 0; --both)
#pragma unroll
                for (int x = both; x >= 0; --x) o[m] = product(v[x], p[c][both - x], o[m], E());
        }
    };
    auto multiply_values = [&](const unsigned char* v_tile) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < kTile / 16; ++c)
#pragma unroll
            for (int m = 0; m < kSlabs; ++m) {
                u32x4 v[kTermsC];
                values_of(v_tile, c, m, v);
                multiply_by(v, c, m);
            }
    };
    if constexpr (FEW) {
        // Up to 32 rows in all: each wavefront takes every kWaves-th 32 tokens for itself.  Keys go through a part of LDS of its own, so that their rows are read from
        // memory whole (32 bytes a row and load, as the products want them, take 2 us more for 256 tokens).  Values come as the products want
        // them: lane (n, h) has of each of its tokens the n-th kFewV values, whose e-th ones are row n of the e-th product, dimension kFewV n + e.
        constexpr int kKLoads = kRowPieces / 2, kVWords = kFewV * (int)sizeof(C) / 4;
        constexpr std::integral_constant<int, kFewV> kAcc;
        using K = Near<DP * (int)sizeof(C) / 2>;
        static_assert(kWaves * 32 * K::kPitch <= kNear, "");
        unsigned char* const k_mine = near + wave * 32 * K::kPitch;
        u32x4 k[kKLoads];
        uint32_t v[16][kVWords];
        auto entry_at = [&](uint32_t t0) __attribute__((always_inline)) -> int32_t {
            const uint32_t t = t0 + n;
            return t < end ? table[divided(t, a.block)] : -1;
        };
        auto find_few = [&](uint32_t t0, int32_t entry, int slot) __attribute__((always_inline)) -> uint32_t {
            const uint32_t t = t0 + n;
            const int64_t at = paged_row(view, entry, (int32_t)(t - divided(t, a.block) * a.block.by));
            if (h == 0) offsets[wave][slot][n] = at < 0 ? 0 : at;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            return (uint32_t)__builtin_amdgcn_ballot_w64(at >= 0);
        };
        // (Larger heads leave no registers for these places: held ahead of the loop they cost scratch.  64 single tokens over 4000, 32 heads over 8 of 192, bf16: 762 us, made
        // again 292; of 256, 493 and 401; but 204 and 200 for 128, 24.5 and 26.7 for 16 tokens over 2000 of 128.)
        auto key_lane = [&]() __attribute__((always_inline)) -> uint32_t { return DP > 128 ? again(lane) : lane; };
        auto load_k = [&](int slot) __attribute__((always_inline)) {
            const uint32_t mine = key_lane();
#pragma unroll
            for (int i = 0; i < kKLoads; ++i) {
                const uint32_t x = i * 64 + mine, row = x / kRowPieces, piece = x - row * kRowPieces;
                k[i] = *(const u32x4*)(keys + offsets[wave][slot][row] + (piece * 16 < D * (uint32_t)sizeof(C) ? piece * (16 / (uint32_t)sizeof(C)) : 0));
            }
        };
        auto store_k = [&]() __attribute__((always_inline)) {
            const uint32_t mine = key_lane();
#pragma unroll
            for (int i = 0; i < kKLoads; ++i) {
                const uint32_t x = i * 64 + mine, row = x / kRowPieces, piece = x - row * kRowPieces;
                *(u32x4*)(k_mine + K::at(row, piece)) = piece * 16 < D * (uint32_t)sizeof(C) ? k[i] : u32x4{0, 0, 0, 0};
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        };
        auto load_v = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const C* const from = values + offsets[wave][slot][16 * (j >> 3) + 8 * (j >> 2 & 1) + 4 * h + (j & 3)] + (kFewV * n < D ? kFewV * n : 0);
                if constexpr (kVWords == 1) {
                    v[j][0] = *(const uint32_t*)from;
                } else if constexpr (kVWords == 2) {
                    const u32x2 x = *(const u32x2*)from;
                    v[j][0] = x[0];
                    v[j][1] = x[1];
                } else {
#pragma unroll
                    for (int w = 0; w < kVWords; w += 4) {
                        const u32x4 x = *(const u32x4*)(from + w * 4 / (int)sizeof(C));
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[j][w + i] = x[i];
                    }
                }
            }
        };
        constexpr uint32_t kStep = kWaves * 32;
        uint32_t t0 = begin + wave * 32, odd_from = ~0u, odd_to = 0, there = 0;
        int slot = 0;
        int32_t entry = t0 < end ? entry_at(t0) : -1;
        if (t0 < end) {
            there = find_few(t0, entry, 0);
            entry = t0 + kStep < end ? entry_at(t0 + kStep) : -1;
            load_k(0);
            load_v(0);
        }
        for (; t0 < end; t0 += kStep) {
            const bool more = t0 + kStep < end;
            const uint32_t there_now = there;
            store_k();
            if (more) {
                there = find_few(t0 + kStep, entry, slot ^ 1);
                entry = t0 + 2 * kStep < end ? entry_at(t0 + 2 * kStep) : -1;
                load_k(slot ^ 1);
            }
            f32x16 s[1];
#pragma unroll
            for (int i = 0; i < 16; ++i) s[0][i] = 0.0f;
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
                if constexpr (kTermsC == 1) {
                    const u32x4 x = *(const u32x4*)(k_mine + (K::at(n, h) ^ c * 32));
#pragma unroll
                    for (int i = kTermsQ - 1; i >= 0; --i) s[0] = product(x, q[i][c], s[0], E());
                } else {
                    u32x4 x[3];
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const f32x4 z = *(const f32x4*)(k_mine + (K::at(n, 2 * h + y) ^ c * 64));
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            uint32_t t[3];
                            terms(z[2 * w], z[2 * w + 1], t, E());
#pragma unroll
                            for (int i = 0; i < 3; ++i) x[i][2 * y + w] = t[i];
                        }
                    }
#pragma unroll
                    for (int both = 2; both >= 0; --both)
#pragma unroll
                        for (int i = both; i >= 0; --i) s[0] = product(x[i], q[both - i][c], s[0], E());
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            shrunk(s);
            const bool by_all = t0 >= all_lo && t0 + 32 <= all_hi;
            if (!by_all || there_now != ~0u) hide(s, t0, there_now);
            refer(largest(s), kAcc);
            approach(s);
            weigh(s);
            if (there_now != ~0u) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (!(there_now >> (4 * h) >> (16 * (j >> 3) + 8 * (j >> 2 & 1) + (j & 3)) & 1)) {
#pragma unroll
                        for (int w = 0; w < kVWords; ++w) v[j][w] = 0;
                    }
            }
            if (!by_all) {               // (as in store())
                bool found = false;
#pragma unroll
                for (int j = 0; j < 16; ++j)
#pragma unroll
                    for (int w = 0; w < kVWords; ++w) {
                        const uint32_t keep = keep_of(v[j][w], C());
                        found |= keep != ~0u;
                        v[j][w] &= keep;
                    }
                if (__builtin_amdgcn_ballot_w64(found)) {
                    odd_from = min(odd_from, t0);
                    odd_to = t0 + 32;
                }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < kFewV; ++e) {
                    u32x4 x[kTermsC];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int j = c * 8 + 2 * w;
                        if constexpr (kTermsC == 1) {
                            x[0][w] = __builtin_amdgcn_perm(v[j + 1][e / 2], v[j][e / 2], e & 1 ? 0x07060302 : 0x05040100);
                        } else {
                            uint32_t t[3];
                            terms(__uint_as_float(v[j][e]), __uint_as_float(v[j + 1][e]), t, E());
#pragma unroll
                            for (int i = 0; i < 3; ++i) x[i][w] = t[i];
                        }
                    }
                    if constexpr (kTermsC == 1) {
#pragma unroll
                        for (int i = kTermsP - 1; i >= 0; --i) o[e] = product(x[0], p[c][i], o[e], E());
                    } else {
#pragma unroll
                        for (int both = 2; both >= 0; --both)
#pragma unroll
                            for (int i = both; i >= 0; --i) o[e] = product(x[i], p[c][both - i], o[e], E());
                    }
                }
            slot ^= 1;
            if (more) load_v(slot);
        }
        for (uint32_t t = odd_from; t < min(end, odd_to); ++t) {
            const uint32_t page = divided(t, a.block);
            const int64_t at = paged_row(view, table[page], (int32_t)(t - page * a.block.by));
            if (at < 0 || !(t >= lo && t < hi)) continue;
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
                for (int e = 0; e < kFewV; ++e) {
                    const int dim = kFewV * (8 * (i >> 2) + 4 * h + (i & 3)) + e;
                    if (!(fabsf((float)values[at + (dim < D ? dim : 0)]) < INFINITY)) o[e][i] = NAN;
                }
        }
        // The wavefronts that had tokens, joined: neighbouring dimensions of a row next to each other, lane after lane; then a unit of them a thread.
        constexpr int kUnit = kFewV < 4 ? kFewV : 4, kUnits = kFewV / kUnit * 16;
        typedef float UnitF __attribute__((ext_vector_type(kUnit)));
        typedef Q UnitQ __attribute__((ext_vector_type(kUnit)));
        l = other_sum(l);
        const int waves = min((int)((end - begin + 31) / 32), kWaves);
        float2* const stats = (float2*)offsets;
        __syncthreads();                 // (the places are read)
        if (wave < waves) {
            if (h == 0) stats[wave * 32 + n] = make_float2(R, l);
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
                for (int e = 0; e < kFewV; e += kUnit) {
                    UnitF x;
#pragma unroll
                    for (int y = 0; y < kUnit; ++y) x[y] = o[e + y][i];
                    ((UnitF*)near)[(wave * kUnits + i * (kFewV / kUnit) + e / kUnit) * 64 + lane] = x;
                }
        }
        __syncthreads();
        float top = -INFINITY, sum = 0.0f, weight[kWaves];
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
            if (w < waves) top = fmaxf(top, stats[w * 32 + n].x);
        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            weight[w] = 0.0f;
            if (w < waves) {
                const float2 x = stats[w * 32 + n];
                weight[w] = __builtin_amdgcn_exp2f(x.x - base);
                sum += weight[w] * x.y;
            }
        }
        if (!valid) return;
        const int64_t at = ((int64_t)(it.slot + it.share) * d.cache.kv_heads + kvh) * kTileRows + n;
        const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
        Q* const to = (Q*)a.out + out_row * d.out_stride + head * d.out_head_stride;
        for (int u = wave; u < kUnits; u += kWaves) {
            const int i = u / (kFewV / kUnit), dim = kFewV * (8 * (i >> 2) + 4 * h + (i & 3)) + (u - i * (kFewV / kUnit)) * kUnit;
            if (dim >= D) continue;
            UnitF all = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w)
                if (w < waves) all += weight[w] * ((const UnitF*)near)[(w * kUnits + u) * 64 + lane];
            if (it.shares > 1) {
                *(UnitF*)(a.parts + at * D + dim) = all;
            } else {
                UnitQ x;
#pragma unroll
                for (int y = 0; y < kUnit; ++y) x[y] = (Q)(all[y] * f);
                *(UnitQ*)(to + dim) = x;
            }
        }
        if (wave == 0 && h == 0) {
            if (it.shares > 1) a.stats[at] = make_float2(top == -INFINITY ? -INFINITY : top - kGrow, sum);
            else if (a.lse) a.lse[out_row * d.heads + head] = sum == 0.0f ? -INFINITY : (top + (__log2f(sum) - kGrow)) * kLn2;
        }
        return;
    }

    const uint32_t count = (end - begin + kTile - 1) / kTile;
    auto seen_by_all = [&](uint32_t j, uint64_t there) __attribute__((always_inline)) {
        return begin + j * kTile >= all_lo && begin + (j + 1) * kTile <= all_hi && there == kAll;
    };
    // the same of the workgroup's rows, but for tokens that are not there
    const uint32_t first_place = (uint32_t)r.cached + divided((uint32_t)it.tile * kTileRows, a.by_group);
    const uint32_t last_place = (uint32_t)r.cached + divided(min((uint32_t)(it.tile + 1) * kTileRows, rows) - 1, a.by_group);
    auto inside_all = [&](uint32_t j) __attribute__((always_inline)) {
        const uint32_t t0 = begin + j * kTile;
        return t0 + kTile <= first_place + 1 && last_place < (uint32_t)r.n && (!d.window || t0 + (uint32_t)d.window > last_place);
    };
    // Tile j + 1's keys and tile j's values on their way, and into LDS.
    uint64_t there = 0, there_next = 0;      // of tiles j and j + 1
    auto ask = [&](uint32_t j, auto parity) __attribute__((always_inline)) {
        constexpr int kNow = decltype(parity)::value;          // j % 2
        if (j + 1 < count) {
            there_next = find(begin + (j + 1) * kTile, entry, kNow ^ 1);
            entry = j + 2 < count ? entry_of(begin + (j + 2) * kTile) : -1;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            load(keys, k_on_way, kNow ^ 1);
        }
        load(values, v_on_way, kNow);
    };
    auto take = [&](uint32_t j, auto parity) __attribute__((always_inline)) {
        constexpr int kNow = decltype(parity)::value;
        if (j + 1 < count) store(k_near + (kNow ^ 1) * kBuffer, k_on_way, there_next, false, 0);
        if constexpr (kValues == 1) __syncthreads();
        store(v_near + (kValues == 2 ? kNow : 0) * kBuffer, v_on_way, there, !inside_all(j), j);
        __syncthreads();
        there = there_next;
    };
    constexpr std::integral_constant<int, 0> kEvenOnes;
    constexpr std::integral_constant<int, 1> kOddOnes;
    if (count) {
        if (threadIdx.x == 0) {
            odd_first = ~0u;
            odd_end = 0;
        }
        there = find(begin, entry, 0);
        entry = count > 1 ? entry_of(begin + kTile) : -1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        load(keys, k_on_way, 0);
        store(k_near, k_on_way, there, false, 0);
        __syncthreads();
        if (some_hi == 0) {                  // no rows: this wavefront only brings keys and values
            for (uint32_t j = 0; j < count; j += 2) {
                ask(j, kEvenOnes);
                take(j, kEvenOnes);
                if (j + 1 == count) break;
                ask(j + 1, kOddOnes);
                take(j + 1, kOddOnes);
            }
            if (it.shares == 1 && !valid) return;
        } else {
            f32x16 even[kSub], odd[kSub];    // scores of even and odd tiles
            auto look = [&](uint32_t j, f32x16 (&s)[kSub], float top) __attribute__((always_inline)) {
                if (!seen_by_all(j, there)) {
                    hide(s, begin + j * kTile, there);
                    top = largest(s);
                }
                refer(top, std::integral_constant<int, kSlabs>());
            };
            // Weights of tile j - 1 go to its values while the scores of tile j are made.
            auto step = [&](uint32_t j, f32x16 (&s)[kSub], f32x16 (&next)[kSub], auto parity) __attribute__((always_inline)) {
                constexpr int kNow = decltype(parity)::value;
                ask(j, parity);
                approach(s);
                multiply_keys(next, k_near + kNow * kBuffer);
                weigh(s);
                multiply_values(v_near + (kValues == 2 ? kNow ^ 1 : 0) * kBuffer);
                shrunk(next);
                look(j, next, largest(next));
                take(j, parity);
            };
            auto end_with = [&](f32x16 (&s)[kSub], int parity) __attribute__((always_inline)) {
                approach(s);
                weigh(s);
                multiply_values(v_near + (kValues == 2 ? parity : 0) * kBuffer);
            };
            ask(0, kEvenOnes);
            multiply_keys(even, k_near);
            shrunk(even);
            look(0, even, largest(even));
            take(0, kEvenOnes);
            uint32_t j = 1;
            for (; j + 1 < count; j += 2) {
                step(j, even, odd, kOddOnes);
                step(j + 1, odd, even, kEvenOnes);
            }
            if (j < count) {
                step(j, even, odd, kOddOnes);
#pragma unroll
                for (int u = 0; u < kSub; ++u) even[u] = odd[u];
            }
            end_with(even, (count - 1) & 1);
            // Rows that see an infinity or a NaN among values have NaN.  (Rare: the values are read again, token after token.)
            for (uint32_t t = begin + min(odd_first, odd_end) * kTile; t < min(end, begin + odd_end * kTile); ++t) {
                const uint32_t page = divided(t, a.block);
                const int64_t at = paged_row(view, table[page], (int32_t)(t - page * a.block.by));
                if (at < 0 || !(t >= lo && t < hi)) continue;
#pragma unroll
                for (int m = 0; m < kSlabs; ++m)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int dim = m * 32 + 8 * (i >> 2) + 4 * h + (i & 3);
                        if (!(fabsf((float)values[at + (dim < D ? dim : 0)]) < INFINITY)) o[m][i] = NAN;
                    }
            }
        }
    }

    l = other_sum(l);
    if (it.shares > 1) {
        const int64_t at = ((int64_t)(it.slot + it.share) * d.cache.kv_heads + kvh) * kTileRows + in_tile;
        if (h == 0) a.stats[at] = make_float2(R == -INFINITY ? -INFINITY : R - kGrow, l);
#pragma unroll
        for (int m = 0; m < kSlabs; ++m)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int dim = m * 32 + i * 2 + h * 4;
                if (dim < D) *(f32x4*)(a.parts + at * D + dim) = f32x4{o[m][i], o[m][i + 1], o[m][i + 2], o[m][i + 3]};
            }
        return;
    }
    if (!valid) return;
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    Q* const to = (Q*)a.out + out_row * d.out_stride + head * d.out_head_stride;
#pragma unroll
    for (int m = 0; m < kSlabs; ++m)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int dim = m * 32 + i * 2 + h * 4;
            if (dim < D) put4(to + dim, o[m][i] * f, o[m][i + 1] * f, o[m][i + 2] * f, o[m][i + 3] * f);
        }
    if (h == 0 && a.lse) a.lse[out_row * d.heads + head] = l == 0.0f ? -INFINITY : (R + (__log2f(l) - kGrow)) * kLn2;
}

constexpr int kThreads = 1024;               // of the join
// The shares of a tile, one cache head: a workgroup for each of its slots, which take the tile's rows among them, a quad of a row a thread, share after share.
template <class Q>
__global__ void __launch_bounds__(kThreads) join_shares(Args a) {
    const reef_chunk_attention_desc& d = a.d;
    const int D = d.cache.head_dim, quads = D / 4;
    const uint32_t kv_heads = (uint32_t)d.cache.kv_heads, works = (uint32_t)*a.used * kv_heads;
    for (uint32_t work = blockIdx.x; work < works; work += gridDim.x) {
        const int32_t id = (int32_t)(work / kv_heads), kvh = (int32_t)(work - (uint32_t)id * kv_heads);
        const int4 job = a.jobs[id];
        const Request r = request_of(a, job.x);
        const int32_t rows = min(a.tile_rows, r.added * a.group - job.y * a.tile_rows), slot = id - job.z, shares = job.w;
        const int32_t from = (int32_t)((int64_t)rows * quads * job.z / job.w), to = (int32_t)((int64_t)rows * quads * (job.z + 1) / job.w);
        const int64_t step = (int64_t)d.cache.kv_heads * a.tile_rows;
        for (int32_t x = from + (int32_t)threadIdx.x; x < to; x += kThreads) {
            const int32_t i = x / quads, dim = (x - i * quads) * 4;
            const int64_t at = ((int64_t)slot * d.cache.kv_heads + kvh) * a.tile_rows + i;
            float R = -INFINITY, l = 0.0f;
            f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
            for (int32_t s = 0; s < shares; ++s) {
                const float2 stat = a.stats[at + s * step];
                const f32x4 mine = *(const f32x4*)(a.parts + (at + s * step) * D + dim);
                const float next = fmaxf(R, stat.x), base = next == -INFINITY ? 0.0f : next;
                const float f = __builtin_amdgcn_exp2f(R - base), g = __builtin_amdgcn_exp2f(stat.x - base);
                R = next;
                l = l * f + stat.y * g;
                o = o * f + mine * g;
            }
            const uint32_t row = (uint32_t)(job.y * a.tile_rows + i), token = divided(row, a.by_group);
            const int32_t head = kvh * a.group + (int32_t)(row - token * a.by_group.by);
            const int64_t out_row = (int64_t)r.first + token;
            const float f = l == 0.0f ? 0.0f : 1.0f / l;
            put4((Q*)a.out + out_row * d.out_stride + head * d.out_head_stride + dim, o[0] * f, o[1] * f, o[2] * f, o[3] * f);
            if (dim == 0 && a.lse) a.lse[out_row * d.heads + head] = l == 0.0f ? -INFINITY : (R + __log2f(l)) * kLn2;
        }
    }
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

// What the host asks of a shape.
struct Waves {
    int few, each, at_once, products;
};
template <class Q, class C>
Waves waves_of(int dim) {
    auto of = [](auto dp) {
        using Sh = Shape<Q, C, decltype(dp)::value>;
        return Waves{Sh::kFewWaves, Sh::kWaves, Sh::kPair ? 2 * kCus : kCus, Sh::kTermsC == 3 ? 6 : Sh::kTermsQ};
    };
    return dim <= 64 ? of(std::integral_constant<int, 64>()) : dim <= 96 ? of(std::integral_constant<int, 96>()) : dim <= 128 ? of(std::integral_constant<int, 128>())
         : dim <= 192 ? of(std::integral_constant<int, 192>()) : of(std::integral_constant<int, 256>());
}
Waves waves_of(const reef_chunk_attention_desc& d) {
    const int dim = d.cache.head_dim;
    if (d.type != REEF_TYPE_F32) return d.type == REEF_TYPE_F16 ? waves_of<_Float16, _Float16>(dim) : waves_of<__bf16, __bf16>(dim);
    return d.cache.type == REEF_TYPE_F32 ? waves_of<float, float>(dim) : d.cache.type == REEF_TYPE_F16 ? waves_of<float, _Float16>(dim) : waves_of<float, __bf16>(dim);
}

// How a call is laid out.
struct Plan {
    int32_t tile_rows, at_once, looked, budget;
    float join;
    bool few;               // tiles of 32 rows in all
    int64_t items, slots, groups;      // groups: workgroups
    size_t info_bytes, list_bytes, jobs_bytes, stats_bytes, bytes;
};
Plan plan_of(const reef_chunk_attention_desc& d) {
    const int32_t group = d.heads / d.cache.kv_heads, kv = d.cache.kv_heads;
    const int64_t rows = (int64_t)d.tokens * group;
    Plan p{};
    // Up to 32 rows a request on the average: tiles of so many, whose wavefronts share the tokens, else tiles of so many for each wavefront, which share keys and values.
    const Waves waves = waves_of(d);
    p.few = rows <= (int64_t)kRows * d.requests && waves.few;
    p.tile_rows = p.few ? kRows : waves.each * kRows;
    p.at_once = p.few ? kCus : waves.at_once;
    p.looked = p.few ? kLookedFew : waves.products > 1 ? kLooked * 2 / 3 : kLooked;
    p.join = p.few ? 0.0f : kJoin / (float)waves.products;
    int64_t longest = (int64_t)d.max_blocks * d.cache.block_size;
    if (d.longest && d.longest < longest) longest = d.longest;
    if (d.window) longest = std::min(longest, (int64_t)d.window + p.tile_rows / group);
    p.items = rows / p.tile_rows + d.requests;
    const int64_t least = p.few ? kLeastFew : kLeast;
    // tokens that a workgroup has at most where all are the longest; of one request the cut is known
    const int64_t most = p.items * kv * longest / p.at_once;
    bool whole = false;
    if (d.requests == 1) {
        const float tokens = (float)std::min<int64_t>(d.tokens, longest);
        const Cut c = cut_for((float)most * (1.0f - 0.5f * tokens / (float)longest), p.join, p.few);
        whole = (float)longest <= c.whole + 0.7f * c.tokens + 0.5f * p.join;
    }
    if (longest > p.looked && !whole) {
        // Workgroups that find no item take 2 us a round for their look (four prompts of 2048: 74 us without, 80 with three rounds): there are no more than are likely to have one.
        const int64_t shares = (longest + least - 1) / least, tiles = p.items;
        p.budget = p.at_once * (tiles * kv <= p.at_once / 2 ? 1 : (int32_t)std::max<int64_t>(1, std::min<int64_t>(3, most * waves.products / 1000)));
        p.items = std::min(tiles * shares, tiles + (p.budget + kv - 1) / kv);
        // (a tile that is cut has two shares at least, so that these are what tiles may be cut into beside one each, twice: a slot of 256 rows, heads of 128, has 133 KB)
        p.slots = std::min<int64_t>(p.items, 2ll * ((p.budget + kv - 1) / kv));
        p.jobs_bytes = 16 * (size_t)(1 + p.slots);
        p.stats_bytes = (size_t)p.slots * kv * p.tile_rows * 8;
    }
    p.groups = p.items * kv;
    if (d.requests > kFewRequests) {
        p.info_bytes = ((size_t)d.requests * 8 + 15) / 16 * 16;
        p.list_bytes = ((size_t)(kListHead + p.items) * 4 + 15) / 16 * 16;
    }
    p.bytes = p.info_bytes + p.list_bytes + p.jobs_bytes + p.stats_bytes + (size_t)p.slots * kv * p.tile_rows * d.cache.head_dim * 4;
    return p;
}

template <class Q, class C, int DP>
int run_heads(const char* what, const Args& a, const Plan& p, unsigned groups, void* stream) {
    using Sh = Shape<Q, C, DP>;
    if constexpr (Sh::kFewWaves != 0)
        if (p.few) return launch(what, chunk_attention<Q, C, DP, true>, dim3(groups), dim3(Sh::kFewWaves * 64), a, stream);
    return launch(what, chunk_attention<Q, C, DP, false>, dim3(groups), dim3(Sh::kWaves * 64), a, stream);
}
template <class Q, class C>
int run(const char* what, const Args& a, const Plan& p, void* stream) {
    const int D = a.d.cache.head_dim;
    const unsigned groups = (unsigned)p.groups;
    if (a.list)
        if (int rc = launch(what, list_items, dim3(1), dim3(kListThreads), a, stream)) return rc;
    const int rc = D <= 64    ? run_heads<Q, C, 64>(what, a, p, groups, stream)
                   : D <= 96  ? run_heads<Q, C, 96>(what, a, p, groups, stream)
                   : D <= 128 ? run_heads<Q, C, 128>(what, a, p, groups, stream)
                   : D <= 192 ? run_heads<Q, C, 192>(what, a, p, groups, stream)
                              : run_heads<Q, C, 256>(what, a, p, groups, stream);
    if (rc || !p.budget) return rc;
    return launch(what, join_shares<Q>, dim3((unsigned)std::min<int64_t>(p.slots * a.d.cache.kv_heads, 2 * kCus)), dim3(kThreads), a, stream);
}

}  // namespace

extern "C" int64_t reef_ops_chunk_attention_workspace(const reef_chunk_attention_desc* d) {
    if (check("reef_ops_chunk_attention_workspace", d)) return -1;
    return (int64_t)plan_of(*d).bytes;
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
    const Plan p = plan_of(*d);
    // (2^32 threads are refused by the launch, which may be the call's second one)
    if (p.groups >= 1ll << 23) return refuse(what, "%lld workgroups are too many", (long long)p.groups);
    if (p.bytes && (!rows16(workspace) || workspace_bytes < (int64_t)p.bytes))
        return refuse(what, "a workspace of %zu bytes on 16 is needed, %lld are given", p.bytes, (long long)workspace_bytes);
    char* const w = (char*)workspace;
    const size_t list = p.info_bytes, jobs = list + p.list_bytes, stats = jobs + p.jobs_bytes, parts = stats + p.stats_bytes;
    const int32_t group = d->heads / d->cache.kv_heads;
    const Args a{*d, query, key_cache, value_cache, table, starts, cached, lengths, out, lse, (int2*)w, p.list_bytes ? (int32_t*)(w + list) : nullptr, (float*)(w + parts),
                 (float2*)(w + stats), d->scale == 0.0f ? kLog2e : std::fabs(d->scale) * kLog2e, d->scale < 0.0f ? (d->type == REEF_TYPE_F32 ? 0x80000000u : 0x80008000u) : 0u,
                 d->scale == 0.0f, group, p.tile_rows, p.at_once, p.looked, p.join, p.budget, (int32_t)p.items, (int32_t)p.slots, (int32_t*)(w + jobs), (int4*)(w + jobs) + 1,
                 divider((uint32_t)d->cache.block_size), divider((uint32_t)group)};
    switch (d->type * 4 + d->cache.type) {
        case REEF_TYPE_F32 * 4 + REEF_TYPE_F32: return run<float, float>(what, a, p, stream);
        case REEF_TYPE_F32 * 4 + REEF_TYPE_F16: return run<float, _Float16>(what, a, p, stream);
        case REEF_TYPE_F32 * 4 + REEF_TYPE_BF16: return run<float, __bf16>(what, a, p, stream);
        case REEF_TYPE_F16 * 4 + REEF_TYPE_F16: return run<_Float16, _Float16>(what, a, p, stream);
        default: return run<__bf16, __bf16>(what, a, p, stream);
    }
}
