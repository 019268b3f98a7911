// Attention of one new token a request over a paged key-value cache (reef_ops_paged_attention).
#include <algorithm>
#include <cmath>

#include "ops_common.h"
#include "paged_shares.h"

namespace {
using namespace reef_ops;

constexpr int kThreads = 256;                // of a workgroup of four wavefronts, and of the join's
// Workgroups that the shares of all sequences are to make: what runs at once (two a CU; one for heads over 128) less an eighth, as each
// sequence's number of shares is rounded up.  Just above what runs at once the last round is nearly empty: of 224 .. 3584, 448 takes
// 80 us for 12 x 8000 tokens, 8 cache heads of 128, bf16 (672: 87, 1344: 88), 21 where these lengths are the longest (672: 26).
// Where the heads of all sequences are as many by themselves most have one or two shares, and the few long ones decide: twice as many
// take 95 us instead of 103 for 90 sequences of up to 8000 tokens, 149 instead of 158 for 300 with 4 heads, 306 instead of 326 for
// 50 x 8000, the same for 300 x 1500, 2 % more for 90 x 8000; 64 x 9000 with heads of 64, which just run at once uncut, lose most: 262
// instead of 240 (the rule has no term for batches that do).  Four times as many win little more (306 -> 303) and lose 7 % for 300 x 8000, heads of 64.
constexpr int kGroups = 448, kFiner = 2;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Args {
    reef_paged_attention_desc d;
    const void *query, *key_cache, *value_cache;
    const int32_t *table, *lengths;
    void* out;
    float* lse;
    float* parts;           // [share][head][head_dim], sums that are not divided yet
    float2* stats;          // [share][head]: maximum (of scores * log2 e) and sum
    int2* info;             // [request]: its first share and how many they are
    int32_t* list;          // more than kFewRequests: the number of shares, then the request of each; otherwise null
    int32_t group, tiles;   // query heads a cache head; tiles of 16 of them
    int32_t budget;         // shares that all tokens are cut into, beside one a request; 0: sequences are not split
    Divider block;          // by the block size
    int32_t heads_each;     // of a workgroup of the join
    int32_t units, together;   // workgroups in `units` groups of `together`, each group on one XCD
};

struct Share {
    int32_t request, number, first, count;   // the number-th of `count` shares of the request, which start with share `first` of all
};

__device__ inline int32_t seen_tokens(const Args& a, int32_t r) {
    const int32_t held = held_length(a.lengths[r], a.d.max_blocks, a.d.cache.block_size);
    return a.d.window && held > a.d.window ? a.d.window : held;
}

// Up to kFewRequests every workgroup adds up the lengths for itself, more are listed by a launch ahead (4096 requests of 8 heads would be
// read by 33000 workgroups).
constexpr int32_t kFewRequests = 256, kListHead = 1;

// Adds up over the workgroup, exclusively; *all: the sum.
template <int WAVES>
__device__ inline int32_t scan(int32_t v, int32_t* counts, int32_t* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t at = v;
    for (int x = 1; x < 64; x <<= 1) {
        const int32_t o = __shfl_up(at, x);
        if (lane >= x) at += o;
    }
    if (lane == 63) counts[wave] = at;
    __syncthreads();
    at -= v;
    *all = 0;
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) at += counts[w];
        *all += counts[w];
    }
    return at;
}
template <int WAVES>
__device__ inline float sum_of(float v, float* sums) {
    for (int x = 32; x; x >>= 1) v += __shfl_xor(v, x);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
    for (int w = 0; w < WAVES; ++w) v += sums[w];
    return v;
}

// Share `id` of all; number < 0: there is no such share.
__device__ inline Share find_share(const Args& a, int32_t id) {
    if (a.list) {
        if (id >= a.list[0]) return {0, -1, 0, 0};
        const int32_t r = a.list[kListHead + id];
        const int2 info = a.info[r];
        return {r, id - info.x, info.x, info.y};
    }
    if (a.d.requests <= 64) {                // a request a lane, each wavefront for itself
        const int lane = threadIdx.x & 63;
        const int32_t n = lane < a.d.requests ? seen_tokens(a, lane) : 0;
        float total = (float)n;
        for (int x = 32; x; x >>= 1) total += __shfl_xor(total, x);
        const int32_t tokens = tokens_of(total, a.budget), mine = lane < a.d.requests ? shares_of(n, tokens) : 0;
        int32_t at = mine;
        for (int x = 1; x < 64; x <<= 1) {
            const int32_t o = __shfl_up(at, x);
            if (lane >= x) at += o;
        }
        at -= mine;
        const uint64_t who = __builtin_amdgcn_ballot_w64(id >= at && id < at + mine);
        if (!who) return {0, -1, 0, 0};
        const int r = __builtin_amdgcn_readfirstlane(__builtin_ctzll(who));
        const int32_t first = __builtin_amdgcn_readlane(at, r);
        return {r, id - first, first, __builtin_amdgcn_readlane(mine, r)};
    }
    constexpr int kWaves = kThreads / 64;    // a request a thread
    __shared__ float sums[kWaves];
    __shared__ int32_t counts[kWaves];
    __shared__ Share found;
    const int32_t r = threadIdx.x, n = r < a.d.requests ? seen_tokens(a, r) : 0;
    if (r == 0) found.number = -1;
    const int32_t tokens = tokens_of(sum_of<kWaves>((float)n, sums), a.budget), mine = r < a.d.requests ? shares_of(n, tokens) : 0;
    int32_t all;
    const int32_t at = scan<kWaves>(mine, counts, &all);
    if (id >= at && id < at + mine) found = {r, id - at, at, mine};
    __syncthreads();
    return found;
}

// The list of shares, by one workgroup: `per` requests a thread.
constexpr int kListThreads = 1024;
__global__ void __launch_bounds__(kListThreads) list_shares(Args a) {
    constexpr int kWaves = kListThreads / 64;
    __shared__ float sums[kWaves];
    __shared__ int32_t counts[kWaves];
    const int32_t R = a.d.requests, per = (R + kListThreads - 1) / kListThreads, lo = min(R, (int32_t)threadIdx.x * per), hi = min(R, lo + per);
    float total = 0.0f;
    for (int32_t r = lo; r < hi; ++r) total += (float)seen_tokens(a, r);
    const int32_t tokens = tokens_of(sum_of<kWaves>(total, sums), a.budget);
    int32_t mine = 0, all;
    for (int32_t r = lo; r < hi; ++r) mine += shares_of(seen_tokens(a, r), tokens);
    int32_t at = scan<kWaves>(mine, counts, &all);
    for (int32_t r = lo; r < hi; ++r) {
        const int32_t n = shares_of(seen_tokens(a, r), tokens);
        a.info[r] = make_int2(at, n);
        for (int32_t i = 0; i < n; ++i) a.list[kListHead + at + i] = r;
        at += n;
    }
    if (threadIdx.x == 0) a.list[0] = all;
}

// Four values of an output row: divided by the sum of the weights and rounded once, 0 where there are none.
template <class Q>
__device__ inline void put4(Q* to, f32x4 v, float sum) {
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    typedef Q Q4 __attribute__((ext_vector_type(4)));
    const Q4 x = {(Q)(v[0] * f), (Q)(v[1] * f), (Q)(v[2] * f), (Q)(v[3] * f)};
    *(Q4*)to = x;
}

// The maximum or sum over the 16 lanes of a row, for all of them.
template <int BY>
__device__ inline float rotated(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x120 | BY, 0xF, 0xF, true));
}
__device__ inline float over_lanes_max(float x) {
    x = fmaxf(x, rotated<8>(x));
    x = fmaxf(x, rotated<4>(x));
    x = fmaxf(x, rotated<2>(x));
    return fmaxf(x, rotated<1>(x));
}
__device__ inline float over_lanes_sum(float x) {
    x += rotated<8>(x);
    x += rotated<4>(x);
    x += rotated<2>(x);
    return x + rotated<1>(x);
}

// The maximum or sum over the four rows of 16 lanes.
__device__ inline float over_rows_max(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ inline float over_rows_sum(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

template <class C>
__device__ inline float to_float(uint32_t word, int odd) {
    if constexpr (__is_same(C, __bf16)) return __uint_as_float(odd ? word & 0xFFFF0000u : word << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)(odd ? word >> 16 : word));
}

__device__ inline f32x4 product(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ inline f32x4 product(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ inline f32x4 product(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Two values as `N` terms of a 16-bit type each, whose sums they are but for what the last rounds off: two terms keep 16 (bf16) or
// 22 (fp16) bits, three all 24.  All but the last are cut, so that what is left has their sign.
template <int N>
__device__ inline void terms(float a, float b, uint32_t (&t)[N], __bf16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < N - 1; ++i) {
        t[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
        a -= __uint_as_float(__float_as_uint(a) & 0xFFFF0000u);
        b -= __uint_as_float(__float_as_uint(b) & 0xFFFF0000u);
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

// Tokens of a tile: 32, or 16 where 32 take too many registers.
constexpr int tile_of(int bytes) { return bytes == 2 ? 32 : 16; }

// One share of a sequence, one cache head, up to 16 of its query heads: a workgroup whose wavefronts take tiles of 32 tokens (16
// of a 32-bit cache) in turn, each with a running maximum, sum and output, and join at the end.
//
// Both products are 16x16 MFMAs whose operands come from memory as they lie there, 16 bytes a lane, with no way
// through LDS:  S^T[token][head] = K Q^T, then O^T[dim][head] = V^T P^T.  A product does not care in which order its k runs:
//   K Q^T: lane (row r, quarter g) loads pieces 4s + g of token r; the same pieces of Q are the other operand.
//   V^T P^T: S^T leaves lane (head, g) the tokens 4g..4g+3 of a tile, so these are its k; lane (m, g) loads of each
//   of them the m-th piece, whose e-th values are row m of the e-th product (dim = pieces * m + e).
// So weights stay in the lane that made them, and a head's maximum, sum and rescaling are one value a lane.
// 16-bit caches use 16x16x32 products.  Weights are two terms of the cache's type (a single one would put 2^-9 on bf16 outputs that are
// off by 2^-9 at most from their own rounding); 32-bit queries are three terms, and so are their weights, which keeps all 24
// bits at a fifth of the time of 16x16x4 products on 32-bit values.  Terms of fp16 need room below: queries are scaled by a power of
// two to 2^13 a head (for bf16 those below 2^-100 to that), weights are up to 2^14.  32-bit caches use the 16x16x4 products, but for FEW query heads a cache head, where
// these would be nearly all padding: there the same pieces are multiplied and added by the lanes, a head after the other.
template <class Q, class C, int DP, bool WHOLE, int WAVES, int FEW>
__global__ void __launch_bounds__(WAVES * 64, WAVES == 4 && DP < 256 ? 2 : 1) paged_attention(Args a) {
    constexpr bool kNarrow = sizeof(C) == 2;                  // products in the cache's 16-bit type
    constexpr bool kHalf = __is_same(C, _Float16);
    constexpr int kTermsQ = sizeof(Q) == sizeof(C) ? 1 : 3, kTermsP = sizeof(Q) == 2 ? 2 : 3;
    constexpr float kGrow = kHalf ? 0x1p14f : 1.0f;           // weights are up to that
    constexpr int kPiece = 16 / sizeof(C);                    // values of 16 bytes
    constexpr int kTile = tile_of(sizeof(C)), kSub = kTile / 16;
    constexpr int kSteps = DP / (4 * kPiece);                 // pieces of a key row a lane
    constexpr int kV = DP / 16 < kPiece ? DP / 16 : kPiece;   // values of a value row a lane and slab
    constexpr int kSlabs = DP / (16 * kV), kVWords = kV * sizeof(C) / 4;
    constexpr int kRow = DP + 4;                              // of the join, against bank conflicts

    const reef_paged_attention_desc& d = a.d;
    int32_t id = blockIdx.x;
    if (a.together > 1) {                    // (workgroups go to the 8 XCDs in turn)
        const int32_t eights = id / 8, unit = eights / a.together * 8 + id % 8;
        if (unit >= a.units) return;
        id = unit * a.together + eights % a.together;
    }
    const int tile16 = id % a.tiles;
    id /= a.tiles;
    const int kvh = id % d.cache.kv_heads;
    id /= d.cache.kv_heads;
    Share of = {id, 0, 0, 1};
    if (WAVES == 4 && a.budget) {            // (wide workgroups do not split)
        of = find_share(a, id);
        if (of.number < 0) return;
        if (!a.list && of.number == 0 && kvh == 0 && tile16 == 0 && threadIdx.x == 0) a.info[of.request] = make_int2(of.first, of.count);
    }
    const int32_t r = of.request;
    const int32_t held = held_length(a.lengths[r], d.max_blocks, d.cache.block_size);
    const int32_t first = d.window && held > d.window ? held - d.window : 0;
    int32_t begin = first, end = held;
    if (WAVES == 4 && of.count > 1) {
        begin = first + begin_of(held - first, of.number, of.count);
        if (of.number + 1 < of.count) end = first + begin_of(held - first, of.number + 1, of.count);
    }

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const int D = d.cache.head_dim;
    const int heads = min(16, a.group - tile16 * 16), head0 = kvh * a.group + tile16 * 16;
    const PagedView view{d.cache.blocks, d.cache.block_stride, d.cache.slot_stride};
    const C* keys = (const C*)a.key_cache + kvh * d.cache.head_stride;
    const C* values = (const C*)a.value_cache + kvh * d.cache.head_stride;
    const int32_t* table = a.table + (int64_t)r * d.table_stride;

    __shared__ int64_t offsets[WAVES][2][kTile];
    constexpr int kHeads = FEW ? FEW : 16;
    __shared__ float o_part[WAVES][kHeads][kRow];
    __shared__ float m_part[WAVES][kHeads], l_part[WAVES][kHeads];

    // the table's entry of one token of a tile a lane; -1: no token
    auto entry_of = [&](int32_t t0) -> int32_t {
        const int64_t t = (int64_t)t0 + lane;
        return lane < kTile && t < end ? table[divided((uint32_t)t, a.block)] : -1;
    };
    constexpr int32_t kStride = WAVES * kTile;
    int32_t t0 = first_of(begin, end, wave * kTile);
    // (asked for ahead of the queries: keys and values wait for them)
    int32_t entry = t0 < end ? entry_of(t0) : -1;

    // the queries: head n, the pieces that this lane's keys have
    float scale = d.scale * kLog2e, shrink = 1.0f;           // scores: products * shrink * scale
    u32x4 q[FEW ? 1 : kTermsQ][FEW ? 1 : kSteps];
    float fq[FEW ? FEW : 1][kSteps][4];
    if constexpr (FEW) {                      // (for each head)
#pragma unroll
        for (int h = 0; h < FEW; ++h)
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int at = (s * 4 + g) * kPiece;
                f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
                if (h < heads && at < D) v = *(const f32x4*)((const float*)a.query + r * d.query_stride + (head0 + h) * d.query_head_stride + at);
#pragma unroll
                for (int e = 0; e < 4; ++e) fq[h][s][e] = v[e];
            }
    } else {
        const Q* query = (const Q*)a.query + r * d.query_stride + (head0 + n) * d.query_head_stride;
        constexpr int kWords = kPiece * sizeof(Q) / 4;
        uint32_t raw[kSteps][kWords];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int at = (s * 4 + g) * kPiece;
#pragma unroll
            for (int w = 0; w < kWords; w += 4) {
                u32x4 v = {0, 0, 0, 0};
                if (n < heads && at < D) v = *(const u32x4*)(query + at + w * 4 / sizeof(Q));
#pragma unroll
                for (int i = 0; i < 4; ++i) raw[s][w + i] = v[i];
            }
        }
        if constexpr (kTermsQ == 1) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) q[0][s] = {raw[s][0], raw[s][1], raw[s][2], raw[s][3]};
        } else {
            float grow = 1.0f, top = 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
#pragma unroll
                for (int w = 0; w < kWords; ++w) top = fmaxf(top, fabsf(__uint_as_float(raw[s][w])));
            top = over_rows_max(top);
            if (top > 0.0f && top < INFINITY) {
                // (-114 .. 126, so both factors are normal numbers; bf16 lacks room below 2^-133 only, and keys may be 2^127)
                const int power = (int)(__float_as_uint(top) >> 23) - 127, by = kHalf ? min(126, 13 - power) : max(0, -100 - power);
                grow = __uint_as_float((uint32_t)(127 + by) << 23);
                const float back = __uint_as_float((uint32_t)(127 - by) << 23);
                // One factor where it is one: large queries and a large scale may pass 32 bits together where a product is 0.
                if (back > 1.0f && fabsf(scale) > 1.0f) shrink = back;
                else scale *= back;
            }
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t t[kTermsQ];
                    terms(__uint_as_float(raw[s][2 * w]) * grow, __uint_as_float(raw[s][2 * w + 1]) * grow, t, C());
#pragma unroll
                    for (int x = 0; x < kTermsQ; ++x) q[x][s][w] = t[x];
                }
        }
    }

    float m = -INFINITY, l = 0.0f;
    f32x4 o[FEW ? 1 : kSlabs][FEW ? 1 : kV];
    float fm[FEW ? FEW : 1], fl[FEW ? FEW : 1], fo[FEW ? FEW : 1][kSlabs][kV];   // FEW: of each head; fo over this row's tokens
#pragma unroll
    for (int s = 0; s < (FEW ? 1 : kSlabs); ++s)
#pragma unroll
        for (int e = 0; e < (FEW ? 1 : kV); ++e) o[s][e] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int h = 0; h < (FEW ? FEW : 1); ++h) {
        fm[h] = -INFINITY;
        fl[h] = 0.0f;
#pragma unroll
        for (int c = 0; c < kSlabs; ++c)
#pragma unroll
            for (int e = 0; e < kV; ++e) fo[h][c][e] = 0.0f;
    }

    // that token's place, for all lanes to read; which of the tile's tokens there are
    auto place = [&](int32_t t0, int32_t entry, int buffer) -> uint32_t {
        int64_t at = -1;
        if (lane < kTile) {
            const uint32_t t = (uint32_t)t0 + lane;
            at = paged_row(view, entry, (int32_t)(t - divided(t, a.block) * a.block.by));
            offsets[wave][buffer][lane] = at < 0 ? 0 : at;
        }
        return (uint32_t)__builtin_amdgcn_ballot_w64(at >= 0);
    };
    u32x4 k[kSub][kSteps];
    uint32_t v[kSub][4][kSlabs][kVWords];
    auto load_k = [&](int buffer) {
#pragma unroll
        for (int t = 0; t < kSub; ++t) {
            const C* row = keys + offsets[wave][buffer][t * 16 + n];
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int at = (s * 4 + g) * kPiece;
                k[t][s] = *(const u32x4*)(row + (WHOLE || at < D ? at : 0));
            }
        }
    };
    auto load_v = [&](int buffer) {
#pragma unroll
        for (int t = 0; t < kSub; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const C* row = values + offsets[wave][buffer][t * 16 + g * 4 + i];
#pragma unroll
                for (int s = 0; s < kSlabs; ++s) {
                    const int at = (s * 16 + n) * kV;
                    const C* p = row + (WHOLE || at < D ? at : 0);
                    if constexpr (kVWords == 4) {
                        const u32x4 x = *(const u32x4*)p;
#pragma unroll
                        for (int w = 0; w < 4; ++w) v[t][i][s][w] = x[w];
                    } else {
                        const u32x2 x = *(const u32x2*)p;
                        v[t][i][s][0] = x[0];
                        v[t][i][s][1] = x[1];
                    }
                }
            }
    };

    uint32_t there = 0, there_next = 0;
    int buffer = 0;
    if (t0 < end) {
        there = place(t0, entry, 0);
        entry = t0 < end - kStride ? entry_of(t0 + kStride) : -1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        load_k(0);
        load_v(0);
    }
    while (t0 < end) {
        const bool more = t0 < end - kStride;
        if (more) {
            there_next = place(t0 + kStride, entry, buffer ^ 1);
            entry = t0 < end - 2 * kStride ? entry_of(t0 + 2 * kStride) : -1;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        const bool all = there == (kTile == 32 ? 0xFFFFFFFFu : 0xFFFFu);
        if constexpr (FEW) {
            // scores: token n of each 16, the same in all rows
            float p[FEW][kSub];
#pragma unroll
            for (int t = 0; t < kSub; ++t)
#pragma unroll
                for (int h = 0; h < FEW; ++h) {
                    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int c = 0; c < kSteps; ++c)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (WHOLE || (c * 4 + g) * kPiece < D) x[e] = fmaf(__uint_as_float(k[t][c][e]), fq[h][c][e], x[e]);
                    p[h][t] = over_rows_sum((x[0] + x[1]) + (x[2] + x[3])) * scale;
                    if (!all && !(there >> (t * 16 + n) & 1)) p[h][t] = -INFINITY;
                }
            if (more) load_k(buffer ^ 1);
#pragma unroll
            for (int h = 0; h < FEW; ++h) {
                static_assert(kSub == 1, "32-bit caches have tiles of 16 tokens");
                const float top = fmaxf(over_lanes_max(p[h][0]), fm[h]);
                const float base = top == -INFINITY ? 0.0f : top, f = __builtin_amdgcn_exp2f(fm[h] - base);
                fm[h] = top;
                fl[h] *= f;
#pragma unroll
                for (int c = 0; c < kSlabs; ++c)
#pragma unroll
                    for (int e = 0; e < kV; ++e) fo[h][c][e] *= f;
#pragma unroll
                for (int t = 0; t < kSub; ++t) {
                    p[h][t] = __builtin_amdgcn_exp2f(p[h][t] - base);
                    fl[h] += p[h][t];
                }
            }
            // values of places that are no tokens may be anything, and 0 times that too
            if (!all) {
#pragma unroll
                for (int t = 0; t < kSub; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!(there >> (t * 16 + g * 4 + i) & 1)) {
#pragma unroll
                            for (int c = 0; c < kSlabs; ++c)
#pragma unroll
                                for (int w = 0; w < kVWords; ++w) v[t][i][c][w] = 0;
                        }
            }
#pragma unroll
            for (int t = 0; t < kSub; ++t)
#pragma unroll
                for (int h = 0; h < FEW; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float w = __shfl(p[h][t], g * 4 + i);
#pragma unroll
                        for (int c = 0; c < kSlabs; ++c)
#pragma unroll
                            for (int e = 0; e < kV; ++e) fo[h][c][e] = fmaf(__uint_as_float(v[t][i][c][e]), w, fo[h][c][e]);
                    }
        } else {
            // scores
            f32x4 s[kSub];
#pragma unroll
            for (int t = 0; t < kSub; ++t) s[t] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < kSteps; ++c)
#pragma unroll
                for (int t = 0; t < kSub; ++t) {
                    u32x4 kk = k[t][c];
                    if constexpr (!WHOLE)
                        if ((c * 4 + g) * kPiece >= D) kk = {0, 0, 0, 0};
                    if constexpr (kNarrow) {
                        typedef C C8 __attribute__((ext_vector_type(8)));
#pragma unroll
                        for (int x = kTermsQ - 1; x >= 0; --x) s[t] = product(__builtin_bit_cast(C8, kk), __builtin_bit_cast(C8, q[x][c]), s[t]);
                    } else {
#pragma unroll
                        for (int e = 0; e < kPiece; ++e) s[t] = product(__uint_as_float(kk[e]), __uint_as_float(q[0][c][e]), s[t]);
                    }
                }
            if constexpr (kTermsQ > 1) {
                // An infinite key times a term that is 0 or of the other sign: the sum is made again on 32-bit values, as it is written.
                bool odd = false;
#pragma unroll
                for (int t = 0; t < kSub; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) odd |= s[t][i] != s[t][i];
                if (__builtin_amdgcn_ballot_w64(odd)) {
#pragma unroll
                    for (int t = 0; t < kSub; ++t) s[t] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int c = 0; c < kSteps; ++c)
#pragma unroll
                        for (int e = 0; e < kPiece; ++e) {
                            float x = 0.0f;
#pragma unroll
                            for (int i = kTermsQ - 1; i >= 0; --i) {
                                uint32_t y = q[i][c][e / 2];
                                asm volatile("" : "+v"(y));       // (or the sums are made ahead of the loop, and held in registers for it)
                                x += to_float<C>(y, e & 1);
                            }
#pragma unroll
                            for (int t = 0; t < kSub; ++t) {
                                const bool inside = WHOLE || (c * 4 + g) * kPiece < D;
                                s[t] = product(inside ? to_float<C>(k[t][c][e / 2], e & 1) : 0.0f, x, s[t]);
                            }
                        }
                }
            }
            if (more) load_k(buffer ^ 1);
            // weights
            float top = m;
#pragma unroll
            for (int t = 0; t < kSub; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (kHalf && kTermsQ > 1) s[t][i] *= shrink;
                    s[t][i] *= scale;
                    if (!all && !(there >> (t * 16 + g * 4 + i) & 1)) s[t][i] = -INFINITY;
                    top = fmaxf(top, s[t][i]);
                }
            top = over_rows_max(top);
            const float base = top == -INFINITY ? 0.0f : top;
            if (__builtin_amdgcn_ballot_w64(top != m)) {
                const float f = __builtin_amdgcn_exp2f(m - base);
                l *= f;
#pragma unroll
                for (int c = 0; c < kSlabs; ++c)
#pragma unroll
                    for (int e = 0; e < kV; ++e) o[c][e] *= f;
            }
            m = top;
#pragma unroll
            for (int t = 0; t < kSub; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[t][i] = __builtin_amdgcn_exp2f(s[t][i] - base);
                    if constexpr (kHalf) s[t][i] *= kGrow;    // (not by the exponent: base - 14 would be rounded where scores are large)
                    l += s[t][i];
                }
            // values of places that are no tokens may be anything, and 0 times that too
            if (!all) {
#pragma unroll
                for (int t = 0; t < kSub; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!(there >> (t * 16 + g * 4 + i) & 1)) {
#pragma unroll
                            for (int c = 0; c < kSlabs; ++c)
#pragma unroll
                                for (int w = 0; w < kVWords; ++w) v[t][i][c][w] = 0;
                        }
            }
            if constexpr (kNarrow) {
                typedef C C8 __attribute__((ext_vector_type(8)));
                u32x4 p[kTermsP];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t x[kTermsP];
                    terms(s[w >> 1][(w & 1) * 2], s[w >> 1][(w & 1) * 2 + 1], x, C());
#pragma unroll
                    for (int i = 0; i < kTermsP; ++i) p[i][w] = x[i];
                }
#pragma unroll
                for (int c = 0; c < kSlabs; ++c)
#pragma unroll
                    for (int e = 0; e < kV; ++e) {
                        u32x4 x;
#pragma unroll
                        for (int w = 0; w < 4; ++w)
                            x[w] = __builtin_amdgcn_perm(v[w >> 1][(w & 1) * 2 + 1][c][e / 2], v[w >> 1][(w & 1) * 2][c][e / 2], e & 1 ? 0x07060302 : 0x05040100);
#pragma unroll
                        for (int i = kTermsP - 1; i >= 0; --i) o[c][e] = product(__builtin_bit_cast(C8, x), __builtin_bit_cast(C8, p[i]), o[c][e]);
                    }
            } else {
#pragma unroll
                for (int t = 0; t < kSub; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int c = 0; c < kSlabs; ++c)
#pragma unroll
                            for (int e = 0; e < kV; ++e)
                                o[c][e] = product(__uint_as_float(v[t][i][c][e]), s[t][i], o[c][e]);
            }
        }
        if (more) load_v(buffer ^ 1);
        there = there_next;
        buffer ^= 1;
        if (!more) break;
        t0 += kStride;
    }

    // the wavefronts' parts
    if constexpr (FEW) {
#pragma unroll
        for (int h = 0; h < FEW; ++h) {
#pragma unroll
            for (int c = 0; c < kSlabs; ++c) {
                f32x4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = over_rows_sum(fo[h][c][e]);
                if (g == 0) *(f32x4*)&o_part[wave][h][(c * 16 + n) * kV] = x;
            }
            const float sum = over_lanes_sum(fl[h]);
            if (lane == 0) {
                m_part[wave][h] = fm[h];
                l_part[wave][h] = sum;
            }
        }
    } else {
        l = over_rows_sum(l) * (1.0f / kGrow);
        if (n < heads) {
#pragma unroll
            for (int c = 0; c < kSlabs; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < kV; e += 4) {
                        f32x4 x = {o[c][e][i], o[c][e + 1][i], o[c][e + 2][i], o[c][e + 3][i]};
                        if constexpr (kHalf) x *= 1.0f / kGrow;
                        *(f32x4*)&o_part[wave][n][(c * 16 + g * 4 + i) * kV + e] = x;
                    }
            if (g == 0) {
                m_part[wave][n] = m;
                l_part[wave][n] = l;
            }
        }
    }
    __syncthreads();
    const int quads = D / 4;
    for (int x = threadIdx.x; x < heads * quads; x += WAVES * 64) {
        const int h = x / quads, at = (x - h * quads) * 4;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, m_part[w][h]);
        const float base = top == -INFINITY ? 0.0f : top;
        f32x4 all = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f(m_part[w][h] - base);
            sum += f * l_part[w][h];
            all += f * *(const f32x4*)&o_part[w][h][at];
        }
        if (of.count > 1) {
            const int64_t row = (int64_t)(of.first + of.number) * d.heads + head0 + h;
            *(f32x4*)(a.parts + row * D + at) = all;
            if (at == 0) a.stats[row] = make_float2(top, sum);
        } else {
            put4((Q*)a.out + r * d.out_stride + (head0 + h) * d.out_head_stride + at, all, sum);
            if (at == 0 && a.lse) a.lse[(int64_t)r * d.heads + head0 + h] = sum == 0.0f ? -INFINITY : (top + __log2f(sum)) * kLn2;
        }
    }
}

// The shares of a sequence of one query head: a workgroup, lanes over quads of the head, groups of them over the shares.  `heads_each`
// heads one after the other: most requests of a large batch are not split, and their workgroups only find that out.
template <class Q>
__global__ void __launch_bounds__(kThreads) join_shares(Args a) {
    constexpr int kWaves = kThreads / 64;
    const reef_paged_attention_desc& d = a.d;
    const int blocks = (d.heads + a.heads_each - 1) / a.heads_each, r = blockIdx.x / blocks, D = d.cache.head_dim;
    const int2 of = a.info[r];
    if (of.y <= 1) return;
    __shared__ float weight[kFiner * kGroups + 2];
    __shared__ float red[2][kWaves];
    __shared__ f32x4 sums[kThreads];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h1 = min(d.heads, ((int)blockIdx.x % blocks + 1) * a.heads_each);
    for (int h = (int)blockIdx.x % blocks * a.heads_each; h < h1; ++h) {
        const float2* stats = a.stats + (int64_t)of.x * d.heads + h;
        const float* parts = a.parts + ((int64_t)of.x * d.heads + h) * D;
        const int64_t step = (int64_t)d.heads * D;
        const int quads = D / 4, groups = kThreads / quads, mine = tid / quads, at = (tid - mine * quads) * 4;
        constexpr int kAhead = 4;                // of a group's parts, on their way while the weights are made
        f32x4 ahead[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int s = mine + u * groups;
            ahead[u] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (mine < groups && s < of.y) ahead[u] = *(const f32x4*)(parts + s * step + at);
        }
        float m = -INFINITY, l = 0.0f;
        for (int s = tid; s < of.y; s += kThreads) m = fmaxf(m, stats[(int64_t)s * d.heads].x);
        for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
        if (lane == 0) red[0][wave] = m;
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, red[0][w]);
        const float base = m == -INFINITY ? 0.0f : m;
        for (int s = tid; s < of.y; s += kThreads) {
            const float2 x = stats[(int64_t)s * d.heads];
            weight[s] = __builtin_amdgcn_exp2f(x.x - base);
            l += weight[s] * x.y;
        }
        for (int x = 32; x; x >>= 1) l += __shfl_xor(l, x);
        if (lane == 0) red[1][wave] = l;
        __syncthreads();
        l = 0.0f;
        for (int w = 0; w < kWaves; ++w) l += red[1][w];
        f32x4 all = {0.0f, 0.0f, 0.0f, 0.0f};
        if (mine < groups) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (mine + u * groups < of.y) all += weight[mine + u * groups] * ahead[u];
#pragma unroll 4
            for (int s = mine + kAhead * groups; s < of.y; s += groups) all += weight[s] * *(const f32x4*)(parts + s * step + at);
        }
        sums[tid] = all;
        __syncthreads();
        if (!mine) {
            for (int x = 1; x < groups; ++x) all += sums[x * quads + tid];
            put4((Q*)a.out + r * d.out_stride + h * d.out_head_stride + at, all, l);
            if (tid == 0 && a.lse) a.lse[(int64_t)r * d.heads + h] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2;
        }
        __syncthreads();                         // (the next head's weights and sums go where these are)
    }
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
    if (!std::isfinite(d->scale * kLog2e)) return refuse(what, "scale %g is not a finite number, or not one as a power of two", (double)d->scale);
    const int bytes = type_bytes(d->type);
    if (!stride16(d->requests, d->query_stride, bytes) || !stride16(d->requests, d->out_stride, bytes) || !stride16(d->heads, d->query_head_stride, bytes) ||
        !stride16(d->heads, d->out_head_stride, bytes))
        return refuse(what, "strides of query or out are not multiples of 16 bytes");
    // rows of out: heads inside requests or requests inside heads, none over another
    const bool heads_first = d->requests <= 1 || (d->heads > 1 && d->out_head_stride <= d->out_stride);
    const int64_t count[2] = {heads_first ? d->heads : d->requests, heads_first ? d->requests : d->heads};
    const int64_t stride[2] = {heads_first ? d->out_head_stride : d->out_stride, heads_first ? d->out_stride : d->out_head_stride};
    __int128 extent = d->cache.head_dim;
    for (int i = 0; i < 2; ++i) {
        if (count[i] <= 1) continue;
        if (stride[i] < extent) return refuse(what, "a stride of %lld elements lets rows of out overlap", (long long)stride[i]);
        extent += (__int128)stride[i] * (count[i] - 1);
    }
    return 0;
}

// How a call is laid out.
struct Plan {
    int32_t tiles, budget;
    bool wide;              // workgroups of more wavefronts
    int64_t groups;         // workgroups
    int32_t units, together;
    size_t info_bytes, list_bytes, stats_bytes, bytes;
};
// Wavefronts of a wide workgroup: as many as the registers allow a CU; with matrix products for heads over 128 those of any.
constexpr int wide_waves(int dp, bool terms, int few) {
    return dp <= 64 && !terms && few <= 1 ? 16 : dp <= 128 ? 8 : 4;
}
// Whether lanes do the work of the matrix instructions: 32-bit caches, query heads a cache head up to 4 for heads up to 64, 2 for heads up to 128.
constexpr int few_of(bool narrow, int dp, int group) {
    return narrow || dp > 128 ? 0 : group <= 2 ? group : group <= 4 && dp <= 64 ? 4 : 0;
}
Plan plan_of(const reef_paged_attention_desc& d) {
    const int32_t group = d.heads / d.cache.kv_heads, tiles = (group + 15) / 16, rows = d.cache.kv_heads * tiles;
    int64_t longest = (int64_t)d.max_blocks * d.cache.block_size;
    if (d.longest && d.longest < longest) longest = d.longest;
    if (d.window && d.window < longest) longest = d.window;
    const int64_t all = (int64_t)d.requests * rows;
    const int D = d.cache.head_dim, few = few_of(d.cache.type != REEF_TYPE_F32, D, group), tile = tile_of(type_bytes(d.cache.type)),
              wide = wide_waves(D, d.type != d.cache.type, few);
    Plan p{};
    p.tiles = tiles;
    // Whole sequences where a wide workgroup takes the longest in few rounds.  3 / 4 / 5 rounds against shares, heads of 128, bf16: 48 heads in all
    // 12 / 15 / 17 us against 13 / 14 / 15 (11 / 13 / 16 against 11 where that is the longest), 256 heads 18 / 24 / 33 against 25 / 30 / 39 (12 / 15 / 17
    // against 13 / 16 / 17).  Eight wavefronts for heads up to 64 have short rounds: 32-bit queries over bf16, 48 heads, 9 / 10 / 12 against 12 / 12 / 13,
    // 32-bit caches of 4 query heads, 20 heads, 9 / 11 / 12 (6 rounds: 14) against 12.  (Between 48 and 256 heads nothing was measured.)
    const int rounds = all >= 192 || (wide == 8 && D <= 64) ? 5 : 3;
    p.wide = all < kGroups && longest <= (int64_t)rounds * wide * tile;
    p.groups = all;
    // The tiles of a cache head, which read the same, go to one XCD and meet in its L2 (32 query heads a cache head, 4 x 30000 tokens: 45 -> 35 us), and
    // so do the heads of a share where rows end inside lines, if there are shares enough for all XCDs (heads of 80, bf16, 64 x 1000 tokens: 46 -> 39).
    auto spread = [&](int64_t shares) {
        const bool lines = d.cache.head_stride < d.cache.slot_stride && d.cache.head_stride * type_bytes(d.cache.type) % 128 != 0;
        p.together = lines && shares >= 32 ? rows : tiles;
        const int64_t units = p.groups / p.together;
        p.units = (int32_t)std::min<int64_t>(units, INT32_MAX);
        if (p.together > 1) p.groups = (units + 7) / 8 * 8 * p.together;
    };
    if (p.wide || longest <= 4 * 4 * tile) {
        spread(d.requests);
        return p;
    }
    const bool finer = all >= kGroups * 7 / 8 && longest >= 4096;     // (90 sequences of up to 1500 tokens: 29 us, 30 with twice as many)
    p.budget = std::max(1, (D > 128 ? kGroups / 2 : kGroups) * (finer ? kFiner : 1) / rows);
    const int64_t shares = (int64_t)p.budget + d.requests;
    p.groups = shares * rows;
    spread(shares);
    p.info_bytes = ((size_t)d.requests * 8 + 15) / 16 * 16;
    p.stats_bytes = ((size_t)shares * d.heads * 8 + 15) / 16 * 16;
    if (d.requests > kFewRequests) p.list_bytes = ((size_t)(kListHead + shares) * 4 + 15) / 16 * 16;
    p.bytes = p.info_bytes + p.list_bytes + p.stats_bytes + (size_t)shares * d.heads * D * 4;
    return p;
}

template <class Q, class C, int DP, bool WHOLE, int FEW>
int run_waves(const char* what, const Args& a, const Plan& p, void* stream) {
    constexpr int kWide = wide_waves(DP, sizeof(Q) != sizeof(C), FEW);
    const dim3 grid((unsigned)p.groups);
    if (p.wide && kWide > 4) return launch(what, paged_attention<Q, C, DP, WHOLE, kWide, FEW>, grid, dim3(kWide * 64), a, stream);
    return launch(what, paged_attention<Q, C, DP, WHOLE, 4, FEW>, grid, dim3(kThreads), a, stream);
}

template <class Q, class C, int DP, bool WHOLE>
int run_heads(const char* what, const Args& a, const Plan& p, void* stream) {
    if constexpr (sizeof(C) == 4) {
        const int few = few_of(false, DP, a.group);
        if constexpr (DP <= 128) {
            if (few == 1) return run_waves<Q, C, DP, WHOLE, 1>(what, a, p, stream);
            if (few == 2) return run_waves<Q, C, DP, WHOLE, 2>(what, a, p, stream);
        }
        if constexpr (DP <= 64)
            if (few == 4) return run_waves<Q, C, DP, WHOLE, 4>(what, a, p, stream);
    }
    return run_waves<Q, C, DP, WHOLE, 0>(what, a, p, stream);
}

template <class Q, class C>
int run(const char* what, const Args& a, const Plan& p, void* stream) {
    const int D = a.d.cache.head_dim;
    if (a.list)
        if (int rc = launch(what, list_shares, dim3(1), dim3(kListThreads), a, stream)) return rc;
    const int rc = D == 64    ? run_heads<Q, C, 64, true>(what, a, p, stream)
                   : D < 64   ? run_heads<Q, C, 64, false>(what, a, p, stream)
                   : D == 128 ? run_heads<Q, C, 128, true>(what, a, p, stream)
                   : D < 128  ? run_heads<Q, C, 128, false>(what, a, p, stream)
                   : D == 256 ? run_heads<Q, C, 256, true>(what, a, p, stream)
                              : run_heads<Q, C, 256, false>(what, a, p, stream);
    if (rc || !p.budget) return rc;
    return launch(what, join_shares<Q>, dim3((unsigned)(a.d.requests * ((a.d.heads + a.heads_each - 1) / a.heads_each))), dim3(kThreads), a, stream);
}

}  // namespace

extern "C" int64_t reef_ops_paged_attention_workspace(const reef_paged_attention_desc* d) {
    if (check("reef_ops_paged_attention_workspace", d)) return -1;
    return (int64_t)plan_of(*d).bytes;
}

extern "C" int reef_ops_paged_attention(const reef_paged_attention_desc* d, const void* query, const void* key_cache, const void* value_cache,
                                        const int32_t* table, const int32_t* lengths, void* out, float* lse, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
    const char* what = "reef_ops_paged_attention";
    if (int rc = check(what, d)) return rc;
    if (!d->requests) return 0;
    if (!rows16(query) || !rows16(key_cache) || !rows16(value_cache) || !rows16(out) || !words(table) || !words(lengths) || !aligned(lse, 4))
        return refuse(what, "null or unaligned argument");
    const Plan p = plan_of(*d);
    // (2^32 threads are refused by the launch, which may be the call's second one)
    if (p.groups >= 1ll << 24) return refuse(what, "%lld workgroups are too many", (long long)p.groups);
    if (p.bytes && (!rows16(workspace) || workspace_bytes < (int64_t)p.bytes))
        return refuse(what, "a workspace of %zu bytes on 16 is needed, %lld are given", p.bytes, (long long)workspace_bytes);
    char* w = (char*)workspace;
    const size_t list = p.info_bytes, stats = list + p.list_bytes, parts = stats + p.stats_bytes;
    const Args a{*d, query, key_cache, value_cache, table, lengths, out, lse, (float*)(w + parts), (float2*)(w + stats), (int2*)w,
                 p.list_bytes ? (int32_t*)(w + list) : nullptr, d->heads / d->cache.kv_heads, p.tiles, p.budget, divider((uint32_t)d->cache.block_size),
                 d->requests > kFewRequests ? std::min(d->heads, 8) : 1, p.units, p.together};
    switch (d->type * 4 + d->cache.type) {
        case REEF_TYPE_F32 * 4 + REEF_TYPE_F32: return run<float, float>(what, a, p, stream);
        case REEF_TYPE_F32 * 4 + REEF_TYPE_F16: return run<float, _Float16>(what, a, p, stream);
        case REEF_TYPE_F32 * 4 + REEF_TYPE_BF16: return run<float, __bf16>(what, a, p, stream);
        case REEF_TYPE_F16 * 4 + REEF_TYPE_F16: return run<_Float16, _Float16>(what, a, p, stream);
        default: return run<__bf16, __bf16>(what, a, p, stream);
    }
}
