// Log probabilities of given tokens, their ranks, the entropy and the best alternatives (reef_ops_token_scores).
#include <algorithm>
#include <type_traits>

#include "ops_common.h"

namespace {
using namespace reef_ops;

constexpr int kMaxTop = 128;
constexpr float kLog2e = 1.4426950408889634f;

constexpr int kGroups = 1024;                // maxima of groups that are held
// Groups of neighbours: 2^bits lanes' 16 bytes of the units that a wavefront reads at once (a batch), and of `per` batches where there are more than 256.
struct Groups {
    int32_t batches, per, bits, groups;
};
Groups groups_of(int32_t units, int32_t loads) {
    Groups g{(units + loads - 1) / loads, 1, 0, 0};
    while (g.bits < 4 && g.batches * 64 > kGroups << g.bits) ++g.bits;
    g.per = (g.batches + kGroups / 4 - 1) / (kGroups / 4);
    g.groups = (g.batches + g.per - 1) / g.per * (64 >> g.bits);
    return g;
}
struct Args {
    reef_token_scores_desc d;
    const void* logits;
    const int32_t* tokens;
    float* scores;
    int32_t* ranks;
    float* entropy;
    int32_t* top_tokens;
    float* top_scores;
    struct Part* parts;     // [row][slice]
    uint32_t* maxima;       // [row][groups]
    int32_t slices, slice_units;
    Groups by;
    int32_t loads;
};
// What a part of a row comes to: its maximum, the sums relative to it, values that come before the given token.
struct Part {
    double s, near;
    float m;
    int32_t rank;
};

// A NaN counts as -infinity.
__device__ inline float cleaned(float v) { return v == v ? v : -INFINITY; }
// Whole numbers that are ordered as values are (-0 as 0), and with a token behind them, the lower first.
__device__ inline uint32_t order_of(float v) {
    const uint32_t bits = __float_as_uint(v + 0.0f);
    return bits >> 31 ? ~bits : bits | 1u << 31;
}
__device__ inline float value_of(uint32_t order) { return __uint_as_float(order >> 31 ? order & ~(1u << 31) : ~order); }
__device__ inline uint64_t key_of(uint32_t order, int32_t token) { return (uint64_t)order << 32 | (uint32_t)~token; }

// v - m, or what has an exponential of 0 all the same where that is below, or is an infinity less itself.
__device__ inline float less(float v, float m) { return fmaxf(v - m, -1000.0f); }
// Exponentials relative to m are 2^(v c - M), c = log2 e and M = m c of 32 bits each, so that one rounding makes the exponent: larger by
// 2^(m c - M) than they should be, which is taken off at the end.  Where M is so large that this could be much they are 2^((v - m) c).
__device__ inline bool plain(float M) { return fabsf(M) < 0x1p20f; }
__device__ inline float exponent(float v, float m, float M) { return plain(M) ? fmaxf(fmaf(v, kLog2e, -M), -1000.0f) : less(v, m) * kLog2e; }
__device__ inline float excess(float m, float M) { return plain(M) ? fmaf(m, kLog2e, -M) : 0.0f; }
// By which power of two sums relative to m0 are to be multiplied to be such relative to m1 >= m0.
__device__ inline float step(float m0, float m1) {
    const float M0 = m0 * kLog2e, M1 = m1 * kLog2e;
    return plain(M0) && plain(M1) ? fmaxf(M0 - M1, -1000.0f) : less(m0, m1) * kLog2e + excess(m1, M1) - excess(m0, M0);
}
// A signalling NaN as a quiet one, which maxima pass over.
__device__ inline float quiet(float v) {
    float x;
    asm("v_max_f32 %0, %1, %1" : "=v"(x) : "v"(v));
    return x;
}
// The largest of three, of which none signals.
__device__ inline float largest(float a, float b, float c) {
    float x;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(x) : "v"(a), "v"(b), "v"(c));
    return x;
}

// Sums and maxima over lanes without LDS: rows of 16 turned by 8, 4, 2, 1 lanes, then halves of halves and halves exchanged.
template <int CONTROL, class V>
__device__ inline V moved(V x) {
    uint32_t w[sizeof(V) / 4];
    __builtin_memcpy(w, &x, sizeof(V));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(V) / 4); ++i) w[i] = __builtin_amdgcn_update_dpp(0, w[i], CONTROL, 0xF, 0xF, true);
    __builtin_memcpy(&x, w, sizeof(V));
    return x;
}
template <bool HALVES, class V>
__device__ inline V swapped(V x) {
    uint32_t w[sizeof(V) / 4];
    __builtin_memcpy(w, &x, sizeof(V));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(V) / 4); ++i) {
        const auto y = HALVES ? __builtin_amdgcn_permlane32_swap(w[i], w[i], false, false) : __builtin_amdgcn_permlane16_swap(w[i], w[i], false, false);
        // one of the two is this lane's own: the other's
        w[i] = (threadIdx.x & (HALVES ? 32 : 16)) ? y[0] : y[1];
    }
    __builtin_memcpy(&x, w, sizeof(V));
    return x;
}
// lane i ^ 1; i ^ 2; 7 - i of eight, where fours have the same; i - 8 of sixteen
constexpr int kOne = 0xB1, kTwo = 0x4E, kFour = 0x141, kEight = 0x128;
template <class V, class Join>
__device__ inline V over_wave(V x, Join join) {
    x = join(x, moved<kOne>(x));
    x = join(x, moved<kTwo>(x));
    x = join(x, moved<kFour>(x));
    x = join(x, moved<kEight>(x));
    x = join(x, swapped<false>(x));
    return join(x, swapped<true>(x));
}
struct Max {
    __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Sum {
    template <class V>
    __device__ V operator()(V a, V b) const { return a + b; }
};

// What stands behind a row's end, and how far above it a lane's largest has to be for its exponential to be 0: 1000 powers of two.
constexpr float kBehind = -0x1p18f, kAbove = 1024.0f;        // (plain)
constexpr int kHeld = 2048;                  // candidates that are held

// A row a workgroup, read once: a lane keeps its 16 bytes of a batch of units, their maximum m and sums relative to the largest so far; how many values come
// before the given token is counted by the wavefront.  Exponentials are those of 32 bits, off by 2^-23 of themselves; those of 16 bytes are
// added in 32 bits, up to seven roundings, and everything else in 64.
//
// The lanes' operations are nearly as long as the reads (1000 rows of 128257, bf16, without the best tokens: 62 us, 4.1 TB/s), so nothing is cleaned
// ahead: maxima pass over a NaN, and the bound that makes exponents no less than -1000 is what a NaN and -infinity come to.  A batch with +infinity, or with
// a maximum so large that M is not plain, is read again and taken with care.
//
// The best tokens: of the maxima of groups of neighbours (up to 16 lanes of a batch), held near, as many as wanted reach a bound that is
// found by halving; only groups that reach it are read again.  Their values that reach it are candidates.  Where there are more than are held (values that ascend with their
// numbers, many alike) the bound is raised by halving again, down to one value, and of the tokens that have it the first ones are taken in order.
//
// Few long rows are read in slices by as many workgroups, and looked at by one each in a second launch.
enum { kWhole, kSlice, kJoin };
// LOADS: of a wavefront in flight, 1 KiB each, a unit.
template <class T, int WAVES, int LOADS, int STAGE>
__global__ void __launch_bounds__(WAVES * 64) token_scores(Args a) {
    constexpr int kLoads = LOADS, kThreads = WAVES * 64, kE = 16 / sizeof(T), kUnit = 64 * kE, kMine = kGroups / 64, kLoadBits = __builtin_ctz(LOADS);
    constexpr int kShift = sizeof(T) == 4 ? 0 : __is_same(T, _Float16) ? 13 : 16;
    typedef T Raw __attribute__((ext_vector_type(kE), aligned(sizeof(T))));
    const reef_token_scores_desc& d = a.d;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = STAGE == kSlice ? blockIdx.x / (uint32_t)a.slices : blockIdx.x;
    const T* x = (const T*)a.logits + row * d.logits_stride;
    const int32_t units = (d.vocab + kUnit - 1) / kUnit;
    const int32_t per = a.by.per, bits = a.by.bits, wide = 1 << bits, in_batch = 64 >> bits, groups = a.by.groups;

    __shared__ uint32_t maxima[kGroups];
    __shared__ uint64_t held[kHeld];
    __shared__ double sums[2][WAVES];
    __shared__ float tops[WAVES];
    __shared__ int32_t counts[2][WAVES], n_held;
    __shared__ uint16_t chosen[WAVES][64];

    const int32_t t = a.tokens[row];
    const bool given = (uint32_t)t < (uint32_t)d.vocab;
    const float mine = given ? cleaned((float)x[t]) : INFINITY;
    const int32_t slice = STAGE == kSlice ? (int32_t)(blockIdx.x - row * a.slices) : 0, first_unit = slice * a.slice_units;
    const int32_t end_unit = STAGE == kSlice ? min(units, first_unit + a.slice_units) : STAGE == kJoin ? 0 : units;
    if (STAGE != kJoin && d.top && per > 1) {
        for (int i = tid; i < groups; i += kThreads) maxima[i] = 0;
        __syncthreads();
    }
    float m = -INFINITY;
    double s = 0.0, near = 0.0;
    int32_t rank = 0;
    // (as a NaN comes after all values but -infinity, and with -infinity by its number)
    const bool lowest = mine == -INFINITY;
    const float mine_before = lowest ? NAN : mine;
    // 16 bytes from value i of the row on, and what is behind its end
    auto fetch = [&](int32_t i, float (&v)[kE], float behind) __attribute__((always_inline)) {
        if (i + kE <= d.vocab) {
            const Raw raw = *(const Raw*)(x + i);
#pragma unroll
            for (int e = 0; e < kE; ++e) v[e] = (float)raw[e];
        } else {
#pragma unroll
            for (int e = 0; e < kE; ++e) v[e] = i + e < d.vocab ? (float)x[i + e] : behind;
        }
    };
    for (int32_t u0 = first_unit + wave * kLoads; u0 < end_unit; u0 += WAVES * kLoads) {
        float v[kLoads][kE];
        const bool full = (u0 + kLoads) * kUnit <= d.vocab;
        // behind the end: no infinity, none that comes before the given token, and (in front of a lane's real values) none that is its largest
        const float behind = fminf(mine, kBehind);
        if (full) {
            Raw raw[kLoads];
#pragma unroll
            for (int u = 0; u < kLoads; ++u) raw[u] = *(const Raw*)(x + (u0 + u) * kUnit + lane * kE);
#pragma unroll
            for (int u = 0; u < kLoads; ++u)
#pragma unroll
                for (int e = 0; e < kE; ++e) v[u][e] = (float)raw[u][e];
        } else {
#pragma unroll
            for (int u = 0; u < kLoads; ++u) fetch((u0 + u) * kUnit + lane * kE, v[u], behind);
        }
        // those that come before the given token: at least as large in front of it, larger behind it
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            const int32_t first = (u0 + u) * kUnit;
            if (t >= first + kUnit) {
#pragma unroll
                for (int e = 0; e < kE; ++e) rank += (int32_t)__popcll(__builtin_amdgcn_ballot_w64(v[u][e] >= mine_before));
            } else if (t < first) {
#pragma unroll
                for (int e = 0; e < kE; ++e) rank += (int32_t)__popcll(__builtin_amdgcn_ballot_w64(v[u][e] > mine));
            } else {
#pragma unroll
                for (int e = 0; e < kE; ++e)
                    rank += (int32_t)__popcll(__builtin_amdgcn_ballot_w64(first + lane * kE + e < t ? v[u][e] >= mine_before : v[u][e] > mine));
            }
        }
        constexpr bool kQuiet = __is_same(T, _Float16);       // (conversions make them so)
        auto value = [&](int i) __attribute__((always_inline)) { return kQuiet ? v[i / kE][i % kE] : quiet(v[i / kE][i % kE]); };
        float all = -INFINITY;
#pragma unroll
        for (int i = 0; i < kLoads * kE; i += 2) all = largest(all, value(i), value(i + 1));
        const float next = largest(m, m, all), base = next * kLog2e;
        float e1[kLoads], e2[kLoads];
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            e1[u] = e2[u] = 0.0f;
#pragma unroll
            for (int e = 0; e < kE; ++e) {
                const float y = fmaxf(fmaf(v[u][e], kLog2e, -base), -1000.0f), w = __builtin_amdgcn_exp2f(y);    // (-1000 for a NaN)
                e1[u] += w;
                e2[u] = fmaf(w, y, e2[u]);
            }
        }
        const bool any = full || u0 * kUnit + lane * kE < d.vocab;           // of the lane's values are real
        if (__builtin_amdgcn_ballot_w64(any && !((plain(base) || next == -INFINITY) && (full || all > kBehind + kAbove))) == 0) {
            if (any) {
                if (next > m) {
                    const float y = step(m, next), f = __builtin_amdgcn_exp2f(y);
                    near = (near + s * (double)y) * f;
                    s *= f;
                    m = next;
                }
#pragma unroll
                for (int u = 0; u < kLoads; ++u) {
                    s += (double)e1[u];
                    near += (double)e2[u];
                }
            } else {
                all = -INFINITY;
            }
        } else {
            all = -INFINITY;
#pragma unroll 1
            for (int u = 0; u < kLoads; ++u) {
                float z[kE], top = -INFINITY;
                fetch((u0 + u) * kUnit + lane * kE, z, -INFINITY);
#pragma unroll
                for (int e = 0; e < kE; ++e) {
                    z[e] = cleaned(z[e]);
                    top = fmaxf(top, z[e]);
                }
                all = fmaxf(all, top);
                if (top > m) {
                    const float y = step(m, top), f = __builtin_amdgcn_exp2f(y);
                    near = (near + s * (double)y) * f;
                    s *= f;
                    m = top;
                }
                const float M = m * kLog2e;
                float sum = 0.0f, sum2 = 0.0f;
#pragma unroll
                for (int e = 0; e < kE; ++e) {
                    const float y = exponent(z[e], m, M), w = __builtin_amdgcn_exp2f(y);
                    sum += w;
                    sum2 = fmaf(w, y, sum2);
                }
                s += (double)sum;
                near += (double)sum2;
            }
        }
        if (d.top) {
            float of = all;
            if (wide > 1) of = fmaxf(of, moved<kOne>(of));
            if (wide > 2) of = fmaxf(of, moved<kTwo>(of));
            if (wide > 4) of = fmaxf(of, moved<kFour>(of));
            if (wide > 8) of = fmaxf(of, moved<kEight>(of));
            if ((lane & (wide - 1)) == 0) {
                uint32_t* const to = &maxima[(per == 1 ? u0 / kLoads : u0 / kLoads / per) * in_batch + (lane >> bits)];
                if (per == 1) *to = order_of(of);
                else atomicMax(to, order_of(of));
            }
        }
    }
    if (STAGE != kJoin && lowest && slice == 0 && wave == 0) rank += t;
    if constexpr (STAGE == kJoin) {          // a slice a thread
        if (tid < a.slices) {
            const Part part = a.parts[row * a.slices + tid];
            m = part.m;
            s = part.s;
            near = part.near;
            rank = part.rank;
        }
        if (d.top)
            for (int i = tid; i < groups; i += kThreads) maxima[i] = a.maxima[row * groups + i];
    }
    // the row's: first of the wavefront's lanes, then of the wavefronts
    float all = over_wave(m, Max());
    if constexpr (STAGE == kJoin) rank = over_wave(rank, Sum());
    if (lane == 0) {
        tops[wave] = all;
        counts[0][wave] = rank;
    }
    if (tid == 0) n_held = 0;
    __syncthreads();
    rank = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        all = fmaxf(all, tops[w]);
        rank += counts[0][w];
    }
    const bool none = !(all > -INFINITY && all < INFINITY);
    if (m > -INFINITY && !none) {
        const float y = step(m, all);
        const double f = (double)__builtin_amdgcn_exp2f(y);
        near = (near + s * (double)y) * f;
        s *= f;
    } else {
        s = near = 0.0;
    }
    s = over_wave(s, Sum());
    near = over_wave(near, Sum());
    if (lane == 0) {
        sums[0][wave] = s;
        sums[1][wave] = near;
    }
    __syncthreads();
    s = near = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        s += sums[0][w];
        near += sums[1][w];
    }
    if constexpr (STAGE == kSlice) {
        if (tid == 0) a.parts[row * a.slices + slice] = {s, near, all, rank};
        if (d.top)
            for (int i = first_unit / (kLoads * per) * in_batch + tid; i < (end_unit + kLoads * per - 1) / (kLoads * per) * in_batch; i += kThreads)
                a.maxima[row * groups + i] = maxima[i];
        return;
    }
    const double off = excess(all, all * kLog2e);
    const double log_s = none ? (double)NAN : log(s) - off * 0.6931471805599453;
    auto score = [&](float v) { return (float)((double)v - (double)all - log_s); };
    if (tid == 0) {
        a.scores[row] = given ? score(mine) : -INFINITY;
        a.ranks[row] = given ? rank : -1;
        a.entropy[row] = (float)(log_s - (near / s - off) / (double)kLog2e);
    }
    if (!d.top) return;

    // A bound that `top` groups or more reach, not many more.  (0 is below all.)  Every wavefront finds it for itself.
    // Bounds are orders without the bits that no value of the type has.
    uint32_t near_me[kMine];
#pragma unroll
    for (int k = 0; k < kMine; ++k) near_me[k] = k * 64 + lane < groups ? maxima[k * 64 + lane] >> kShift : 0;
    auto groups_from = [&](uint32_t bound) __attribute__((always_inline)) {
        int32_t n = 0;
#pragma unroll
        for (int k = 0; k < kMine; ++k)
            n += (int32_t)__popcll(__builtin_amdgcn_ballot_w64(near_me[k] >= bound));
        return n;
    };
    const uint32_t best = order_of(all) >> kShift;
    const int32_t enough = d.top + d.top / 2 + 8;
    uint32_t low = 0, high = best + 1;       // groups_from(low) >= top (or all there are), groups_from(high) < top
    if (groups >= d.top) {
        // down from the best by steps that double, then halving
        for (uint32_t step = (1u << 18) >> kShift; low == 0 && step; step <<= 1) {
            const uint32_t bound = best > step ? best - step : 1;
            const int32_t n = groups_from(bound);
            if (n >= d.top) {
                low = bound;
                if (n <= enough) break;
            } else {
                high = bound;
            }
            if (bound == 1) break;
        }
        while (high - low > 1) {
            const uint32_t bound = low + (high - low) / 2;
            const int32_t n = groups_from(bound);
            if (n >= d.top) {
                low = bound;
                if (n <= enough) break;
            } else {
                high = bound;
            }
        }
    }
    // The values of those groups from a bound on: all are counted, some are held.
    const uint32_t groups_bound = low;
    auto values_from = [&](uint32_t bound) __attribute__((always_inline)) {
        auto offer = [&](int32_t i) __attribute__((always_inline)) {
            float v[kE];
            fetch(i, v, -INFINITY);
#pragma unroll
            for (int e = 0; e < kE; ++e) {
                const uint32_t o = order_of(cleaned(v[e]));
                if (o >> kShift >= bound && i + e < d.vocab) {
                    const int32_t at = atomicAdd(&n_held, 1);
                    if (at < kHeld) held[at] = key_of(o, i + e);
                }
            }
        };
        for (int g0 = wave * 64; g0 < groups; g0 += WAVES * 64) {
            const bool is = g0 + lane < groups && maxima[min(g0 + lane, groups - 1)] >> kShift >= groups_bound;
            const uint64_t who = __builtin_amdgcn_ballot_w64(is);
            const int32_t many = (int32_t)__popcll(who);
            if (is) chosen[wave][__popcll(who & ((1ull << lane) - 1))] = (uint16_t)(g0 + lane);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            const int32_t team_bits = min(6, bits + kLoadBits), team = 1 << team_bits;       // lanes a group
            for (int32_t k = lane >> team_bits; k < many; k += 64 >> team_bits) {
                const int32_t g = chosen[wave][k], first = (g >> (6 - bits)) * per * kLoads, end = min(units, first + per * kLoads);
                for (int32_t u = first + ((lane & (team - 1)) >> bits); u < end; u += team >> bits) {
                    const int32_t i = u * kUnit + (((g & (in_batch - 1)) << bits) + (lane & (wide - 1))) * kE;
                    if (i < d.vocab) offer(i);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        __syncthreads();
        return n_held;
    };
    auto again_from = [&](uint32_t bound) {
        __syncthreads();
        if (tid == 0) n_held = 0;
        __syncthreads();
        return values_from(bound);
    };
    int32_t n = values_from(low);
    int32_t ties = 0;
    if (n > kHeld) {
        high = best + 1;                     // values_from(low) > kHeld, values_from(high) < top
        while (high - low > 1) {
            const uint32_t bound = low + (high - low) / 2;
            n = again_from(bound);
            if (n < d.top) high = bound;
            else low = bound;
            if (n >= d.top && n <= kHeld) break;
        }
        if (n > kHeld || n < d.top) {
            n = high > best ? 0 : again_from(high);            // fewer than top
            ties = d.top - n;
        }
    }
    if (ties) {
        // of the tokens whose value is `low` the first ones, in order
        int turn = 0;
        __syncthreads();
        for (int32_t i0 = 0; ties && i0 < d.vocab; i0 += kThreads) {
            const int32_t i = i0 + tid;
            const uint32_t o = i < d.vocab ? order_of(cleaned((float)x[i])) : 0;
            const bool is = i < d.vocab && o >> kShift == low;
            const uint64_t who = __builtin_amdgcn_ballot_w64(is);
            if (lane == 0) counts[turn][wave] = (int32_t)__popcll(who);
            __syncthreads();
            int32_t before = (int32_t)__popcll(who & ((1ull << lane) - 1)), found = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                if (w < wave) before += counts[turn][w];
                found += counts[turn][w];
            }
            turn ^= 1;
            if (is && before < ties) held[n + before] = key_of(o, i);
            n += min(found, ties);
            ties -= min(found, ties);
        }
        __syncthreads();
    }
    auto put = [&](int32_t place, uint64_t key) {
        a.top_tokens[row * d.top + place] = (int32_t)~(uint32_t)key;
        a.top_scores[row * d.top + place] = score(value_of((uint32_t)(key >> 32)));
    };
    if (n <= 512) {                          // ranked, eight lanes a candidate
        for (int i0 = 0; i0 < n; i0 += kThreads / 8) {
            const int i = i0 + (tid >> 3);
            const uint64_t key = held[min(i, n - 1)];
            int32_t place = 0;
#pragma unroll 4
            for (int j = tid & 7; j < n; j += 8) place += held[j] > key;
            place += __shfl_xor(place, 1);
            place += __shfl_xor(place, 2);
            place += __shfl_xor(place, 4);
            if (i < n && (tid & 7) == 0 && place < d.top) put(place, key);
        }
        return;
    }
    int size = 1024;                         // sorted
    while (size < n) size <<= 1;
    for (int i = n + tid; i < size; i += kThreads) held[i] = 0;
    __syncthreads();
    for (int run = 2; run <= size; run <<= 1)
        for (int step = run >> 1; step; step >>= 1) {
            for (int k = tid; k < size / 2; k += kThreads) {
                const int i = (k / step) * 2 * step + k % step, j = i + step;
                const uint64_t p = held[i], q = held[j];
                if ((q > p) == ((i & run) == 0)) {
                    held[i] = q;
                    held[j] = p;
                }
            }
            __syncthreads();
        }
    for (int i = tid; i < d.top; i += kThreads) put(i, held[i]);
}

// How a call is laid out: slices of 128 units, which sixteen wavefronts read at once, where rows are few and have more of them (a row of 150001, f32: 24 us
// whole, 17.6 in slices; 16 of 128257, bf16: 24.3 and 22.2).
// Units that a wavefront reads at once: as few as leave none idle (123 rows of 1270, bf16: 10.6 us, with eight 17.4; 500 of 8000: 12.8 and 16.1), eight,
// or four where rows fill the device, for longer ones.
int32_t loads_of(int32_t rows, int32_t units) {
    const int32_t waves = rows <= 256 ? 16 : 8;
    return units <= waves ? 1 : units <= 2 * waves ? 2 : rows <= 512 ? 8 : 4;
}
struct Plan {
    int32_t slices, slice_units;
    Groups by;
    int32_t loads;
    int64_t parts_bytes, bytes;
};
Plan plan_of(const reef_token_scores_desc& d) {
    const int32_t unit = 1024 / type_bytes(d.type), units = (d.vocab + unit - 1) / unit, loads = loads_of(d.rows, units);
    Plan p{1, units, groups_of(units, loads), loads, 0, 0};
    if (d.rows > 128 || units <= 192) return p;
    const int32_t most = std::min(256 / d.rows, (units + 127) / 128);
    const int32_t step = p.by.per * loads;        // no group and no batch reaches into the next slice
    p.slice_units = ((units + most - 1) / most + step - 1) / step * step;
    p.slices = (units + p.slice_units - 1) / p.slice_units;
    if (p.slices <= 1) return p;
    p.parts_bytes = (int64_t)d.rows * p.slices * (int64_t)sizeof(Part);
    p.bytes = p.parts_bytes + (d.top ? 4ll * d.rows * p.by.groups : 0);
    return p;
}
// Sixteen wavefronts a row where rows are few, four where they fill the device (1000 rows of 128257, bf16: 72 us, 3.6 TB/s; eight 81, sixteen 104; 2000
// of 5000: 25, 44, 84).
template <class T>
int run(const char* what, const Args& a, const Plan& p, void* stream) {
    const dim3 rows((unsigned)a.d.rows);
    if (p.bytes) {
        if (int rc = launch(what, token_scores<T, 16, 8, kSlice>, dim3((unsigned)(a.d.rows * p.slices)), dim3(16 * 64), a, stream)) return rc;
        return launch(what, token_scores<T, 16, 8, kJoin>, rows, dim3(16 * 64), a, stream);
    }
    auto go = [&](auto loads) {
        constexpr int kLoads = decltype(loads)::value;
        if (a.d.rows <= 256) return launch(what, token_scores<T, 16, kLoads, kWhole>, rows, dim3(16 * 64), a, stream);
        if (a.d.rows <= 512) return launch(what, token_scores<T, 8, kLoads, kWhole>, rows, dim3(8 * 64), a, stream);
        return launch(what, token_scores<T, 4, kLoads == 8 ? 4 : kLoads, kWhole>, rows, dim3(4 * 64), a, stream);
    };
    if (a.loads == 1) return go(std::integral_constant<int, 1>());
    if (a.loads == 2) return go(std::integral_constant<int, 2>());
    return go(std::integral_constant<int, 8>());
}

int check(const char* what, const reef_token_scores_desc* d) {
    if (!d) return refuse(what, "null argument");
    if (!type_bytes(d->type)) return refuse(what, "unknown type %d", d->type);
    if (d->rows < 0 || d->rows >= 1 << 24 || d->vocab < 1 || d->vocab >= 1 << 24) return refuse(what, "bad sizes: %d rows of %d tokens", d->rows, d->vocab);
    if (d->top < 0 || d->top > kMaxTop || d->top > d->vocab) return refuse(what, "the first %d of %d tokens cannot be given (up to %d)", d->top, d->vocab, kMaxTop);
    if (d->rows > 1 && d->logits_stride < d->vocab) return refuse(what, "rows of logits overlap");
    if ((int64_t)d->rows * d->vocab >= 1ll << 40) return refuse(what, "more than 2^40 logits");
    return 0;
}

}  // namespace

extern "C" int64_t reef_ops_token_scores_workspace(const reef_token_scores_desc* d) {
    if (check("reef_ops_token_scores_workspace", d)) return -1;
    return d->rows ? plan_of(*d).bytes : 0;
}

extern "C" int reef_ops_token_scores(const reef_token_scores_desc* d, const void* logits, const int32_t* tokens, float* scores, int32_t* ranks, float* entropy,
                                     int32_t* top_tokens, float* top_scores, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "reef_ops_token_scores";
    if (int rc = check(what, d)) return rc;
    if (!d->rows) return 0;
    if (!logits || !aligned(logits, type_bytes(d->type)) || !words(tokens) || !words(scores) || !words(ranks) || !words(entropy) ||
        (d->top && (!words(top_tokens) || !words(top_scores))))
        return refuse(what, "null or unaligned argument");
    const int64_t n = d->rows, need = plan_of(*d).bytes;
    if (need && (!rows16(workspace) || workspace_bytes < need))
        return refuse(what, "a workspace of %lld bytes on 16 is needed, %lld are given", (long long)need, (long long)workspace_bytes);
    const Span out[] = {{scores, 4 * n}, {ranks, 4 * n}, {entropy, 4 * n}, {top_tokens, 4 * n * d->top}, {top_scores, 4 * n * d->top}, {workspace, need}};
    const Span in[] = {{logits, ((n - 1) * d->logits_stride + d->vocab) * type_bytes(d->type)}, {tokens, 4 * n}};
    if (overlap(out, in)) return refuse(what, "an output overlaps an input");
    const Plan p = plan_of(*d);
    const Args a{*d, logits, tokens, scores, ranks, entropy, top_tokens, top_scores, (Part*)workspace, (uint32_t*)((char*)workspace + p.parts_bytes), p.slices, p.slice_units, p.by, p.loads};
    switch (d->type) {
        case REEF_TYPE_F32: return run<float>(what, a, p, stream);
        case REEF_TYPE_F16: return run<_Float16>(what, a, p, stream);
        default: return run<__bf16>(what, a, p, stream);
    }
}
