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
    double* sums;           // [row][piece]: sum of exp(x - maximum)
    float* tops;            // [row][piece]: maximum
    int32_t n_pieces;       // of a row
};

// A piece: 1 KiB of a row, counted from its first value.  (Not from a line of 128 bytes on: rows of an odd length start anywhere, and rows that
// hold the same values have to have the same sums, to the bit.)
template <class T>
constexpr int kPiece = 1024 / sizeof(T);

// A candidate, in two whole numbers: its score, in an order that whole numbers have too, and its place, beam then token.
struct Offer {
    uint64_t key, place;
};
__device__ inline uint64_t key_of(double score) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, score + 0.0);      // (-0 counts as 0)
    return bits >> 63 ? ~bits : bits | 1ull << 63;
}
__device__ inline double score_of(uint64_t key) { return __builtin_bit_cast(double, key >> 63 ? key & ~(1ull << 63) : ~key); }
__device__ inline bool before(const Offer& a, const Offer& b) { return (a.key > b.key) | ((a.key == b.key) & (a.place < b.place)); }
// Anything that is not a finite number counts as -infinity.
__device__ inline double offered(double s) { return s < INFINITY && s > -INFINITY ? s : -INFINITY; }

__device__ inline bool lives(const SelectArgs& a, int64_t row) { return !(a.ended && a.ended[row]); }

// Eight values a lane, reduced over the wavefront: lanes 8 u .. 8 u + 7 have the u-th.  At each of three steps half of the values go to the other half of
// the lanes, which leaves one; all of it without LDS (through it row_pieces takes 28.6 instead of 20.9 us).
template <int CONTROL>
__device__ inline uint32_t moved(uint32_t x) { return __builtin_amdgcn_update_dpp(0, x, CONTROL, 0xF, 0xF, true); }
template <int CONTROL>
__device__ inline float moved(float x) { return __uint_as_float(moved<CONTROL>(__float_as_uint(x))); }
template <int CONTROL>
__device__ inline double moved(double x) {
    const u32x2 w = __builtin_bit_cast(u32x2, x), m = {moved<CONTROL>(w[0]), moved<CONTROL>(w[1])};
    return __builtin_bit_cast(double, m);
}
// The upper half of p's lanes against the lower half of q's: of all lanes, or of each 32.
__device__ inline void swap_words(uint32_t& p, uint32_t& q, bool halves) {
    const auto x = halves ? __builtin_amdgcn_permlane32_swap(p, q, false, false) : __builtin_amdgcn_permlane16_swap(p, q, false, false);
    p = x[0];
    q = x[1];
}
template <class V>
__device__ inline void swap_lanes(V& p, V& q, bool halves) {
    if constexpr (sizeof(V) == 4) {
        uint32_t a = __builtin_bit_cast(uint32_t, p), b = __builtin_bit_cast(uint32_t, q);
        swap_words(a, b, halves);
        p = __builtin_bit_cast(V, a);
        q = __builtin_bit_cast(V, b);
    } else {
        u32x2 a = __builtin_bit_cast(u32x2, p), b = __builtin_bit_cast(u32x2, q);
        for (int i = 0; i < 2; ++i) {
            uint32_t x = a[i], y = b[i];
            swap_words(x, y, halves);
            a[i] = x;
            b[i] = y;
        }
        p = __builtin_bit_cast(V, a);
        q = __builtin_bit_cast(V, b);
    }
}
template <class V, class Join>
__device__ inline V over_wave(V (&v)[8], Join join) {
    constexpr int kTurn8 = 0x128, kMirror8 = 0x141, kNext1 = 0xB1, kNext2 = 0x4E;    // rows of 16 by 8 lanes; lane i to 7 - i, i ^ 1, i ^ 2
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        swap_lanes(v[j], v[j + 4], true);
        v[j] = join(v[j], v[j + 4]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        swap_lanes(v[j], v[j + 2], false);
        v[j] = join(v[j], v[j + 2]);
    }
    const bool upper = threadIdx.x & 8;
    const V keep = upper ? v[1] : v[0], give = upper ? v[0] : v[1];
    V x = join(keep, moved<kTurn8>(give));
    x = join(x, moved<kMirror8>(x));
    x = join(x, moved<kNext1>(x));
    return join(x, moved<kNext2>(x));
}

// Everything that a choice needs of a row beside single values: of each piece the maximum and the sum over it.  A wavefront has eight pieces, 1 KiB a
// load; a lane keeps its 64 (32) values, so the row is read once, and the sum needs no rescaling.  A row that does not begin
// at a line costs a ninth line a load.  Exponentials are those of 32 bits, off by 2^-23 of themselves (exp2) and three roundings of the argument, 2^-22 (1 + |x - maximum|)
// in all; 64 bits would take 38 us instead of 21 for 48 x 8 rows of 128257 (bf16).  They are added in 64 bits, so that rows
// that differ in one unlikely token have different sums (in 32 bits, in pieces from a line on: 18.6 us).  Bound by memory: 4.2 TB/s, some fourteen operations a value.
template <class T>
__global__ void __launch_bounds__(kThreads) row_pieces(SelectArgs a) {
    constexpr int kE = 16 / sizeof(T);
    typedef T Raw __attribute__((ext_vector_type(kE), aligned(sizeof(T))));
    const reef_beam_select_desc& d = a.d;
    const int lane = threadIdx.x & 63;
    const int32_t rounds = (a.n_pieces + 7) / 8;
    const int64_t id = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6), row = id / rounds;
    if (row >= (int64_t)d.requests * d.beams || !lives(a, row)) return;
    const int32_t piece0 = (int32_t)(id - row * rounds) * 8, at = piece0 * kPiece<T> + lane * kE;
    const T* x = (const T*)a.logits + row * d.logits_stride;
    float v[8][kE];
    if ((piece0 + 8) * kPiece<T> <= d.vocab) {
        Raw raw[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) raw[u] = *(const Raw*)(x + at + u * kPiece<T>);
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int e = 0; e < kE; ++e) v[u][e] = (float)raw[u][e];
    } else {                                  // the row ends in here
        Raw raw[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int32_t i = at + u * kPiece<T>;
            if (i + kE <= d.vocab) raw[u] = *(const Raw*)(x + i);
            else if (i < d.vocab) {
#pragma unroll
                for (int e = 0; e < kE; ++e) raw[u][e] = x[min(i + e, d.vocab - 1)];
            }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int e = 0; e < kE; ++e) v[u][e] = at + u * kPiece<T> + e < d.vocab ? (float)raw[u][e] : -INFINITY;
    }
    float top[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        top[u] = -INFINITY;                   // (where all are NaN)
#pragma unroll
        for (int e = 0; e < kE; ++e) top[u] = fmaxf(top[u], v[u][e]);
    }
    const float m = over_wave(top, [](float p, float q) { return fmaxf(p, q); });
    double sum[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const float of = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(m), u * 8)), base = of == -INFINITY ? 0.0f : of;
        sum[u] = 0.0;
#pragma unroll
        for (int e = 0; e < kE; ++e) sum[u] += (double)__builtin_amdgcn_exp2f((v[u][e] - base) * 1.4426950408889634f);
    }
    const double s = over_wave(sum, [](double p, double q) { return p + q; });
    const int32_t piece = piece0 + (lane >> 3);
    if ((lane & 7) == 0 && piece < a.n_pieces) {
        a.sums[row * a.n_pieces + piece] = s;
        a.tops[row * a.n_pieces + piece] = m;
    }
}

constexpr int kChoose = 512, kChooseWaves = kChoose / 64;
constexpr int kBuffer = 2048;                 // candidates held; at least kMaxSelect and a piece
constexpr int kNear = 4096;                   // pieces that are held near; more are read from memory again

// The choice of one request.  The maxima of the pieces, as scores, bound what a piece can hold: the select-th best of 256 groups'
// best maxima lies below or at the select-th best offer, and only pieces that reach it are read again, some `select` of
// them.  Their offers that pass the bound go to a buffer; where it would run over (many equal values) it is cut to its
// best `select`, whose last one is the bound from then on.  Bound by latency: two trips to memory and some 15 barriers.
template <class T>
__global__ void __launch_bounds__(kChoose) beam_choose(SelectArgs a) {
    constexpr int kE = kPiece<T> / 64, kTwo = 2;   // values of a piece a lane; pieces a wavefront and step
    const reef_beam_select_desc& d = a.d;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row0 = (int64_t)blockIdx.x * d.beams;
    __shared__ double lse[kMaxBeams], score[kMaxBeams];
    __shared__ bool alive[kMaxBeams];
    __shared__ __align__(16) uint32_t tops[kChoose];
    __shared__ int ranks[kChoose];
    __shared__ Offer buffer[kBuffer], kept[kMaxSelect], bound;
    __shared__ int32_t list[kNear];
    __shared__ float near[kNear];
    __shared__ int held, listed, wave_count[kChooseWaves];

    const int32_t pieces = d.beams * a.n_pieces;
    const float* far = a.tops + row0 * a.n_pieces;
    const double* sums = a.sums + row0 * a.n_pieces;
#pragma unroll
    for (int k = 0; k < kNear / kChoose; ++k) {
        const int32_t i = k * kChoose + tid;
        if (i < pieces) near[i] = far[i];     // (of an ended beam: never used)
    }
    constexpr int kAhead = 4;                 // sums a lane of the wavefront's first beam, on their way beside the maxima
    double ahead[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
        const int i = k * 64 + lane;
        ahead[k] = sums[min(min(wave, d.beams - 1) * a.n_pieces + i, pieces - 1)];
    }
    for (int b = tid; b < d.beams; b += kChoose) {
        alive[b] = lives(a, row0 + b);
        score[b] = offered((double)a.scores[row0 + b]);
    }
    if (tid == 0) {
        held = listed = 0;
        bound = {key_of(-INFINITY), 0};       // whatever is above -infinity passes
    }
    __syncthreads();
    auto row_of = [&](int b) { return (const T*)a.logits + (row0 + b) * d.logits_stride; };
    auto piece = [&](int32_t i) { return i < kNear ? near[i] : far[i]; };
    for (int b = wave; b < d.beams; b += kChooseWaves) {
        if (!alive[b]) continue;
        const int32_t p0 = b * a.n_pieces;
        float m = -INFINITY;
        for (int i = lane; i < a.n_pieces; i += 64) m = fmaxf(m, piece(p0 + i));
        for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
        const float base = m == -INFINITY ? 0.0f : m;
        double sum = 0.0;
        // (the same roundings in both places: beams with the same values have the same sum)
        auto add = [&](int i, double s) { sum = __builtin_fma(s, (double)__builtin_amdgcn_exp2f((piece(p0 + i) - base) * 1.4426950408889634f), sum); };
        int i = lane;
        if (b == wave) {
#pragma unroll
            for (int k = 0; k < kAhead; ++k, i += 64)
                if (i < a.n_pieces) add(i, ahead[k]);
        }
        for (; i < a.n_pieces; i += 64) add(i, sums[p0 + i]);
        for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
        if (lane == 0) lse[b] = (double)m + log(sum);
    }
    __syncthreads();
    // what beam b offers for a logit; the best that a piece of it offers
    auto offer = [&](int b, float x) { return offered(score[b] + ((double)x - lse[b])); };
    auto best_of = [&](int32_t i) -> double {
        const int b = i / a.n_pieces, p = i - b * a.n_pieces;
        if (alive[b]) return offer(b, piece(i));
        return d.end_token >= 0 && d.end_token < d.vocab && d.end_token / kPiece<T> == p ? score[b] : -INFINITY;
    };
    double best[kNear / kChoose], top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kNear / kChoose; ++k) {
        const int32_t i = k * kChoose + tid;
        best[k] = i < pieces ? best_of(i) : -INFINITY;
        top = fmax(top, best[k]);
    }
    for (int64_t i = kNear + tid; i < pieces; i += kChoose) top = fmax(top, best_of((int32_t)i));

    // Raises the bound by one offer a thread (or -infinity), of the first `threads`: the maxima of groups of neighbours, `want` of them at
    // least if there are so many threads, rounded down to 22 bits and made unique by their numbers, are ranked by all threads
    // together, and the select-th best is the bound.
    auto raise = [&](double top, int threads, int want) {
        int per = 16, places = 64;
        while (per > 1 && threads / per < want) per >>= 1;
        const int groups = (threads + per - 1) / per;
        while (places < groups) places <<= 1;
        float low = (float)top;
        low -= fabsf(low) * 0x1p-23f + 1e-37f;
        if (top == -INFINITY) low = -INFINITY;
        for (int x = 1; x < per; x <<= 1) low = fmaxf(low, __shfl_xor(low, x));
        if (tid % per == 0 && tid / per < places) {
            const uint32_t bits = __float_as_uint(low), order = low == -INFINITY ? 0 : bits >> 31 ? ~bits : bits | 1u << 31;
            tops[tid / per] = tid / per < groups ? (order & ~1023u) | (1023 - tid / per) : 0;
            ranks[tid / per] = 0;
        }
        __syncthreads();
        // (threads that have no group of their own write what their slice does not have)
        const int mine = tid & (places - 1), slices = kChoose / places, others = ((groups + slices - 1) / slices + 3) / 4 * 4, o0 = tid / places * others;
        if (mine < groups) {
            const uint32_t value = tops[mine];
            int rank = 0;
#pragma unroll 4
            for (int o = o0; o < min(places, o0 + others); o += 4) {
                const u32x4 t = *(const u32x4*)&tops[o];
                rank += (int)(t[0] > value) + (int)(t[1] > value) + (int)(t[2] > value) + (int)(t[3] > value);
            }
            if (rank) atomicAdd(&ranks[mine], rank);
        }
        __syncthreads();
        if (tid < groups && ranks[tid] == d.select - 1) {
            const uint32_t order = tops[tid] & ~1023u;
            const double least = (double)__uint_as_float(order >> 31 ? order & ~(1u << 31) : ~order);
            if (order && key_of(least) > bound.key) bound = {key_of(least), ~0ull};
        }
        __syncthreads();
    };
    // (up to as many groups a beam as are chosen: often one beam has them all)
    raise(top, min(pieces, kChoose), max(2 * d.select, min(256, d.beams * d.select)));

    // The best `select` of the buffer, in order; the last of them bounds what follows.
    auto cut = [&]() {
        const int n = held, m = min(n, d.select);
        __syncthreads();
        if (n <= 512) {                                       // ranked, eight lanes a candidate
            for (int i0 = 0; i0 < n; i0 += kChoose / 8) {
                const int i = i0 + (tid >> 3);
                const Offer mine = buffer[min(i, n - 1)];
                int rank = 0;
#pragma unroll 4
                for (int j = tid & 7; j < n; j += 8) rank += before(buffer[j], mine);
                rank += __shfl_xor(rank, 1);
                rank += __shfl_xor(rank, 2);
                rank += __shfl_xor(rank, 4);
                if (i < n && (tid & 7) == 0 && rank < d.select) kept[rank] = mine;
            }
            __syncthreads();
            if (tid < m) buffer[tid] = kept[tid];
        } else {                                              // sorted (2048 candidates: 170 us ranked)
            const int size = n <= 1024 ? 1024 : 2048;
            for (int i = n + tid; i < size; i += kChoose) buffer[i] = {0, ~0ull};
            __syncthreads();
            for (int run = 2; run <= size; run <<= 1)
                for (int step = run >> 1; step; step >>= 1) {
                    for (int t = tid; t < size / 2; t += kChoose) {
                        const int i = (t / step) * 2 * step + t % step, j = i + step;
                        const Offer x = buffer[i], y = buffer[j];
                        if (before(y, x) == ((i & run) == 0)) {
                            buffer[i] = y;
                            buffer[j] = x;
                        }
                    }
                    __syncthreads();
                }
        }
        if (tid == 0) {
            held = m;
            if (m == d.select) bound = n <= 512 ? kept[m - 1] : buffer[m - 1];
        }
        __syncthreads();
    };
    for (int64_t i0 = 0; i0 < pieces; i0 += kNear) {
        const double least = score_of(bound.key);
#pragma unroll
        for (int k = 0; k < kNear / kChoose; ++k) {
            const int64_t i = i0 + k * kChoose + tid;
            if (i >= pieces) continue;
            const double x = i0 ? best_of((int32_t)i) : best[k];
            if (x > -INFINITY && x >= least) list[atomicAdd(&listed, 1)] = (int32_t)i;
        }
        __syncthreads();
        const int n = listed;
        for (int j0 = 0; j0 < n; j0 += kChooseWaves * kTwo) {
            float x[kTwo][kE];
            double own[kTwo], norm[kTwo];
            int beam[kTwo], v0[kTwo];
            bool live[kTwo];
            T raw[kTwo][kE];
            const double least_now = score_of(bound.key);
#pragma unroll
            for (int u = 0; u < kTwo; ++u) {                  // all loads before any of them is looked at
                const int j = j0 + u * kChooseWaves + wave;
                beam[u] = -1;
                own[u] = norm[u] = 0.0;
                live[u] = false;
                v0[u] = 0;
                if (j >= n || best_of(list[j]) < least_now) continue;     // (the bound rises on the way)
                const int32_t i = list[j], b = i / a.n_pieces;
                const T* row = row_of(b);
                beam[u] = b;
                v0[u] = (i - b * a.n_pieces) * kPiece<T> + lane;
#pragma unroll
                for (int e = 0; e < kE; ++e) raw[u][e] = row[max(0, min(v0[u] + e * 64, d.vocab - 1))];
                live[u] = alive[b];
                own[u] = score[b];
                norm[u] = live[u] ? lse[b] : 0.0;
            }
#pragma unroll
            for (int u = 0; u < kTwo; ++u) {
#pragma unroll
                for (int e = 0; e < kE; ++e) {
                    const int32_t v = v0[u] + e * 64;
                    x[u][e] = beam[u] < 0 || (uint32_t)v >= (uint32_t)d.vocab ? -INFINITY : live[u] ? (float)raw[u][e] : v == d.end_token ? 0.0f : -INFINITY;
                }
            }
            auto one = [&](int u, int e) -> Offer {
                return {key_of(live[u] ? offered(own[u] + ((double)x[u][e] - norm[u])) : own[u]), (uint64_t)beam[u] << 32 | (uint32_t)(v0[u] + e * 64)};
            };
            // What a value must at least be for its offer to pass, a little lower than it is: few are looked at in 64 bits
            // (by the roundings of both sides: offers of a beam whose score is large may be equal for many values).
            float least_x[kTwo];
            auto near_enough = [&](int u, int e) { return x[u][e] > -INFINITY && x[u][e] >= least_x[u]; };
            int had = 0;                                      // held before this step
            auto count = [&]() {
                const double limit = score_of(bound.key);
                int mine = 0;
#pragma unroll
                for (int u = 0; u < kTwo; ++u) {
                    if (beam[u] < 0) continue;
                    const double f = limit - own[u] + norm[u];
                    const double slack = fabs(f) * 0x1p-20 + (fabs(limit) + fabs(own[u]) + fabs(norm[u])) * 0x1p-49;
                    least_x[u] = live[u] && limit > -INFINITY && own[u] > -INFINITY ? (float)(f - slack) : -INFINITY;
#pragma unroll
                    for (int e = 0; e < kE; ++e) mine += __popcll(__builtin_amdgcn_ballot_w64(near_enough(u, e)));
                }
                if (lane == 0) wave_count[wave] = mine;
                __syncthreads();
                had = held;
                int all = had;
                for (int w = 0; w < kChooseWaves; ++w) all += wave_count[w];
                __syncthreads();
                return all;
            };
            int all = count();
            if (all > had + d.select + 128) {
                // pieces are few or alike: each lane's best offer is a bound of its own (16 beams of 500 tokens, 32 chosen: 600 -> 25 us)
                double mine = -INFINITY;
#pragma unroll
                for (int u = 0; u < kTwo; ++u) {
                    float high = -INFINITY;
#pragma unroll
                    for (int e = 0; e < kE; ++e) high = fmaxf(high, x[u][e]);
                    if (high > -INFINITY) mine = fmax(mine, live[u] ? offered(own[u] + ((double)high - norm[u])) : own[u]);
                }
                raise(mine, min(n - j0, kChooseWaves) * 64, max(2 * d.select, min(128, 8 * d.select)));
                all = count();
            }
            auto push = [&](int u) {                          // one place in the buffer for all that pass
                if (beam[u] < 0) return;
                const Offer now = bound;
                uint64_t who[kE];
                int total = 0;
#pragma unroll
                for (int e = 0; e < kE; ++e) {
                    who[e] = 0;
                    if (__builtin_amdgcn_ballot_w64(near_enough(u, e))) who[e] = __builtin_amdgcn_ballot_w64(near_enough(u, e) && before(one(u, e), now));
                    total += __popcll(who[e]);
                }
                if (!total) return;
                int at = 0;
                if (lane == 0) at = atomicAdd(&held, total);
                at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
                for (int e = 0; e < kE; ++e) {
                    if (who[e] >> lane & 1) buffer[at + __popcll(who[e] & ((1ull << lane) - 1))] = one(u, e);
                    at += __popcll(who[e]);
                }
            };
            if (all <= kBuffer) {
#pragma unroll
                for (int u = 0; u < kTwo; ++u) push(u);
                __syncthreads();
            } else {
                for (int w = 0; w < kChooseWaves; ++w)        // one piece after another, cut in between
#pragma unroll
                    for (int u = 0; u < kTwo; ++u) {
                        const bool full = held + kPiece<T> > kBuffer;
                        __syncthreads();                      // (all have read it)
                        if (full) cut();
                        if (wave == w) push(u);
                        __syncthreads();
                    }
            }
        }
        __syncthreads();
        if (tid == 0) listed = 0;
        __syncthreads();
    }
    cut();
    const int found = held;
    const int64_t out = (int64_t)blockIdx.x * d.select;
    if (tid < found) {
        a.best[out + tid] = (float)score_of(buffer[tid].key);
        a.parents[out + tid] = (int32_t)(row0 + (buffer[tid].place >> 32));
        a.tokens[out + tid] = (int32_t)buffer[tid].place;
    }
    if (found == d.select) return;
    // Fewer offers than places: the rest at -infinity, in order.  All offers above it are in the buffer, fewer than
    // select, so the first 2 * select places hold enough of the others.
    int rank = found;
    const int64_t p = tid;
    bool none = false;
    if (p < 2 * d.select && p < (int64_t)d.beams * d.vocab) {
        const int b = (int)(p / d.vocab);
        const int32_t v = (int32_t)(p - (int64_t)b * d.vocab);
        none = true;
        for (int j = 0; j < found; ++j) none = none && buffer[j].place != ((uint64_t)b << 32 | (uint32_t)v);
    }
    const uint64_t who = __builtin_amdgcn_ballot_w64(none);
    if (lane == 0) wave_count[wave] = __popcll(who);
    __syncthreads();
    for (int w = 0; w < wave; ++w) rank += wave_count[w];
    rank += __popcll(who & ((1ull << lane) - 1));
    if (none && rank < d.select) {
        a.best[out + rank] = -INFINITY;
        a.parents[out + rank] = (int32_t)(row0 + p / d.vocab);
        a.tokens[out + rank] = (int32_t)(p % d.vocab);
    }
}

template <class T>
int run_select(const char* what, SelectArgs a, void* stream) {
    const int64_t waves = (int64_t)a.d.requests * a.d.beams * ((a.n_pieces + 7) / 8);
    if (int rc = launch(what, row_pieces<T>, dim3((unsigned)((waves + 3) / 4)), dim3(kThreads), a, stream)) return rc;
    return launch(what, beam_choose<T>, dim3((unsigned)a.d.requests), dim3(kChoose), a, stream);
}

int32_t pieces_of(const reef_beam_select_desc& d) { return (int32_t)(((int64_t)d.vocab * type_bytes(d.type) + 1023) / 1024); }

int check_select(const char* what, const reef_beam_select_desc* d) {
    if (!d) return refuse(what, "null argument");
    if (!type_bytes(d->type)) return refuse(what, "unknown type %d", d->type);
    if (d->requests < 0 || d->beams < 1 || d->beams > kMaxBeams || d->vocab < 1 || d->vocab >= 1 << 24 || (int64_t)d->requests * d->beams >= 1 << 24)
        return refuse(what, "bad sizes: %d requests, %d beams (up to %d), %d tokens", d->requests, d->beams, kMaxBeams, d->vocab);
    if (d->select < 1 || d->select > kMaxSelect || d->select > (int64_t)d->beams * d->vocab)
        return refuse(what, "%d of %d beams of %d tokens cannot be selected (up to %d)", d->select, d->beams, d->vocab, kMaxSelect);
    if ((int64_t)d->requests * d->beams > 1 && d->logits_stride < d->vocab) return refuse(what, "rows of logits overlap");
    if ((int64_t)d->requests * d->beams * d->vocab >= 1ll << 40) return refuse(what, "more than 2^40 logits");
    return 0;
}

struct ReorderArgs {
    reef_beam_reorder_desc d;
    const int32_t *parents, *lengths, *table, *spare;
    int32_t *table_out, *lengths_out;
    void *key_cache, *value_cache;
};

// A workgroup: one row's table, or the tokens of its last block in one layer of one pool, four 16-byte pieces a thread in flight.  What
// is to be moved takes three loads in a row to find out, which many small workgroups hide best: 256 rows, 24 layers 43 us = 3.8 TB/s, with
// two pools a workgroup 46, with six 70.
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
    const uint32_t bytes = d.cache.type == REEF_TYPE_F32 ? 4 : 2, heads = d.cache.kv_heads, pieces = d.cache.head_dim * bytes / 16;
    const uint32_t part = blockIdx.y - 1, total = rest * heads * pieces;
    const int64_t from = source * d.cache.block_stride, to = target * d.cache.block_stride;
    unsigned char* pool = (unsigned char*)(part & 1 ? a.value_cache : a.key_cache) + (int64_t)(part >> 1) * d.layer_stride * bytes;
    for (uint32_t k0 = threadIdx.x; k0 < total; k0 += 4 * kThreads) {
        unsigned char* at[4];
        u32x4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t k = min(k0 + u * kThreads, total - 1), th = k / pieces, t = th / heads, h = th - t * heads;
            at[u] = pool + (t * d.cache.slot_stride + h * d.cache.head_stride) * bytes + (k - th * pieces) * 16;
            v[u] = *(const u32x4*)(at[u] + from * bytes);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (k0 + u * kThreads < total) *(u32x4*)(at[u] + to * bytes) = v[u];
    }
}

}  // namespace

extern "C" int64_t reef_ops_beam_select_workspace(const reef_beam_select_desc* d) {
    if (check_select("reef_ops_beam_select_workspace", d)) return -1;
    return (int64_t)d->requests * d->beams * pieces_of(*d) * (int64_t)(sizeof(double) + sizeof(float));
}

extern "C" int reef_ops_beam_select(const reef_beam_select_desc* d, const void* logits, const float* scores, const uint8_t* ended, float* best,
                                    int32_t* parents, int32_t* tokens, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "reef_ops_beam_select";
    if (int rc = check_select(what, d)) return rc;
    if (!d->requests) return 0;
    if (!logits || !aligned(logits, type_bytes(d->type)) || !words(scores) || !words(best) || !words(parents) || !words(tokens))
        return refuse(what, "null or unaligned argument");
    const int64_t n = (int64_t)d->requests * d->beams, picks = 4ll * d->requests * d->select;
    const Span out[] = {{best, picks}, {parents, picks}, {tokens, picks}, {workspace, reef_ops_beam_select_workspace(d)}};
    const Span in[] = {{logits, ((n - 1) * d->logits_stride + d->vocab) * type_bytes(d->type)}, {scores, 4 * n}, {ended, ended ? n : 0}};
    if (overlap(out, in)) return refuse(what, "an output overlaps an input");
    double* const sums = (double*)workspace;
    const SelectArgs a{*d, logits, scores, ended, best, parents, tokens, sums, (float*)(sums + n * pieces_of(*d)), pieces_of(*d)};
    const int64_t need = reef_ops_beam_select_workspace(d);
    if (!rows16(workspace) || workspace_bytes < need)
        return refuse(what, "a workspace of %lld bytes on 16 is needed, %lld are given", (long long)need, (long long)workspace_bytes);
    switch (d->type) {
        case REEF_TYPE_F32: return run_select<float>(what, a, stream);
        case REEF_TYPE_F16: return run_select<_Float16>(what, a, stream);
        default: return run_select<__bf16>(what, a, stream);
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
    if ((int64_t)d->cache.block_size * d->cache.kv_heads * d->cache.head_dim >= 1 << 30) return refuse(what, "blocks of %d tokens are too large", d->cache.block_size);
    if (!d->rows) return 0;
    if (!words(parents) || !words(lengths) || !words(table) || !words(spare) || !words(table_out) || !words(lengths_out) || !rows16(key_cache) ||
        !rows16(value_cache))
        return refuse(what, "null or unaligned argument");
    const Span out[] = {{table_out, 4 * ((d->rows - 1ll) * d->out_stride + d->max_blocks)}, {lengths_out, 4ll * d->rows}};
    const Span in[] = {{table, 4 * ((d->table_rows - 1ll) * d->table_stride + d->max_blocks)}, {lengths, 4ll * d->table_rows}, {parents, 4ll * d->rows}, {spare, 4ll * d->rows}};
    if (overlap(out, in)) return refuse(what, "an output overlaps an input");
    const ReorderArgs a{*d, parents, lengths, table, spare, table_out, lengths_out, key_cache, value_cache};
    return launch(what, beam_reorder, dim3((unsigned)d->rows, 1 + 2 * d->layers), dim3(kThreads), a, stream);
}
