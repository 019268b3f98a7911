// Log probabilities of given tokens, their ranks, the entropy and the best alternatives (reef_ops_token_scores).
#include "ops_common.h"

namespace {
using namespace reef_ops;

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxTop = 128;
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
    reef_token_scores_desc d;
    const void* logits;
    const int32_t* tokens;
    float* scores;
    int32_t* ranks;
    float* entropy;
    int32_t* top_tokens;
    float* top_scores;
};

// A NaN counts as -infinity.
template <class T>
__device__ inline float value_of(T x) {
    const float v = (float)x;
    return v == v ? v : -INFINITY;
}

template <class V, class Join>
__device__ inline V over_group(V v, V* parts, Join join) {
    for (int x = 32; x; x >>= 1) v = join(v, (V)__shfl_xor(v, x));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = v;
    __syncthreads();
    v = parts[0];
    for (int w = 1; w < kWaves; ++w) v = join(v, parts[w]);
    return v;
}

template <class T>
__global__ void __launch_bounds__(kThreads) token_scores(Args a) {
    const reef_token_scores_desc& d = a.d;
    const int64_t row = blockIdx.x;
    const T* x = (const T*)a.logits + row * d.logits_stride;
    __shared__ float parts[kWaves];
    __shared__ double sums[kWaves];
    __shared__ int32_t counts[kWaves];
    __shared__ uint64_t keys[kWaves];
    const int32_t t = a.tokens[row];
    const bool given = (uint32_t)t < (uint32_t)d.vocab;
    const float mine = given ? value_of(x[t]) : 0.0f;
    float m = -INFINITY;
    int32_t rank = 0;
    for (int32_t i = threadIdx.x; i < d.vocab; i += kThreads) {
        const float v = value_of(x[i]);
        m = fmaxf(m, v);
        rank += v > mine || (v == mine && i < t);
    }
    m = over_group(m, parts, [](float p, float q) { return fmaxf(p, q); });
    rank = over_group(rank, counts, [](int32_t p, int32_t q) { return p + q; });
    double s = 0.0, near = 0.0;
    for (int32_t i = threadIdx.x; i < d.vocab; i += kThreads) {
        const float y = value_of(x[i]) - m, e = __builtin_amdgcn_exp2f(y * kLog2e);
        s += e;
        if (e > 0.0f) near += (double)e * y;
    }
    s = over_group(s, sums, [](double p, double q) { return p + q; });
    near = over_group(near, sums, [](double p, double q) { return p + q; });
    const bool none = !(m > -INFINITY && m < INFINITY);
    const double log_s = none ? NAN : log(s);
    if (threadIdx.x == 0) {
        a.scores[row] = given ? (float)((double)mine - (double)m - log_s) : -INFINITY;
        a.ranks[row] = given ? rank : -1;
        a.entropy[row] = (float)(log_s - near / s);
    }
    uint64_t last = ~0ull;                   // an order of values, the larger first, then of tokens
    for (int k = 0; k < d.top; ++k) {
        uint64_t best = 0;
        for (int32_t i = threadIdx.x; i < d.vocab; i += kThreads) {
            const uint32_t bits = __float_as_uint(value_of(x[i]) + 0.0f);
            const uint64_t key = (uint64_t)(bits >> 31 ? ~bits : bits | 1u << 31) << 32 | (uint32_t)~i;
            if (key < last && key > best) best = key;
        }
        last = over_group(best, keys, [](uint64_t p, uint64_t q) { return p > q ? p : q; });
        if (threadIdx.x == 0) {
            const int32_t i = (int32_t)~(uint32_t)last;
            a.top_tokens[row * d.top + k] = i;
            a.top_scores[row * d.top + k] = (float)((double)value_of(x[i]) - (double)m - log_s);
        }
    }
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
    return 0;
}

extern "C" int reef_ops_token_scores(const reef_token_scores_desc* d, const void* logits, const int32_t* tokens, float* scores, int32_t* ranks, float* entropy,
                                     int32_t* top_tokens, float* top_scores, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "reef_ops_token_scores";
    if (int rc = check(what, d)) return rc;
    if (!d->rows) return 0;
    if (!logits || !aligned(logits, type_bytes(d->type)) || !words(tokens) || !words(scores) || !words(ranks) || !words(entropy) ||
        (d->top && (!words(top_tokens) || !words(top_scores))))
        return refuse(what, "null or unaligned argument");
    const int64_t n = d->rows, need = reef_ops_token_scores_workspace(d);
    if (need && (!rows16(workspace) || workspace_bytes < need))
        return refuse(what, "a workspace of %lld bytes on 16 is needed, %lld are given", (long long)need, (long long)workspace_bytes);
    const Span out[] = {{scores, 4 * n}, {ranks, 4 * n}, {entropy, 4 * n}, {top_tokens, 4 * n * d->top}, {top_scores, 4 * n * d->top}, {workspace, need}};
    const Span in[] = {{logits, ((n - 1) * d->logits_stride + d->vocab) * type_bytes(d->type)}, {tokens, 4 * n}};
    if (overlap(out, in)) return refuse(what, "an output overlaps an input");
    const Args a{*d, logits, tokens, scores, ranks, entropy, top_tokens, top_scores};
    const dim3 grid((unsigned)n), block(kThreads);
    switch (d->type) {
        case REEF_TYPE_F32: return launch(what, token_scores<float>, grid, block, a, stream);
        case REEF_TYPE_F16: return launch(what, token_scores<_Float16>, grid, block, a, stream);
        default: return launch(what, token_scores<__bf16>, grid, block, a, stream);
    }
}
