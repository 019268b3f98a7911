// What the operators on plain device pointers share: refusals, launches, the layout of a paged cache.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "reef_c.h"
#include "reef_hal.h"

namespace reef_ops {

inline int refuse(const char* what, const char* format, ...) {
    char msg[256];
    const int n = std::snprintf(msg, sizeof(msg), "%s: ", what);
    va_list args;
    va_start(args, format);
    std::vsnprintf(msg + n, sizeof(msg) - n, format, args);
    va_end(args);
    reef_hal_set_error(msg);
    return 1;   // Status::Fail
}

template <class Args>
int launch(const char* what, void (*kernel)(Args), dim3 grid, dim3 block, Args args, void* stream) {
    void* p[] = {&args};
    const hipError_t e = hipLaunchKernel((const void*)kernel, grid, block, p, 0, (hipStream_t)stream);
    return e == hipSuccess ? 0 : refuse(what, "%s", hipGetErrorString(e));
}

inline int type_bytes(int type) { return type == REEF_TYPE_F32 ? 4 : type == REEF_TYPE_F16 || type == REEF_TYPE_BF16 ? 2 : 0; }
__host__ __device__ inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
// Two int32 arrays and the like: a pointer that is there and aligned.
inline bool words(const void* p) { return p && aligned(p, 4); }
inline bool rows16(const void* p) { return p && aligned(p, 16); }

// Whether an output shares memory with an input.
struct Span {
    const void* p;
    int64_t bytes;
};
template <int N, int M>
bool overlap(const Span (&out)[N], const Span (&in)[M]) {
    for (const Span& o : out)
        for (const Span& i : in)
            if (o.bytes > 0 && i.bytes > 0 && (const char*)o.p < (const char*)i.p + i.bytes && (const char*)i.p < (const char*)o.p + o.bytes) return true;
    return false;
}

// Whether `count` steps of `stride` elements keep to 16 bytes.
inline bool stride16(int64_t count, int64_t stride, int bytes) { return count <= 1 || (stride >= 0 && stride * bytes % 16 == 0); }

// Whether rows of `dim` values overlap, `n` and `m` steps of two strides that are not negative where there is more than one.
inline bool rows_overlap(int64_t n, int64_t stride_n, int64_t m, int64_t stride_m, int64_t dim) {
    const bool m_first = n <= 1 || (m > 1 && stride_m <= stride_n);
    const int64_t count[2] = {m_first ? m : n, m_first ? n : m}, stride[2] = {m_first ? stride_m : stride_n, m_first ? stride_n : stride_m};
    __int128 extent = dim;
    for (int i = 0; i < 2; ++i) {
        if (count[i] <= 1) continue;
        if (stride[i] < extent) return true;
        extent += (__int128)stride[i] * (count[i] - 1);
    }
    return false;
}

// A layout that the kernels take: rows of 16-byte pieces, none over another, offsets that fit 60 bits.
inline int check_layout(const char* what, const reef_cache_layout& c, int64_t layers = 1, int64_t layer_stride = 0) {
    const int bytes = type_bytes(c.type);
    if (!bytes) return refuse(what, "unknown cache type %d", c.type);
    if (c.blocks < 1 || c.block_size < 1 || c.kv_heads < 1 || (int64_t)c.blocks * c.block_size >= (1ll << 31))
        return refuse(what, "bad cache: %d blocks of %d tokens, %d heads", c.blocks, c.block_size, c.kv_heads);
    if (c.head_dim < 8 || c.head_dim > 256 || c.head_dim % 8) return refuse(what, "head_dim %d is not a multiple of 8 up to 256", c.head_dim);
    int64_t count[4] = {c.kv_heads, c.block_size, c.blocks, layers}, stride[4] = {c.head_stride, c.slot_stride, c.block_stride, layer_stride};
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j + 1 < 4 - i; ++j)
            if (count[j] > 1 && (count[j + 1] <= 1 || stride[j] > stride[j + 1])) {   // (steps of one place go first)
                const int64_t n = count[j], s = stride[j];
                count[j] = count[j + 1], stride[j] = stride[j + 1], count[j + 1] = n, stride[j + 1] = s;
            }
    __int128 extent = c.head_dim;
    for (int i = 0; i < 4; ++i) {
        if (count[i] <= 1) continue;
        if (!stride16(count[i], stride[i], bytes)) return refuse(what, "a cache stride of %lld elements is not a multiple of 16 bytes", (long long)stride[i]);
        if (stride[i] < extent) return refuse(what, "a cache stride of %lld elements lets rows overlap", (long long)stride[i]);
        extent += (__int128)stride[i] * (count[i] - 1);
        if (extent >= (__int128)1 << 60) return refuse(what, "cache too large");
    }
    return 0;
}

// ---- places in a paged cache, the same on both sides ----------------------------------------------
// Element offset of the first head of a block's token `place`, or -1: a block number outside the pool.  (That a token lies within the
// entries of its row is for callers to see to.)
struct PagedView {
    int32_t blocks;
    int64_t block_stride, slot_stride;
};
__host__ __device__ inline int64_t paged_row(const PagedView& v, int32_t entry, int32_t place) {
    return (uint32_t)entry < (uint32_t)v.blocks ? (int64_t)entry * v.block_stride + (int64_t)place * v.slot_stride : -1;
}
// t / by for 0 <= t < 2^31, without a division: with 2^(l-1) < by <= 2^l, floor(t m / 2^(31+l)) for m = floor(2^(31+l) / by) + 1, whose
// excess of at most by over the true quotient's multiple is too small to count below 2^31.  m = 0: by is 1.
struct Divider {
    uint32_t by, m, shift;
};
inline Divider divider(uint32_t by) {
    if (by <= 1) return {1, 0, 0};
    uint32_t l = 1;
    while (l < 31 && (1ull << l) < by) ++l;
    return {by, (uint32_t)((1ull << (31 + l)) / by + 1), l - 1};
}
__host__ __device__ inline uint32_t divided(uint32_t t, const Divider& d) { return d.m ? (uint32_t)((uint64_t)t * d.m >> 32) >> d.shift : t; }

// What a request's length counts for: [0, what a row of the table holds].
__host__ __device__ inline int32_t held_length(int32_t n, int32_t max_blocks, int32_t block_size) {
    const int64_t room = (int64_t)max_blocks * block_size;
    return n < 0 ? 0 : (int64_t)n > room ? (int32_t)room : n;
}

// ---- values in their types --------------------------------------------------------------------------
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

}  // namespace reef_ops
