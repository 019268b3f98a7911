// How paged attention cuts a sequence into shares, and a share into the tiles of its wavefronts: the arithmetic, the same on both sides.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace reef_ops {

constexpr int32_t kLeast = 128;              // tokens a share at least

// Sequences are cut into shares of at most so many tokens, equal ones, so that long sequences among short ones, or few of them, keep
// the device as busy as many.  With the sum of the lengths rounded up by more than its 32-bit additions lose,
// sum ceil(seen / tokens) <= budget + requests, the size of the grid.
// (2^24 requests are 2^14 additions a thread, each off by 2^-24 of the sum at most)
__host__ __device__ inline int32_t tokens_of(float total, int32_t budget) {
    const float each = total * 1.02f / (float)budget;
    if (!(each < 2.0e9f)) return INT32_MAX;
    const int32_t tokens = ((int32_t)each + 32) / 32 * 32;
    return tokens < kLeast ? kLeast : tokens;
}
__host__ __device__ inline int32_t shares_of(int32_t n, int32_t tokens) {
    const int32_t shares = (int32_t)(((uint32_t)n + tokens - 1) / (uint32_t)tokens);
    return shares < 1 ? 1 : shares;
}
// Where share `number` of `count` begins among n tokens: whole tiles of 32, one more for the first ones.  (None is
// empty: n > 128 (count - 1), so there are 4 count - 3 tiles or more.)
__host__ __device__ inline int32_t begin_of(int32_t n, int32_t number, int32_t count) {
    const int32_t tiles = (int32_t)(((uint32_t)n + 31) / 32), each = tiles / count, rest = tiles - each * count;
    return (number * each + (number < rest ? number : rest)) * 32;
}
// Where a wavefront begins that leaves out the first `skip` of the tokens [begin, end), or `end` where there are no more.  (The sum alone would
// pass 2^31 for the longest sequences.)
__host__ __device__ inline int32_t first_of(int32_t begin, int32_t end, int32_t skip) { return skip < end - begin ? begin + skip : end; }

}  // namespace reef_ops
