// What the kernels behind the output head share: a token's place in the order of
// its row as one key, and running statistics of a row (token_logprobs.hip).
#pragma once
#include "ops_device.hpp"

namespace stx {

constexpr float kLowest = -3.40282346638528859812e38f, kInf = __builtin_inff();

__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);   // -0 counts as 0
    return uint64_t(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | uint32_t(~id);
}
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t b = uint32_t(key >> 32);
    return __builtin_bit_cast(float, b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}
__device__ __forceinline__ uint32_t id_of(uint64_t key) { return ~uint32_t(key); }

struct Stats {
    float m, n, s, h;
};
constexpr Stats kNothing = {kLowest, 0.0f, 0.0f, 0.0f};

// Distances past 2^24 have no weight at any admitted scale (2^24 times 2^-16
// log2 e is over 300); kept finite, a weight of 0 times one is 0.
__device__ __forceinline__ float power(float d, float c) { return fmaxf(d, -0x1p24f) * c; }

// Statistics p against the larger maximum m.
__device__ __forceinline__ Stats against(const Stats& p, float m, float c) {
    const float d = power(p.m - m, c), f = __builtin_amdgcn_exp2f(d), t = p.n + p.s;
    return p.m == m ? p : Stats{m, 0.0f, f * t, f * __builtin_fmaf(t, d, p.h)};
}
__device__ __forceinline__ void join(Stats& a, const Stats& b, float c) {
    const float m = fmaxf(a.m, b.m);
    const Stats x = against(a, m, c), y = against(b, m, c);
    a = {m, x.n + y.n, x.s + y.s, x.h + y.h};
}
// Joins the lanes' statistics; every lane gets the result.
__device__ __forceinline__ Stats join_lanes(const Stats& mine, float c) {
    const float m = wave_max(mine.m);
    const Stats x = against(mine, m, c);
    return {m, wave_sum(x.n), wave_sum(x.s), wave_sum(x.h)};
}

}  // namespace stx
