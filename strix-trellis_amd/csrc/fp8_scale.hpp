// The quotients of the e4m3 rounding rule, RN32(most / 448) and RN32(1 / s), in fewer
// steps than a division takes that has to reach every pair of operands.  Plain arithmetic, which
// the kernels share with a host test that tries every mantissa.  (Templates, as a plain constexpr
// function, which either side may call, cannot name an fma.)
#pragma once
#include <cstdint>

namespace stx {

// RN32(x / 448), x not infinite: a product corrected once by its residual.
template <class Float>
constexpr Float over_448(Float x) {
    constexpr Float kBy = 1.0f / 448.0f;
    const Float q = x * kBy;
    return __builtin_fmaf(__builtin_fmaf(-448.0f, q, x), kBy, q);
}

// RN32(1 / s) of a normal s with a normal inverse, from a float y at most one unit from it: two Newton
// steps, which end on it for every mantissa but one.  s = 2^k (2 - 2^-23), all bits set, has its
// inverse 2^-(k + 1) (1 + 2^-24 + ..) a hair above the middle of two floats, and the steps may
// end on the lower one, 2^-(k + 1), whose last bit is then set; the upper one has it set.
template <class Float>
constexpr Float inverse_from(Float s, Float y) {
    constexpr uint32_t kMantissa = 0x7FFFFF;
    y = __builtin_fmaf(__builtin_fmaf(-s, y, 1.0f), y, y);
    y = __builtin_fmaf(__builtin_fmaf(-s, y, 1.0f), y, y);
    const bool full = (__builtin_bit_cast(uint32_t, s) & kMantissa) == kMantissa;
    return __builtin_bit_cast(Float, __builtin_bit_cast(uint32_t, y) | uint32_t(full));
}

}  // namespace stx
