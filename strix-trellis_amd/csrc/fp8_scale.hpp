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
// steps, the last one's residual a unit of its own higher.  Without that they end on it for every mantissa
// but one: s = 2^k (2 - 2^-23) has its inverse 2^-(k + 1) (1 + 2^-24 + 2^-48 ..) a hair above the middle of two floats,
// from the lower of which the residual, 2^-24, loses that hair and leads to the middle, which goes down.
template <class Float>
constexpr Float inverse_from(Float s, Float y) {
    y = __builtin_fmaf(__builtin_fmaf(-s, y, 1.0f), y, y);
    const Float e = __builtin_fmaf(-s, y, 1.0f);
    return __builtin_fmaf(__builtin_fmaf(__builtin_fabsf(e), 0x1.8p-24f, e), y, y);   // 0.75 to 1.5 units of e
}

}  // namespace stx
