// Tries every mantissa of the e4m3 scales' quotients (csrc/fp8_scale.hpp) against quotients in 64 bits, rounded once: a
// quotient of two floats is never so near the middle of two floats that its 64-bit value falls on the other side.
#include <cstdio>
#include <initializer_list>

#include "fp8_scale.hpp"

namespace {

constexpr uint32_t kMantissas = 1u << 23;
long failures = 0;

float of_bits(uint32_t b) { return __builtin_bit_cast(float, b); }
uint32_t bits_of(float x) { return __builtin_bit_cast(uint32_t, x); }

void expect(const char* what, float x, float got, float want) {
    if (bits_of(got) == bits_of(want)) return;
    if (++failures <= 10) std::printf("%s(%a) = %a, not %a\n", what, double(x), double(got), double(want));
}

// From every float that is at most a unit away.
void inverses(uint32_t exponent) {
    for (uint32_t m = 0; m < kMantissas; ++m) {
        const float s = of_bits(exponent << 23 | m), want = float(1.0 / double(s));
        for (int unit = -1; unit <= 1; ++unit)
            expect("1 / ", s, stx::inverse_from(s, of_bits(bits_of(want) + uint32_t(unit))), want);
    }
}

// Below the least scale, 2^-126, only that it is below counts.
void quotients(uint32_t exponent) {
    auto least = [](float s) { return s < 0x1p-126f ? 0x1p-126f : s; };
    for (uint32_t m = 0; m < kMantissas; ++m) {
        const float x = of_bits(exponent << 23 | m);
        expect("over_448", x, least(stx::over_448(x)), least(float(double(x) / 448.0)));
    }
}

}  // namespace

int main() {
    // scales: 2^-126 to 2^128 / 448, biased exponents 1 to 246; the steps do not depend on the exponent between
    for (uint32_t e : {1u, 127u, 246u}) inverses(e);
    // largest values: those about the least scale and those at both ends
    for (uint32_t e : {0u, 1u, 8u, 9u, 10u, 127u, 254u}) quotients(e);
    if (failures) return std::printf("%ld failures\n", failures), 1;
    std::printf("all mantissas passed\n");
    return 0;
}
