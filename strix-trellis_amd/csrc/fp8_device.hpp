// Device parts that the kernels of the e4m3 layers share: rounding to e4m3 with a
// scale, fragments of blocks, and what becomes of the sums.
#pragma once
#include "fp8.hpp"
#include "fp8_scale.hpp"
#include "ops_device.hpp"

namespace stx {

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

constexpr float kLeastScale = 0x1p-126f;

__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// s = max(RN32(most / 448), 2^-126) and its inverse; a block with an infinity or
// a NaN has most = inf or NaN (the maximum passes NaN on), and with it s; its
// values become NaN (inf * 0, x * NaN) or meet that s in the sum.
struct BlockScale {
    float s, inv;
};
// Both quotients are the rounded ones (fp8_scale.hpp), given that the instruction's reciprocal is off by at
// most a unit.  Only an infinity needs a step of its own.
__device__ __forceinline__ BlockScale block_scale(float most) {
    BlockScale r;
    const bool infinite = most == __builtin_inff();
    const float s = maximum(over_448(most), kLeastScale);
    r.s = infinite ? most : s;
    r.inv = infinite ? 0.0f : inverse_from(s, __builtin_amdgcn_rcpf(s));
    return r;
}
// e4m3 of RN32(v * inv), four to a word.  |v * inv| <= 448 (1 + 2^-22), which rounds to 448.
__device__ __forceinline__ uint32_t round4(const float (&v)[4], float inv) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, r, true));
}

// Largest of a half-wave's 32 lanes, to all of them.
__device__ __forceinline__ float half_wave_max(float v) {
    v = maximum(v, dpp<0xB1>(v));    // quad_perm 1,0,3,2
    v = maximum(v, dpp<0x4E>(v));    // quad_perm 2,3,0,1
    v = maximum(v, dpp<0x141>(v));   // row_half_mirror
    v = maximum(v, dpp<0x140>(v));   // row_mirror
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return maximum(__builtin_bit_cast(float, uint32_t(a[0])), __builtin_bit_cast(float, uint32_t(a[1])));
}
// Largest of lanes l, l ^ 16, l ^ 32 and l ^ 48, to all of them.
__device__ __forceinline__ float across_rows_max(float v) {
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = maximum(__builtin_bit_cast(float, uint32_t(a[0])), __builtin_bit_cast(float, uint32_t(a[1])));
    u = __builtin_bit_cast(uint32_t, v);
    const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return maximum(__builtin_bit_cast(float, uint32_t(b[0])), __builtin_bit_cast(float, uint32_t(b[1])));
}

// ---- products of a block ----
// The 8-bit MFMAs (f8f6f4, at twice the rate of the 16-bit ones) align the products of eight
// neighbouring inputs of a lane to the largest of them and drop what lies below 2^-13 of it:
// 1.25e-5 of a random block's sum in the 2-norm, measured, where FP32 sums have 1e-7.
// That is far below a 16-bit output's half step (2^-12 of the value for F16, 2^-9 for BF16), and those
// outputs take them.  F32 outputs do not, nor e4m3 ones, which come with F32 scales: their operands are
// converted to FP16, which holds every e4m3 value, and the 16-bit MFMAs sum their
// products in FP32 (1.3e-8 of a random block's sum, measured).
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ i32x8 operand(u32x4 a, u32x4 b) {
    return i32x8{int(a[0]), int(a[1]), int(a[2]), int(a[3]), int(b[0]), int(b[1]), int(b[2]), int(b[3])};
}
// Eight e4m3 values as FP16.
__device__ __forceinline__ f16x8 widened(uint32_t a, uint32_t b) {
    const f16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true)};
    return f16x8{v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
}
__device__ __forceinline__ f16x4 widened4(uint32_t a) {
    const f16x2 v[2] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true)};
    return f16x4{v[0][0], v[0][1], v[1][0], v[1][1]};
}
// 16 channels x 16 rows: a lane's 32 inputs of either operand.
__device__ __forceinline__ f32x4 product16(const u32x4 (&w)[2], const f16x8 (&x)[4]) {
    f32x4 p{};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        p = __builtin_amdgcn_mfma_f32_16x16x32_f16(widened(w[i / 2][i % 2 * 2], w[i / 2][i % 2 * 2 + 1]), x[i], p, 0, 0, 0);
    return p;
}
template <bool EXACT>
__device__ __forceinline__ f32x4 product16(const u32x4 (&w)[2], const u32x4 (&x)[2]) {
    f32x4 p{};
    if constexpr (EXACT) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            p = __builtin_amdgcn_mfma_f32_16x16x32_f16(widened(w[i / 2][i % 2 * 2], w[i / 2][i % 2 * 2 + 1]),
                                                       widened(x[i / 2][i % 2 * 2], x[i / 2][i % 2 * 2 + 1]), p, 0, 0, 0);
    } else {
        p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w[0], w[1]), operand(x[0], x[1]), p, 0, 0, 0, 0, 0, 0);
    }
    return p;
}
// A value that is the same for a whole wave and that no kernel running meanwhile writes:
// a scalar load, which does not count among the vector loads in flight.
__device__ __forceinline__ float ld_uniform(const float* p) {
    return *(const __attribute__((address_space(4))) float*)(p);
}

struct Fp8Args {
    const uint8_t* w;         // blocks of weights
    const uint8_t* x;         // blocks of rows
    const float *t, *s;       // scales of weights, of rows ([k_blocks][s_pitch], or as given)
    const float* bias;        // null: none
    void* y;
    uint64_t y_stride;
    float* y_scales;          // wide cores, e4m3 output
    uint32_t y_type;
    uint32_t rows, output, k_blocks, s_pitch;   // s_pitch: padded rows
    uint32_t t_up, bias_up;   // where a pair's up scales and biases start
    uint32_t activation;
    float alpha, beta;
    uint32_t n_tiles, m_tiles;
};

// act(g) u.  silu(g) = g sigmoid(g); the tanh form of gelu is g sigmoid(2 z) with
// z = sqrt(2 / pi) (g + 0.044715 g^3), as (1 + tanh z) / 2 = sigmoid(2 z).
__device__ __forceinline__ float gated(float g, float u, uint32_t activation) {
    constexpr float kTwo = 1.59576912160573071176f;   // 2 sqrt(2 / pi)
    return g * sigmoid(activation == kSilu ? g : kTwo * __builtin_fmaf(0.044715f * g * g, g, g)) * u;
}

// 16 bytes of a row of `width`, at its column n.
__device__ __forceinline__ void store_bytes(uint8_t* row, uint32_t n, uint32_t width, u32x4 q) {
    if (n + 16 <= width) {
        st_packed<16>(row + n, __builtin_bit_cast(Packed<uint8_t, 16>::type, q));
    } else {
#pragma unroll
        for (int i = 0; i < 15; ++i)
            if (n + i < width) st_global(row + n + i, uint8_t(q[i / 4] >> (8 * (i % 4))));
    }
}

template <class T>
__device__ __forceinline__ void emit4(const Fp8Args& a, uint32_t m, uint32_t n, f32x4 v, bool linear) {
    T* row = static_cast<T*>(a.y) + uint64_t(m) * a.y_stride;
    float o[4], old[4];
    const bool add = linear && a.beta != 0.0f;
    if (add) load4(static_cast<const T*>(row), n, a.output, false).to(old);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        o[i] = linear ? v[i] * a.alpha : v[i];
        if (add) o[i] += a.beta * old[i];
    }
    store4(row, n, a.output, o);
}
// Channels n .. n + 3 of row m, from their sums with the bias.
__device__ __forceinline__ void emit(const Fp8Args& a, uint32_t m, uint32_t n, f32x4 v, bool linear) {
    if (a.y_type == kF32) emit4<float>(a, m, n, v, linear);
    else if (a.y_type == kBF16) emit4<__bf16>(a, m, n, v, linear);
    else emit4<_Float16>(a, m, n, v, linear);
}
__device__ __forceinline__ f32x4 with_bias(const Fp8Args& a, uint32_t at, f32x4 v) {
    return a.bias ? v + ld_global(reinterpret_cast<const f32x4*>(a.bias + at)) : v;
}
__device__ __forceinline__ f32x4 gated4(const Fp8Args& a, uint32_t n, f32x4 g, f32x4 u) {
    g = with_bias(a, n, g);
    u = with_bias(a, a.bias_up + n, u);
    f32x4 h;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = gated(g[i], u[i], a.activation);
    return h;
}

}  // namespace stx
