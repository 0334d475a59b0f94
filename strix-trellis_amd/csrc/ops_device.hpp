// Device helpers of the operators around the trellis layers: rows of F32, F16,
// BF16 or I8 elements at any element alignment, and wave reductions.
#pragma once
#include <type_traits>

#include "ops.hpp"
#include "trellis.hpp"

namespace stx {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <class T>
constexpr uint32_t op_type = std::is_same_v<T, float>      ? uint32_t(kF32)
                             : std::is_same_v<T, _Float16> ? uint32_t(kF16)
                             : std::is_same_v<T, __bf16>   ? uint32_t(kBF16)
                                                           : uint32_t(kI8);

// N consecutive elements from an address aligned to one element only: gfx950
// serves vector accesses at any alignment, so rows of odd widths and strides
// take the same loads as aligned ones.
template <class T, int N>
struct Packed {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <int N, class T>
__device__ __forceinline__ typename Packed<T, N>::type ld_packed(const T* p) {
    return *(const __attribute__((address_space(1))) typename Packed<T, N>::type*)(p);
}
template <int N, class T>
__device__ __forceinline__ void st_packed(T* p, typename Packed<T, N>::type v) {
    *(__attribute__((address_space(1))) typename Packed<T, N>::type*)(p) = v;
}
template <class T>
__device__ __forceinline__ void st_global(T* p, T v) {
    *(__attribute__((address_space(1))) T*)(p) = v;
}

// Four elements as loaded, converted only where they are used, so that a wait
// for them stands behind every load issued in between.
template <class T>
struct Raw4 {
    typename Packed<T, 4>::type v;
    __device__ __forceinline__ void to(float (&f)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = float(v[i]);
    }
};

// Elements [k, k + 4) of a row of `width`, zeros past its end.  A group that
// lies inside by construction (`full`) is one load.  Otherwise the load is
// moved back into the row and its elements shifted down, without a branch;
// rows of fewer than four elements go one by one.
template <class T>
__device__ __forceinline__ Raw4<T> load4(const T* row, uint32_t k, uint32_t width, bool full) {
    Raw4<T> r;
    if (full) {
        r.v = ld_packed<4>(row + k);
        return r;
    }
    if (width < 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.v[i] = k + i < width ? ld_global(row + k + i) : T(0);
        return r;
    }
    const uint32_t at = k < width - 4 ? k : width - 4, by = k - at;   // by >= 4: nothing is left
    r.v = ld_packed<4>(row + at);
    if constexpr (sizeof(T) == 2) {
        const uint64_t u = __builtin_bit_cast(uint64_t, r.v);
        r.v = __builtin_bit_cast(decltype(r.v), by < 4 ? u >> (16 * (by & 3)) : uint64_t(0));
    } else {
        T e[4] = {r.v[0], r.v[1], r.v[2], r.v[3]};
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = by & 1 ? (i < 3 ? e[i + 1] : T(0)) : e[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = by & 2 ? (i < 2 ? e[i + 2] : T(0)) : e[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) r.v[i] = by < 4 ? e[i] : T(0);
    }
    return r;
}
template <class T>
__device__ __forceinline__ void store4(T* row, uint32_t k, uint32_t width, const float (&f)[4]) {
    if (k + 4 <= width) {
        typename Packed<T, 4>::type x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = T(f[i]);
        st_packed<4>(row + k, x);
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (k + i < width) st_global(row + k + i, T(f[i]));
    }
}

// Wave-wide reductions (every lane gets the result): neighbours, quads, halves
// of a row of 16 and rows through DPP operands, then rows against each other
// through the swaps of 16 and 32 lanes.  No LDS round trip.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <class F>
__device__ __forceinline__ float wave_reduce(float v, F op) {
    v = op(v, dpp<0xB1>(v));    // quad_perm 1,0,3,2
    v = op(v, dpp<0x4E>(v));    // quad_perm 2,3,0,1
    v = op(v, dpp<0x141>(v));   // row_half_mirror
    v = op(v, dpp<0x140>(v));   // row_mirror
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = op(__builtin_bit_cast(float, uint32_t(a[0])), __builtin_bit_cast(float, uint32_t(a[1])));
    u = __builtin_bit_cast(uint32_t, v);
    const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return op(__builtin_bit_cast(float, uint32_t(b[0])), __builtin_bit_cast(float, uint32_t(b[1])));
}
__device__ __forceinline__ float wave_sum(float v) {
    return wave_reduce(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_max(float v) {
    return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}

}  // namespace stx
