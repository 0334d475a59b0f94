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

// Elements [k, k + N) of a row of `width`, as floats; `fill` past its end.
template <int N, class T>
__device__ __forceinline__ void load_row(const T* row, uint32_t k, uint32_t width, float fill, float (&v)[N]) {
    if (k + N <= width) {
        const auto x = ld_packed<N>(row + k);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = float(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = k + i < width ? float(ld_global(row + k + i)) : fill;
    }
}
template <int N, class T>
__device__ __forceinline__ void store_row(T* row, uint32_t k, uint32_t width, const float (&v)[N]) {
    if (k + N <= width) {
        typename Packed<T, N>::type x;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = T(v[i]);
        st_packed<N>(row + k, x);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (k + i < width) st_global(row + k + i, T(v[i]));
    }
}

// Wave-wide sum and maximum (every lane gets the result).
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int s = 32; s; s >>= 1) v = fmaxf(v, __shfl_xor(v, s));
    return v;
}

}  // namespace stx
