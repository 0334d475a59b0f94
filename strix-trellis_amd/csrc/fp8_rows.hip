// Rows into the e4m3 layers' blocks, with a scale per row and block of 128
// inputs, and weights with a scale per 128 x 128 block.
//
//   s = max(RN32(max |x| / 448), 2^-126)   q = e4m3(RN32(x * RN32(1 / s))), ties to even
#include "fp8_device.hpp"

namespace stx {

namespace {

// A lane's 32 inputs of a block: 16 piece + 0..15 of either half, of row l % 16.
// Blocks inside the row take whole loads; the last one may end before its 128.
template <class T>
struct Inputs {
    static constexpr int kWidth = 16 / sizeof(T);   // elements of a 16-byte load
    typename Packed<T, kWidth>::type raw[2][16 / kWidth];

    __device__ __forceinline__ void load(const T* row, uint32_t k, uint32_t width, bool full) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 16 / kWidth; ++i) {
                const uint32_t at = k + j * 64 + i * kWidth;
                if (full) {
                    raw[j][i] = ld_packed<kWidth>(row + at);
                } else {
#pragma unroll
                    for (int e = 0; e < kWidth; ++e) raw[j][i][e] = at + e < width ? ld_global(row + at + e) : T(0);
                }
            }
    }
    __device__ __forceinline__ float at(int j, int e) const { return float(raw[j][e / kWidth][e % kWidth]); }
    __device__ __forceinline__ float most() const {
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) m = maximum(m, fabsf(at(j, e)));
        return m;
    }
    __device__ __forceinline__ u32x4 rounded(int j, float inv) const {
        if constexpr (std::is_same_v<T, uint8_t>) {
            return __builtin_bit_cast(u32x4, raw[j][0]);
        } else {
            u32x4 q;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float v[4] = {at(j, 4 * i), at(j, 4 * i + 1), at(j, 4 * i + 2), at(j, 4 * i + 3)};
                q[i] = round4(v, inv);
            }
            return q;
        }
    }
};

__device__ __forceinline__ void put_block(uint8_t* block, int lane, u32x4 a, u32x4 b) {
    st_global(reinterpret_cast<u32x4*>(block + lane * 16), a);
    st_global(reinterpret_cast<u32x4*>(block + 1024 + lane * 16), b);
}

// One wave per block of 16 rows x 128 inputs: a lane rounds 32 inputs of one row, the
// four lanes of a row share its maximum, and the block is written as it lies.  Rows
// past the last repeat it (their products go nowhere).  2048 x 4096 BF16: 6-7 us, 3.9 TB/s of rows and blocks; hundreds
// of rows are one round trip, 3-4 us.
template <class T>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const T* x, uint64_t stride, uint32_t input, uint32_t k_blocks,
                                                       const float* given, uint8_t* blocks, float* scales,
                                                       uint32_t rows, uint32_t s_pitch) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t kb = blockIdx.x * 4 + w, rb = blockIdx.y;
    if (kb >= k_blocks) return;
    const uint32_t m = rb * 16 + (lane & 15), row = m < rows ? m : rows - 1;
    Inputs<T> in;
    in.load(x + row * stride, kb * 128 + (lane >> 4) * 16, input, kb * 128 + 128 <= input);
    float inv = 0.0f, s;
    if constexpr (std::is_same_v<T, uint8_t>) {
        s = ld_global(given + uint64_t(row) * k_blocks + kb);
    } else {
        const BlockScale r = block_scale(across_rows_max(in.most()));
        s = r.s;
        inv = r.inv;
    }
    put_block(blocks + (uint64_t(rb) * k_blocks + kb) * 2048, lane, in.rounded(0, inv), in.rounded(1, inv));
    if (lane < 16 && m < rows) st_global(scales + uint64_t(kb) * s_pitch + m, s);
}

// One workgroup per 128 x 128 block of weights: eight blocks of 16 channels, two to
// a wave.  Channels past the last are zeros.  At preparation only: 129280 x 5120 in e4m3 290 us, 4.6 TB/s.
template <class T>
__global__ __launch_bounds__(256) void fp8_weights_kernel(const T* w, uint64_t stride, uint64_t rows, uint32_t input,
                                                          uint32_t k_blocks, const float* given, uint8_t* blocks,
                                                          uint32_t step, float* scales) {
    __shared__ float wave_most[4];
    const int lane = threadIdx.x & 63, v = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t kb = blockIdx.x, nb = blockIdx.y;
    const bool full = kb * 128 + 128 <= input;
    Inputs<T> in[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint64_t n = uint64_t(nb) * 128 + (v * 2 + i) * 16 + (lane & 15);
        in[i].load(w + (n < rows ? n : rows - 1) * stride, kb * 128 + (lane >> 4) * 16, input, full);
        if (n >= rows) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) in[i].raw[j][e / Inputs<T>::kWidth][e % Inputs<T>::kWidth] = T(0);
        }
    }
    float inv = 0.0f, s;
    if constexpr (std::is_same_v<T, uint8_t>) {
        s = ld_global(given + uint64_t(nb) * k_blocks + kb);
    } else {
        const float most = wave_reduce(maximum(in[0].most(), in[1].most()), maximum);
        if (lane == 0) wave_most[v] = most;
        __syncthreads();
        const BlockScale r =
            block_scale(maximum(maximum(wave_most[0], wave_most[1]), maximum(wave_most[2], wave_most[3])));
        s = r.s;
        inv = r.inv;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint64_t rb = uint64_t(nb) * 8 + v * 2 + i;
        if (rb * 16 >= (rows + 31) / 32 * 32) continue;
        put_block(blocks + ((rb / 2 * step * 2 + rb % 2) * k_blocks + kb) * 2048, lane, in[i].rounded(0, inv),
                  in[i].rounded(1, inv));
    }
    if (threadIdx.x == 0) st_global(scales + uint64_t(nb) * k_blocks + kb, s);
}

// F32 rows to e4m3 rows with a scale per 128 channels: eight lanes share 128 channels
// of a row, 16 each.  Bytes: five a value.
__global__ __launch_bounds__(256) void fp8_round_kernel(const float* h, uint32_t width, uint8_t* y, uint64_t y_stride,
                                                        float* scales, uint32_t rows, uint32_t blocks) {
    const uint64_t unit = uint64_t(blockIdx.x) * 32 + (threadIdx.x >> 3);
    const uint32_t row = uint32_t(unit / blocks), b = uint32_t(unit % blocks), n = b * 128 + (threadIdx.x & 7) * 16;
    if (row >= rows) return;
    const float* from = h + uint64_t(row) * width;
    float v[4][4], most = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        load4(from, n + 4 * i, width, false).to(v[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) most = maximum(most, fabsf(v[i][e]));
    }
    most = maximum(most, dpp<0xB1>(most));    // quad_perm 1,0,3,2
    most = maximum(most, dpp<0x4E>(most));    // quad_perm 2,3,0,1
    most = maximum(most, dpp<0x141>(most));   // row_half_mirror
    const BlockScale r = block_scale(most);
    u32x4 q;
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = round4(v[i], r.inv);
    store_bytes(y + uint64_t(row) * y_stride, n, width, q);
    if ((threadIdx.x & 7) == 0) st_global(scales + uint64_t(row) * blocks + b, r.s);
}

template <class T>
hipError_t rows_of(const OpRows& x, uint64_t rows, uint32_t input, const float* given, uint8_t* blocks, float* scales,
                   hipStream_t stream) {
    const uint32_t kbs = fp8_k_blocks(input);
    hipLaunchKernelGGL(fp8_rows_kernel<T>, dim3((kbs + 3) / 4, uint32_t((rows + 15) / 16)), dim3(256), 0, stream,
                       static_cast<const T*>(x.data), x.stride, input, kbs, given, blocks, scales, uint32_t(rows),
                       uint32_t(fp8_padded_rows(rows)));
    return hipGetLastError();
}

template <class T>
hipError_t weights_of(const OpRows& w, uint64_t rows, uint32_t input, const float* given, uint8_t* blocks,
                      uint32_t step, float* scales, hipStream_t stream) {
    // a launch holds fewer than 2^32 threads, and its grid 2^16 - 1 rows of workgroups
    const uint32_t kbs = fp8_k_blocks(input);
    const uint64_t most = (uint64_t(1) << 23) / kbs, at_once = (most < 32768 ? most : 32768) * 128;
    for (uint64_t n = 0; n < rows; n += at_once) {
        const uint64_t part = rows - n < at_once ? rows - n : at_once;
        hipLaunchKernelGGL(fp8_weights_kernel<T>, dim3(kbs, uint32_t((part + 127) / 128)), dim3(256), 0, stream,
                           static_cast<const T*>(w.data) + n * w.stride, w.stride, part, input, kbs,
                           given ? given + n / 128 * kbs : nullptr, blocks + n / 16 * step * kbs * 2048, step,
                           scales + n / 128 * kbs);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_fp8_rows(const OpRows& x, uint64_t rows, uint32_t input, const float* given, uint8_t* blocks,
                           float* scales, hipStream_t stream) {
    switch (x.type) {
        case kF32: return rows_of<float>(x, rows, input, given, blocks, scales, stream);
        case kF16: return rows_of<_Float16>(x, rows, input, given, blocks, scales, stream);
        case kBF16: return rows_of<__bf16>(x, rows, input, given, blocks, scales, stream);
        case kE4M3: return rows_of<uint8_t>(x, rows, input, given, blocks, scales, stream);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_fp8_weights(const OpRows& w, uint64_t rows, uint32_t input, const float* given, uint8_t* blocks,
                              uint32_t step, float* scales, hipStream_t stream) {
    switch (w.type) {
        case kF32: return weights_of<float>(w, rows, input, given, blocks, step, scales, stream);
        case kF16: return weights_of<_Float16>(w, rows, input, given, blocks, step, scales, stream);
        case kBF16: return weights_of<__bf16>(w, rows, input, given, blocks, step, scales, stream);
        case kE4M3: return weights_of<uint8_t>(w, rows, input, given, blocks, step, scales, stream);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_fp8_round(const float* hidden, uint32_t width, uint8_t* y, uint64_t y_stride, float* scales,
                            uint64_t rows, hipStream_t stream) {
    const uint32_t blocks = (width + 127) / 128;
    hipLaunchKernelGGL(fp8_round_kernel, dim3(uint32_t((rows * blocks + 31) / 32)), dim3(256), 0, stream, hidden, width,
                       y, y_stride, scales, uint32_t(rows), blocks);
    return hipGetLastError();
}

}  // namespace stx
