// Norms and residual sum between two blocks, in one pass over the rows:
//   u = residual_scale * residual + block_scale * channel_scale * act(gate) * norm(block)
//   n = norm(u)
// One workgroup per row; each thread holds its channels in registers from the
// first load to the last store, so every element is read and written once and
// outputs may take the place of the inputs.  Sums are FP32: a thread's
// channels, then its wave's lanes, then the waves, in that order always.
#include "ops_device.hpp"

namespace stx {

namespace {

// Sum over the workgroup, the same in every thread.  `slot` is scratch of 16
// words that no earlier sum of the launch used.
template <int THREADS>
__device__ __forceinline__ float group_sum(float v, float* slot) {
    v = wave_sum(v);
    if constexpr (THREADS > 64) {
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < THREADS / 64; ++i) v += slot[i];
    }
    return v;
}

// v -> norm(v) * (offset + weight) + bias over the row.
template <int THREADS, int C>
__device__ __forceinline__ void normalise(float (&v)[C][4], const NormCall& a, const float* weight, const float* bias,
                                          float* slots) {
    const uint32_t width = a.width;
    float mean = 0.0f;
    if (a.layer) {
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) s += v[c][i];   // channels past the width are 0
        mean = group_sum<THREADS>(s, slots) / float(width);
    }
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t k = (c * THREADS + threadIdx.x) * 4 + i;
            if (a.layer) v[c][i] = k < width ? v[c][i] - mean : 0.0f;
            s = __builtin_fmaf(v[c][i], v[c][i], s);
        }
    s = group_sum<THREADS>(s, slots + 16) / float(width);
    const float inv = 1.0f / sqrtf(s + a.eps);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t k = (c * THREADS + threadIdx.x) * 4;
        if (k >= width) continue;
        float w[4], b[4] = {};
        load_row<4>(weight, k, width, 0.0f, w);
        if (bias) load_row<4>(bias, k, width, 0.0f, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[c][i] = v[c][i] * inv * (a.weight_offset + w[i]);
            if (bias) v[c][i] += b[i];
        }
    }
}

template <class T, int THREADS, int C>
__global__ __launch_bounds__(THREADS) void block_norm_kernel(NormCall a) {
    __shared__ float slots[64];
    const uint64_t row = blockIdx.x;
    const uint32_t width = a.width;
    auto at = [&](const OpRows& r) { return static_cast<const T*>(r.data) + row * r.stride; };
    auto chan = [&](int c) { return (c * THREADS + threadIdx.x) * 4; };
    float v[C][4], g[C][4], h[C][4];
    if (a.block.data) {
#pragma unroll
        for (int c = 0; c < C; ++c) load_row<4>(at(a.block), chan(c), width, 0.0f, v[c]);
    }
    // every load ahead of the first sum
    if (a.residual.data) {
#pragma unroll
        for (int c = 0; c < C; ++c) load_row<4>(at(a.residual), chan(c), width, 0.0f, h[c]);
    }
    float row_gate = 1.0f;
    const bool full_gate = a.gate.data && !a.gate_per_row;
    if (full_gate) {
#pragma unroll
        for (int c = 0; c < C; ++c) load_row<4>(at(a.gate), chan(c), width, 0.0f, g[c]);
    } else if (a.gate.data) {
        row_gate = float(ld_global(at(a.gate)));
        if (a.sigmoid) row_gate = 1.0f / (1.0f + expf(-row_gate));
    }
    if (a.block.data && a.post_weight) normalise<THREADS>(v, a, a.post_weight, a.post_bias, slots);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t k = chan(c);
        if (a.block.data) {
            float cs[4];
            if (a.channel_scale) load_row<4>(a.channel_scale, k, width, 0.0f, cs);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float t = v[c][i] * row_gate;
                if (full_gate) t *= a.sigmoid ? 1.0f / (1.0f + expf(-g[c][i])) : g[c][i];
                if (a.channel_scale) t *= cs[i];
                v[c][i] = a.block_scale * t;
                if (a.residual.data) v[c][i] = __builtin_fmaf(a.residual_scale, h[c][i], v[c][i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[c][i] = a.residual_scale * h[c][i];
        }
        if (a.hidden.data) store_row<4>(const_cast<T*>(at(a.hidden)), k, width, v[c]);
    }
    if (!a.normed.data) return;
    // channels past the width: 0 again, whatever a gate made of them
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = chan(c) + i < width ? v[c][i] : 0.0f;
    normalise<THREADS>(v, a, a.pre_weight, a.pre_bias, slots + 32);
#pragma unroll
    for (int c = 0; c < C; ++c) store_row<4>(const_cast<T*>(at(a.normed)), chan(c), width, v[c]);
}

template <class T>
hipError_t dispatch(const NormCall& a, hipStream_t stream) {
    const dim3 grid{uint32_t(a.rows)};
    auto go = [&](auto kernel, uint32_t threads) {
        hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, stream, a);
        return hipGetLastError();
    };
    const uint32_t width = a.width;
    if (width <= 256) return go(block_norm_kernel<T, 64, 1>, 64);
    if (width <= 1024) return go(block_norm_kernel<T, 256, 1>, 256);
    if (width <= 2048) return go(block_norm_kernel<T, 256, 2>, 256);
    if (width <= 5120) return go(block_norm_kernel<T, 256, 5>, 256);
    if (width <= 8192) return go(block_norm_kernel<T, 512, 4>, 512);
    if (width <= 16384) return go(block_norm_kernel<T, 1024, 4>, 1024);
    if (width <= 32768) return go(block_norm_kernel<T, 1024, 8>, 1024);
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_block_norm(const NormCall& call, uint32_t type, hipStream_t stream) {
    // a launch holds fewer than 2^32 threads
    constexpr uint64_t kRows = 1u << 20;
    NormCall part = call;
    for (uint64_t left = call.rows; left;) {
        part.rows = left < kRows ? left : kRows;
        hipError_t e = hipErrorInvalidValue;
        switch (type) {
            case kF32: e = dispatch<float>(part, stream); break;
            case kF16: e = dispatch<_Float16>(part, stream); break;
            case kBF16: e = dispatch<__bf16>(part, stream); break;
        }
        if (e != hipSuccess) return e;
        left -= part.rows;
        for (OpRows* r : {&part.block, &part.residual, &part.gate, &part.hidden, &part.normed})
            if (r->data) r->data = static_cast<const char*>(r->data) + part.rows * r->stride * (type == kF32 ? 4 : 2);
    }
    return hipSuccess;
}

}  // namespace stx
