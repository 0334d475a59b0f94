// Norms and residual sum between two blocks, in one pass over the rows:
//   u = residual_scale * residual + block_scale * channel_scale * act(gate) * norm(block)
//   n = norm(u)
// One workgroup per row; each thread holds its channels in registers from the
// first load to the last store, so every element is read and written once and
// outputs may take the place of the inputs.  Sums are FP32: a thread's
// channels, then its wave's lanes, then the waves, in that order always.
//
// Many rows are bound by their bytes: 4096 x 5120 F32 with both norms takes 63.8 us,
// 5.3 TB/s, the rate of a large copy; in BF16, half the bytes, 42 us, 4.0 TB/s, so there
// the chain of a row's latencies counts as well.  512 rows of 16384 F32 29.4 us, 4.6 TB/s;
// of 32768 63 us, 4.3 TB/s (the F32 instance above 28672 channels spills 16 registers).  Few
// rows are bound by one chain of latencies, launch, loads, two to four sums over the
// workgroup, stores: one row 4.0 us, of which a launch that copies it is 2.9; 333 x 4099
// F16 6.3 us with the two sums of RMS, 7.9 with the four of LAYER, 9.7 with gate, biases and
// channel scale, at 1.3 workgroups a compute unit (8.7 at 4096 channels, without a third
// group for three of them).  So a row has as many threads as leave each two or
// three groups of four channels (5120 at 512), and every load is ahead of the first
// sum; reading the row a second time for the second norm instead of holding it
// would cost another round trip.
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


// A thread's share of a row (or of a vector): groups of four channels, the
// workgroup's groups side by side.  Every group but the last lies inside the
// row: C is the least that covers the width.  A wave whose last group lies
// behind the row leaves it out (`tail`, uniform).
template <int THREADS, int C>
__device__ __forceinline__ bool tail_of_wave(uint32_t width) {
    return ((C - 1) * THREADS + __builtin_amdgcn_readfirstlane(threadIdx.x & ~63u)) * 4 < width;
}
template <class T, int THREADS, int C>
struct Share {
    Raw4<T> raw[C];
    __device__ __forceinline__ void load(const T* row, uint32_t width) {
#pragma unroll
        for (int c = 0; c + 1 < C; ++c) raw[c] = load4(row, (c * THREADS + threadIdx.x) * 4, width, true);
        if (tail_of_wave<THREADS, C>(width)) raw[C - 1] = load4(row, ((C - 1) * THREADS + threadIdx.x) * 4, width, false);
        else raw[C - 1].v = typename Packed<T, 4>::type{};
    }
};

// v -> norm(v) * (offset + weight) + bias over the row.  Channels past the
// width are 0 before and after.  A weight that is not there yet (`late`) is
// loaded behind the sums' inputs, so it arrives while they are added up.
//
// Sums or squares past FP32's range are taken again of the values times a power
// of two; every thread has the same sum, so the whole workgroup does, and rows in
// range pay one comparison for each sum (4096 x 5120 F32 63.9 us with it and
// without).  Only scalars differ behind it: scaling the values themselves took
// 13 registers more, and 65.8 us.
// A LAYER row whose sum reaches 2^103 goes on at 2^-20 of its size (32768 values
// at most then add up to less than 2^124; below 2^103 no value minus the mean leaves
// the range either).  Squares are taken of values times 2^-80, and the reciprocal
// keeps 2^8 that the weights give back, since 1 / 2^128 is below the normal range.
// Infinities and NaN come out as they would without.
template <int THREADS, int C>
__device__ __forceinline__ void normalise(float (&v)[C][4], const NormCall& a, Share<float, THREADS, C>& weight,
                                          const float* late, Share<float, THREADS, C>& bias, const float* with_bias,
                                          bool late_bias, float* slots) {
    const uint32_t width = a.width;
    float eps = a.eps;
    if (late) weight.load(late, width);
    if (a.layer) {
        float s = 0.0f, size = 1.0f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) s += v[c][i];
        s = group_sum<THREADS>(s, slots);
        if (!(fabsf(s) < 0x1p103f)) {
            size = 0x1p-20f;
            eps = fmaxf(eps * size * size, 0x1p-126f);   // beside such a row's deviations, if it has any, nothing
            s = 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) s = __builtin_fmaf(v[c][i], size, s);
            s = group_sum<THREADS>(s, slots + 32);
        }
        const float mean = s / float(width);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t k = (c * THREADS + threadIdx.x) * 4 + i;
                v[c][i] = c + 1 < C || k < width ? __builtin_fmaf(v[c][i], size, -mean) : 0.0f;
            }
    }
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) s = __builtin_fmaf(v[c][i], v[c][i], s);
    s = group_sum<THREADS>(s, slots + 16);
    float back = 1.0f, up = 1.0f;
    if (!(s < __builtin_inff())) {
        constexpr float kDown = 0x1p-80f;
        eps = eps * kDown * kDown;
        up = kDown * 0x1p8f;
        back = 0x1p-8f;
        s = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) s = __builtin_fmaf(v[c][i] * kDown, v[c][i] * kDown, s);
        s = group_sum<THREADS>(s, slots + 48);
    }
    const float inv = up / sqrtf(s / float(width) + eps), offset = a.weight_offset * back;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = v[c][i] * inv * __builtin_fmaf(weight.raw[c].v[i], back, offset);
    if (with_bias) {
        if (late_bias) bias.load(with_bias, width);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[c][i] += bias.raw[c].v[i];
    }
}

// A row's latency is one round trip to memory if every load is issued ahead of
// the first sum, but the loads have to fit the registers.  kEarly: all but
// biases and channel scales, which are loaded where they are used; kAll: those
// too (few calls have them); kLate: rows too wide for either also load the gate
// and the weights where they are used.
enum Loads { kLate, kEarly, kAll };
template <class T, int THREADS, int C, Loads LOADS>
__global__ __launch_bounds__(THREADS) void block_norm_kernel(NormCall a) {
    __shared__ float slots[128];
    const uint64_t row = blockIdx.x;
    const uint32_t width = a.width;
    auto at = [&](const OpRows& r) { return static_cast<const T*>(r.data) + row * r.stride; };
    Share<T, THREADS, C> block, residual, gate;
    Share<float, THREADS, C> post, pre, post_bias, pre_bias, channel;
    constexpr bool EARLY = LOADS != kLate, ALL = LOADS == kAll;
    const bool tail = tail_of_wave<THREADS, C>(width);
    const bool full_gate = a.gate.data && !a.gate_per_row;
    float row_gate = 1.0f;
    if (a.block.data) block.load(at(a.block), width);
    if (EARLY && a.post_weight) post.load(a.post_weight, width);
    if (a.residual.data) residual.load(at(a.residual), width);
    if (EARLY && full_gate) gate.load(at(a.gate), width);
    if (a.gate.data && !full_gate) row_gate = float(ld_global(at(a.gate)));
    if (EARLY && a.pre_weight) pre.load(a.pre_weight, width);
    if (ALL && a.post_bias) post_bias.load(a.post_bias, width);
    if (ALL && a.channel_scale) channel.load(a.channel_scale, width);
    if (ALL && a.pre_bias) pre_bias.load(a.pre_bias, width);

    float v[C][4];
    if (a.block.data) {
#pragma unroll
        for (int c = 0; c < C; ++c) block.raw[c].to(v[c]);
        if (a.post_weight)
            normalise<THREADS>(v, a, post, EARLY ? nullptr : a.post_weight, post_bias, a.post_bias, !ALL, slots);
        if (!EARLY && full_gate) gate.load(at(a.gate), width);
        auto act = [&](float g) { return a.sigmoid ? sigmoid(g) : g; };
        if (!full_gate) row_gate = a.block_scale * (a.gate.data ? act(row_gate) : 1.0f);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (c + 1 == C && !tail) continue;
            float g[4];
            if (full_gate) gate.raw[c].to(g);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[c][i] *= full_gate ? a.block_scale * act(g[i]) : row_gate;
        }
        if (a.channel_scale) {
            if (!ALL) channel.load(a.channel_scale, width);
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[c][i] *= channel.raw[c].v[i];
        }
    } else {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[c][i] = 0.0f;
    }
    if (a.residual.data) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float h[4];
            residual.raw[c].to(h);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[c][i] = __builtin_fmaf(a.residual_scale, h[i], v[c][i]);
        }
    }
    auto store = [&](const OpRows& to) {
        T* out = const_cast<T*>(at(to));
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (c + 1 < C || tail) store4(out, (c * THREADS + threadIdx.x) * 4, width, v[c]);
    };
    if (a.hidden.data) store(a.hidden);
    if (!a.normed.data) return;
    // channels past the width: 0 again, whatever a gate or a bias made of them
#pragma unroll
    for (int i = 0; i < 4; ++i) v[C - 1][i] = ((C - 1) * THREADS + threadIdx.x) * 4 + i < width ? v[C - 1][i] : 0.0f;
    normalise<THREADS>(v, a, pre, EARLY ? nullptr : a.pre_weight, pre_bias, a.pre_bias, !ALL, slots + 64);
    store(a.normed);
}

template <class T>
hipError_t dispatch(const NormCall& a, hipStream_t stream) {
    const dim3 grid{uint32_t(a.rows)};
    auto go = [&](auto kernel, uint32_t threads) {
        hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, stream, a);
        return hipGetLastError();
    };
    const uint32_t w = a.width;
    const bool all = a.post_bias || a.pre_bias || a.channel_scale;
    auto early = [&](auto threads, auto c) {
        constexpr int THREADS = decltype(threads)::value, C = decltype(c)::value;
        return all ? go(block_norm_kernel<T, THREADS, C, kAll>, THREADS)
                   : go(block_norm_kernel<T, THREADS, C, kEarly>, THREADS);
    };
    using std::integral_constant;
    if (w <= 256) return early(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (w <= 1024) return early(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    if (w <= 2048) return early(integral_constant<int, 512>{}, integral_constant<int, 1>{});
    if (w <= 4096) return early(integral_constant<int, 512>{}, integral_constant<int, 2>{});
    if (w <= 6144) return early(integral_constant<int, 512>{}, integral_constant<int, 3>{});
    if (w <= 8192) return early(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
    if (w <= 12288) return early(integral_constant<int, 1024>{}, integral_constant<int, 3>{});
    if (w <= 16384) return go(block_norm_kernel<T, 1024, 4, kLate>, 1024);
    if (w <= 20480) return go(block_norm_kernel<T, 1024, 5, kLate>, 1024);
    if (w <= 24576) return go(block_norm_kernel<T, 1024, 6, kLate>, 1024);
    if (w <= 28672) return go(block_norm_kernel<T, 1024, 7, kLate>, 1024);
    if (w <= 32768) return go(block_norm_kernel<T, 1024, 8, kLate>, 1024);
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
