// 8-bit integer linear layer: y = alpha * (s[m] t[n] sum_i q[m][i] w[n][i] + bias[n]) + beta * y.
//
// Activations are rounded to int8 per token (int8_stage_kernel) into the same
// block order the prepared weights have, so that both MFMA operands are read
// as whole 1 KiB blocks, 16 bytes per lane.  The integer sums are exact, so
// neither the split of K nor the tile a row falls into changes a bit.
#include "ops_device.hpp"

namespace stx {

namespace {

constexpr float kLeastScale = 0x1p-126f;

// q = x / s to the nearest integer, ties to even.  The estimate x * (1 / s) is
// off by less than 2^-16, so its nearest integer is off by one at most; r = x -
// q s is exact in the fma (a multiple of ulp(s) / 2 below 2 s), so its
// comparison with s / 2 decides the exact quotient's rounding.
__device__ __forceinline__ int quotient(float x, float s, float inv) {
    const float q0 = rintf(x * inv);
    const float r = __builtin_fmaf(-q0, s, x), half = 0.5f * s;
    const int q = int(q0);
    const int up = r > half || (r == half && (q & 1)), down = r < -half || (r == -half && (q & 1));
    return q + up - down;
}

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    return uint32_t(a & 255) | uint32_t(b & 255) << 8 | uint32_t(c & 255) << 16 | uint32_t(d) << 24;
}

// ---- rows into blocks ----
// One wave per row; a lane takes 16 consecutive inputs at a time (one 16-byte
// piece of a block).  With ROUNDS > 0 the row stays in registers between the
// maximum and the rounding (rows of up to 1024 ROUNDS inputs), otherwise it is
// read twice.  Rows past the last and inputs past the width become zeros.
template <class T, int ROUNDS>
__global__ __launch_bounds__(256) void int8_stage_kernel(const T* x, uint64_t stride, uint64_t rows, uint32_t input,
                                                         uint32_t k_blocks, const float* given, int8_t* blocks,
                                                         float* scales) {
    const int lane = threadIdx.x & 63;
    const uint64_t row = uint64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const uint32_t padded = k_blocks * 64, k0 = lane * 16;
    int8_t* to = blocks + (row >> 4) * k_blocks * 1024 + (row & 15) * 16;
    // the piece of inputs k .. k + 15
    auto put = [&](uint32_t k, u32x4 v) {
        st_global(reinterpret_cast<u32x4*>(to + uint64_t(k >> 6) * 1024 + ((k >> 4) & 3) * 256), v);
    };
    if (row >= rows) {
        for (uint32_t k = k0; k < padded; k += 1024) put(k, u32x4{});
        return;
    }
    const T* from = x + row * stride;
    if constexpr (std::is_same_v<T, int8_t>) {
        for (uint32_t k = k0; k < padded; k += 1024) {
            u32x4 v{};
            if (k + 16 <= input) {
                v = __builtin_bit_cast(u32x4, ld_packed<16>(from + k));
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (k + i < input) v[i / 4] |= uint32_t(uint8_t(ld_global(from + k + i))) << (8 * (i & 3));
            }
            put(k, v);
        }
        if (given && lane == 0) st_global(scales + row, ld_global(given + row));
    } else {
        constexpr int R = ROUNDS ? ROUNDS : 1;
        float v[R][16];
        float most = 0.0f, bad = 0.0f;   // bad: 0, or NaN once an infinity or a NaN was seen
        auto look = [&](const float (&u)[16]) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                most = fmaxf(most, fabsf(u[i]));
                bad += u[i] * 0.0f;
            }
        };
        if constexpr (ROUNDS > 0) {
#pragma unroll
            for (int c = 0; c < R; ++c) load_row<16>(from, k0 + c * 1024, input, 0.0f, v[c]);
#pragma unroll
            for (int c = 0; c < R; ++c) look(v[c]);
        } else {
            for (uint32_t k = k0; k < input; k += 1024) {
                load_row<16>(from, k, input, 0.0f, v[0]);
                look(v[0]);
            }
        }
        most = wave_max(most);
        bad = wave_sum(bad);
        const bool fine = bad == 0.0f;
        float s = fmaxf(most / 127.0f, kLeastScale);
        const float inv = 1.0f / s;
        auto round16 = [&](const float (&u)[16]) {
            u32x4 q;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                q[j] = pack4(quotient(u[4 * j], s, inv), quotient(u[4 * j + 1], s, inv),
                             quotient(u[4 * j + 2], s, inv), quotient(u[4 * j + 3], s, inv));
            return fine ? q : u32x4{};
        };
        if constexpr (ROUNDS > 0) {
#pragma unroll
            for (int c = 0; c < R; ++c)
                if (k0 + c * 1024 < padded) put(k0 + c * 1024, round16(v[c]));
        } else {
            for (uint32_t k = k0; k < padded; k += 1024) {
                load_row<16>(from, k, input, 0.0f, v[0]);
                put(k, round16(v[0]));
            }
        }
        if (lane == 0) st_global(scales + row, fine ? s : __builtin_nanf(""));
    }
}

// ---- products ----
struct Int8Args {
    const int8_t* w;          // [N/16][k_blocks][1 KiB]
    const int8_t* x;          // [M/16][k_blocks][1 KiB]
    const float *t, *s, *bias;
    void* y;
    uint64_t y_stride;
    uint32_t y_type;
    uint32_t rows, output, k_blocks;
    float alpha, beta;
};

// Channels n .. n + 3 of row m from their integer sums.  Channels past the
// last read padded scales; their values go nowhere.
struct Channels {
    f32x4 t, b;
    bool bias;
};
__device__ __forceinline__ Channels channels_of(const Int8Args& a, uint32_t n) {
    Channels c;
    c.t = ld_global(reinterpret_cast<const f32x4*>(a.t + n));
    c.bias = a.bias != nullptr;
    c.b = c.bias ? ld_global(reinterpret_cast<const f32x4*>(a.bias + n)) : f32x4{};
    return c;
}

template <class T>
__device__ __forceinline__ void emit4(const Int8Args& a, uint32_t m, uint32_t n, i32x4 acc, float s,
                                      const Channels& c) {
    T* row = static_cast<T*>(a.y) + uint64_t(m) * a.y_stride;
    float v[4], old[4];
    if (a.beta != 0.0f) load_row<4>(row, n, a.output, 0.0f, old);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = float(acc[i]) * s * c.t[i];
        if (c.bias) v[i] += c.b[i];
        v[i] *= a.alpha;
        if (a.beta != 0.0f) v[i] += a.beta * old[i];
    }
    store_row<4>(row, n, a.output, v);
}
__device__ __forceinline__ void emit(const Int8Args& a, uint32_t m, uint32_t n, i32x4 acc, float s,
                                     const Channels& c) {
    if (a.y_type == kF32) emit4<float>(a, m, n, acc, s, c);
    else if (a.y_type == kBF16) emit4<__bf16>(a, m, n, acc, s, c);
    else emit4<_Float16>(a, m, n, acc, s, c);
}

// Few rows (1..16): one workgroup per 16 channels, its eight waves split K and
// add their sums in LDS.
__global__ __launch_bounds__(512) void int8_rows16_kernel(Int8Args a) {
    __shared__ i32x4 part[8][64];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t kb0 = a.k_blocks * w / 8, kb1 = a.k_blocks * (w + 1) / 8;
    const auto wr = make_rsrc(a.w + uint64_t(blockIdx.x) * a.k_blocks * 1024, kb1 * 1024);
    const auto xr = make_rsrc(a.x, kb1 * 1024);
    constexpr int U = 10;
    i32x4 acc{};
    for (uint32_t kb = kb0; kb < kb1; kb += U) {
        u32x4 f[U], g[U];   // blocks past kb1 read zeros
#pragma unroll
        for (int u = 0; u < U; ++u)
            f[u] = __builtin_amdgcn_raw_buffer_load_b128(wr, (kb + u) * 1024 + lane * 16, 0, 0);
#pragma unroll
        for (int u = 0; u < U; ++u)
            g[u] = __builtin_amdgcn_raw_buffer_load_b128(xr, (kb + u) * 1024 + lane * 16, 0, 0);
#pragma unroll
        for (int u = 0; u < U; ++u)
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, f[u]),
                                                        __builtin_bit_cast(i32x4, g[u]), acc, 0, 0, 0);
    }
    part[w][lane] = acc;
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int j = 1; j < 8; ++j) acc += part[j][lane];
    const uint32_t m = lane & 15, n = blockIdx.x * 16 + 4 * (lane >> 4);
    if (m < a.rows) emit(a, m, n, acc, ld_global(a.s + m), channels_of(a, n));
}

// Tiles of 128 channels x 128 rows, four waves of 64 x 64, both operands in a
// ring of LDS stages of 64 inputs.
__global__ __launch_bounds__(256) void int8_tile_kernel(Int8Args a, uint32_t n_tiles) {
    constexpr int kStage = 16384, kRing = 4;
    __shared__ __align__(16) unsigned char ring[kRing * kStage];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t nt = blockIdx.x % n_tiles, mt = blockIdx.x / n_tiles;
    const uint32_t nb = (a.output + 31) / 32 * 2, mb = (a.rows + 31) / 32 * 2, kbs = a.k_blocks;
    const uint32_t nb0 = nt * 8, mb0 = mt * 8;
    const uint32_t nbn = nb - nb0 < 8 ? nb - nb0 : 8, mbn = mb - mb0 < 8 ? mb - mb0 : 8;
    const auto wr = make_rsrc(a.w + uint64_t(nb0) * kbs * 1024, nbn * kbs * 1024);
    const auto xr = make_rsrc(a.x + uint64_t(mb0) * kbs * 1024, mbn * kbs * 1024);
    const uint32_t pair = kbs * 1024;
    auto dma = [&](uint32_t kb) {
        unsigned char* base = ring + (kb % kRing) * kStage + 2 * w * 1024;
        const uint32_t off = (kb < kbs ? kb * 1024 + lane * 16 : 0x80000000u);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (__attribute__((address_space(3))) void*)(base + j * 1024), 16,
                                                     off + (2 * w + j) * pair, 0, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                xr, (__attribute__((address_space(3))) void*)(base + 8192 + j * 1024), 16, off + (2 * w + j) * pair, 0, 0,
                0);
        }
    };
    const int wn = w & 1, wm = w >> 1, h = lane >> 5, r16 = lane & 15, hi = (lane >> 4) & 1;
    i32x16 acc[2][2] = {};
    dma(0);
    dma(1);
    dma(2);
    for (uint32_t kb = 0; kb < kbs; ++kb) {
        asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        dma(kb + 3);
        const unsigned char* st = ring + (kb % kRing) * kStage;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            i32x4 f[2], g[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                f[i] = *reinterpret_cast<const i32x4*>(st + (wn * 4 + i * 2 + hi) * 1024 + ((2 * j + h) * 16 + r16) * 16);
                g[i] = *reinterpret_cast<const i32x4*>(st + 8192 + (wm * 4 + i * 2 + hi) * 1024 +
                                                       ((2 * j + h) * 16 + r16) * 16);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) acc[i][k] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f[i], g[k], acc[i][k], 0, 0, 0);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint32_t m = mt * 128 + wm * 64 + k * 32 + (lane & 31);
        if (m >= a.rows) continue;
        const float s = ld_global(a.s + m);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t n = nt * 128 + wn * 64 + i * 32 + 8 * q + 4 * h;
                if (n < a.output)
                    emit(a, m, n, i32x4{acc[i][k][4 * q], acc[i][k][4 * q + 1], acc[i][k][4 * q + 2], acc[i][k][4 * q + 3]}, s,
                         channels_of(a, n));
            }
    }
}

__global__ __launch_bounds__(256) void copy_f32_kernel(const float* from, float* to, uint64_t count) {
    const uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x;
    if (i < count) st_global(to + i, ld_global(from + i));
}

template <class T>
void stage(const OpRows& x, uint64_t rows, uint32_t input, const float* given, int8_t* blocks, float* scales,
           hipStream_t stream) {
    const dim3 grid(uint32_t(int8_row_blocks(rows) * 4)), block(256);
    const uint32_t kb = int8_k_blocks(input);
    const T* from = static_cast<const T*>(x.data);
    if (input <= 5120)
        hipLaunchKernelGGL((int8_stage_kernel<T, 5>), grid, block, 0, stream, from, x.stride, rows, input, kb, given,
                           blocks, scales);
    else
        hipLaunchKernelGGL((int8_stage_kernel<T, 0>), grid, block, 0, stream, from, x.stride, rows, input, kb, given,
                           blocks, scales);
}

}  // namespace

hipError_t launch_copy_f32(const float* from, float* to, uint64_t count, hipStream_t stream) {
    hipLaunchKernelGGL(copy_f32_kernel, dim3(uint32_t((count + 255) / 256)), dim3(256), 0, stream, from, to, count);
    return hipGetLastError();
}

hipError_t launch_int8_stage(const OpRows& x, uint64_t rows, uint32_t input, const float* given, int8_t* blocks,
                             float* scales, hipStream_t stream) {
    switch (x.type) {
        case kF32: stage<float>(x, rows, input, given, blocks, scales, stream); break;
        case kF16: stage<_Float16>(x, rows, input, given, blocks, scales, stream); break;
        case kBF16: stage<__bf16>(x, rows, input, given, blocks, scales, stream); break;
        case kI8: stage<int8_t>(x, rows, input, given, blocks, scales, stream); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

static hipError_t launch_pass(const Int8Layer& w, const Int8Call& call, hipStream_t stream) {
    auto* blocks = static_cast<int8_t*>(call.workspace);
    auto* scales = reinterpret_cast<float*>(blocks + int8_block_bytes(call.rows, w.input));
    const hipError_t e = launch_int8_stage(call.x, call.rows, w.input, call.x_scales, blocks, scales, stream);
    if (e != hipSuccess) return e;
    Int8Args a{};
    a.w = w.blocks;
    a.x = blocks;
    a.t = w.scales;
    a.s = scales;
    a.bias = w.bias;
    a.y = const_cast<void*>(call.y.data);
    a.y_stride = call.y.stride;
    a.y_type = call.y.type;
    a.rows = uint32_t(call.rows);
    a.output = w.output;
    a.k_blocks = int8_k_blocks(w.input);
    a.alpha = call.alpha;
    a.beta = call.beta;
    if (call.rows <= 16) {
        hipLaunchKernelGGL(int8_rows16_kernel, dim3((w.output + 15) / 16), dim3(512), 0, stream, a);
    } else {
        const uint32_t nt = (w.output + 127) / 128;
        const uint32_t tiles = nt * uint32_t((call.rows + 127) / 128);
        hipLaunchKernelGGL(int8_tile_kernel, dim3(tiles), dim3(256), 0, stream, a, nt);
    }
    return hipGetLastError();
}

hipError_t launch_int8_linear(const Int8Layer& w, const Int8Call& call, hipStream_t stream) {
    auto bytes = [](uint32_t type) { return type == kF32 ? 4u : type == kI8 ? 1u : 2u; };
    const uint64_t pass = int8_pass_rows(call.rows, w.output);
    Int8Call part = call;
    for (uint64_t left = call.rows; left; left -= part.rows) {
        part.rows = left < pass ? left : pass;
        const hipError_t e = launch_pass(w, part, stream);
        if (e != hipSuccess) return e;
        part.x.data = static_cast<const char*>(part.x.data) + part.rows * part.x.stride * bytes(part.x.type);
        part.y.data = static_cast<const char*>(part.y.data) + part.rows * part.y.stride * bytes(part.y.type);
        if (part.x_scales) part.x_scales += part.rows;
    }
    return hipSuccess;
}

}  // namespace stx
