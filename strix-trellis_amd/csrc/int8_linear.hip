// 8-bit integer linear layer: y = alpha * (s[m] t[n] sum_i q[m][i] w[n][i] + bias[n]) + beta * y.
//
// Activations are rounded to int8 per token (int8_stage_kernel) into the same
// block order the prepared weights have, so that both MFMA operands are read
// as whole 1 KiB blocks, 16 bytes per lane.  The integer sums are exact, so
// neither the split of K nor the tile a row falls into changes a bit.
#include <utility>

#include "ops_device.hpp"

namespace stx {

namespace {

constexpr float kLeastScale = 0x1p-126f;

// ---- rounding of a row ----
// s = max(RN32(most / 127), 2^-126); a row with an infinity or a NaN has most =
// inf or NaN (the maximum passes NaN on).
struct RowScale {
    float s, inv, half;
    bool fine;
};
__device__ __forceinline__ RowScale row_scale(float most) {
    RowScale r;
    r.fine = most < __builtin_inff();
    r.s = fmaxf(most / 127.0f, kLeastScale);
    r.inv = 1.0f / r.s;
    r.half = 0.5f * r.s;
    return r;
}
__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// The largest magnitude of a lane's inputs.  Magnitudes of 16-bit floats are in
// the order of their bits, so those go two to an operation without conversions.
template <class T>
struct Most {
    float m = 0.0f;
    __device__ __forceinline__ void look(const Raw4<T>& x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = maximum(m, fabsf(x.v[i]));
    }
    __device__ __forceinline__ float value() const { return m; }
};
template <class T>
    requires(sizeof(T) == 2)
struct Most<T> {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 m = 0;
    __device__ __forceinline__ void look(const Raw4<T>& x) {
        const u32x2 u = __builtin_bit_cast(u32x2, x.v) & 0x7FFF7FFFu;
        const uint32_t lo = u[0], hi = u[1];
        m = __builtin_elementwise_max(m, __builtin_elementwise_max(__builtin_bit_cast(u16x2, lo), __builtin_bit_cast(u16x2, hi)));
    }
    __device__ __forceinline__ float value() const {
        const uint16_t most = m[0] > m[1] ? m[0] : m[1];
        return float(__builtin_bit_cast(T, most));
    }
};

// Four inputs as int8 in one word.  q = x / s to the nearest integer, ties to
// even: t = x * inv + 1.5 2^23 rounds x * inv to an integer in its low mantissa
// bits, whose last byte is q.  inv is off by half a step, so q is the nearest
// integer of the exact quotient unless that lies within 2^-16 of a tie: then
// |x - q s| >= s / 2, and x - q s is exact in the fma (a multiple of ulp(s) / 2
// below 2^24 of them, or beyond s / 2), so comparing it with s / 2 decides.
template <class T>
__device__ __forceinline__ uint32_t round4(const Raw4<T>& x, const RowScale& r) {
    constexpr float kMagic = 12582912.0f;
    float v[4], t[4], d[4];
    x.to(v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        t[i] = __builtin_fmaf(v[i], r.inv, kMagic);
        d[i] = __builtin_fmaf(kMagic - t[i], r.s, v[i]);
    }
    const float farthest = fmaxf(fmaxf(fabsf(d[0]), fabsf(d[1])), fmaxf(fabsf(d[2]), fabsf(d[3])));
    if (__any(farthest >= r.half)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool odd = __builtin_bit_cast(uint32_t, t[i]) & 1;
            const float by = fabsf(d[i]) > r.half || (fabsf(d[i]) == r.half && odd) ? 1.0f : 0.0f;
            t[i] += __builtin_copysignf(by, d[i]);
        }
    }
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __builtin_bit_cast(uint32_t, t[i]);
    // bytes 0 of the four words
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0c);
    return r.fine ? lo | hi : 0;
}
__device__ __forceinline__ uint32_t word_of(const Raw4<int8_t>& x) { return __builtin_bit_cast(uint32_t, x.v); }

// ---- rows into blocks ----
// One workgroup per row.  A lane takes four consecutive inputs at a time, a wave
// 256 (one coalesced load, 16 pieces of blocks), the waves every fourth 256.
// With HELD > 0 a wave's share stays in registers between the maximum and the
// rounding (rows of up to 1024 HELD inputs), otherwise it is read twice.  Inputs
// past the width become zeros; rows past the last are left as they are (they
// meet only outputs that are not written).  Eight rows share a 128-byte line of
// the blocks, so the 16 rows of a block go to workgroups of one XCD (workgroup i
// runs on XCD i % 8), whose L2 puts the lines together: in row order, with a
// piece of every line in each L2, 2048 float rows of 4096 took 16.2 us for 12.7
// (12288 int8 rows, a layer's weights, 48 for 24).
template <class T, int HELD>
__global__ __launch_bounds__(256) void int8_stage_kernel(const T* x, uint64_t stride, uint32_t input,
                                                         uint32_t k_blocks, const float* given, int8_t* blocks,
                                                         float* scales, uint64_t rows) {
    __shared__ float wave_most[4];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t row = blockIdx.x / 128 * 128 + blockIdx.x % 8 * 16 + blockIdx.x / 8 % 16;
    if (row >= rows) return;
    const uint32_t padded = k_blocks * 64;
    int8_t* to = blocks + (row >> 4) * k_blocks * 1024 + (row & 15) * 16;
    constexpr int kAtOnce = HELD ? HELD : 5;   // loads in flight
    const T* from = x + row * stride;
    // inputs c .. c + 255 of the wave: every 1024; the last may reach past the end
    const uint32_t c0 = w * 256, inside = input / 256 * 256;
    const bool at_end = input > inside && (inside - c0) % 1024 == 0 && inside >= c0;
    auto put = [&](uint32_t c, uint32_t q) {
        const uint32_t k = c + lane * 4;
        if (k < padded)
            st_global(reinterpret_cast<uint32_t*>(to + uint64_t(k >> 6) * 1024 + ((k >> 4) & 3) * 256 + (k & 12)), q);
    };
    Raw4<T> raw[kAtOnce], end;
    auto load_some = [&](uint32_t c) {
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
            if (c + j * 1024 < inside) raw[j] = load4(from, c + j * 1024 + lane * 4, input, true);
    };
    if (at_end) end = load4(from, inside + lane * 4, input, false);
    if constexpr (std::is_same_v<T, int8_t>) {
        for (uint32_t c = c0; c < inside; c += kAtOnce * 1024) {
            load_some(c);
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j)
                if (c + j * 1024 < inside) put(c + j * 1024, word_of(raw[j]));
        }
        if (at_end) put(inside, word_of(end));
        if (given && threadIdx.x == 0) st_global(scales + row, ld_global(given + row));
    } else {
        Most<T> of_lane;
        for (uint32_t c = c0; c < inside; c += kAtOnce * 1024) {
            load_some(c);
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j)
                if (c + j * 1024 < inside) of_lane.look(raw[j]);
        }
        if (at_end) of_lane.look(end);
        const float most = wave_reduce(of_lane.value(), maximum);
        if (lane == 0) wave_most[w] = most;
        __syncthreads();
        const RowScale r = row_scale(maximum(maximum(wave_most[0], wave_most[1]), maximum(wave_most[2], wave_most[3])));
        for (uint32_t c = c0; c < inside; c += kAtOnce * 1024) {
            if (!HELD) load_some(c);
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j)
                if (c + j * 1024 < inside) put(c + j * 1024, round4(raw[j], r));
        }
        if (at_end) put(inside, round4(end, r));
        if (threadIdx.x == 0) st_global(scales + row, r.fine ? r.s : __builtin_nanf(""));
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
    uint32_t n_tiles, m_tiles;
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

// A token's scale as s * by, with `by` a power of two that comes last: the sum
// (below 2^31) times s stays finite for every s, and in the normal range where
// the scale itself is below it, so only the output's own range counts.  By is 1
// for scales of 2^-126 to 2^96; above, sum * s is at least 2^64, so that no channel
// scale takes it below the normal range.
struct TokenScale {
    float s, by;
};
__device__ __forceinline__ TokenScale token_scale(float s) {
    const float a = fabsf(s);
    const bool large = a >= 0x1p96f, small = a < 0x1p-126f;
    return {s * (large ? 0x1p-32f : small ? 0x1p32f : 1.0f), large ? 0x1p32f : small ? 0x1p-32f : 1.0f};
}

template <class T>
__device__ __forceinline__ void emit4(const Int8Args& a, uint32_t m, uint32_t n, i32x4 acc, float s,
                                      const Channels& c) {
    T* row = static_cast<T*>(a.y) + uint64_t(m) * a.y_stride;
    float v[4], old[4];
    if (a.beta != 0.0f) load4(static_cast<const T*>(row), n, a.output, false).to(old);
    const TokenScale ts = token_scale(s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = float(acc[i]) * ts.s * c.t[i] * ts.by;
        if (c.bias) v[i] += c.b[i];
        v[i] *= a.alpha;
        if (a.beta != 0.0f) v[i] += a.beta * old[i];
    }
    store4(row, n, a.output, v);
}
__device__ __forceinline__ void emit(const Int8Args& a, uint32_t m, uint32_t n, i32x4 acc, float s,
                                     const Channels& c) {
    if (a.y_type == kF32) emit4<float>(a, m, n, acc, s, c);
    else if (a.y_type == kBF16) emit4<__bf16>(a, m, n, acc, s, c);
    else emit4<_Float16>(a, m, n, acc, s, c);
}

// ---- a few rows ----
// One launch: every workgroup rounds the rows itself, into LDS, while its
// weights (16 channels) are on their way.  Eight waves; the waves split K and add
// their sums in LDS.  M: rows, rounded up to a power of two; 8 / M waves round one
// row.  Bound by the weights' bytes where there are many channels (4096 -> 12288
// one row 7.7 us, 6.5 TB/s) and by one chain of latencies, launch, row, rounding,
// products, where there are few (4096^2 3.4 us).  The figures of this note and of
// the sizing rule are of one layer again and again, which the last-level cache holds
// (but for 5120 -> 129280); three layers of 4096^2 in turn take 4.1 to 4.5 us each.
// U: K blocks of a wave's part, all in flight at once, and with them the row's
// share of each lane, which stays in registers between the maximum and the
// rounding.  Every block that a wave asks for and does not have costs issue slots
// and registers, and so workgroups per compute unit: 4096 -> 12288 one / four rows
// take 7.7 / 9.1 us with U = 8 for 8.5 / 10.0 with U = 10 (5120^2 the other way:
// 4.2 with 10, 5.6 with 8, in two batches), 1152 -> 5120 3.2 with 4, 4.0 with 10.
// LONG: parts of several batches of U; the row is read twice, from the caches.
// Its loads have code of their own: loads that may or may not have been followed
// by others are waited for as if they had been, here with all the weights.
template <class T, int M, int U, bool LONG>
__global__ __launch_bounds__(512, 4) void int8_decode_kernel(Int8Args a, const T* x, uint64_t stride, uint32_t input) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int G = 8 / M;                  // waves per row
    __shared__ i32x4 part[8][64];
    __shared__ float wave_most[8], row_s[8];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t kbs = a.k_blocks, kb0 = kbs * w / 8, kb1 = kbs * (w + 1) / 8;
    const uint32_t pitch = kbs * 64 + 64;     // bytes of a row in LDS: rows 16 banks apart
    u32x4 f[U];
    const auto wr = make_rsrc(a.w + uint64_t(blockIdx.x) * kbs * 1024, kb1 * 1024);
    // blocks kb .. kb + U - 1; past the wave's part they read zeros
    auto load_w = [&](uint32_t kb) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            f[u] = __builtin_amdgcn_raw_buffer_load_b128(wr, (kb + u) * 1024 + lane * 16, 0, 0);
    };

    // ---- rows into LDS ----
    {
        const int m = w / G, part_of = w % G;
        const bool live = uint32_t(m) < a.rows;
        const T* from = x + (live ? m : 0) * stride;
        const uint32_t padded = kbs * 64, step = G * 256;
        unsigned char* to = smem + m * pitch;
        auto put = [&](uint32_t b, uint32_t q) {
            if (b + lane * 4 < padded) *reinterpret_cast<uint32_t*>(to + b + lane * 4) = q;
        };
        // the wave's groups of 256 inputs: b0, b0 + step, ..; the last may reach past the end
        const uint32_t b0 = part_of * 256, inside = input / 256 * 256;
        const bool at_end = input > inside && inside >= b0 && (inside - b0) % step == 0;
        constexpr int kHeld = (U * M + 3) / 4;   // the row's groups of U K blocks a wave
        Raw4<T> raw[kHeld], end;
        auto load_some = [&](uint32_t b) {
#pragma unroll
            for (int c = 0; c < kHeld; ++c)
                if (b + c * step < inside) raw[c] = load4(from, b + c * step + lane * 4, input, true);
        };
        // the weights behind the row: loads arrive in order, and the row's come first
        load_some(b0);
        if (at_end) end = load4(from, inside + lane * 4, input, false);
        __builtin_amdgcn_sched_barrier(0);
        load_w(kb0);
        __builtin_amdgcn_sched_barrier(0);
        auto each = [&](uint32_t b, auto&& use) __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < kHeld; ++c)
                if (b + c * step < inside) use(b + c * step, raw[c]);
        };
        auto others = [&](uint32_t b, auto&& use) __attribute__((always_inline)) {
            for (; b < inside; b += kHeld * step) {
                load_some(b);
                each(b, use);
            }
        };
        if constexpr (std::is_same_v<T, int8_t>) {
            auto copy = [&](uint32_t b, const Raw4<T>& r) __attribute__((always_inline)) { put(b, word_of(r)); };
            if (live) {
                each(b0, copy);
                if (LONG) others(b0 + kHeld * step, copy);
                if (at_end) put(inside, word_of(end));
                if (lane == 0 && part_of == 0) row_s[m] = ld_global(a.s + m);
            }
        } else {
            Most<T> of_lane;
            auto look = [&](uint32_t, const Raw4<T>& r) __attribute__((always_inline)) { of_lane.look(r); };
            each(b0, look);
            if (LONG) others(b0 + kHeld * step, look);
            if (at_end) of_lane.look(end);
            float most = wave_reduce(of_lane.value(), maximum);
            if constexpr (G > 1) {
                if (lane == 0) wave_most[w] = most;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < G; ++i) most = maximum(most, wave_most[m * G + i]);
            }
            const RowScale r = row_scale(most);
            auto round = [&](uint32_t b, const Raw4<T>& x4) __attribute__((always_inline)) { put(b, round4(x4, r)); };
            if (live) {
                if (LONG) others(b0, round);
                else each(b0, round);
                if (at_end) put(inside, round4(end, r));
                if (lane == 0 && part_of == 0) row_s[m] = r.fine ? r.s : __builtin_nanf("");
            }
        }
    }
    __syncthreads();

    // ---- products ----
    const uint32_t m = lane & 15, n = blockIdx.x * 16 + 4 * (lane >> 4);
    const unsigned char* xr = smem + (m < a.rows ? m : 0) * pitch + (lane >> 4) * 16;   // dead columns repeat row 0
    i32x4 acc{};
    for (uint32_t kb = kb0;;) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // past the wave's part the weights are zeros, whatever lies in LDS
            const uint32_t at = kb + u < kbs ? kb + u : kbs - 1;
            const i32x4 q = *reinterpret_cast<const i32x4*>(xr + at * 64);
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, f[u]), q, acc, 0, 0, 0);
        }
        kb += U;
        if (!LONG || kb >= kb1) break;
        load_w(kb);
    }
    part[w][lane] = acc;
    __syncthreads();
    if (w || m >= a.rows || n >= a.output) return;
#pragma unroll
    for (int j = 1; j < 8; ++j) acc += part[j][lane];
    emit(a, m, n, acc, row_s[m], channels_of(a, n));
}

// ---- up to sixteen rows ----
// One workgroup per 16 channels; its eight waves split K and add their sums in
// LDS.  U: K blocks of a wave in flight, as in the decode kernel.  Bound by the
// weights' bytes behind one round trip (5120^2 7.3 us for 26 MB, and 2.7 for the
// rounding); 32 x 32 tiles instead are 0.2 us faster there, 1.1 slower at 4096^2, 5.5
// slower at 12288 -> 4096.
template <int U>
__global__ __launch_bounds__(512) void int8_rows16_kernel(Int8Args a) {
    __shared__ i32x4 part[8][64];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t kb0 = a.k_blocks * w / 8, kb1 = a.k_blocks * (w + 1) / 8;
    const auto wr = make_rsrc(a.w + uint64_t(blockIdx.x) * a.k_blocks * 1024, kb1 * 1024);
    const auto xr = make_rsrc(a.x, kb1 * 1024);
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
    if (m < a.rows && n < a.output) emit(a, m, n, acc, ld_global(a.s + m), channels_of(a, n));
}

// ---- tens to hundreds of rows ----
// Tiles of 32 TN channels x 32 TM rows, few and short: the tile's K is split over
// the workgroup's eight waves, each of which multiplies the whole tile over its
// part with operands straight from the caches (both are in MFMA order, 1 KiB per
// load), two batches of U blocks in flight and no barrier.  The sums meet in
// LDS, [wave][row][channel] with 16-byte units at unit ^ row, and leave as whole
// rows of the tile.  Bound by the caches' latency and rate, so what counts is how
// many waves a compute unit holds: the two small tiles run with one block in flight
// twice and few registers, four and two workgroups to a compute unit (5120^2 24 /
// 48 rows 9.7 us in 32 x 32, 11.3 in 32 x 64; with 4 and 3 blocks, one workgroup
// each, 11.6 and 12.6).  64 x 64 has the LDS of a compute unit to itself.
template <int TN, int TM>
__global__ __launch_bounds__(512, TN * TM == 1 ? 8 : TN * TM == 2 ? 4 : 2) void int8_direct_kernel(Int8Args a) {
    constexpr int BN = 32 * TN, BM = 32 * TM, U = TN * TM <= 2 ? 1 : 2;
    constexpr int kUnits = BN / 4, kPlane = BM * BN * 4;
    extern __shared__ __align__(16) unsigned char smem[];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    // The row tiles of a channel tile run on one XCD (workgroup i on XCD i % 8), whose
    // L2 then reads the weights once.
    const uint32_t j = blockIdx.x / 8, nt = j / a.m_tiles * 8 + blockIdx.x % 8, mt = j % a.m_tiles;
    if (nt >= a.n_tiles) return;
    const uint32_t kbs = a.k_blocks, kb0 = kbs * w / 8, kb1 = kbs * (w + 1) / 8, pair = kbs * 1024;
    const uint32_t nb = (a.output + 31) / 32 * 2 - nt * 2 * TN, mb = (a.rows + 31) / 32 * 2 - mt * 2 * TM;
    // blocks of channels or rows past the last read zeros
    const auto wr = make_rsrc(a.w + uint64_t(nt) * 2 * TN * pair, (nb < 2 * TN ? nb : 2 * TN) * pair);
    const auto xr = make_rsrc(a.x + uint64_t(mt) * 2 * TM * pair, (mb < 2 * TM ? mb : 2 * TM) * pair);
    const int h = lane >> 5, r16 = lane & 15, hi = (lane >> 4) & 1;
    const uint32_t piece = hi * pair + (h * 16 + r16) * 16;
    struct Operands {
        u32x4 f[U][2][TN], g[U][2][TM];
    };
    auto load = [&](Operands& o, uint32_t kb) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool live = kb + u < kb1;   // past the wave's part: out of range, zeros
            const uint32_t at = piece + (live ? (kb + u) * 1024 : 0x80000000u);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int i = 0; i < TN; ++i)
                    o.f[u][j][i] = __builtin_amdgcn_raw_buffer_load_b128(wr, at + 2 * i * pair + j * 512, 0, 0);
#pragma unroll
                for (int i = 0; i < TM; ++i)
                    o.g[u][j][i] = __builtin_amdgcn_raw_buffer_load_b128(xr, at + 2 * i * pair + j * 512, 0, 0);
            }
        }
    };
    i32x16 acc[TN][TM] = {};
    auto multiply = [&](const Operands& o) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < TN; ++i)
#pragma unroll
                    for (int k = 0; k < TM; ++k)
                        acc[i][k] = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, o.f[u][j][i]),
                                                                          __builtin_bit_cast(i32x4, o.g[u][j][k]),
                                                                          acc[i][k], 0, 0, 0);
    };
    Operands o[2];
    load(o[0], kb0);
    for (uint32_t kb = kb0; kb < kb1; kb += 2 * U) {
        // the next batch's loads stay ahead of this one's products
        load(o[1], kb + U);
        __builtin_amdgcn_sched_barrier(0);
        multiply(o[0]);
        __builtin_amdgcn_sched_barrier(0);
        load(o[0], kb + 2 * U);
        __builtin_amdgcn_sched_barrier(0);
        multiply(o[1]);
        __builtin_amdgcn_sched_barrier(0);
    }
    auto place = [&](int row, int unit) { return row * (BN * 4) + ((unit ^ row) & (kUnits - 1)) * 16; };
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int k = 0; k < TM; ++k)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<i32x4*>(smem + w * kPlane + place(k * 32 + (lane & 31), i * 8 + 2 * q + h)) =
                    i32x4{acc[i][k][4 * q], acc[i][k][4 * q + 1], acc[i][k][4 * q + 2], acc[i][k][4 * q + 3]};
    __syncthreads();
#pragma unroll
    for (int c = 0; c < (BM * kUnits + 511) / 512; ++c) {
        const int item = c * 512 + threadIdx.x, row = item / kUnits, unit = item % kUnits;
        const uint32_t m = mt * BM + row, n = nt * BN + unit * 4;
        if (row >= BM || m >= a.rows || n >= a.output) continue;
        i32x4 sum{};
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += *reinterpret_cast<const i32x4*>(smem + j * kPlane + place(row, unit));
        emit(a, m, n, sum, ld_global(a.s + m), channels_of(a, n));
    }
}

// ---- many rows ----
// Tiles of 64 TN channels x 64 TM rows, four waves (two along each side) of 32 TN x
// 32 TM, both operands in a ring of LDS stages of 64 inputs that the DMA fills
// kRing - 1 stages ahead.  A stage is two K32 steps; the fragments of a step are
// read while the step before multiplies.  The barrier stands between a stage's
// steps: behind it every wave has read the whole stage, so its buffer takes the
// DMA of the stage kRing ahead, and the next stage has landed.
//
// 4096 -> 12288, 2048 F32 rows: 108-130 us on different cards with the rounding of
// the rows (13), 2.0 POPS at 8192 rows.  Two things are seen to cost.  The clock under
// the matrix pipes' load: the same launch takes 80 us on zeros (3.0 POPS at 8192 rows)
// and 112 on random bytes, at 1.6 GHz.  And the feed: the pipes are busy half the cycles,
// 85 us are left of 110 without the DMA (105 without the LDS reads), 189 MB are fetched
// for 59, and the library's product, whose outputs are the sums as they are, is 10 %
// faster on random bytes at 8192 rows.  Tiles of 192 x 256, with three quarters of the
// traffic into LDS, run at the same 2.0 POPS there and lose where the tiles are few.
template <int TN, int TM, int RING>
struct WideShape {
    static constexpr int kBN = 64 * TN, kBM = 64 * TM, kStage = (TN + TM) * 4096, kRing = RING;
    static constexpr size_t kLds = size_t(kRing) * kStage;
    static_assert(kLds >= 4u * (32 * 128 * TN + 128), "the epilogue's turn");
};

template <int TN, int TM, int RING>
__global__ __launch_bounds__(256, 2) void int8_wide_kernel(Int8Args a) {
    using S = WideShape<TN, TM, RING>;
    extern __shared__ __align__(16) unsigned char smem[];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    // XCD-aware order: workgroup i runs on XCD i % 8, which takes a contiguous run of
    // tiles, rows first in bands of up to eight row tiles, so its workgroups share
    // both operands in its L2.
    const uint32_t tiles = a.n_tiles * a.m_tiles, per = tiles / 8;
    uint32_t t = blockIdx.x;
    if (t < per * 8) t = (t % 8) * per + t / 8;
    const uint32_t band = t / (8 * a.n_tiles), in_band = t - band * 8 * a.n_tiles;
    const uint32_t height = a.m_tiles - band * 8 < 8 ? a.m_tiles - band * 8 : 8;
    const uint32_t mt = band * 8 + in_band % height, nt = in_band / height;
    const uint32_t kbs = a.k_blocks, pair = kbs * 1024;
    const uint32_t nb = (a.output + 31) / 32 * 2 - nt * 4 * TN, mb = (a.rows + 31) / 32 * 2 - mt * 4 * TM;
    // blocks of channels or rows past the last read zeros
    const auto wr = make_rsrc(a.w + uint64_t(nt) * 4 * TN * pair, (nb < 4 * TN ? nb : 4 * TN) * pair);
    const auto xr = make_rsrc(a.x + uint64_t(mt) * 4 * TM * pair, (mb < 4 * TM ? mb : 4 * TM) * pair);
    // a stage: 4 TN blocks of channels, 4 TM of rows; wave w moves blocks w, w + 4, ..
    const uint32_t lane_off = lane * 16 + w * pair;
    auto dma = [&](uint32_t kb, uint32_t slot) {
        unsigned char* base = smem + slot * S::kStage + w * 1024;
        const uint32_t off = lane_off + (kb < kbs ? kb * 1024 : 0x80000000u);   // past the end: out of range
#pragma unroll
        for (int j = 0; j < TN; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (__attribute__((address_space(3))) void*)(base + j * 4096), 16,
                                                     off + j * 4 * pair, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < TM; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                xr, (__attribute__((address_space(3))) void*)(base + (TN + j) * 4096), 16, off + j * 4 * pair, 0, 0, 0);
    };
    const int wn = w & 1, wm = w >> 1, h = lane >> 5, r16 = lane & 15, hi = (lane >> 4) & 1;
    const uint32_t piece = hi * 1024 + (h * 16 + r16) * 16;
    i32x4 f[2][TN], g[2][TM];
    auto read = [&](uint32_t slot, int j) {
        const unsigned char* st = smem + slot * S::kStage + piece + j * 512;
#pragma unroll
        for (int i = 0; i < TN; ++i) f[j][i] = *reinterpret_cast<const i32x4*>(st + (wn * 2 * TN + i * 2) * 1024);
#pragma unroll
        for (int i = 0; i < TM; ++i)
            g[j][i] = *reinterpret_cast<const i32x4*>(st + (4 * TN + wm * 2 * TM + i * 2) * 1024);
    };
    i32x16 acc[TN][TM] = {};
    auto multiply = [&](int j) {
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int k = 0; k < TM; ++k) acc[i][k] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f[j][i], g[j][k], acc[i][k], 0, 0, 0);
        // the reads behind the first MFMAs (0x008: MFMA, 0x100: LDS read)
        constexpr int kReads = TN + TM, kEach = TN * TM >= kReads ? 1 : 2;
#pragma unroll
        for (int i = 0; i < kReads / kEach; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, kEach, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, TN * TM - kReads / kEach, 0);
    };
    constexpr int kLoads = TN + TM;
#pragma unroll
    for (int i = 0; i < RING; ++i) dma(i, i);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((RING - 1) * kLoads) : "memory");
    read(0, 0);
    for (uint32_t kb = 0, slot = 0; kb < kbs; ++kb) {
        const uint32_t ahead = slot + 1 == RING ? 0 : slot + 1;
        __builtin_amdgcn_sched_barrier(0);
        read(slot, 1);
        multiply(0);
        __builtin_amdgcn_sched_barrier(0);
        // all but the next stage's DMAs may still be on their way
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((RING - 2) * kLoads) : "memory");
        dma(kb + RING, slot);
        __builtin_amdgcn_sched_barrier(0);
        read(ahead, 0);   // past the last stage: zeros of the DMA, not used
        multiply(1);
        slot = ahead;
    }
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

    // A lane holds four consecutive channels of 32 rows here and there; each 32-row
    // block of a wave turns around in the wave's own part of LDS (16-byte unit u
    // of row r at unit u ^ r), after which a store covers whole rows of the
    // block (512 contiguous bytes of two rows at TN = 4).  A wave's LDS operations
    // are in order: no barrier.  The row loop stays a loop: written out for every
    // type and edge the epilogue took 95 KB of code, more than the instruction
    // cache holds.
    constexpr int kUnits = 8 * TN, kRowsAtOnce = 64 / kUnits, kTurn = 32 * kUnits * 16;
    unsigned char* turn = smem + w * (kTurn + 128);
    float* row_s = reinterpret_cast<float*>(turn + kTurn);
    const uint32_t unit = lane % kUnits, sub = lane / kUnits;
    const uint32_t n = nt * S::kBN + wn * 32 * TN + unit * 4, m_wave = mt * S::kBM + wm * 32 * TM;
    const bool inside = n < a.output;
    const Channels c = channels_of(a, inside ? n : 0);
    float s[TM];
#pragma unroll
    for (int k = 0; k < TM; ++k) {
        const uint32_t m = m_wave + k * 32 + (lane & 31);
        s[k] = ld_global(a.s + (m < a.rows ? m : 0));
    }
#pragma unroll
    for (int k = 0; k < TM; ++k) {
        if (lane < 32) row_s[lane] = s[k];
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<i32x4*>(turn + (lane & 31) * (kUnits * 16) +
                                          (((i * 8 + 2 * q + h) ^ lane) & (kUnits - 1)) * 16) =
                    i32x4{acc[i][k][4 * q], acc[i][k][4 * q + 1], acc[i][k][4 * q + 2], acc[i][k][4 * q + 3]};
#pragma unroll 4
        for (uint32_t row = sub; row < 32; row += kRowsAtOnce) {
            const uint32_t m = m_wave + k * 32 + row;
            const i32x4 v = *reinterpret_cast<const i32x4*>(turn + row * (kUnits * 16) + ((unit ^ row) & (kUnits - 1)) * 16);
            if (m < a.rows && inside) emit(a, m, n, v, row_s[row], c);
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
    const dim3 grid{uint32_t((rows + 127) / 128 * 128)}, block(256);
    const uint32_t kb = int8_k_blocks(input);
    const T* from = static_cast<const T*>(x.data);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, block, 0, stream, from, x.stride, input, kb, given, blocks, scales, rows);
    };
    if (input <= 5 * 1024) go(int8_stage_kernel<T, 5>);
    else if (input <= 8 * 1024) go(int8_stage_kernel<T, 8>);
    else go(int8_stage_kernel<T, 0>);
}

template <class T>
hipError_t decode(const Int8Args& a, const OpRows& x, uint32_t input, hipStream_t stream) {
    const size_t lds = size_t(a.rows) * (a.k_blocks * 64 + 64);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((a.output + 15) / 16), dim3(512), lds, stream, a,
                           static_cast<const T*>(x.data), x.stride, input);
        return hipGetLastError();
    };
    // U: K blocks of a wave, an eighth of all
    auto go_rows = [&](auto rows) {
        constexpr int M = decltype(rows)::value;
        if (a.k_blocks <= 32) return go(int8_decode_kernel<T, M, 4, false>);
        if (a.k_blocks <= 64) return go(int8_decode_kernel<T, M, 8, false>);
        if (a.k_blocks <= 80) return go(int8_decode_kernel<T, M, 10, false>);
        return go(int8_decode_kernel<T, M, 8, true>);
    };
    using std::integral_constant;
    if (a.rows <= 1) return go_rows(integral_constant<int, 1>{});
    if (a.rows <= 2) return go_rows(integral_constant<int, 2>{});
    if (a.rows <= 4) return go_rows(integral_constant<int, 4>{});
    return a.k_blocks <= 32 ? go(int8_decode_kernel<T, 8, 4, false>) : hipErrorInvalidValue;
}

template <class F>
hipError_t launch_core(F kernel, uint32_t tiles, uint32_t threads, size_t lds, const Int8Args& a, hipStream_t stream) {
    hipLaunchKernelGGL(kernel, dim3(tiles), dim3(threads), lds, stream, a);
    return hipGetLastError();
}

using Wide256x128 = WideShape<4, 2, 3>;
using Wide128x128 = WideShape<2, 2, 3>;

hipError_t launch_pass(const Int8Layer& w, const Int8Call& call, hipStream_t stream) {
    const Int8Plan plan = int8_plan(call.rows, w.input, w.output);
    auto* blocks = static_cast<int8_t*>(call.workspace);
    Int8Args a{};
    a.w = w.blocks;
    a.x = blocks;
    a.t = w.scales;
    a.bias = w.bias;
    a.y = const_cast<void*>(call.y.data);
    a.y_stride = call.y.stride;
    a.y_type = call.y.type;
    a.rows = uint32_t(call.rows);
    a.output = w.output;
    a.k_blocks = int8_k_blocks(w.input);
    a.alpha = call.alpha;
    a.beta = call.beta;
    a.n_tiles = plan.n_tiles;
    a.m_tiles = plan.m_tiles;
    if (plan.core == kInt8Decode) {
        a.s = call.x_scales;
        switch (call.x.type) {
            case kF32: return decode<float>(a, call.x, w.input, stream);
            case kF16: return decode<_Float16>(a, call.x, w.input, stream);
            case kBF16: return decode<__bf16>(a, call.x, w.input, stream);
            case kI8: return decode<int8_t>(a, call.x, w.input, stream);
            default: return hipErrorInvalidValue;
        }
    }
    auto* scales = reinterpret_cast<float*>(blocks + plan.scales_at);
    a.s = scales;
    const hipError_t e = launch_int8_stage(call.x, call.rows, w.input, call.x_scales, blocks, scales, stream);
    if (e != hipSuccess) return e;
    const uint32_t tiles = plan.n_tiles * plan.m_tiles, spread = (plan.n_tiles + 7) / 8 * 8 * plan.m_tiles;
    switch (plan.core) {
        case kInt8Rows16:
            if (a.k_blocks <= 32) return launch_core(int8_rows16_kernel<4>, tiles, 512, 0, a, stream);
            if (a.k_blocks <= 64 || a.k_blocks > 80) return launch_core(int8_rows16_kernel<8>, tiles, 512, 0, a, stream);
            return launch_core(int8_rows16_kernel<10>, tiles, 512, 0, a, stream);
        case kInt8Direct32x32: return launch_core(int8_direct_kernel<1, 1>, spread, 512, 8 * 4096, a, stream);
        case kInt8Direct32x64: return launch_core(int8_direct_kernel<1, 2>, spread, 512, 8 * 8192, a, stream);
        case kInt8Direct64x64: return launch_core(int8_direct_kernel<2, 2>, spread, 512, 8 * 16384, a, stream);
        case kInt8Wide256x128: return launch_core(int8_wide_kernel<4, 2, 3>, tiles, 256, Wide256x128::kLds, a, stream);
        case kInt8Wide128x128: return launch_core(int8_wide_kernel<2, 2, 3>, tiles, 256, Wide128x128::kLds, a, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t int8_allow_lds() {
    const std::pair<void (*)(Int8Args), size_t> large[] = {{int8_direct_kernel<2, 2>, 8 * 16384},
                                                           {int8_wide_kernel<4, 2, 3>, Wide256x128::kLds}};
    for (const auto& [kernel, lds] : large) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, int(lds));
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_copy_f32(const float* from, float* to, uint64_t count, hipStream_t stream) {
    hipLaunchKernelGGL(copy_f32_kernel, dim3(uint32_t((count + 255) / 256)), dim3(256), 0, stream, from, to, count);
    return hipGetLastError();
}

hipError_t launch_int8_stage(const OpRows& x, uint64_t rows, uint32_t input, const float* given, int8_t* blocks,
                             float* scales, hipStream_t stream) {
    constexpr uint64_t kRows = 1u << 20;   // a launch holds fewer than 2^32 threads
    OpRows part = x;
    for (uint64_t left = rows; left;) {
        const uint64_t n = left < kRows ? left : kRows;
        switch (x.type) {
            case kF32: stage<float>(part, n, input, given, blocks, scales, stream); break;
            case kF16: stage<_Float16>(part, n, input, given, blocks, scales, stream); break;
            case kBF16: stage<__bf16>(part, n, input, given, blocks, scales, stream); break;
            case kI8: stage<int8_t>(part, n, input, given, blocks, scales, stream); break;
            default: return hipErrorInvalidValue;
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        left -= n;
        part.data = static_cast<const char*>(part.data) + n * x.stride * (x.type == kF32 ? 4 : x.type == kI8 ? 1 : 2);
        if (given) given += n;
        blocks += n / 16 * int8_k_blocks(input) * 1024;
        scales += n;
    }
    return hipSuccess;
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
