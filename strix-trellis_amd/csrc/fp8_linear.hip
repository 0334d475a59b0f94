// Products of the e4m3 layers: y = alpha (sum_b s[m][b] t[n / 128][b] p[m][n][b] + bias[n]) + beta y with
// p the sum of products within a block of 128 inputs, and the gated pair act(g) u.
//
// A block's p comes out of the MFMA from an accumulator of zero and enters the
// FP32 sum with one fma per element, so the scales cost no rounding of the
// operands.  A row's bits depend on the core that its call takes (the order of
// the FP32 sums does), not on the other rows.
#include <utility>

#include "fp8_device.hpp"

namespace stx {

namespace {

// ---- a few rows ----
// One launch: every workgroup rounds the rows itself while its weights (16
// channels, of both projections in a pair) are on their way.  Eight waves split
// K in whole blocks; a wave rounds its own part of every row, so nothing is
// shared before the sums meet in LDS.  M: rows, rounded up to a power of two.  U:
// blocks of a wave's part, all in flight at once.  LONG: parts of several
// batches of U.
template <class T, int M, int U, bool PAIR, bool LONG>
__global__ __launch_bounds__(512) void fp8_decode_kernel(Fp8Args a, const T* x, uint64_t stride, uint32_t input) {
    constexpr int P = PAIR ? 2 : 1, kGroups = (U + 1) / 2;   // of two blocks
    constexpr bool kGiven = std::is_same_v<T, uint8_t>;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ f32x4 part[P][8][64];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t kbs = a.k_blocks, kb0 = kbs * w / 8, kb1 = kbs * (w + 1) / 8;
    const uint32_t pitch = kbs * 128 + 64;   // bytes of a row in LDS: rows 16 banks apart
    float* row_s = reinterpret_cast<float*>(smem + M * pitch);   // [M][kbs]
    const uint32_t c = blockIdx.x;           // 16 channels
    // blocks past the wave's part read zeros
    const auto gr = make_rsrc(a.w + uint64_t(PAIR ? c / 2 * 4 + c % 2 : c) * kbs * 2048, kb1 * 2048);
    const auto ur = make_rsrc(a.w + uint64_t(c / 2 * 4 + c % 2 + 2) * kbs * 2048, kb1 * 2048);
    const float* t[2] = {a.t + uint64_t(c / 8) * kbs, a.t + a.t_up + uint64_t(c / 8) * kbs};
    u32x4 f[P][U][2];
    const uint32_t m = lane & 15;
    const unsigned char* xr = smem + (m < a.rows ? m : 0) * pitch + (lane >> 4) * 16;   // dead columns repeat row 0
    const float* xs = row_s + (m < a.rows ? m : 0) * kbs;
    f32x4 acc[P] = {};
    for (uint32_t kb = kb0; kb < kb1; kb += U) {
        // The rows first: loads arrive in order.  A lane has four inputs of a group of
        // two blocks; a half-wave has a block.
        Raw4<T> raw[M][kGroups];
#pragma unroll
        for (int r = 0; r < M; ++r)
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const uint32_t k = (kb + 2 * g) * 128;
                if (uint32_t(r) < a.rows && kb + 2 * g < kb1)
                    raw[r][g] = load4(x + r * stride, k + lane * 4, input, k + 256 <= input);
            }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    f[p][u][j] = __builtin_amdgcn_raw_buffer_load_b128(
                        p ? ur : gr, (kb + u) * 2048 + j * 1024 + lane * 16, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < M; ++r)
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const uint32_t at = kb + 2 * g + (lane >> 5);
                if (uint32_t(r) >= a.rows || kb + 2 * g >= kb1) continue;
                uint32_t q;
                float s;
                if constexpr (kGiven) {
                    q = __builtin_bit_cast(uint32_t, raw[r][g].v);
                    s = at < kbs ? ld_global(a.s + uint64_t(r) * kbs + at) : 0.0f;
                } else {
                    float v[4];
                    raw[r][g].to(v);
                    const BlockScale b = block_scale(half_wave_max(
                        maximum(maximum(fabsf(v[0]), fabsf(v[1])), maximum(fabsf(v[2]), fabsf(v[3])))));
                    q = round4(v, b.inv);
                    s = b.s;
                }
                if (at < kb1) {   // the second block may be another wave's
                    *reinterpret_cast<uint32_t*>(smem + r * pitch + at * 128 + (lane & 31) * 4) = q;
                    if ((lane & 31) == 0) row_s[r * kbs + at] = s;
                }
            }
        // a wave reads what it wrote itself: its LDS operations are in order
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (kb + u >= kb1) break;
            const u32x4 q[2] = {*reinterpret_cast<const u32x4*>(xr + (kb + u) * 128),
                                *reinterpret_cast<const u32x4*>(xr + (kb + u) * 128 + 64)};
            const float s = xs[kb + u];
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const f32x4 v = product16<true>(f[p][u], q);
                const float st = s * ld_global(t[p] + kb + u);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[p][i] = __builtin_fmaf(v[i], st, acc[p][i]);
            }
        }
        if (!LONG) break;
    }
#pragma unroll
    for (int p = 0; p < P; ++p) part[p][w][lane] = acc[p];
    __syncthreads();
    const uint32_t n = c * 16 + 4 * (lane >> 4);
    if (w || m >= a.rows || n >= a.output) return;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int j = 1; j < 8; ++j) acc[p] += part[p][j][lane];
    if constexpr (PAIR) emit(a, m, n, gated4(a, n, acc[0], acc[1]), false);
    else emit(a, m, n, with_bias(a, n, acc[0]), true);
}

// ---- up to sixteen rows ----
// One workgroup per 16 channels (of both projections in a pair); its eight waves
// split K and add their sums in LDS.  U: blocks of a wave in flight.
template <int U, bool PAIR>
__global__ __launch_bounds__(512) void fp8_rows16_kernel(Fp8Args a) {
    constexpr int P = PAIR ? 2 : 1;
    __shared__ f32x4 part[P][8][64];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t kbs = a.k_blocks, kb0 = kbs * w / 8, kb1 = kbs * (w + 1) / 8, c = blockIdx.x;
    const auto xr = make_rsrc(a.x, kb1 * 2048);
    const auto gr = make_rsrc(a.w + uint64_t(PAIR ? c / 2 * 4 + c % 2 : c) * kbs * 2048, kb1 * 2048);
    const auto ur = make_rsrc(a.w + uint64_t(c / 2 * 4 + c % 2 + 2) * kbs * 2048, kb1 * 2048);
    const float* t[2] = {a.t + uint64_t(c / 8) * kbs, a.t + a.t_up + uint64_t(c / 8) * kbs};
    const uint32_t m = lane & 15;
    const float* s = a.s + fp8_scale_at(m);
    f32x4 acc[P] = {};
    for (uint32_t kb = kb0; kb < kb1; kb += U) {
        u32x4 f[P][U][2], g[U][2];   // blocks past kb1 read zeros
        float st[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t at = (kb + u) * 2048 + j * 1024 + lane * 16;
                f[0][u][j] = __builtin_amdgcn_raw_buffer_load_b128(gr, at, 0, 0);
                if (PAIR) f[P - 1][u][j] = __builtin_amdgcn_raw_buffer_load_b128(ur, at, 0, 0);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            st[u] = ld_global(s + uint64_t(kb + u < kb1 ? kb + u : kb1 - 1) * a.s_pitch);
#pragma unroll
            for (int j = 0; j < 2; ++j)
                g[u][j] = __builtin_amdgcn_raw_buffer_load_b128(xr, (kb + u) * 2048 + j * 1024 + lane * 16, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (kb + u >= kb1) break;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const f32x4 v = product16<true>(f[p][u], g[u]);
                const float by = st[u] * ld_global(t[p] + kb + u);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[p][i] = __builtin_fmaf(v[i], by, acc[p][i]);
            }
        }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) part[p][w][lane] = acc[p];
    __syncthreads();
    const uint32_t n = c * 16 + 4 * (lane >> 4);
    if (w || m >= a.rows || n >= a.output) return;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int j = 1; j < 8; ++j) acc[p] += part[p][j][lane];
    if constexpr (PAIR) emit(a, m, n, gated4(a, n, acc[0], acc[1]), false);
    else emit(a, m, n, with_bias(a, n, acc[0]), true);
}

// ---- tens to hundreds of rows ----
// Tiles of 32 TN rows of weights (a pair: 16 TN channels of either projection) x 32
// TM rows, few and short: the tile's K is split over the workgroup's eight
// waves, each of which multiplies the whole tile over its part with operands
// straight from the caches (both are in MFMA order), two blocks in flight and no
// barrier.  The sums meet in LDS, [wave][row][channel] with 16-byte units at
// unit ^ row, and leave as whole rows of the tile.
template <int TN, int TM, bool PAIR, bool EXACT>
__global__ __launch_bounds__(512, TN * TM == 1 ? 4 : 2) void fp8_direct_kernel(Fp8Args a) {
    static_assert(!PAIR || TN == 2);
    constexpr int BN = 32 * TN, BM = 32 * TM;
    constexpr int kUnits = BN / 4, kPlane = BM * BN * 4;
    extern __shared__ __align__(16) unsigned char smem[];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    // The row tiles of a channel tile run on one XCD (workgroup i on XCD i % 8), whose
    // L2 then reads the weights once.
    const uint32_t b = blockIdx.x / 8, nt = b / a.m_tiles * 8 + blockIdx.x % 8, mt = b % a.m_tiles;
    if (nt >= a.n_tiles) return;
    const uint32_t kbs = a.k_blocks, kb0 = kbs * w / 8, kb1 = kbs * (w + 1) / 8, pair = kbs * 2048;
    const uint32_t weight_rows = PAIR ? (a.output + 31) / 32 * 64 : a.output;
    const uint32_t nb = (weight_rows + 31) / 32 * 2 - nt * 2 * TN, mb = (a.rows + 31) / 32 * 2 - mt * 2 * TM;
    // blocks of channels or rows past the last read zeros
    const auto wr = make_rsrc(a.w + uint64_t(nt) * 2 * TN * pair, (nb < 2 * TN ? nb : 2 * TN) * pair);
    const auto xr = make_rsrc(a.x + uint64_t(mt) * 2 * TM * pair, (mb < 2 * TM ? mb : 2 * TM) * pair);
    const int h = lane >> 5, r16 = lane & 15, hi = (lane >> 4) & 1;
    const uint32_t piece = hi * pair + (2 * h * 16 + r16) * 16;
    const float* s[TM];
    const float* t[TN];
#pragma unroll
    for (int k = 0; k < TM; ++k) s[k] = a.s + fp8_scale_at(mt * BM + k * 32 + (lane & 31));
#pragma unroll
    for (int i = 0; i < TN; ++i) {
        // channels of a tile past the last have no scales of their own
        const uint32_t n = PAIR ? nt * 32 : nt * BN + i * 32, block = (n < a.output ? n : 0) / 128;
        t[i] = a.t + (PAIR && i ? a.t_up : 0) + uint64_t(block) * kbs;
    }
    struct Operands {
        u32x4 f[TN][2][2], g[TM][2][2];
        float s[TM];
    };
    auto load = [&](Operands& o, uint32_t kb) {
        const bool live = kb < kb1;   // past the wave's part: out of range, zeros
        const uint32_t at = piece + (live ? kb * 2048 : 0x80000000u);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int i = 0; i < TN; ++i)
                    o.f[i][j][e] = __builtin_amdgcn_raw_buffer_load_b128(wr, at + 2 * i * pair + j * 1024 + e * 256, 0, 0);
#pragma unroll
                for (int k = 0; k < TM; ++k)
                    o.g[k][j][e] = __builtin_amdgcn_raw_buffer_load_b128(xr, at + 2 * k * pair + j * 1024 + e * 256, 0, 0);
            }
#pragma unroll
        for (int k = 0; k < TM; ++k) o.s[k] = live ? ld_global(s[k] + uint64_t(kb) * a.s_pitch) : 0.0f;
    };
    f32x16 acc[TN][TM] = {};
    auto multiply = [&](const Operands& o, uint32_t kb) {
        if (kb >= kb1) return;
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const float by = ld_global(t[i] + kb);
#pragma unroll
            for (int k = 0; k < TM; ++k) {
                const f32x16 p = product32<EXACT>(o.f[i], o.g[k]);
                const float st = o.s[k] * by;
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][k][e] = __builtin_fmaf(p[e], st, acc[i][k][e]);
            }
        }
    };
    Operands o[2];
    load(o[0], kb0);
    for (uint32_t kb = kb0; kb < kb1; kb += 2) {
        // the next block's loads stay ahead of this one's products
        load(o[1], kb + 1);
        __builtin_amdgcn_sched_barrier(0);
        multiply(o[0], kb);
        __builtin_amdgcn_sched_barrier(0);
        load(o[0], kb + 2);
        __builtin_amdgcn_sched_barrier(0);
        multiply(o[1], kb + 1);
        __builtin_amdgcn_sched_barrier(0);
    }
    auto place = [&](int row, int unit) { return row * (BN * 4) + ((unit ^ row) & (kUnits - 1)) * 16; };
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int k = 0; k < TM; ++k)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<f32x4*>(smem + w * kPlane + place(k * 32 + (lane & 31), i * 8 + 2 * q + h)) =
                    f32x4{acc[i][k][4 * q], acc[i][k][4 * q + 1], acc[i][k][4 * q + 2], acc[i][k][4 * q + 3]};
    __syncthreads();
    constexpr int kOut = PAIR ? kUnits / 2 : kUnits;   // units of a row that leaves
#pragma unroll
    for (int c = 0; c < (BM * kOut + 511) / 512; ++c) {
        const int item = c * 512 + threadIdx.x, row = item / kOut, unit = item % kOut;
        const uint32_t m = mt * BM + row, n = nt * (kOut * 4) + unit * 4;
        if (row >= BM || m >= a.rows || n >= a.output) continue;
        f32x4 sum{}, up{};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sum += *reinterpret_cast<const f32x4*>(smem + j * kPlane + place(row, unit));
            if (PAIR) up += *reinterpret_cast<const f32x4*>(smem + j * kPlane + place(row, unit + kOut));
        }
        if constexpr (PAIR) emit(a, m, n, gated4(a, n, sum, up), false);
        else emit(a, m, n, with_bias(a, n, sum), true);
    }
}

template <class T, bool PAIR>
hipError_t decode(const Fp8Args& a, const OpRows& x, uint32_t input, hipStream_t stream) {
    auto go = [&](auto kernel, uint32_t rows) {
        const size_t lds = size_t(rows) * (a.k_blocks * 132 + 64);
        hipLaunchKernelGGL(kernel, dim3((a.output + 15) / 16), dim3(512), lds, stream, a,
                           static_cast<const T*>(x.data), x.stride, input);
        return hipGetLastError();
    };
    // U: blocks of a wave, an eighth of all
    auto go_rows = [&](auto rows) {
        constexpr int M = decltype(rows)::value;
        if (a.k_blocks <= 16) return go(fp8_decode_kernel<T, M, 2, PAIR, false>, M);
        if (a.k_blocks <= 32) return go(fp8_decode_kernel<T, M, 4, PAIR, false>, M);
        if (a.k_blocks <= 40) return go(fp8_decode_kernel<T, M, 5, PAIR, false>, M);
        return go(fp8_decode_kernel<T, M, 4, PAIR, true>, M);
    };
    using std::integral_constant;
    if (a.rows <= 1) return go_rows(integral_constant<int, 1>{});
    if (a.rows <= 2) return go_rows(integral_constant<int, 2>{});
    if (a.rows <= 4) return go_rows(integral_constant<int, 4>{});
    return a.k_blocks <= 16 ? go(fp8_decode_kernel<T, 8, 2, PAIR, false>, 8) : hipErrorInvalidValue;
}

template <class F>
hipError_t launch_core(F kernel, uint32_t tiles, uint32_t threads, size_t lds, const Fp8Args& a, hipStream_t stream) {
    hipLaunchKernelGGL(kernel, dim3(tiles), dim3(threads), lds, stream, a);
    return hipGetLastError();
}

template <bool PAIR, bool EXACT>
hipError_t launch_cores(const Fp8Plan& plan, const Fp8Layer& w, const Fp8Call& call, Fp8Args& a, hipStream_t stream) {
    if (plan.core == kFp8Decode) {
        a.s = call.x_scales;
        switch (call.x.type) {
            case kF32: return decode<float, PAIR>(a, call.x, w.input, stream);
            case kF16: return decode<_Float16, PAIR>(a, call.x, w.input, stream);
            case kBF16: return decode<__bf16, PAIR>(a, call.x, w.input, stream);
            case kE4M3: return decode<uint8_t, PAIR>(a, call.x, w.input, stream);
            default: return hipErrorInvalidValue;
        }
    }
    auto* blocks = static_cast<uint8_t*>(call.workspace);
    auto* scales = reinterpret_cast<float*>(blocks + plan.scales_at);
    a.x = blocks;
    a.s = scales;
    a.s_pitch = uint32_t(fp8_padded_rows(call.rows));
    const hipError_t e = launch_fp8_rows(call.x, call.rows, w.input, call.x_scales, blocks, scales, stream);
    if (e != hipSuccess) return e;
    const uint32_t spread = (plan.n_tiles + 7) / 8 * 8 * plan.m_tiles;
    switch (plan.core) {
        case kFp8Rows16: {
            const uint32_t groups = (w.output + 15) / 16;
            if (a.k_blocks <= 32) return launch_core(fp8_rows16_kernel<4, PAIR>, groups, 512, 0, a, stream);
            return launch_core(fp8_rows16_kernel<5, PAIR>, groups, 512, 0, a, stream);
        }
        case kFp8Direct32x32:
            if constexpr (!PAIR) return launch_core(fp8_direct_kernel<1, 1, false, EXACT>, spread, 512, 8 * 4096, a, stream);
            return hipErrorInvalidValue;
        case kFp8Direct32x64:
            if constexpr (!PAIR) return launch_core(fp8_direct_kernel<1, 2, false, EXACT>, spread, 512, 8 * 8192, a, stream);
            return hipErrorInvalidValue;
        case kFp8Direct64x32: return launch_core(fp8_direct_kernel<2, 1, PAIR, EXACT>, spread, 512, 8 * 8192, a, stream);
        case kFp8Direct64x64: return launch_core(fp8_direct_kernel<2, 2, PAIR, EXACT>, spread, 512, 8 * 16384, a, stream);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_pass(const Fp8Layer& w, const Fp8Call& call, hipStream_t stream) {
    const bool rounded = call.y.type == kE4M3;
    const Fp8Plan plan = fp8_plan(call.rows, w.input, w.output, w.pair, rounded);
    Fp8Args a{};
    a.w = w.blocks;
    a.t = w.scales;
    a.bias = w.bias;
    a.rows = uint32_t(call.rows);
    a.output = w.output;
    a.k_blocks = fp8_k_blocks(w.input);
    a.t_up = (w.output + 127) / 128 * a.k_blocks;
    a.bias_up = (w.output + 31) / 32 * 32;
    a.activation = call.activation;
    a.alpha = call.alpha;
    a.beta = call.beta;
    a.n_tiles = plan.n_tiles;
    a.m_tiles = plan.m_tiles;
    a.y = const_cast<void*>(call.y.data);
    a.y_stride = call.y.stride;
    a.y_type = call.y.type;
    a.y_scales = call.y_scales;
    float* hidden = nullptr;
    if (rounded) {
        a.y = hidden = reinterpret_cast<float*>(static_cast<char*>(call.workspace) + plan.hidden_at);
        a.y_stride = w.output;
        a.y_type = kF32;
    }
    const bool exact = call.y.type == kF32;
    const hipError_t e = w.pair ? exact ? launch_cores<true, true>(plan, w, call, a, stream)
                                        : launch_cores<true, false>(plan, w, call, a, stream)
                                : exact ? launch_cores<false, true>(plan, w, call, a, stream)
                                        : launch_cores<false, false>(plan, w, call, a, stream);
    if (e != hipSuccess || !hidden) return e;
    return launch_fp8_round(hidden, w.output, static_cast<uint8_t*>(const_cast<void*>(call.y.data)), call.y.stride,
                            call.y_scales, call.rows, stream);
}

}  // namespace

hipError_t fp8_allow_lds() {
    const std::pair<void (*)(Fp8Args), size_t> large[] = {{fp8_direct_kernel<2, 2, false, false>, 8 * 16384},
                                                          {fp8_direct_kernel<2, 2, false, true>, 8 * 16384},
                                                          {fp8_direct_kernel<2, 2, true, false>, 8 * 16384},
                                                          {fp8_direct_kernel<2, 2, true, true>, 8 * 16384}};
    for (const auto& [kernel, lds] : large) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, int(lds));
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_fp8(const Fp8Layer& w, const Fp8Call& call, hipStream_t stream) {
    auto bytes = [](uint32_t type) { return type == kF32 ? 4u : type == kE4M3 ? 1u : 2u; };
    const uint64_t pass = fp8_pass_rows(call.rows, w.output);
    Fp8Call part = call;
    for (uint64_t left = call.rows; left; left -= part.rows) {
        part.rows = left < pass ? left : pass;
        const hipError_t e = launch_pass(w, part, stream);
        if (e != hipSuccess) return e;
        part.x.data = static_cast<const char*>(part.x.data) + part.rows * part.x.stride * bytes(part.x.type);
        part.y.data = static_cast<const char*>(part.y.data) + part.rows * part.y.stride * bytes(part.y.type);
        if (part.x_scales) part.x_scales += part.rows * fp8_k_blocks(w.input);
        if (part.y_scales) part.y_scales += part.rows * ((w.output + 127) / 128);
    }
    return hipSuccess;
}

}  // namespace stx
