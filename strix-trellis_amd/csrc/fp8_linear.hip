// Products of the e4m3 layers: y = alpha (sum_b s[m][b] t[n / 128][b] p[m][n][b] + bias[n]) + beta y with
// p the sum of products within a block of 128 inputs, and the gated pair act(g) u.
//
// A block's p comes out of the MFMA from an accumulator of zero and enters the
// FP32 sum with one fma per element, so the scales cost no rounding of the
// operands.  A row's bits depend on the core that its call takes (the order of
// the FP32 sums does), not on the other rows.
#include <utility>

#include "fp8_device.hpp"
#include "fp8_wide.hpp"

namespace stx {

namespace {

// ---- a few rows ----
// One launch: every workgroup rounds the rows itself while its weights (16
// channels, of both projections in a pair) are on their way.  Eight waves split
// K in whole blocks; a wave rounds its own part of every row, so nothing is
// shared before the sums meet in LDS; what a wave writes for its own lanes is FP16, which
// every e4m3 value is, and which the products take.  M: rows, rounded up to a power of two.  U:
// blocks of a wave's part, all in flight at once.  LONG: parts of several
// batches of U.
// Bound by the weights' bytes where there are many (5120 -> 129280, four BF16 rows: 117 us, 5.7 TB/s;
// of the vector units' time 70 % goes into rounding four rows in every workgroup), by the chain of
// launch, row, rounding, products and sums where there are few (4096^2, one row: 4.9 us).
template <class T, int M, int U, bool PAIR, bool LONG>
__global__ __launch_bounds__(512) void fp8_decode_kernel(Fp8Args a, const T* x, uint64_t stride, uint32_t input) {
    constexpr int P = PAIR ? 2 : 1, kGroups = (U + 1) / 2;   // of two blocks
    constexpr bool kGiven = std::is_same_v<T, uint8_t>;
    // A wave's batch of rows as the products take it, the rows' starts spread over the banks.
    constexpr int kBatch = M * U * 256 + (M - 1) / 2 * 128 + 16;
    auto place = [](uint32_t row) { return row * (U * 256) + row % 2 * 16 + row / 2 * 128; };
    __shared__ __align__(16) unsigned char smem[8][kBatch];
    __shared__ float row_s[8][M][U];
    __shared__ f32x4 part[P][8][64];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t kbs = a.k_blocks, kb0 = kbs * w / 8, kb1 = kbs * (w + 1) / 8;
    const uint32_t c = blockIdx.x;           // 16 channels
    // blocks past the wave's part read zeros
    const auto gr = make_rsrc(a.w + uint64_t(PAIR ? c / 2 * 4 + c % 2 : c) * kbs * 2048, kb1 * 2048);
    const auto ur = make_rsrc(a.w + uint64_t(c / 2 * 4 + c % 2 + 2) * kbs * 2048, kb1 * 2048);
    const float* t[2] = {a.t + uint64_t(c / 8) * kbs, a.t + a.t_up + uint64_t(c / 8) * kbs};
    u32x4 f[P][U][2];
    const uint32_t m = lane & 15;
    const uint32_t of = m < a.rows ? m : 0;   // dead columns repeat row 0
    const unsigned char* xr = smem[w] + place(of) + (lane >> 4) * 32;
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
                const int u = 2 * g + (lane >> 5);
                if (U % 2 == 0 || u < U) {
                    *reinterpret_cast<f16x4*>(smem[w] + place(r) + u * 256 + (lane & 31) * 8) = widened4(q);
                    if ((lane & 31) == 0) row_s[w][r][u] = s;
                }
            }
        lanes_meet();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (kb + u >= kb1) break;
            f16x8 q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const f16x8*>(xr + u * 256 + i / 2 * 128 + i % 2 * 16);
            const float s = row_s[w][of][u];
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const f32x4 v = product16(f[p][u], q);
                const float st = s * ld_uniform(t[p] + kb + u);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[p][i] = __builtin_fmaf(v[i], st, acc[p][i]);
            }
        }
        if (!LONG) break;
        lanes_meet();   // read before the next batch is written
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

// ---- up to hundreds of rows ----
// Tiles of 16 TN rows of weights (a pair: half of them of either projection) x 16 TM
// rows, few and short: the tile's K is split over the workgroup's eight waves, each
// of which multiplies the whole tile over its part with operands straight from the
// caches (both are in MFMA order), two batches of U blocks in flight and no
// barrier.  The sums meet in LDS, [wave][row][channel] with 16-byte units at
// unit ^ row, and leave as whole rows of the tile.  Bound by round trips to the caches and the
// operands' way from the L2 (5119 -> 2307, 333 F16 rows, 222 tiles of 64 x 64: 12 us, 145 MB at 12 TB/s; 12288 ->
// 4096, 48 rows in 32 x 32: 11-12.5 us for the weights' 50 MB).  An odd last batch has products of
// its own behind the loop: a second batch of zeros cost the former 3 us.
template <int TN_, int TM_, int U_, int WAVES_>
struct SplitShape {
    static constexpr int TN = TN_, TM = TM_, U = U_, kUnits = 4 * TN, kPlane = 16 * TM * kUnits * 16;
    static constexpr int kSimd = WAVES_;   // waves a SIMD holds
    static constexpr size_t kLds = 8 * size_t(kPlane);
};

template <class S, bool PAIR, bool EXACT>
__global__ __launch_bounds__(512, S::kSimd) void fp8_split_kernel(Fp8Args a) {
    constexpr int TN = S::TN, TM = S::TM, U = S::U;
    static_assert(!PAIR || TN % 2 == 0);
    extern __shared__ __align__(16) unsigned char smem[];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    // The row tiles of a channel tile run on one XCD (workgroup i on XCD i % 8), whose
    // L2 then reads the weights once.
    const uint32_t b = blockIdx.x / 8, nt = b / a.m_tiles * 8 + blockIdx.x % 8, mt = b % a.m_tiles;
    if (nt >= a.n_tiles) return;
    const uint32_t kbs = a.k_blocks, kb0 = kbs * w / 8, kb1 = kbs * (w + 1) / 8, block_row = kbs * 2048;
    // blocks of channels c, c + 1, ..; of a pair the first half are gates, the others their ups
    constexpr int kTiles = PAIR ? TN / 2 : TN;
    const uint32_t c0 = nt * kTiles, blocks = (a.output + 31) / 32 * 2;
    // Uniform offsets of the operands' row blocks.  Blocks past the last repeat it (their sums
    // go nowhere).
    uint32_t w_at[TN], x_at[TM];
    const float* t[TN];
#pragma unroll
    for (int i = 0; i < TN; ++i) {
        const uint32_t c = c0 + i % kTiles < blocks ? c0 + i % kTiles : blocks - 1;
        w_at[i] = (PAIR ? c / 2 * 4 + c % 2 + i / kTiles * 2 - c0 / 2 * 4 : c - c0) * block_row;
        // tiles past the last have no scales of their own
        t[i] = a.t + (PAIR && i >= kTiles ? a.t_up : 0) + uint64_t((c * 16 < a.output ? c : 0) / 8) * kbs;
    }
    const uint32_t m_blocks = (a.rows + 15) / 16 - mt * TM;
#pragma unroll
    for (int k = 0; k < TM; ++k) x_at[k] = (uint32_t(k) < m_blocks ? k : m_blocks - 1) * block_row;
    constexpr uint32_t kSpan = PAIR ? (TN + 3) / 4 * 4 : TN;
    const auto wr = make_rsrc(a.w + uint64_t(PAIR ? c0 / 2 * 4 : c0) * block_row, kSpan * block_row);
    const auto xr = make_rsrc(a.x + uint64_t(mt) * TM * block_row, TM * block_row);
    const auto sr = make_rsrc(a.s, kbs * a.s_pitch * 4);
    const uint32_t s_at = (mt * 16 * TM + (lane & 15)) * 4;
    struct Operands {
        u32x4 f[U][TN][2], g[U][TM][2];
        float s[U][TM];
    };
    auto load = [&](Operands& o, uint32_t kb) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // Past the wave's part: a batch that starts there is not multiplied; of one that ends there
            // the rest is out of range, zeros (scales too: a block's may be infinite).
            const bool live = kb + u < kb1;
            const uint32_t at = live ? kb + u : kb0, past = live || u == 0 ? 0 : 0x80000000u, lane_at = lane * 16 + past;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int i = 0; i < TN; ++i)
                    o.f[u][i][j] = __builtin_amdgcn_raw_buffer_load_b128(wr, lane_at + j * 1024, w_at[i] + at * 2048, 0);
#pragma unroll
                for (int k = 0; k < TM; ++k)
                    o.g[u][k][j] = __builtin_amdgcn_raw_buffer_load_b128(xr, lane_at + j * 1024, x_at[k] + at * 2048, 0);
            }
#pragma unroll
            for (int k = 0; k < TM; ++k)
                o.s[u][k] = __builtin_bit_cast(
                    float, __builtin_amdgcn_raw_buffer_load_b32(sr, (s_at + past) + k * 64, at * a.s_pitch * 4, 0));
        }
    };
    f32x4 acc[TN][TM] = {};
    auto multiply = [&](const Operands& o, uint32_t kb) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool live = u == 0 || kb + u < kb1;
            const uint32_t at = live ? kb + u : kb0;
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                const float by_at = ld_uniform(t[i] + at), by = live ? by_at : 0.0f;
#pragma unroll
                for (int k = 0; k < TM; ++k) {
                    const f32x4 p = product16<EXACT>(o.f[u][i], o.g[u][k]);
                    const float st = o.s[u][k] * by;
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][k][e] = __builtin_fmaf(p[e], st, acc[i][k][e]);
                }
                if (TN * TM >= 8) __builtin_amdgcn_sched_barrier(0);   // more products in flight cost registers
            }
        }
    };
    Operands o[2];
    load(o[0], kb0);
    uint32_t kb = kb0;
    for (; kb + U < kb1; kb += 2 * U) {
        // the next batch's loads stay ahead of this one's products
        load(o[1], kb + U);
        __builtin_amdgcn_sched_barrier(0);
        multiply(o[0], kb);
        __builtin_amdgcn_sched_barrier(0);
        load(o[0], kb + 2 * U);
        __builtin_amdgcn_sched_barrier(0);
        multiply(o[1], kb + U);
        __builtin_amdgcn_sched_barrier(0);
    }
    if (kb < kb1) multiply(o[0], kb);
    constexpr int kUnits = S::kUnits;
    auto place = [&](int row, int unit) { return row * (kUnits * 16) + ((unit ^ row) & (kUnits - 1)) * 16; };
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int k = 0; k < TM; ++k)
            *reinterpret_cast<f32x4*>(smem + w * S::kPlane + place(k * 16 + (lane & 15), i * 4 + (lane >> 4))) = acc[i][k];
    __syncthreads();
    constexpr int kOut = 4 * kTiles;   // units of a row that leaves
#pragma unroll
    for (int c = 0; c < (16 * TM * kOut + 511) / 512; ++c) {
        const int item = c * 512 + threadIdx.x, row = item / kOut, unit = item % kOut;
        const uint32_t m = mt * 16 * TM + row, n = c0 * 16 + unit * 4;
        if (row >= 16 * TM || m >= a.rows || n >= a.output) continue;
        f32x4 sum{}, up{};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sum += *reinterpret_cast<const f32x4*>(smem + j * S::kPlane + place(row, unit));
            if (PAIR) up += *reinterpret_cast<const f32x4*>(smem + j * S::kPlane + place(row, unit + kOut));
        }
        if constexpr (PAIR) emit(a, m, n, gated4(a, n, sum, up), false);
        else emit(a, m, n, with_bias(a, n, sum), true);
    }
}

template <class T, bool PAIR>
hipError_t decode(const Fp8Args& a, const OpRows& x, uint32_t input, hipStream_t stream) {
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((a.output + 15) / 16), dim3(512), 0, stream, a,
                           static_cast<const T*>(x.data), x.stride, input);
        return hipGetLastError();
    };
    // U: blocks of a wave, an eighth of all
    auto go_rows = [&](auto rows) {
        constexpr int M = decltype(rows)::value;
        if (a.k_blocks <= 16) return go(fp8_decode_kernel<T, M, 2, PAIR, false>);
        if (a.k_blocks <= 32) return go(fp8_decode_kernel<T, M, 4, PAIR, false>);
        if (a.k_blocks <= 40) return go(fp8_decode_kernel<T, M, 5, PAIR, false>);
        return go(fp8_decode_kernel<T, M, 4, PAIR, true>);
    };
    using std::integral_constant;
    if (a.rows <= 1) return go_rows(integral_constant<int, 1>{});
    if (a.rows <= 2) return go_rows(integral_constant<int, 2>{});
    if (a.rows <= 4) return go_rows(integral_constant<int, 4>{});
    return a.k_blocks <= 16 ? go(fp8_decode_kernel<T, 8, 2, PAIR, false>) : hipErrorInvalidValue;
}

template <class F>
hipError_t launch_core(F kernel, uint32_t tiles, uint32_t threads, size_t lds, const Fp8Args& a, hipStream_t stream) {
    hipLaunchKernelGGL(kernel, dim3(tiles), dim3(threads), lds, stream, a);
    return hipGetLastError();
}

using Split16x16 = SplitShape<1, 1, 3, 4>;
using Split16x32 = SplitShape<1, 2, 1, 4>;
using Split32x16 = SplitShape<2, 1, 2, 4>;
using Split32x32 = SplitShape<2, 2, 1, 4>;
using Split32x64 = SplitShape<2, 4, 1, 2>;
using Split64x64 = SplitShape<4, 4, 1, 2>;
// Rows of weights x rows.  Two waves along the rows where the widening counts: a wave of 64 x 64 widens
// less for its products than one of 128 x 32, which loads no weights that another loads too.
template <bool EXACT>
using Wide128x128 = WideShape<EXACT ? 4 : 8, EXACT ? 4 : 2, EXACT ? 2 : 1, EXACT ? 2 : 4, EXACT ? 1 : 2, EXACT>;
template <bool EXACT>
using Wide256x128 = WideShape<EXACT ? 4 : 8, EXACT ? 4 : 2, EXACT ? 2 : 1, EXACT ? 4 : 8, EXACT ? 1 : 2, EXACT>;
using Wide256x256 = WideShape<8, 4, 2, 4, 1, false>;

template <class S, bool PAIR, bool ROUNDED>
hipError_t launch_wide(const Fp8Args& a, hipStream_t stream) {
    return launch_core(fp8_wide_kernel<S, PAIR, ROUNDED>, a.n_tiles * a.m_tiles, S::kThreads, S::kLds, a, stream);
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
    auto split = [&](auto shape) {
        using S = decltype(shape);
        if constexpr (PAIR && S::TN % 2) return hipErrorInvalidValue;
        else return launch_core(fp8_split_kernel<S, PAIR, EXACT>, spread, 512, S::kLds, a, stream);
    };
    switch (plan.core) {
        case kFp8Split16x16: return split(Split16x16{});
        case kFp8Split16x32: return split(Split16x32{});
        case kFp8Split32x16: return split(Split32x16{});
        case kFp8Split32x32: return split(Split32x32{});
        case kFp8Split32x64: return split(Split32x64{});
        case kFp8Split64x64: return split(Split64x64{});
        case kFp8Wide128x128: return launch_wide<Wide128x128<EXACT>, PAIR, false>(a, stream);
        case kFp8Wide256x128:
            if constexpr (PAIR && EXACT) {
                if (a.y_type == kE4M3) return launch_wide<Wide256x128<true>, true, true>(a, stream);
            }
            return launch_wide<Wide256x128<EXACT>, PAIR, false>(a, stream);
        case kFp8Wide256x256:
            if constexpr (!EXACT) return launch_wide<Wide256x256, PAIR, false>(a, stream);
            return hipErrorInvalidValue;
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_pass(const Fp8Layer& w, const Fp8Call& call, hipStream_t stream) {
    // e4m3 outputs come with F32 scales, which want F32's precision
    const bool rounded = call.y.type == kE4M3, exact = call.y.type == kF32 || rounded;
    const Fp8Plan plan = fp8_plan(call.rows, w.input, w.output, w.pair, exact, rounded);
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
    if (plan.hidden) {
        a.y = hidden = reinterpret_cast<float*>(static_cast<char*>(call.workspace) + plan.hidden_at);
        a.y_stride = w.output;
        a.y_type = kF32;
    }
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
    hipError_t e = hipSuccess;
    auto allow = [&](auto kernel, size_t lds) {
        if (e == hipSuccess)
            e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                    int(lds));
    };
    auto allow_cores = [&](auto pair) {
        constexpr bool P = decltype(pair)::value;
        allow(fp8_split_kernel<Split64x64, P, false>, Split64x64::kLds);
        allow(fp8_split_kernel<Split64x64, P, true>, Split64x64::kLds);
        allow(fp8_wide_kernel<Wide128x128<false>, P, false>, Wide128x128<false>::kLds);
        allow(fp8_wide_kernel<Wide128x128<true>, P, false>, Wide128x128<true>::kLds);
        allow(fp8_wide_kernel<Wide256x128<false>, P, false>, Wide256x128<false>::kLds);
        allow(fp8_wide_kernel<Wide256x128<true>, P, false>, Wide256x128<true>::kLds);
        allow(fp8_wide_kernel<Wide256x256, P, false>, Wide256x256::kLds);
    };
    allow_cores(std::false_type{});
    allow_cores(std::true_type{});
    allow(fp8_wide_kernel<Wide256x128<true>, true, true>, Wide256x128<true>::kLds);
    return e;
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
