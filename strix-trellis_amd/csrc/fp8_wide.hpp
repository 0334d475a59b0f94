// Products of the e4m3 layers with many rows.
#pragma once
#include "fp8_device.hpp"

namespace stx {

namespace {

// Tiles of 16 TM WM rows x 16 TN WN rows of weights, WM x WN waves of 16 TM x 16 TN.
// The activations go through a ring of LDS stages of 128 inputs that the DMA fills
// ahead; the weights' fragments, which lie in MFMA order, come straight from the
// caches, a stage ahead in registers.
// Calls back to back, with the rounding of their BF16 rows: 2048 rows 4096 -> 12288 in 256 x 128 118 us, of which
// about 111 are this kernel's, 1.9 PFLOP/s (in a kernel trace, which slows it, 113 at the least and 131 in the median); 8192^3 in
// 256 x 256 496 us, 2.2 PFLOP/s (zeros, which cost the clock less: 423).  A third of the waves' time goes into waiting for operands from the
// caches; the rest is shared by matrix steps and the vector steps beside them, of which an 8-bit MFMA hides
// four (there are 4.9) and a 16-bit one one (3.4, with the widening).  EXACT, the gated pair of 2048 rows 4096 -> 2 x 12288:
// 352 us, of which about 346 are this kernel's, 1.2 PFLOP/s.
template <int TM_, int TN_, int WM_, int WN_, int AHEAD_, bool EXACT_>
struct WideShape {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;
    static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves, kBM = 16 * TM * WM, kBN = 16 * TN * WN;
    static constexpr int kAhead = AHEAD_;   // token tiles read ahead of the one that multiplies
    static constexpr bool kExact = EXACT_;
    static constexpr int kRing = 4, kData = kBM * 128, kStage = kData + 1024;   // blocks, scales
    static constexpr int kDma = kData / 1024 / kWaves + 1;   // of a wave and stage: 1 KiB each, and scales
    static constexpr size_t kLds = size_t(kRing) * kStage;
    static_assert((kDma - 1) * kWaves * 1024 == kData && kBM <= 256 && kLds <= 160 * 1024);
    static_assert(kWaves * 16 * TN * 64 <= kLds, "a token tile of every wave in the epilogue");
    static_assert(kBM * (128 + 4 * WN) <= kLds, "rounded rows in the epilogue");
};

// N bytes a lane into LDS, side by side, from the lane's own offset behind a uniform one.
template <int N>
__device__ __forceinline__ void lds_load(__amdgpu_buffer_rsrc_t from, unsigned char* to, uint32_t lane_at, uint32_t at) {
    auto* lds = (__attribute__((address_space(3))) void*)to;
    if constexpr (N == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(from, lds, 16, lane_at, at, 0, 0);
    else __builtin_amdgcn_raw_ptr_buffer_load_lds(from, lds, 4, lane_at, at, 0, 0);
}

template <class S, bool PAIR, bool ROUNDED>
__global__ __launch_bounds__(S::kThreads, 2) void fp8_wide_kernel(Fp8Args a) {
    constexpr bool EXACT = S::kExact;
    static_assert(S::TN == 2 || S::TN == 4, "a wave's channels lie in one block of 128");
    static_assert(!ROUNDED || (PAIR && S::kBN == 256), "a tile holds whole blocks of 128 channels");
    constexpr int TM = S::TM, TN = S::TN;
    extern __shared__ __align__(16) unsigned char smem[];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = w % S::WM, wn = w / S::WM;
    // XCD-aware order: workgroup i runs on XCD i % 8, which takes a contiguous run of
    // tiles, rows first in bands of up to eight row tiles, so its workgroups share
    // both operands in its L2.
    const uint32_t tiles = a.n_tiles * a.m_tiles, per = tiles / 8;
    uint32_t tile = blockIdx.x;
    if (tile < per * 8) tile = (tile % 8) * per + tile / 8;
    const uint32_t band = tile / (8 * a.n_tiles), in_band = tile - band * 8 * a.n_tiles;
    const uint32_t height = a.m_tiles - band * 8 < 8 ? a.m_tiles - band * 8 : 8;
    const uint32_t mt = band * 8 + in_band % height, nt = in_band / height;
    const uint32_t kbs = a.k_blocks, block_row = kbs * 2048;
    // blocks of channels or rows past the last repeat it: their sums go nowhere
    const uint32_t mb = (a.rows + 15) / 16 - mt * (S::kBM / 16);
    const auto wr = make_rsrc(a.w + uint64_t(nt) * (S::kBN / 16) * block_row, S::kBN / 16 * block_row);
    const auto xr = make_rsrc(a.x + uint64_t(mt) * (S::kBM / 16) * block_row, S::kBM / 16 * block_row);
    uint32_t w_at[TN], x_at[S::kDma - 1];   // uniform offsets of what the wave loads
    constexpr int kTiles = PAIR ? TN / 2 : TN;   // of channels that leave; a pair's gates come first, then their ups
    const uint32_t c0 = nt * (S::kBN / 16 / (PAIR ? 2 : 1)) + wn * kTiles, c_last = (a.output + 31) / 32 * 2 - 1;
#pragma unroll
    for (int i = 0; i < TN; ++i) {
        const uint32_t c = c0 + i % kTiles < c_last ? c0 + i % kTiles : c_last;
        w_at[i] = ((PAIR ? c / 2 * 4 + c % 2 + i / kTiles * 2 : c) - nt * (S::kBN / 16)) * block_row;
    }
#pragma unroll
    for (int j = 0; j < S::kDma - 1; ++j) {
        const uint32_t c = w + j * S::kWaves;   // half a block
        x_at[j] = (c / 2 < mb ? c / 2 : mb - 1) * block_row + c % 2 * 1024;
    }
    const auto sr = make_rsrc(a.s, kbs * a.s_pitch * 4);
    // scales of the wave's channels, which lie in one block of 128 (a pair's in one of either projection)
    const uint32_t n0 = c0 * 16;
    constexpr int kScales = PAIR ? 2 : 1;
    const uint32_t n_block = (n0 < a.output ? n0 : 0) / 128;
    const float* t[kScales];
#pragma unroll
    for (int i = 0; i < kScales; ++i) t[i] = a.t + (i ? a.t_up : 0) + uint64_t(n_block) * kbs;

    auto dma = [&](uint32_t kb) {
        unsigned char* base = smem + (kb % S::kRing) * S::kStage;
        // past the end: out of range, zeros
        const uint32_t at = kb < kbs ? kb : 0, past = kb < kbs ? 0 : 0x80000000u;
#pragma unroll
        for (int j = 0; j < S::kDma - 1; ++j)
            lds_load<16>(xr, base + (w + j * S::kWaves) * 1024, lane * 16 + past, x_at[j] + at * 2048);
        // the rows' scales, 64 a wave (waves past the tile's rows repeat others, so that all count alike)
        const uint32_t c = w % (S::kBM / 64);
        lds_load<4>(sr, base + S::kData + c * 256, lane * 4 + past, (at * a.s_pitch + mt * S::kBM + c * 64) * 4);
    };
    u32x4 f[2][TN][2];
    auto load_w = [&](u32x4 (&to)[TN][2], uint32_t kb) {
        const uint32_t at = kb < kbs ? kb : 0, lane_at = lane * 16 + (kb < kbs ? 0 : 0x80000000u);
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                to[i][j] = __builtin_amdgcn_raw_buffer_load_b128(wr, lane_at + j * 1024, w_at[i] + at * 2048, 0);
    };
    // token tiles' fragments and scales: the one that multiplies and the next kAhead
    constexpr int kAhead = S::kAhead, kSlots = kAhead == 1 ? 2 : 4;
    u32x4 g[kSlots][2];
    float s[kSlots];
    auto read_x = [&](int to, uint32_t kb, int k) {
        const unsigned char* st = smem + (kb % S::kRing) * S::kStage;
        const unsigned char* from = st + (wm * TM + k) * 2048 + lane * 16;
#pragma unroll
        for (int j = 0; j < 2; ++j) g[to][j] = *reinterpret_cast<const u32x4*>(from + j * 1024);
        s[to] = *reinterpret_cast<const float*>(st + S::kData + ((wm * TM + k) * 16 + (lane & 15)) * 4);
    };
    float t_at[kScales];
    auto load_t = [&](uint32_t kb) {
        kb = kb < kbs ? kb : 0;
#pragma unroll
        for (int i = 0; i < kScales; ++i) t_at[i] = ld_uniform(t[i] + kb);
    };
    // A tile's products p meet its sums while the next token tile's are in the matrix pipe.
    f32x4 acc[TM][TN] = {}, p[TN] = {};
    float st[kScales] = {};
    auto fold = [&](int k, int i) {
        const float by = st[PAIR && i >= TN / 2];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[k][i][e] = __builtin_fmaf(p[i][e], by, acc[k][i][e]);
    };
    // EXACT: the operands widened, the weights' once a stage, a token tile's while the one before
    // multiplies
    f16x8 fh[EXACT ? TN : 1][4], gh[EXACT ? 2 : 1][4];
    auto widen = [](f16x8 (&to)[4], const u32x4 (&from)[2]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) to[j] = widened(from[j / 2][j % 2 * 2], from[j / 2][j % 2 * 2 + 1]);
    };
    constexpr int kLoads = 2 * TN;
    // Stage kb: the weights of the next one are asked for at its start.  Halfway, every wave
    // has read the stage before, whose buffer the DMA of stage kb + 3 takes, and stage
    // kb + 1 has landed, so its first fragments are read ahead of the last products.
    auto stage = [&](const u32x4 (&now)[TN][2], u32x4 (&next)[TN][2], uint32_t kb) {
        float t_now[kScales];
#pragma unroll
        for (int i = 0; i < kScales; ++i) t_now[i] = t_at[i];
        load_w(next, kb + 1);
#pragma unroll
        for (int k = 0; k < TM; ++k) {
            if (k == TM / 2) {
                __builtin_amdgcn_sched_barrier(0);
                asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(kLoads + S::kDma) : "memory");
                dma(kb + 3);
                load_t(kb + 1);
            }
            __builtin_amdgcn_sched_barrier(0);
            const float s_now = s[k % kSlots];
            // past the last stage: zeros of the DMA, not used
            read_x((k + kAhead) % kSlots, kb + (k + kAhead) / TM, (k + kAhead) % TM);
            const int before = (k + TM - 1) % TM;
            if constexpr (EXACT) {
#pragma unroll
                for (int i = 0; i < TN; i += 2) {
                    fold(before, i);
                    fold(before, i + 1);
                    if (k == 0) {
                        widen(fh[i], now[i]);
                        widen(fh[i + 1], now[i + 1]);
                    }
                    p[i] = p[i + 1] = f32x4{};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        p[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[i][j], gh[k % 2][j], p[i], 0, 0, 0);
                        p[i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[i + 1][j], gh[k % 2][j], p[i + 1], 0, 0, 0);
                    }
                    if (i + 2 == TN) widen(gh[(k + 1) % 2], g[(k + 1) % kSlots]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < TN; ++i) {
                    fold(before, i);
                    p[i] = product16<false>(now[i], g[k % kSlots]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
            for (int i = 0; i < kScales; ++i) st[i] = s_now * t_now[i];
        }
    };
    static_assert(TM % kSlots == 0 && TM / 2 + kAhead <= TM, "a stage's first tiles are read behind the barrier of the one before");
    load_t(0);
    dma(0);
    dma(1);
    load_w(f[0], 0);
    dma(2);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(kLoads + 2 * S::kDma) : "memory");
#pragma unroll
    for (int k = 0; k < kAhead; ++k) read_x(k, 0, k);
    if constexpr (EXACT) widen(gh[0], g[0]);
    uint32_t kb = 0;
    for (; kb + 1 < kbs; kb += 2) {
        stage(f[0], f[1], kb);
        stage(f[1], f[0], kb + 1);
    }
    if (kb < kbs) stage(f[0], f[1], kb);
#pragma unroll
    for (int i = 0; i < TN; ++i) fold(TM - 1, i);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

    // A lane holds channels 4 (lane / 16) + 0..3 of a 16-channel tile, of row lane % 16 of a token
    // tile.
    const uint32_t m0 = mt * S::kBM + wm * 16 * TM, quad = lane >> 4;
    if constexpr (PAIR) {
#pragma unroll
        for (int i = 0; i < TN / 2; ++i) {
            const uint32_t n = n0 + i * 16 + quad * 4;
            const bool inside = n < a.output;
#pragma unroll
            for (int k = 0; k < TM; ++k) {
                acc[k][i] = gated4(a, inside ? n : 0, acc[k][i], acc[k][i + TN / 2]);
                if constexpr (ROUNDED) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (n + e >= a.output) acc[k][i][e] = 0.0f;
                }
            }
        }
    }
    if constexpr (ROUNDED) {
        float* most = reinterpret_cast<float*>(smem + S::kBM * 128);   // [WN][kBM]
#pragma unroll
        for (int k = 0; k < TM; ++k) {
            float v = 0.0f;
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) v = maximum(v, fabsf(acc[k][i][e]));
            v = across_rows_max(v);
            if (lane < 16) most[wn * S::kBM + (wm * TM + k) * 16 + lane] = v;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TM; ++k) {
            const uint32_t row = (wm * TM + k) * 16 + (lane & 15), m = mt * S::kBM + row;
            float v = most[row];
#pragma unroll
            for (int i = 1; i < S::WN; ++i) v = maximum(v, most[i * S::kBM + row]);
            const BlockScale b = block_scale(v);
            if (wn == 0 && lane < 16 && m < a.rows)
                st_global(a.y_scales + uint64_t(m) * ((a.output + 127) / 128) + nt, b.s);
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                const float h[4] = {acc[k][i][0], acc[k][i][1], acc[k][i][2], acc[k][i][3]};
                // 16-byte units of a row at unit ^ row
                *reinterpret_cast<uint32_t*>(smem + row * 128 + (((wn * kTiles + i) ^ row) & 7) * 16 + quad * 4) = round4(h, b.inv);
            }
        }
        __syncthreads();
        for (uint32_t unit = threadIdx.x; unit < S::kBM * 8; unit += S::kThreads) {
            const uint32_t row = unit >> 3, m = mt * S::kBM + row;
            if (m >= a.rows) break;
            store_bytes(static_cast<uint8_t*>(a.y) + uint64_t(m) * a.y_stride, nt * 128 + (unit & 7) * 16, a.output,
                        *reinterpret_cast<const u32x4*>(smem + row * 128 + ((unit ^ row) & 7) * 16));
        }
    } else {
        // Each token tile turns around in the wave's own part of LDS (16-byte unit u of row r
        // at unit u ^ r), so that a store covers whole rows of it.  No barrier.
        constexpr int kUnits = 4 * kTiles, kRowsAtOnce = 64 / kUnits;
        unsigned char* turn = smem + w * (16 * kUnits * 16);
        const uint32_t unit = lane % kUnits, sub = lane / kUnits, n = n0 + unit * 4;
        auto place = [](uint32_t row, uint32_t unit) { return (row * kUnits + ((unit ^ row) & (kUnits - 1))) * 16; };
        const f32x4 bias = !PAIR && a.bias && n < a.output ? ld_global(reinterpret_cast<const f32x4*>(a.bias + n)) : f32x4{};
#pragma unroll
        for (int k = 0; k < TM; ++k) {
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
                *reinterpret_cast<f32x4*>(turn + place(lane & 15, i * 4 + quad)) = acc[k][i];
            lanes_meet();
#pragma unroll
            for (uint32_t row = sub; row < 16; row += kRowsAtOnce) {
                const uint32_t m = m0 + k * 16 + row;
                f32x4 v = *reinterpret_cast<const f32x4*>(turn + place(row, unit));
                if (!PAIR) v += bias;
                if (m < a.rows && n < a.output) emit(a, m, n, v, !PAIR);
            }
            lanes_meet();   // read before the next tile is written
        }
    }
}

}  // namespace

}  // namespace stx
