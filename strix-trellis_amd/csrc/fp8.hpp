// Internal interface between the e4m3 layers' C layer (fp8_api.cpp) and their
// kernels: block-scaled linear, and the gated half of a feed-forward block.
#pragma once
#include "ops.hpp"

namespace stx {

constexpr uint32_t kE4M3 = 17;   // element type beside OpType's, with the ABI's value

// Both operands are held in blocks of 16 rows x 128 inputs: block (rb, kb) is
// 2 KiB at (rb * k_blocks + kb) * 2048, its half j (1 KiB) holds inputs
// 128 kb + 64 j + 0..63, and the 16 bytes at lane l = 16 * piece + row % 16 of a
// half are the inputs 16 piece + 0..15 of it, of row 16 rb + row % 16.  The order
// of the inputs within a block is free in a product as long as both operands
// share it, so the same bytes serve the 16x16x128 8-bit MFMA (a lane's 32 inputs are
// its 16 of either half) and, widened, four 16x16x32 16-bit ones (8 of them each).
// Inputs are padded to whole blocks with zeros; rows to whole 32-row pairs, whose
// other rows hold anything.
constexpr uint32_t fp8_k_blocks(uint64_t input) { return uint32_t((input + 127) / 128); }
constexpr uint64_t fp8_row_blocks(uint64_t rows) { return (rows + 31) / 32 * 2; }
constexpr uint64_t fp8_block_bytes(uint64_t rows, uint64_t input) {
    return fp8_row_blocks(rows) * fp8_k_blocks(input) * 2048;
}
// Scales of rounded rows: [k_blocks][rows padded to 256].
constexpr uint64_t fp8_padded_rows(uint64_t rows) { return (rows + 255) / 256 * 256; }

// One layer, or a pair (the gate and up projections of one feed-forward block)
// whose 32-row pairs of blocks alternate: gate channels 32 g + 0..31 in row
// blocks 4 g and 4 g + 1, up channels in 4 g + 2 and 4 g + 3.
struct Fp8Layer {
    const uint8_t* blocks = nullptr;
    const float* scales = nullptr;   // [ceil(N / 128)][k_blocks]; a pair's up scales behind the gate's
    const float* bias = nullptr;     // [N], padded to 32 channels, or null; likewise
    uint32_t input = 0, output = 0;  // of one projection
    bool pair = false;
};

enum Fp8Activation : uint32_t { kSilu = 0, kGelu = 1 };

struct Fp8Call {
    OpRows x, y;
    const float* x_scales = nullptr;   // e4m3 input: [rows][k_blocks]
    float* y_scales = nullptr;         // e4m3 output: [rows][ceil(N / 128)]
    uint64_t rows = 0;
    float alpha = 1.0f, beta = 0.0f;   // linear
    uint32_t activation = kSilu;       // gated
    void* workspace = nullptr;
};

// Weights of any type into blocks at every `step`-th pair of row blocks, with
// their scales ([ceil(rows / 128)][k_blocks]: copied from `given` for e4m3, or
// from the rule of the ABI).
hipError_t launch_fp8_weights(const OpRows& w, uint64_t rows, uint32_t input, const float* given, uint8_t* blocks,
                              uint32_t step, float* scales, hipStream_t stream);
// Rows of any type into blocks, with their scales.
hipError_t launch_fp8_rows(const OpRows& x, uint64_t rows, uint32_t input, const float* given, uint8_t* blocks,
                           float* scales, hipStream_t stream);
// F32 rows to e4m3 rows with their scales.
hipError_t launch_fp8_round(const float* hidden, uint32_t width, uint8_t* y, uint64_t y_stride, float* scales,
                            uint64_t rows, hipStream_t stream);
// Lets the kernels with more than 64 KiB of LDS have it, on the current device;
// every preparation of weights calls it, so no launch has to.
hipError_t fp8_allow_lds();

// How a pass of `rows` runs: its core, the core's tiles, and what lies where in
// its workspace (the activations' blocks are at 0).
enum Fp8Core : uint32_t {
    kFp8Decode,
    kFp8Split16x16, kFp8Split16x32, kFp8Split32x16, kFp8Split32x32, kFp8Split32x64, kFp8Split64x64,
    kFp8Wide128x128, kFp8Wide256x128, kFp8Wide256x256   // rows of weights x rows
};
struct Fp8Plan {
    Fp8Core core = kFp8Decode;
    uint32_t n_tiles = 0, m_tiles = 0;
    uint64_t scales_at = 0, hidden_at = 0, bytes = 0;
    bool hidden = false;   // F32 rows in the workspace that another launch rounds to e4m3
};
// exact: products in FP32 whole (F32 and e4m3 outputs); rounded: e4m3 output.
uint64_t fp8_pass_rows(uint64_t rows, uint32_t output);
Fp8Plan fp8_plan(uint64_t rows, uint32_t input, uint32_t output, bool pair, bool exact, bool rounded);
uint64_t fp8_workspace_bytes(uint64_t rows, uint32_t input, uint32_t output, bool pair, bool exact, bool rounded);
hipError_t launch_fp8(const Fp8Layer& w, const Fp8Call& call, hipStream_t stream);

}  // namespace stx
