// Internal interface between the operators' C layer (ops_api.cpp) and their
// kernels: 8-bit integer linear, block norm, token log probabilities.  Plain
// structs, host-side sizing and launch functions.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace stx {

// Element types, with the ABI's values.
enum OpType : uint32_t { kF16 = 1, kBF16 = 2, kF32 = 3, kI8 = 16 };

// Rows of device memory (row stride in elements).
struct OpRows {
    const void* data = nullptr;
    uint64_t stride = 0;
    uint32_t type = 0;
};

// ---- 8-bit integer linear ----
// Both operands are held in blocks of 16 rows x 64 inputs, the operand order
// of the 16x16x64 integer MFMA: block (rb, kb) is 1 KiB at
// (rb * k_blocks + kb) * 1024, its 16 bytes at lane l = 16 * piece + row % 16
// are inputs 64 kb + 16 piece + 0..15 of row 16 rb + row % 16.  Rows are
// padded to whole 32-row pairs of blocks, whose other rows hold anything, and
// inputs to 128, with zeros.
constexpr uint32_t int8_k_blocks(uint64_t input) { return uint32_t((input + 127) / 128 * 2); }
constexpr uint64_t int8_row_blocks(uint64_t rows) { return (rows + 31) / 32 * 2; }
constexpr uint64_t int8_block_bytes(uint64_t rows, uint64_t input) {
    return int8_row_blocks(rows) * int8_k_blocks(input) * 1024;
}

struct Int8Layer {
    const int8_t* blocks = nullptr;
    const float* scales = nullptr;   // [N], padded to 32 channels
    const float* bias = nullptr;     // [N], padded, or null
    uint32_t input = 0, output = 0;
};

struct Int8Call {
    OpRows x, y;
    const float* x_scales = nullptr;   // I8 input
    uint64_t rows = 0;
    float alpha = 1.0f, beta = 0.0f;
    void* workspace = nullptr;
};

// Rows of any type into blocks, with their scales ([rows] from the rule of
// the ABI; for I8 rows copied from `given`, or left alone where that is null).
hipError_t launch_int8_stage(const OpRows& x, uint64_t rows, uint32_t input, const float* given, int8_t* blocks,
                             float* scales, hipStream_t stream);
// Lets the kernels with more than 64 KiB of LDS have it, on the current device;
// every preparation of weights calls it, so no launch has to.
hipError_t int8_allow_lds();
hipError_t launch_copy_f32(const float* from, float* to, uint64_t count, hipStream_t stream);
// Rows of one pass (a launch holds fewer than 2^32 threads).
uint64_t int8_pass_rows(uint64_t rows, uint32_t output);
// How a pass of `rows` runs: its core, the core's tiles, and where the scales
// start in its workspace (the activations' blocks are at 0).
enum Int8Core : uint32_t {
    kInt8Decode, kInt8Rows16, kInt8Direct32x32, kInt8Direct32x64, kInt8Direct64x64,   // channels x rows
    kInt8Wide128x128, kInt8Wide256x128
};
struct Int8Plan {
    Int8Core core = kInt8Decode;
    uint32_t n_tiles = 0, m_tiles = 0;
    uint64_t scales_at = 0, bytes = 0;
};
constexpr uint32_t kInt8DecodeLds = 44 * 1024;   // rows of a decode launch in LDS, beside 8 KiB of sums
Int8Plan int8_plan(uint64_t rows, uint32_t input, uint32_t output);
uint64_t int8_workspace_bytes(uint64_t rows, uint32_t input, uint32_t output);
hipError_t launch_int8_linear(const Int8Layer& w, const Int8Call& call, hipStream_t stream);

// ---- block norm ----
struct NormCall {
    OpRows block, residual, gate, hidden, normed;   // data null: absent
    const float *post_weight = nullptr, *post_bias = nullptr, *pre_weight = nullptr, *pre_bias = nullptr,
                *channel_scale = nullptr;
    uint64_t rows = 0;
    uint32_t width = 0;
    uint32_t layer = 0;           // 0 RMS, 1 LAYER
    uint32_t sigmoid = 0;
    uint32_t gate_per_row = 0;    // one value per row (its column stride is 0)
    float eps = 0, weight_offset = 0, residual_scale = 1, block_scale = 1;
};
hipError_t launch_block_norm(const NormCall& call, uint32_t type, hipStream_t stream);

// ---- token log probabilities ----
struct LogprobsCall {
    OpRows logits;
    const int32_t* tokens = nullptr;
    float* logprobs = nullptr;
    int32_t* ranks = nullptr;
    float* entropy = nullptr;
    int32_t* top_ids = nullptr;
    float* top_logprobs = nullptr;
    uint64_t rows = 0;
    uint32_t vocab = 0, top = 0;
    float scale = 1.0f;
    void* workspace = nullptr;
};
// Splits of a row of logits, in whole batches, and the workspace for their
// partial results (none for one split).
constexpr uint32_t kLogprobsBatch = 8192;
uint32_t logprobs_splits(uint64_t rows, uint32_t vocab);
uint64_t logprobs_workspace_bytes(uint64_t rows, uint32_t vocab, uint32_t top);
hipError_t launch_token_logprobs(const LogprobsCall& call, hipStream_t stream);

}  // namespace stx
