// Internal interface between the beam operators' C layer (beam_api.cpp) and their kernels.
#pragma once
#include "ops.hpp"

namespace stx {

struct BeamSelectCall {
    OpRows logits;
    const float* scores = nullptr;
    const int32_t* finished = nullptr;
    float* next_scores = nullptr;
    int32_t* parents = nullptr;
    int32_t* tokens = nullptr;
    uint64_t rows = 0;
    uint32_t vocab = 0, beams = 1, keep = 1;
    int32_t pad = 0;
    float scale = 1.0f;
    void* workspace = nullptr;
};
// How a row of logits is read: in batches of 512 threads x `each` logits, and in splits of whole
// batches, a workgroup each.
struct BeamSplits {
    uint32_t each = 16, splits = 1, length = 0;
};
BeamSplits beam_splits(uint64_t rows, uint32_t vocab, uint32_t type);
uint64_t beam_select_workspace_bytes(uint64_t rows, uint32_t vocab, uint32_t type, uint32_t keep);
hipError_t launch_beam_select(const BeamSelectCall& call, hipStream_t stream);

struct BeamReorderCall {
    const int32_t* parents = nullptr;
    const uint8_t* source = nullptr;
    uint8_t* target = nullptr;
    uint64_t prompts = 0, outer = 0, inner = 0, bytes = 0;
    uint64_t source_strides[3] = {}, target_strides[3] = {};   // outer, row, inner
    uint32_t beams = 1;
    bool in_place = false;
};
hipError_t launch_beam_reorder(const BeamReorderCall& call, hipStream_t stream);

}  // namespace stx
