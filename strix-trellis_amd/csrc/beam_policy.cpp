// Host-side sizing of the beam operators.
#include "beam.hpp"

namespace stx {

uint64_t beam_select_workspace_bytes(uint64_t rows, uint32_t vocab, uint32_t keep) {
    const uint64_t top = keep < vocab ? keep : vocab;
    return (rows * logprobs_splits(rows, vocab) * (32 + top * 8) + 255) / 256 * 256;
}

}  // namespace stx
