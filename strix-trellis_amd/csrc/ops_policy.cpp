// Host-side sizing of the operators around the trellis layers.  Plain host
// code, so that the C layer can be built and tested against a fake HIP runtime
// with these same rules.
#include "ops.hpp"

namespace stx {

uint64_t int8_pass_rows(uint64_t rows, uint32_t output) {
    const uint64_t n_tiles = (uint64_t(output) + 127) / 128, most = (uint64_t(1) << 22) / n_tiles;
    const uint64_t pass = 128 * (most < 2048 ? most : 2048);
    return rows < pass ? rows : pass;
}

uint64_t int8_workspace_bytes(uint64_t rows, uint32_t input, uint32_t output) {
    rows = int8_pass_rows(rows, output);
    return int8_block_bytes(rows, input) + (rows * 4 + 255) / 256 * 256;
}

// Enough workgroups for few rows, whole batches each.
uint32_t logprobs_splits(uint64_t rows, uint32_t vocab) {
    const uint64_t batches = (uint64_t(vocab) + kLogprobsBatch - 1) / kLogprobsBatch;
    uint64_t want = rows >= 512 ? 1 : 512 / rows;
    if (want > batches) want = batches;
    const uint64_t each = (batches + want - 1) / want;
    return uint32_t((batches + each - 1) / each);
}

uint64_t logprobs_workspace_bytes(uint64_t rows, uint32_t vocab, uint32_t top) {
    const uint32_t splits = logprobs_splits(rows, vocab);
    if (splits == 1) return 0;
    return (rows * splits * (32 + uint64_t(top) * 8) + 255) / 256 * 256;
}

}  // namespace stx
