// Host-side sizing of the beam operators.
#include "beam.hpp"

namespace stx {

BeamSplits beam_splits(uint64_t rows, uint32_t vocab, uint32_t type) {
    // Up to 512 workgroups, as many as the chip holds at once; a batch of one 16-byte load a thread where
    // batches of 16 logits are fewer than that.
    BeamSplits s;
    const uint64_t want = rows >= 512 ? 1 : 512 / rows;
    auto batches = [&] { return (uint64_t(vocab) + 512 * s.each - 1) / (512 * s.each); };
    if (batches() < want) s.each = type == kF32 ? 4 : 8;
    uint64_t splits = batches() < want ? batches() : want;
    const uint64_t each = (batches() + splits - 1) / splits;
    splits = (batches() + each - 1) / each;
    s.splits = uint32_t(splits);
    s.length = uint32_t(each) * 512 * s.each;
    return s;
}

uint64_t beam_select_workspace_bytes(uint64_t rows, uint32_t vocab, uint32_t type, uint32_t keep) {
    const uint64_t top = keep < vocab ? keep : vocab;
    return (rows * beam_splits(rows, vocab, type).splits * (8 + top * 8) + 255) / 256 * 256;
}

}  // namespace stx
