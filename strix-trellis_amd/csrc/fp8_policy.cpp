// Host-side sizing of the e4m3 layers.  Plain host code, so that the C layer can
// be built and tested against a fake HIP runtime with these same rules.
#include "fp8.hpp"

namespace stx {

uint64_t fp8_pass_rows(uint64_t rows, uint32_t output) {
    // tiles of 32 x 32 and 512 threads at the least: 2^22 of them (a launch holds fewer
    // than 2^32 threads), 2^16 rows at most
    const uint64_t n_tiles = (uint64_t(output) + 31) / 32, most = (uint64_t(1) << 22) / n_tiles;
    const uint64_t pass = 32 * (most < 2048 ? most : 2048) & ~uint64_t(127);
    return rows < pass ? rows : pass;
}

Fp8Plan fp8_plan(uint64_t rows, uint32_t input, uint32_t output, bool pair, bool rounded) {
    Fp8Plan p;
    const uint64_t kbs = fp8_k_blocks(input);
    auto place_hidden = [&] {
        if (!rounded) return;
        p.hidden_at = p.bytes;
        p.bytes += (rows * output * 4 + 255) & ~uint64_t(255);
    };
    const bool decode = rows <= 2 || (rows <= 4 && input <= 8192) || (rows <= 8 && input <= 2048);
    if (decode && rows * (kbs * 132 + 64) <= kFp8DecodeLds) {
        place_hidden();
        return p;
    }
    p.scales_at = fp8_block_bytes(rows, input);
    p.bytes = p.scales_at + ((kbs * fp8_padded_rows(rows) * 4 + 255) & ~uint64_t(255));
    auto tile = [&](Fp8Core core, uint32_t channels, uint32_t tile_rows) {
        p.core = core;
        p.n_tiles = uint32_t(((pair ? (uint64_t(output) + 31) / 32 * 64 : output) + channels - 1) / channels);
        p.m_tiles = uint32_t((rows + tile_rows - 1) / tile_rows);
        return uint64_t(p.n_tiles) * p.m_tiles;
    };
    if (rows <= 16) tile(kFp8Rows16, pair ? 32 : 16, 16);
    else if (rows <= 32) tile(pair ? kFp8Direct64x32 : kFp8Direct32x32, pair ? 64 : 32, 32);
    else tile(kFp8Direct64x64, 64, 64);
    place_hidden();
    return p;
}

uint64_t fp8_workspace_bytes(uint64_t rows, uint32_t input, uint32_t output, bool pair, bool rounded) {
    // a pass of fewer rows takes another core, and so may the last one: no more than the first
    const uint64_t pass = fp8_pass_rows(rows, output), last = rows % pass;
    const uint64_t first = fp8_plan(pass, input, output, pair, rounded).bytes;
    const uint64_t rest = last ? fp8_plan(last, input, output, pair, rounded).bytes : 0;
    return first > rest ? first : rest;
}

}  // namespace stx
