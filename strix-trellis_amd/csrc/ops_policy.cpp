// Host-side sizing of the operators around the trellis layers.  Plain host
// code, so that the C layer can be built and tested against a fake HIP runtime
// with these same rules.
#include "ops.hpp"

namespace stx {

uint64_t int8_pass_rows(uint64_t rows, uint32_t output) {
    // 64 x 64 tiles of 512 threads: 2^22 of them, 2^16 rows at most (smaller tiles are
    // taken only where they are few)
    const uint64_t n_tiles = (uint64_t(output) + 63) / 64, most = (uint64_t(1) << 22) / n_tiles;
    const uint64_t pass = 64 * (most < 1024 ? most : 1024);
    return rows < pass ? rows : pass;
}

Int8Plan int8_plan(uint64_t rows, uint32_t input, uint32_t output) {
    Int8Plan p;
    const uint64_t kbs = int8_k_blocks(input);
    // A few rows: every 16-channel workgroup rounds the rows itself, which saves a
    // launch but costs each of them the rows' reads.  Against the two launches:
    // 5120^2 one / two / four rows 4.2 / 4.9 / 6.1 us for 7.7, 5120 -> 129280 four
    // rows 111 for 117, 8192^2 four rows 14.3 for 14.8, 2048 -> 8192 eight rows 5.1
    // for 5.9; but 12288 -> 4096 three rows 14.0 for 13.5, 4096 -> 12288 eight rows
    // 11.7 for 10.8.
    const bool decode = rows <= 2 || (rows <= 4 && input <= 8192) || (rows <= 8 && input <= 2048);
    if (decode && rows * (kbs * 64 + 64) <= kInt8DecodeLds) return p;   // needs no workspace
    p.scales_at = int8_block_bytes(rows, input);
    p.bytes = (p.scales_at + rows * 4 + 255) & ~uint64_t(255);
    auto tile = [&](Int8Core core, uint32_t channels, uint32_t tile_rows) {
        p.core = core;
        p.n_tiles = (output + channels - 1) / channels;
        p.m_tiles = uint32_t((rows + tile_rows - 1) / tile_rows);
        return uint64_t(p.n_tiles) * p.m_tiles;
    };
    if (rows <= 16) {
        tile(kInt8Rows16, 16, 16);
        return p;
    }
    // The tile with the least estimated time: a start, and for each round (tiles over
    // 256 compute units, rounded up) a part that is fixed and one that grows with the
    // K blocks.  The figures (us) are fitted to 9 layers, 1152 to 12288 inputs and
    // 512 to 20480 channels, at 17 to 1024 rows: of 135 cases the choice is within 4 % of
    // the fastest in 132, 14 % behind it at worst.  Small tiles fill the compute units with few rows and
    // channels, large ones read less: 5120^2 96 / 192 / 512 rows 12.6 / 19.0 / 39.5 us
    // in 32 x 32 tiles, 14.7 / 16.8 / 38.1 in 32 x 64, 14.7 / 15.8 / 39.7 in 64 x 64,
    // 26.7 / 27.1 / 29.9 in 128 x 128.
    const struct {
        Int8Core core;
        uint32_t channels, rows;
        float start, round, per_block;
    } tiles[] = {{kInt8Direct32x32, 32, 32, 2.2f, 0.35f, 0.036f},
                 {kInt8Direct32x64, 32, 64, 1.8f, 1.3f, 0.046f},
                 {kInt8Direct64x64, 64, 64, 1.5f, 3.5f, 0.08f},
                 {kInt8Wide128x128, 128, 128, 5.5f, 0.0f, 0.215f}};
    float least = 0;
    int best = -1;
    for (int i = 0; i < 4; ++i) {
        const auto& t = tiles[i];
        const uint64_t rounds = (tile(t.core, t.channels, t.rows) + 255) / 256;
        const float us = t.start + float(rounds) * (t.round + t.per_block * float(kbs));
        if (best < 0 || us < least) best = i, least = us;
    }
    tile(tiles[best].core, tiles[best].channels, tiles[best].rows);
    if (tiles[best].core != kInt8Wide128x128) return p;
    // The larger LDS tile where it still fills two rounds: 4096 -> 12288 2048 rows
    // 112 us in 128 x 128, 107 in 256 x 128; 1024 rows 61 and 66.
    if (tile(kInt8Wide256x128, 256, 128) < 640) tile(kInt8Wide128x128, 128, 128);
    return p;
}

uint64_t int8_workspace_bytes(uint64_t rows, uint32_t input, uint32_t output) {
    return int8_plan(int8_pass_rows(rows, output), input, output).bytes;
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
