// Host-side sizing of the e4m3 layers.  Plain host code, so that the C layer can
// be built and tested against a fake HIP runtime with these same rules.
#include <iterator>

#include "fp8.hpp"

namespace stx {

uint64_t fp8_pass_rows(uint64_t rows, uint32_t output) {
    // tiles of 32 x 32 and 512 threads at the least: 2^22 of them (a launch holds fewer
    // than 2^32 threads), 2^16 rows at most
    const uint64_t n_tiles = (uint64_t(output) + 31) / 32, most = (uint64_t(1) << 22) / n_tiles;
    const uint64_t pass = 32 * (most < 2048 ? most : 2048) & ~uint64_t(127);
    return rows < pass ? rows : pass;
}

Fp8Plan fp8_plan(uint64_t rows, uint32_t input, uint32_t output, bool pair, bool exact, bool rounded) {
    Fp8Plan p;
    const uint64_t kbs = fp8_k_blocks(input);
    auto place_hidden = [&] {
        // tiles of whole blocks of 128 channels round them themselves
        p.hidden = rounded && p.core != kFp8Wide256x128;
        if (!p.hidden) return;
        p.hidden_at = p.bytes;
        p.bytes += (rows * output * 4 + 255) & ~uint64_t(255);
    };
    const bool decode = rows <= 2 || (rows <= 4 && input <= 8192) || (rows <= 8 && input <= 2048);
    if (decode) {
        place_hidden();
        return p;
    }
    // The tile with the least estimated time (us): a start, and for each round (tiles over 256 compute
    // units, rounded up; the small ones, whose channel tiles stay with their XCD, over 32 in the fullest of
    // eight) a part that is fixed and one that grows with the K blocks.  The figures are fitted to 9 layers,
    // 1152 to 12288 inputs and 1152 to 16384 channels, at 5 to 4096 rows, each product in its two kinds: of 301
    // cases the choice is 0.5 % behind the fastest on average, 16 % at worst.  Small tiles fill the compute
    // units with few rows and channels, large ones read less: 4096^2 48 / 192 / 1024 / 4096 rows
    // take 8.7 / 15.7 / - / - us in 32 x 32, 12.8 / 14.3 / 43 / - in 64 x 64, - / 30 / 33 / 90 in 128 x 128,
    // - / 58 / 59 / 74 in 256 x 256 (BF16 rows and outputs).
    struct Tile {
        Fp8Core core;
        uint32_t weights, rows;   // rows of weights x rows
        float start, round, per_block;
    };
    static const Tile fast[] = {
        {kFp8Split16x16, 16, 16, 4.68f, 1.04f, 0.0515f}, {kFp8Split16x32, 16, 32, 4.64f, 0.48f, 0.0682f},
        {kFp8Split32x16, 32, 16, 5.56f, 0.76f, 0.0698f}, {kFp8Split32x32, 32, 32, 5.19f, 0.62f, 0.0878f},
        {kFp8Split32x64, 32, 64, 3.48f, 2.61f, 0.1327f}, {kFp8Split64x64, 64, 64, 3.98f, 3.92f, 0.1906f},
        {kFp8Wide128x128, 128, 128, 9.16f, 1.29f, 0.5623f}, {kFp8Wide256x128, 256, 128, 1.38f, 8.29f, 0.8246f},
        {kFp8Wide256x256, 256, 256, 0.0f, 15.42f, 1.3404f}};
    static const Tile whole[] = {
        {kFp8Split16x16, 16, 16, 4.95f, 1.07f, 0.0526f}, {kFp8Split16x32, 16, 32, 4.86f, 0.48f, 0.0698f},
        {kFp8Split32x16, 32, 16, 6.03f, 0.81f, 0.0721f}, {kFp8Split32x32, 32, 32, 5.51f, 0.74f, 0.0935f},
        {kFp8Split32x64, 32, 64, 3.77f, 3.14f, 0.1625f}, {kFp8Split64x64, 64, 64, 4.94f, 4.60f, 0.2392f},
        {kFp8Wide128x128, 128, 128, 11.5f, 0.82f, 0.9506f}, {kFp8Wide256x128, 256, 128, 2.28f, 8.13f, 1.5178f}};
    const Tile* const begin = exact ? std::begin(whole) : std::begin(fast);
    const Tile* const end = exact ? std::end(whole) : std::end(fast);
    const uint64_t weights = pair ? (uint64_t(output) + 31) / 32 * 64 : output;
    auto over = [](uint64_t n, uint64_t each) { return (n + each - 1) / each; };
    auto tile = [&](const Tile& t) {
        p.core = t.core;
        p.n_tiles = uint32_t(over(weights, t.weights));
        p.m_tiles = uint32_t(over(rows, t.rows));
    };
    const Tile* best = nullptr;
    float least = 0;
    for (const Tile* t = begin; t != end; ++t) {
        if (pair && t->weights < 32) continue;   // a tile of both projections
        tile(*t);
        float rounds;
        if (t->core < kFp8Wide128x128) {
            rounds = float(over(over(p.n_tiles, 8) * p.m_tiles, 32));
        } else {
            const uint64_t tiles = uint64_t(p.n_tiles) * p.m_tiles;
            rounds = float(over(tiles, 256));
            // two of these to a compute unit: half a round is not lost
            if (t->core == kFp8Wide128x128) rounds = 0.5f * (rounds + (tiles > 256 ? float(tiles) / 256.0f : 1.0f));
        }
        float us = t->start + rounds * (t->round + t->per_block * float(kbs));
        // a launch of its own, and F32 values written and read
        if (rounded && t->core != kFp8Wide256x128) us += 2.5f + 2e-6f * float(rows) * float(output);
        if (!best || us < least) best = t, least = us;
    }
    tile(*best);
    p.scales_at = fp8_block_bytes(rows, input);
    p.bytes = p.scales_at + ((kbs * fp8_padded_rows(rows) * 4 + 255) & ~uint64_t(255));
    place_hidden();
    return p;
}

uint64_t fp8_workspace_bytes(uint64_t rows, uint32_t input, uint32_t output, bool pair, bool exact, bool rounded) {
    // a pass of fewer rows takes another core, and so may the last one: no more than the first
    const uint64_t pass = fp8_pass_rows(rows, output), last = rows % pass;
    const uint64_t first = fp8_plan(pass, input, output, pair, exact, rounded).bytes;
    const uint64_t rest = last ? fp8_plan(last, input, output, pair, exact, rounded).bytes : 0;
    return first > rest ? first : rest;
}

}  // namespace stx
