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
    // The tile with the least estimated time (us): a start; for each round (tiles over 256 compute
    // units, rounded up; the small ones, whose channel tiles stay with their XCD, over 32 in the fullest of
    // eight; several to a compute unit at once where `resident` says so) a part that is fixed and one that
    // grows with the K blocks; and for tiles that share a compute unit what each adds.  The figures are fitted
    // to 17 layers, 1152 to 16384 inputs and 1024 to 20480 channels, at 5 to 4096 rows, each product in its two
    // kinds: of 333 cases each the choice is 0.8 and 0.6 % behind the fastest on average, 25 and 23 % at
    // worst.  Small tiles fill the compute units with few rows and channels, large ones read less: 4096^2
    // 48 / 200 / 1024 / 4096 rows take 8.3 / 18 / 65 / 338 us in 32 x 32, 12 / 14 / 41 / 206 in 64 x 64,
    // 24 / 26 / 30 / 85 in 128 x 128, - / 52 / 54 / 73 in 256 x 256 (BF16 rows and outputs).
    struct Tile {
        Fp8Core core;
        uint32_t weights, rows, resident;   // rows of weights x rows
        float start, round, round_block, tile_block;
    };
    static const Tile fast[] = {
        {kFp8Split16x16, 16, 16, 2, 5.15f, 0.16f, 0.0484f, 0.0162f}, {kFp8Split16x32, 16, 32, 2, 3.12f, 1.48f, 0.0086f, 0.0627f},
        {kFp8Split32x16, 32, 16, 2, 4.47f, 0.0f, 0.0362f, 0.0596f}, {kFp8Split32x32, 32, 32, 2, 5.23f, 0.47f, 0.0151f, 0.0717f},
        {kFp8Split32x64, 32, 64, 1, 4.43f, 1.02f, 0.1297f, 0.0f}, {kFp8Split64x64, 64, 64, 1, 3.06f, 2.98f, 0.1802f, 0.0f},
        {kFp8Wide128x128, 128, 128, 1, 6.08f, 2.78f, 0.5592f, 0.0f}, {kFp8Wide256x128, 256, 128, 1, 0.91f, 6.51f, 0.9370f, 0.0f},
        {kFp8Wide256x256, 256, 256, 1, 0.32f, 9.59f, 1.4899f, 0.0f}};
    static const Tile whole[] = {
        {kFp8Split16x16, 16, 16, 2, 2.90f, 0.02f, 0.0569f, 0.0538f}, {kFp8Split16x32, 16, 32, 2, 1.78f, 1.11f, 0.0058f, 0.0823f},
        {kFp8Split32x16, 32, 16, 2, 0.83f, 0.0f, 0.3046f, 0.0507f}, {kFp8Split32x32, 32, 32, 2, 4.37f, 0.93f, 0.0014f, 0.0906f},
        {kFp8Split32x64, 32, 64, 1, 3.08f, 2.34f, 0.1707f, 0.0f}, {kFp8Split64x64, 64, 64, 1, 3.65f, 3.07f, 0.2671f, 0.0f},
        {kFp8Wide128x128, 128, 128, 1, 9.85f, 0.46f, 0.9211f, 0.0f}, {kFp8Wide256x128, 256, 128, 1, 0.39f, 5.88f, 1.5156f, 0.0f}};
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
        if (t->weights * t->rows < 1024 && rows > 128) continue;   // measured up to there
        tile(*t);
        if (over(p.n_tiles, 8) * 8 * p.m_tiles >= uint64_t(1) << 23) continue;   // more threads than a launch holds
        float rounds;
        if (t->core < kFp8Wide128x128) {
            rounds = float(over(over(p.n_tiles, 8) * p.m_tiles, 32));
        } else {
            const uint64_t tiles = uint64_t(p.n_tiles) * p.m_tiles;
            rounds = float(over(tiles, 256));
            // two of these to a compute unit: half a round is not lost
            if (t->core == kFp8Wide128x128) rounds = 0.5f * (rounds + (tiles > 256 ? float(tiles) / 256.0f : 1.0f));
        }
        const uint64_t shared = (uint64_t(rounds) + t->resident - 1) / t->resident;
        const float turns = t->resident > 1 ? float(shared) : rounds;
        float us = t->start + turns * (t->round + t->round_block * float(kbs)) + rounds * t->tile_block * float(kbs);
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
