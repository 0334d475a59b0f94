// Fake launchers of the e4m3 layers and the beam operators: each checks that every
// buffer its kernels would touch lies in a live fake allocation, and returns the
// injected launch result.
#include "beam.hpp"
#include "fake.hpp"
#include "fp8.hpp"

#include <cstdio>
#include <cstdlib>

namespace {

uint64_t size_of(uint32_t type) { return type == stx::kF32 ? 4 : type == stx::kE4M3 ? 1 : 2; }

void require(bool ok, const char* what) {
    if (ok) return;
    std::fprintf(stderr, "contract violation: %s\n", what);
    std::abort();
}

void rows_ok(const stx::OpRows& r, uint64_t rows, uint64_t width, const char* what) {
    require(fake::in_live_block(r.data, ((rows - 1) * r.stride + width) * size_of(r.type)), what);
}

hipError_t note(const char* name, uint64_t rows, hipStream_t s) {
    fake::Launch l;
    l.name = name;
    l.rows = rows;
    l.stream = s;
    fake::launches.push_back(l);
    return fake::launch_result();
}

}  // namespace

namespace stx {

hipError_t launch_fp8_weights(const OpRows& w, uint64_t rows, uint32_t input, const float* given, uint8_t* blocks,
                              uint32_t step, float* scales, hipStream_t s) {
    rows_ok(w, rows, input, "weights outside device memory");
    const uint64_t kbs = fp8_k_blocks(input), scales_bytes = (rows + 127) / 128 * kbs * 4;
    // the last pair of row blocks at every step-th
    const uint64_t pairs = fp8_row_blocks(rows) / 2, end = ((pairs - 1) * step * 2 + 2) * kbs * 2048;
    require(fake::in_live_block(blocks, end), "blocks outside device memory");
    require(fake::in_live_block(scales, scales_bytes), "scales outside device memory");
    require((w.type == kE4M3) == (given != nullptr), "scales of weights that are not e4m3");
    require(!given || fake::in_live_block(given, scales_bytes), "given scales outside device memory");
    return note("fp8_weights", rows, s);
}

hipError_t fp8_allow_lds() { return fake::launch_result(); }

hipError_t launch_fp8(const Fp8Layer& w, const Fp8Call& c, hipStream_t s) {
    require(c.rows > 0, "no rows");
    rows_ok(c.x, c.rows, w.input, "input outside device memory");
    rows_ok(c.y, c.rows, w.output, "output outside device memory");
    const uint64_t parts = w.pair ? 2 : 1, kbs = fp8_k_blocks(w.input), nbs = (w.output + 127) / 128;
    require(fake::in_live_block(w.blocks, fp8_block_bytes(w.output, w.input) * parts), "weights outside device memory");
    require(fake::in_live_block(w.scales, kbs * nbs * 4 * parts), "scales outside device memory");
    require(!w.bias || fake::in_live_block(w.bias, fp8_row_blocks(w.output) * 64 * parts), "bias outside device memory");
    require(reinterpret_cast<uintptr_t>(w.bias) % 16 == 0, "bias off its alignment");
    require((c.x.type == kE4M3) == (c.x_scales != nullptr), "input scales");
    require((c.y.type == kE4M3) == (c.y_scales != nullptr), "output scales");
    require(!c.x_scales || fake::in_live_block(c.x_scales, c.rows * kbs * 4), "input scales outside device memory");
    require(!c.y_scales || fake::in_live_block(c.y_scales, c.rows * nbs * 4), "output scales outside device memory");
    const uint64_t need = fp8_workspace_bytes(c.rows, w.input, w.output, w.pair, c.y.type == kE4M3 || c.y.type == kF32, c.y.type == kE4M3);
    require(!need || fake::in_live_block(c.workspace, need), "workspace too small");
    return note(w.pair ? "fp8_gated" : "fp8_linear", c.rows, s);
}

hipError_t launch_beam_select(const BeamSelectCall& c, hipStream_t s) {
    require(c.rows > 0 && c.rows % c.beams == 0 && c.keep >= 1, "no rows");
    rows_ok(c.logits, c.rows, c.vocab, "logits outside device memory");
    require(fake::in_live_block(c.scores, c.rows * 4), "scores outside device memory");
    require(!c.finished || fake::in_live_block(c.finished, c.rows * 4), "flags outside device memory");
    for (const void* v : {(const void*)c.next_scores, (const void*)c.parents, (const void*)c.tokens})
        require(fake::in_live_block(v, c.rows / c.beams * c.keep * 4), "results outside device memory");
    require(fake::in_live_block(c.workspace, beam_select_workspace_bytes(c.rows, c.vocab, c.logits.type, c.keep)), "workspace too small");
    return note("beam_select", c.rows, s);
}

hipError_t launch_beam_reorder(const BeamReorderCall& c, hipStream_t s) {
    const uint64_t rows = c.prompts * c.beams;
    require(rows && c.outer && c.inner && c.bytes, "nothing to move");
    require(fake::in_live_block(c.parents, rows * 4), "parents outside device memory");
    auto end = [&](const uint64_t* strides) {
        return (c.outer - 1) * strides[0] + (rows - 1) * strides[1] + (c.inner - 1) * strides[2] + c.bytes;
    };
    require(fake::in_live_block(c.source, end(c.source_strides)), "source outside device memory");
    require(fake::in_live_block(c.target, end(c.target_strides)), "target outside device memory");
    require(c.in_place == (c.source == c.target), "in place");
    return note("beam_reorder", rows, s);
}

}  // namespace stx
