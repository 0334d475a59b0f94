// Fake launchers of the operators around the trellis layers: each checks that
// every buffer its kernels would touch lies in a live fake allocation, and
// returns the injected launch result.
#include "fake.hpp"
#include "ops.hpp"

#include <cstdio>
#include <cstdlib>

namespace {

uint64_t size_of(uint32_t type) { return type == stx::kF32 ? 4 : type == stx::kI8 ? 1 : 2; }

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

hipError_t launch_int8_stage(const OpRows& x, uint64_t rows, uint32_t input, const float* given, int8_t* blocks,
                             float* scales, hipStream_t s) {
    rows_ok(x, rows, input, "rows outside device memory");
    require(fake::in_live_block(blocks, int8_block_bytes(rows, input)), "blocks outside device memory");
    require(fake::in_live_block(scales, rows * 4), "scales outside device memory");
    require((x.type == kI8) == (given != nullptr), "scales of rows that are not int8");
    require(!given || fake::in_live_block(given, rows * 4), "given scales outside device memory");
    return note("int8_stage", rows, s);
}

hipError_t int8_allow_lds() { return fake::launch_result(); }

hipError_t launch_copy_f32(const float* from, float* to, uint64_t count, hipStream_t s) {
    require(fake::in_live_block(from, count * 4) && fake::in_live_block(to, count * 4), "copy outside device memory");
    return note("copy", count, s);
}

hipError_t launch_int8_linear(const Int8Layer& w, const Int8Call& c, hipStream_t s) {
    require(c.rows > 0, "no rows");
    rows_ok(c.x, c.rows, w.input, "input outside device memory");
    rows_ok(c.y, c.rows, w.output, "output outside device memory");
    require(fake::in_live_block(w.blocks, int8_block_bytes(w.output, w.input)), "weights outside device memory");
    require(fake::in_live_block(w.scales, int8_row_blocks(w.output) * 64), "scales outside device memory");
    require(!w.bias || fake::in_live_block(w.bias, int8_row_blocks(w.output) * 64), "bias outside device memory");
    const uint64_t need = int8_workspace_bytes(c.rows, w.input, w.output);
    require(!need || fake::in_live_block(c.workspace, need), "workspace too small");
    return note("int8_linear", c.rows, s);
}

hipError_t launch_block_norm(const NormCall& c, uint32_t type, hipStream_t s) {
    require(c.rows > 0 && type >= kF16 && type <= kF32, "no rows or type");
    for (const OpRows* r : {&c.block, &c.residual, &c.hidden, &c.normed})
        if (r->data) rows_ok(*r, c.rows, c.width, "rows outside device memory");
    if (c.gate.data) rows_ok(c.gate, c.rows, c.gate_per_row ? 1 : c.width, "gate outside device memory");
    for (const float* v : {c.post_weight, c.post_bias, c.pre_weight, c.pre_bias, c.channel_scale})
        require(!v || fake::in_live_block(v, c.width * 4), "vector outside device memory");
    return note("block_norm", c.rows, s);
}

hipError_t launch_token_logprobs(const LogprobsCall& c, hipStream_t s) {
    require(c.rows > 0 && c.top <= c.vocab, "no rows or too many tokens");
    rows_ok(c.logits, c.rows, c.vocab, "logits outside device memory");
    for (const void* v : {(const void*)c.tokens, (const void*)c.logprobs, (const void*)c.ranks, (const void*)c.entropy})
        require(!v || fake::in_live_block(v, c.rows * 4), "row results outside device memory");
    for (const void* v : {(const void*)c.top_ids, (const void*)c.top_logprobs})
        require(!v || fake::in_live_block(v, c.rows * c.top * 4), "first tokens outside device memory");
    const uint64_t need = logprobs_workspace_bytes(c.rows, c.vocab, c.top);
    require(!need || fake::in_live_block(c.workspace, need), "workspace too small");
    return note("token_logprobs", c.rows, s);
}

}  // namespace stx
