// Decoding with several beams (include/strix_trellis_beam.h): argument checks and plans.
#include <algorithm>

#include "beam.hpp"
#include "ops_internal.hpp"
#include "strix_trellis_beam.h"

using namespace stx_ops;

namespace {

strix_status describe_select(strix_context c, const strix_amd_beam_select_desc* d, bool place,
                             stx::BeamSelectCall& call, uint64_t& need) {
    need = 0;
    Rules r;
    r.then([&] { return versioned(d); });
    if (!r.held()) return r.status();
    Rows x;
    r.then([&] { return read_view(d->logits, false, x); })
        .need(d->scale >= 0x1p-16f && d->scale <= 0x1p16f, STRIX_ERROR_INVALID_ARGUMENT);
    if (!r.held()) return r.status();
    const uint64_t rows = x.rows;
    r.need(is_float(x.at.type) && d->beams >= 1 && d->beams <= STRIX_AMD_MAX_BEAMS && d->keep >= 1 &&
               d->keep <= STRIX_AMD_MAX_TOP && rows % d->beams == 0,
           STRIX_ERROR_UNSUPPORTED_FORMAT);
    if (!r.held()) return r.status();
    need = rows ? stx::beam_select_workspace_bytes(rows, uint32_t(x.width), x.at.type, d->keep) : 0;
    if (!place) return STRIX_SUCCESS;
    const uint64_t places = rows / d->beams * d->keep;
    Span scores, finished, next_scores, parents, tokens, workspace;
    r.then([&] { return read_buffer(d->scores, false, rows, scores); })
        .then([&] { return read_buffer(d->finished, true, rows, finished); })
        .then([&] { return read_buffer(d->next_scores, false, places, next_scores); })
        .then([&] { return read_buffer(d->parents, false, places, parents); })
        .then([&] { return read_buffer(d->tokens, false, places, tokens); })
        .then([&] { return read_workspace(d->workspace, need, workspace); })
        .need(apart({next_scores, parents, tokens, workspace}, {x.span, scores, finished}),
              STRIX_ERROR_INVALID_ARGUMENT);
    if (!r.held()) return r.status();
    call.logits = x.at;
    call.scores = at<const float>(scores);
    call.finished = at<const int32_t>(finished);
    call.next_scores = at<float>(next_scores);
    call.parents = at<int32_t>(parents);
    call.tokens = at<int32_t>(tokens);
    call.rows = rows;
    call.vocab = uint32_t(x.width);
    call.beams = d->beams;
    call.keep = d->keep;
    call.pad = d->pad;
    call.scale = d->scale;
    call.workspace = d->workspace.data;
    if (!rows) return STRIX_SUCCESS;
    r.then([&] { return device_resident(c, x.span, x.align); })
        .then([&] { return resident(c, {scores, finished, next_scores, parents, tokens}, 4); })
        .then([&] { return device_resident(c, workspace, kWorkspaceAlign); });
    return r.status();
}

// The bytes that `s` covers.  apart: its pieces must not overlap each other.
strix_status read_states(const strix_amd_states& s, const strix_amd_beam_reorder_desc& d, bool pieces_apart,
                         Span& out) {
    struct Dim {
        uint64_t count, stride;
    } dims[3] = {{d.outer, s.strides[0]}, {d.prompts * d.beams, s.strides[1]}, {d.inner, s.strides[2]}};
    std::sort(dims, dims + 3, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
    uint64_t extent = d.bytes;
    bool disjoint = true;
    for (const Dim& x : dims) {
        if (x.count <= 1) continue;
        disjoint = disjoint && x.stride >= extent;
        uint64_t last = 0;
        if (!checked_mul(x.count - 1, x.stride, last) || __builtin_add_overflow(extent, last, &extent))
            return STRIX_ERROR_INVALID_ARGUMENT;
    }
    out = Span(s.data, extent);
    Rules r;
    r.need(disjoint || !pieces_apart, STRIX_ERROR_UNSUPPORTED_FORMAT)
        .need(out.addressable(), STRIX_ERROR_INVALID_ARGUMENT)
        .need(extent <= s.buffer_bytes, STRIX_ERROR_INSUFFICIENT_BUFFER)
        .need(s.data != nullptr, STRIX_ERROR_INVALID_ARGUMENT);
    return r.status();
}

strix_status describe_reorder(strix_context c, const strix_amd_beam_reorder_desc* d, stx::BeamReorderCall& call) {
    Rules r;
    r.then([&] { return versioned(d); });
    if (!r.held()) return r.status();
    uint64_t rows = 0;
    r.need(!d->flags, STRIX_ERROR_INVALID_ARGUMENT)
        .need(d->beams >= 1 && d->beams <= STRIX_AMD_MAX_BEAMS && d->prompts <= INT_MAX && d->outer <= INT_MAX &&
                  d->inner <= INT_MAX && d->bytes <= INT64_MAX,
              STRIX_ERROR_UNSUPPORTED_FORMAT)
        .need(checked_mul(d->prompts, d->beams, rows), STRIX_ERROR_INVALID_ARGUMENT);
    if (!r.held()) return r.status();
    if (!rows || !d->outer || !d->inner || !d->bytes) return STRIX_SUCCESS;   // nothing to move
    Span parents, source, target;
    r.then([&] { return read_buffer(d->parents, false, rows, parents); })
        .then([&] { return read_states(d->source, *d, false, source); })
        .then([&] { return read_states(d->target, *d, true, target); });
    if (!r.held()) return r.status();
    const uint64_t counts[3] = {d->outer, rows, d->inner};
    bool same = source.at == target.at;
    for (int i = 0; i < 3; ++i) same = same && (counts[i] == 1 || d->source.strides[i] == d->target.strides[i]);
    r.need(same || !source.meets(target), STRIX_ERROR_INVALID_ARGUMENT)
        .need(!target.meets(parents), STRIX_ERROR_INVALID_ARGUMENT)
        .then([&] { return device_resident(c, parents, 4); })
        .then([&] { return resident(c, {source, target}, 1); });
    if (!r.held()) return r.status();
    call.parents = at<const int32_t>(parents);
    call.source = static_cast<const uint8_t*>(d->source.data);
    call.target = static_cast<uint8_t*>(d->target.data);
    call.prompts = d->prompts;
    call.outer = d->outer;
    call.inner = d->inner;
    call.bytes = d->bytes;
    call.beams = d->beams;
    call.in_place = same;
    for (int i = 0; i < 3; ++i) {
        call.source_strides[i] = counts[i] > 1 ? d->source.strides[i] : 0;
        call.target_strides[i] = counts[i] > 1 ? d->target.strides[i] : 0;
    }
    return STRIX_SUCCESS;
}

struct SelectPlan final : strix_amd_op_plan_impl {
    stx::BeamSelectCall call{};
    strix_status describe(strix_context c, const strix_amd_beam_select_desc* d) {
        uint64_t need = 0;
        return describe_select(c, d, true, call, need);
    }
    hipError_t launch() const override { return call.rows ? stx::launch_beam_select(call, stream) : hipSuccess; }
};
struct ReorderPlan final : strix_amd_op_plan_impl {
    stx::BeamReorderCall call{};
    strix_status describe(strix_context c, const strix_amd_beam_reorder_desc* d) { return describe_reorder(c, d, call); }
    hipError_t launch() const override { return call.prompts ? stx::launch_beam_reorder(call, stream) : hipSuccess; }
};

}  // namespace

extern "C" {

strix_status strix_amd_beam_select_workspace_bytes(strix_context c, const strix_amd_beam_select_desc* d,
                                                   uint64_t* out) {
    stx::BeamSelectCall call;
    return query(c, out, [&](uint64_t& need) { return describe_select(c, d, false, call, need); });
}

strix_status strix_amd_beam_select(strix_context c, const strix_amd_beam_select_desc* d, const strix_stream* stream) {
    return direct<SelectPlan>(c, d, stream);
}

strix_status strix_amd_beam_select_plan_create(strix_context c, const strix_amd_beam_select_desc* d,
                                               const strix_stream* stream, strix_amd_op_plan* out) {
    return create<SelectPlan>(c, d, stream, out);
}

strix_status strix_amd_beam_reorder(strix_context c, const strix_amd_beam_reorder_desc* d,
                                    const strix_stream* stream) {
    return direct<ReorderPlan>(c, d, stream);
}

strix_status strix_amd_beam_reorder_plan_create(strix_context c, const strix_amd_beam_reorder_desc* d,
                                                const strix_stream* stream, strix_amd_op_plan* out) {
    return create<ReorderPlan>(c, d, stream, out);
}

}  // extern "C"
