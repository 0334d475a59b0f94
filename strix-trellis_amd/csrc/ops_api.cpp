// Operators around the trellis layers (include/strix_trellis_ops.h): argument
// checks, the int8 weights, and prepared operators.
//
// Each operator is described by one function, which checks the descriptor and
// the device residence of every buffer and leaves the kernels' arguments; a
// direct call launches with them, a plan keeps them.  The order of the checks
// is the linear calls': device, stream, descriptor, shapes and types,
// overlaps, residence.
#include <climits>
#include <cmath>
#include <new>

#include "api_internal.hpp"
#include "ops.hpp"
#include "strix_trellis_ops.h"

using namespace stx_api;

struct strix_amd_int8_weights_impl {
    strix_context owner = nullptr;
    stx::Int8Layer layer{};
    void* base = nullptr;     // one private allocation: blocks | scales | bias
    uint64_t bytes = 0;
    uint64_t plans = 0;       // live plans retaining these weights
};

namespace {

enum class Op { kInt8, kNorm, kLogprobs };

}  // namespace

// A plan counts among its context's live handles (strix_context_impl::weights_live).
struct strix_amd_op_plan_impl {
    strix_context owner = nullptr;
    hipStream_t stream{};
    Op op = Op::kInt8;
    strix_amd_int8_weights weights = nullptr;
    stx::Int8Call int8{};
    stx::NormCall norm{};
    uint32_t norm_type = 0;
    stx::LogprobsCall logprobs{};
};

namespace {

uint64_t size_of(uint32_t type) {
    return type == stx::kF32 ? 4 : type == stx::kF16 || type == stx::kBF16 ? 2 : type == stx::kI8 ? 1 : 0;
}
bool is_float(uint32_t type) { return type == stx::kF32 || type == stx::kF16 || type == stx::kBF16; }

// A view of the descriptor and the bytes it covers.
struct Rows {
    bool given = false;
    uint64_t rows = 0, width = 0;
    stx::OpRows at{};
    Span span;
    uint64_t align = 1;
};

bool absent(const strix_amd_view& v) {
    static const strix_amd_view none{};
    return std::memcmp(&v, &none, sizeof(v)) == 0;
}

strix_status read_view(const strix_amd_view& v, bool optional, Rows& out) {
    out = {};
    if (optional && absent(v)) return STRIX_SUCCESS;
    const uint64_t size = size_of(v.dtype);
    uint64_t last = 0, elements = 0, bytes = 0;
    Rules r;
    r.then([&] { return versioned(&v); })
        .need(!v.flags, STRIX_ERROR_INVALID_ARGUMENT)
        .need(size && v.rows <= INT_MAX && v.width >= 1 && v.width <= INT_MAX, STRIX_ERROR_UNSUPPORTED_FORMAT);
    if (!r.held()) return r.status();
    // row_stride counts only between rows
    const uint64_t gaps = v.rows ? v.rows - 1 : 0;
    r.need(!gaps || v.row_stride >= v.width, STRIX_ERROR_UNSUPPORTED_FORMAT)
        .need(!v.rows || ((!gaps || checked_mul(gaps, v.row_stride, last)) &&
                          !__builtin_add_overflow(last, v.width, &elements) && checked_mul(elements, size, bytes)),
              STRIX_ERROR_INVALID_ARGUMENT);
    if (!r.held()) return r.status();
    out.given = true;
    out.rows = v.rows;
    out.width = v.width;
    out.at = {v.data, v.rows > 1 ? v.row_stride : v.width, v.dtype};
    out.span = Span(v.data, bytes);
    out.align = size;
    r.need(out.span.addressable(), STRIX_ERROR_INVALID_ARGUMENT)
        .need(bytes <= v.buffer_bytes, STRIX_ERROR_INSUFFICIENT_BUFFER)
        .need(!bytes || (v.data && out.span.aligned(size)), STRIX_ERROR_INVALID_ARGUMENT);
    return r.status();
}

// A buffer of `count` 4-byte elements, or absent where that is allowed.
strix_status read_buffer(const strix_amd_buffer& b, bool optional, uint64_t count, Span& out) {
    out = {};
    if (!b.data && !b.bytes && (optional || !count)) return STRIX_SUCCESS;
    uint64_t bytes = 0;
    Rules r;
    r.need(checked_mul(count, 4, bytes), STRIX_ERROR_INVALID_ARGUMENT)
        .need(b.bytes >= bytes, STRIX_ERROR_INSUFFICIENT_BUFFER);
    if (!r.held()) return r.status();
    out = Span(b.data, bytes);
    r.need(b.data && out.addressable() && out.aligned(4), STRIX_ERROR_INVALID_ARGUMENT);
    return r.status();
}

strix_status read_workspace(const strix_amd_buffer& b, uint64_t need, Span& out) {
    out = Span(b.data, b.bytes);
    Rules r;
    r.need(b.bytes >= need, STRIX_ERROR_INSUFFICIENT_BUFFER)
        .need(out.addressable() && (!b.bytes || (b.data && out.aligned(kWorkspaceAlign))),
              STRIX_ERROR_INVALID_ARGUMENT);
    return r.status();
}

bool apart(std::initializer_list<Span> written, std::initializer_list<Span> read) {
    for (auto w = written.begin(); w != written.end(); ++w) {
        for (auto v = w + 1; v != written.end(); ++v)
            if (w->meets(*v)) return false;
        for (const Span& v : read)
            if (w->meets(v)) return false;
    }
    return true;
}

strix_status resident(strix_context c, std::initializer_list<Span> spans, uint64_t align) {
    for (const Span& s : spans) {
        const strix_status status = device_resident(c, s, align);
        if (status != STRIX_SUCCESS) return status;
    }
    return STRIX_SUCCESS;
}

template <class T>
T* at(const Span& s) {
    return s.size ? static_cast<T*>(s.ptr()) : nullptr;
}

// ---- 8-bit integer linear ----

strix_status describe_int8(strix_context c, const strix_amd_int8_linear_desc* d, bool place, stx::Int8Call& call,
                           uint64_t& need) {
    need = 0;
    Rules r;
    r.then([&] { return versioned(d); });
    if (!r.held()) return r.status();
    const strix_amd_int8_weights w = d->weights;
    r.need(w && w->owner == c && std::isfinite(d->alpha) && std::isfinite(d->beta), STRIX_ERROR_INVALID_ARGUMENT);
    Rows x, y;
    Span scales, workspace;
    r.then([&] { return read_view(d->input, false, x); }).then([&] { return read_view(d->output, false, y); });
    if (!r.held()) return r.status();
    const bool integers = x.at.type == stx::kI8;
    r.need(x.width == w->layer.input && y.width == w->layer.output && x.rows == y.rows && is_float(y.at.type),
           STRIX_ERROR_UNSUPPORTED_FORMAT)
        .need(integers || (!d->input_scales.data && !d->input_scales.bytes), STRIX_ERROR_INVALID_ARGUMENT)
        .then([&] { return read_buffer(d->input_scales, !integers, integers ? x.rows : 0, scales); });
    if (!r.held()) return r.status();
    need = x.rows ? stx::int8_workspace_bytes(x.rows, w->layer.input, w->layer.output) : 0;
    if (!place) return STRIX_SUCCESS;
    r.then([&] { return read_workspace(d->workspace, need, workspace); })
        .need(apart({y.span, workspace}, {x.span, scales, Span(w->base, w->bytes)}) &&
                  !x.span.meets(Span(w->base, w->bytes)),
              STRIX_ERROR_INVALID_ARGUMENT);
    if (!r.held()) return r.status();
    call.x = x.at;
    call.y = y.at;
    call.x_scales = at<const float>(scales);
    call.rows = x.rows;
    call.alpha = d->alpha;
    call.beta = d->beta;
    call.workspace = d->workspace.data;
    if (!x.rows) return STRIX_SUCCESS;
    r.then([&] { return device_resident(c, x.span, x.align); })
        .then([&] { return device_resident(c, y.span, y.align); })
        .then([&] { return device_resident(c, scales, 4); })
        .then([&] { return device_resident(c, workspace, kWorkspaceAlign); });
    return r.status();
}

// ---- block norm ----

strix_status describe_norm(strix_context c, const strix_amd_block_norm_desc* d, stx::NormCall& call, uint32_t& type) {
    Rules r;
    r.then([&] { return versioned(d); });
    if (!r.held()) return r.status();
    Rows block, residual, gate, hidden, normed;
    r.then([&] { return read_view(d->block, true, block); })
        .then([&] { return read_view(d->residual, true, residual); })
        .then([&] { return read_view(d->gate, true, gate); })
        .then([&] { return read_view(d->hidden, true, hidden); })
        .then([&] { return read_view(d->normed, true, normed); })
        .need(std::isfinite(d->eps) && d->eps > 0 && std::isfinite(d->weight_offset) &&
                  std::isfinite(d->residual_scale) && std::isfinite(d->block_scale),
              STRIX_ERROR_INVALID_ARGUMENT)
        .need(d->norm <= STRIX_AMD_NORM_LAYER && d->gate_activation <= STRIX_AMD_GATE_SIGMOID,
              STRIX_ERROR_UNSUPPORTED_FORMAT)
        .need((block.given || residual.given) && (hidden.given || normed.given), STRIX_ERROR_INVALID_ARGUMENT);
    if (!r.held()) return r.status();
    const Rows& first = block.given ? block : residual;
    const uint64_t rows = first.rows, width = first.width;
    type = first.at.type;
    for (const Rows* v : {&block, &residual, &hidden, &normed})
        r.need(!v->given || (v->rows == rows && v->width == width && v->at.type == type),
               STRIX_ERROR_UNSUPPORTED_FORMAT);
    r.need(is_float(type) && width <= STRIX_AMD_NORM_MAX_WIDTH, STRIX_ERROR_UNSUPPORTED_FORMAT)
        .need(!gate.given || (gate.at.type == type && (gate.rows == rows || gate.rows == 1) &&
                              (gate.width == width || gate.width == 1)),
              STRIX_ERROR_UNSUPPORTED_FORMAT);
    const bool post = d->post_weight.data, pre = d->pre_weight.data;
    // parts that would have nothing to work on
    r.need(block.given || (!gate.given && !post && !d->channel_scale.data), STRIX_ERROR_INVALID_ARGUMENT)
        .need(gate.given || d->gate_activation == STRIX_AMD_GATE_LINEAR, STRIX_ERROR_INVALID_ARGUMENT)
        .need((post || !d->post_bias.data) && (pre || !d->pre_bias.data) && pre == normed.given,
              STRIX_ERROR_INVALID_ARGUMENT);
    Span vec[5];
    const strix_amd_buffer* given[5] = {&d->post_weight, &d->post_bias, &d->pre_weight, &d->pre_bias,
                                        &d->channel_scale};
    for (int i = 0; i < 5; ++i) r.then([&] { return read_buffer(*given[i], true, width, vec[i]); });
    // An output may take exactly the place of block or residual.
    auto place_ok = [&](const Rows& out) {
        for (const Rows* in : {&block, &residual}) {
            const bool same = in->at.data == out.at.data && in->at.stride == out.at.stride;
            if (!same && out.span.meets(in->span)) return false;
        }
        for (const Span& v : vec)
            if (out.span.meets(v)) return false;
        return !out.span.meets(gate.span);
    };
    r.need(place_ok(hidden) && place_ok(normed) && !hidden.span.meets(normed.span), STRIX_ERROR_INVALID_ARGUMENT);
    if (!r.held()) return r.status();
    call.block = block.at;
    call.residual = residual.at;
    call.gate = gate.at;
    if (gate.given && gate.rows == 1) call.gate.stride = 0;
    call.gate_per_row = gate.given && gate.width == 1 && width > 1;
    call.hidden = hidden.at;
    call.normed = normed.at;
    call.post_weight = at<const float>(vec[0]);
    call.post_bias = at<const float>(vec[1]);
    call.pre_weight = at<const float>(vec[2]);
    call.pre_bias = at<const float>(vec[3]);
    call.channel_scale = at<const float>(vec[4]);
    call.rows = rows;
    call.width = uint32_t(width);
    call.layer = d->norm == STRIX_AMD_NORM_LAYER;
    call.sigmoid = d->gate_activation == STRIX_AMD_GATE_SIGMOID;
    call.eps = d->eps;
    call.weight_offset = d->weight_offset;
    call.residual_scale = d->residual_scale;
    call.block_scale = d->block_scale;
    if (!rows) return STRIX_SUCCESS;
    r.then([&] {
         return resident(c, {block.span, residual.span, gate.span, hidden.span, normed.span}, first.align);
     }).then([&] { return resident(c, {vec[0], vec[1], vec[2], vec[3], vec[4]}, 4); });
    return r.status();
}

// ---- token log probabilities ----

strix_status describe_logprobs(strix_context c, const strix_amd_token_logprobs_desc* d, bool place,
                               stx::LogprobsCall& call, uint64_t& need) {
    need = 0;
    Rules r;
    r.then([&] { return versioned(d); });
    if (!r.held()) return r.status();
    Rows x;
    r.then([&] { return read_view(d->logits, false, x); })
        .need(d->scale >= 0x1p-16f && d->scale <= 0x1p16f, STRIX_ERROR_INVALID_ARGUMENT);
    if (!r.held()) return r.status();
    const uint64_t rows = x.rows;
    r.need(is_float(x.at.type) && d->top <= STRIX_AMD_MAX_TOP && d->top <= x.width, STRIX_ERROR_UNSUPPORTED_FORMAT);
    if (!r.held()) return r.status();
    need = rows ? stx::logprobs_workspace_bytes(rows, uint32_t(x.width), d->top) : 0;
    if (!place) return STRIX_SUCCESS;
    Span tokens, logprobs, ranks, entropy, top_ids, top_logprobs, workspace;
    const bool by_token = d->logprobs.data || d->ranks.data, tops = d->top_ids.data || d->top_logprobs.data;
    r.need(!rows || by_token || tops || d->entropy.data, STRIX_ERROR_INVALID_ARGUMENT)
        .need(!by_token || d->tokens.data, STRIX_ERROR_INVALID_ARGUMENT)
        .need(!tops || d->top, STRIX_ERROR_INVALID_ARGUMENT)
        .then([&] { return read_buffer(d->tokens, true, rows, tokens); })
        .then([&] { return read_buffer(d->logprobs, true, rows, logprobs); })
        .then([&] { return read_buffer(d->ranks, true, rows, ranks); })
        .then([&] { return read_buffer(d->entropy, true, rows, entropy); })
        .then([&] { return read_buffer(d->top_ids, true, rows * d->top, top_ids); })
        .then([&] { return read_buffer(d->top_logprobs, true, rows * d->top, top_logprobs); })
        .then([&] { return read_workspace(d->workspace, need, workspace); })
        .need(apart({logprobs, ranks, entropy, top_ids, top_logprobs, workspace}, {x.span, tokens}),
              STRIX_ERROR_INVALID_ARGUMENT);
    if (!r.held()) return r.status();
    call.logits = x.at;
    call.tokens = at<const int32_t>(tokens);
    call.logprobs = at<float>(logprobs);
    call.ranks = at<int32_t>(ranks);
    call.entropy = at<float>(entropy);
    call.top_ids = at<int32_t>(top_ids);
    call.top_logprobs = at<float>(top_logprobs);
    call.rows = rows;
    call.vocab = uint32_t(x.width);
    call.top = tops ? d->top : 0;
    call.scale = d->scale;
    call.workspace = d->workspace.data;
    if (!rows) return STRIX_SUCCESS;
    r.then([&] { return device_resident(c, x.span, x.align); })
        .then([&] { return resident(c, {tokens, logprobs, ranks, entropy, top_ids, top_logprobs}, 4); })
        .then([&] { return device_resident(c, workspace, kWorkspaceAlign); });
    return r.status();
}

// ---- calls and plans ----

hipError_t launch(const strix_amd_op_plan_impl& p) {
    switch (p.op) {
        case Op::kInt8:
            return p.int8.rows ? stx::launch_int8_linear(p.weights->layer, p.int8, p.stream) : hipSuccess;
        case Op::kNorm: return p.norm.rows ? stx::launch_block_norm(p.norm, p.norm_type, p.stream) : hipSuccess;
        case Op::kLogprobs:
            return p.logprobs.rows ? stx::launch_token_logprobs(p.logprobs, p.stream) : hipSuccess;
    }
    return hipErrorInvalidValue;
}

strix_status describe(strix_context c, const strix_amd_int8_linear_desc* d, strix_amd_op_plan_impl& p) {
    uint64_t need = 0;
    const strix_status s = describe_int8(c, d, true, p.int8, need);
    if (s != STRIX_SUCCESS) return s;
    p.op = Op::kInt8;
    p.weights = d->weights;
    return STRIX_SUCCESS;
}
strix_status describe(strix_context c, const strix_amd_block_norm_desc* d, strix_amd_op_plan_impl& p) {
    p.op = Op::kNorm;
    return describe_norm(c, d, p.norm, p.norm_type);
}
strix_status describe(strix_context c, const strix_amd_token_logprobs_desc* d, strix_amd_op_plan_impl& p) {
    uint64_t need = 0;
    p.op = Op::kLogprobs;
    return describe_logprobs(c, d, true, p.logprobs, need);
}

template <class Desc>
strix_status direct(strix_context c, const Desc* d, const strix_stream* stream) {
    strix_amd_op_plan_impl p;
    Rules r;
    r.then([&] { return on_context_device(c); })
        .then([&] { return borrowed_stream(c, stream, p.stream); })
        .then([&] { return describe(c, d, p); })
        .then([&] { return status_of(launch(p)); });
    return r.status();
}

template <class Desc>
strix_status create(strix_context c, const Desc* d, const strix_stream* stream, strix_amd_op_plan* out) {
    if (!out) return STRIX_ERROR_INVALID_ARGUMENT;
    *out = nullptr;
    strix_amd_op_plan_impl p;
    Rules r;
    r.then([&] { return on_context_device(c); })
        .then([&] { return borrowed_stream(c, stream, p.stream); })
        .then([&] { return describe(c, d, p); });
    if (!r.held()) return r.status();
    p.owner = c;
    auto* plan = new (std::nothrow) strix_amd_op_plan_impl(p);
    if (!plan) return STRIX_ERROR_OUT_OF_MEMORY;
    if (plan->weights) ++plan->weights->plans;
    ++c->weights_live;
    *out = plan;
    return STRIX_SUCCESS;
}

template <class F>
strix_status query(strix_context c, uint64_t* out, F&& describe) {
    if (!out) return STRIX_ERROR_INVALID_ARGUMENT;
    *out = 0;
    uint64_t need = 0;
    Rules r;
    r.then([&] { return on_context_device(c); }).then([&] { return describe(need); });
    if (r.held()) *out = need;
    return r.status();
}

}  // namespace

extern "C" {

strix_status strix_amd_int8_weights_prepare(strix_context c, const strix_amd_int8_weights_desc* d,
                                            const strix_stream* stream, strix_amd_int8_weights* out) {
    if (!out) return STRIX_ERROR_INVALID_ARGUMENT;
    *out = nullptr;
    hipStream_t hs{};
    Rows w;
    Span scales, bias;
    Rules r;
    r.then([&] { return on_context_device(c); })
        .then([&] { return borrowed_stream(c, stream, hs); })
        .then([&] { return versioned(d); });
    if (!r.held()) return r.status();
    r.then([&] { return read_view(d->weights, false, w); });
    if (!r.held()) return r.status();
    const bool integers = w.at.type == stx::kI8;
    r.need(w.rows >= 1 && w.rows <= STRIX_AMD_INT8_MAX_OUTPUT && w.width <= STRIX_AMD_INT8_MAX_INPUT,
           STRIX_ERROR_UNSUPPORTED_FORMAT)
        .need(integers || (!d->scales.data && !d->scales.bytes), STRIX_ERROR_INVALID_ARGUMENT)
        .then([&] { return read_buffer(d->scales, !integers, integers ? w.rows : 0, scales); })
        .then([&] { return read_buffer(d->bias, true, w.rows, bias); })
        .then([&] { return device_resident(c, w.span, w.align); })
        .then([&] { return resident(c, {scales, bias}, 4); });
    if (!r.held()) return r.status();
    auto* impl = new (std::nothrow) strix_amd_int8_weights_impl;
    if (!impl) return STRIX_ERROR_OUT_OF_MEMORY;
    const uint32_t input = uint32_t(w.width), output = uint32_t(w.rows);
    hipError_t e = stx::int8_allow_lds();
    if (e != hipSuccess) {
        delete impl;
        return status_of(e);
    }
    const uint64_t padded = stx::int8_row_blocks(w.rows) * 16, blocks = stx::int8_block_bytes(w.rows, input);
    impl->bytes = blocks + (bias.size ? 2 : 1) * padded * 4;
    e = hipMalloc(&impl->base, impl->bytes);
    if (e != hipSuccess) {
        delete impl;
        return status_of(e);
    }
    auto* base = static_cast<unsigned char*>(impl->base);
    auto* t = reinterpret_cast<float*>(base + blocks);
    auto* b = bias.size ? t + padded : nullptr;
    e = stx::launch_int8_stage(w.at, w.rows, input, at<const float>(scales), reinterpret_cast<int8_t*>(base), t, hs);
    if (e == hipSuccess && b) e = stx::launch_copy_f32(at<const float>(bias), b, w.rows, hs);
    const hipError_t drained = hipStreamSynchronize(hs);
    if (e == hipSuccess) e = drained;
    if (e != hipSuccess) {
        (void)hipFree(impl->base);
        delete impl;
        return status_of(e);
    }
    impl->owner = c;
    impl->layer = {reinterpret_cast<const int8_t*>(base), t, b, input, output};
    ++c->weights_live;
    *out = impl;
    return STRIX_SUCCESS;
}

strix_status strix_amd_int8_weights_destroy(strix_amd_int8_weights w) {
    if (!w || w->plans) return STRIX_ERROR_INVALID_ARGUMENT;
    const strix_status device = on_context_device(w->owner);
    if (device != STRIX_SUCCESS) return device;
    const hipError_t e = hipFree(w->base);
    if (e != hipSuccess) return status_of(e);
    --w->owner->weights_live;
    delete w;
    return STRIX_SUCCESS;
}

strix_status strix_amd_int8_linear_workspace_bytes(strix_context c, const strix_amd_int8_linear_desc* d,
                                                   uint64_t* out) {
    stx::Int8Call call;
    return query(c, out, [&](uint64_t& need) { return describe_int8(c, d, false, call, need); });
}

strix_status strix_amd_int8_linear(strix_context c, const strix_amd_int8_linear_desc* d, const strix_stream* stream) {
    return direct(c, d, stream);
}

strix_status strix_amd_int8_linear_plan_create(strix_context c, const strix_amd_int8_linear_desc* d,
                                               const strix_stream* stream, strix_amd_op_plan* out) {
    return create(c, d, stream, out);
}

strix_status strix_amd_block_norm(strix_context c, const strix_amd_block_norm_desc* d, const strix_stream* stream) {
    return direct(c, d, stream);
}

strix_status strix_amd_block_norm_plan_create(strix_context c, const strix_amd_block_norm_desc* d,
                                              const strix_stream* stream, strix_amd_op_plan* out) {
    return create(c, d, stream, out);
}

strix_status strix_amd_token_logprobs_workspace_bytes(strix_context c, const strix_amd_token_logprobs_desc* d,
                                                      uint64_t* out) {
    stx::LogprobsCall call;
    return query(c, out, [&](uint64_t& need) { return describe_logprobs(c, d, false, call, need); });
}

strix_status strix_amd_token_logprobs(strix_context c, const strix_amd_token_logprobs_desc* d,
                                      const strix_stream* stream) {
    return direct(c, d, stream);
}

strix_status strix_amd_token_logprobs_plan_create(strix_context c, const strix_amd_token_logprobs_desc* d,
                                                  const strix_stream* stream, strix_amd_op_plan* out) {
    return create(c, d, stream, out);
}

strix_status strix_amd_op_plan_submit(strix_amd_op_plan p) {
    if (!p) return STRIX_ERROR_INVALID_ARGUMENT;
    const strix_status device = on_context_device(p->owner);
    return device != STRIX_SUCCESS ? device : status_of(launch(*p));
}

strix_status strix_amd_op_plan_destroy(strix_amd_op_plan p) {
    if (!p) return STRIX_ERROR_INVALID_ARGUMENT;
    if (p->weights) --p->weights->plans;
    --p->owner->weights_live;
    delete p;
    return STRIX_SUCCESS;
}

}  // extern "C"
