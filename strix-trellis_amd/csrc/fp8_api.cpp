// Layers in 8-bit floating point (include/strix_trellis_fp8.h): argument checks,
// weights, plans.
#include "ops_internal.hpp"
#include "strix_trellis_fp8.h"

using namespace stx_ops;

struct strix_amd_fp8_weights_impl {
    strix_context owner = nullptr;
    stx::Fp8Layer layer{};
    void* base = nullptr;     // one private allocation: blocks | scales | bias
    uint64_t bytes = 0;
    uint64_t plans = 0;       // live plans retaining these weights
};

namespace {

bool is_input(uint32_t type) { return is_float(type) || type == stx::kE4M3; }
uint64_t blocks_of(uint64_t n) { return (n + 127) / 128; }

// One matrix of a weights descriptor, with its scales and bias.
struct Matrix {
    Rows w;
    Span scales, bias;
    bool scaled() const { return w.at.type == stx::kE4M3; }
};

strix_status read_matrix(const strix_amd_view& view, const strix_amd_buffer& scales, const strix_amd_buffer& bias,
                         Matrix& out) {
    Rules r;
    r.then([&] { return read_view(view, false, out.w, true); });
    if (!r.held()) return r.status();
    const Rows& w = out.w;
    r.need(is_input(w.at.type) && w.rows >= 1 && w.rows <= STRIX_AMD_FP8_MAX_OUTPUT &&
               w.width <= STRIX_AMD_FP8_MAX_INPUT,
           STRIX_ERROR_UNSUPPORTED_FORMAT)
        .need(out.scaled() || (!scales.data && !scales.bytes), STRIX_ERROR_INVALID_ARGUMENT)
        .then([&] {
            return read_buffer(scales, !out.scaled(), out.scaled() ? blocks_of(w.rows) * blocks_of(w.width) : 0,
                               out.scales);
        })
        .then([&] { return read_buffer(bias, true, w.rows, out.bias); });
    return r.status();
}

// What the linear and the gated call share: rows in, rows out, their scales and
// the workspace.
template <class Desc>
strix_status describe_rows(strix_context c, const Desc* d, bool pair, const strix_amd_buffer& output_scales,
                           bool place, stx::Fp8Call& call, uint64_t& need) {
    const strix_amd_fp8_weights w = d->weights;
    Rules r;
    Rows x, y;
    Span scales, out_scales, workspace;
    r.then([&] { return read_view(d->input, false, x, true); })
        .then([&] { return read_view(d->output, false, y, pair); });
    if (!r.held()) return r.status();
    const uint64_t I = w->layer.input, N = w->layer.output;
    const bool scaled = x.at.type == stx::kE4M3, rounded = y.at.type == stx::kE4M3;
    r.need(is_input(x.at.type) && x.width == I && y.width == N && x.rows == y.rows &&
               (is_float(y.at.type) || rounded),
           STRIX_ERROR_UNSUPPORTED_FORMAT)
        .need(scaled || (!d->input_scales.data && !d->input_scales.bytes), STRIX_ERROR_INVALID_ARGUMENT)
        .need(rounded || (!output_scales.data && !output_scales.bytes), STRIX_ERROR_INVALID_ARGUMENT)
        .then([&] { return read_buffer(d->input_scales, !scaled, scaled ? x.rows * blocks_of(I) : 0, scales); })
        .then([&] { return read_buffer(output_scales, !rounded, rounded ? x.rows * blocks_of(N) : 0, out_scales); });
    if (!r.held()) return r.status();
    need = x.rows ? stx::fp8_workspace_bytes(x.rows, uint32_t(I), uint32_t(N), pair, y.at.type == stx::kF32 || rounded, rounded) : 0;
    if (!place) return STRIX_SUCCESS;
    const Span held(w->base, w->bytes);
    r.then([&] { return read_workspace(d->workspace, need, workspace); })
        .need(apart({y.span, out_scales, workspace}, {x.span, scales, held}) && !x.span.meets(held) &&
                  !scales.meets(held),
              STRIX_ERROR_INVALID_ARGUMENT);
    if (!r.held()) return r.status();
    call.x = x.at;
    call.y = y.at;
    call.x_scales = at<const float>(scales);
    call.y_scales = at<float>(out_scales);
    call.rows = x.rows;
    call.workspace = d->workspace.data;
    if (!x.rows) return STRIX_SUCCESS;
    r.then([&] { return device_resident(c, x.span, x.align); })
        .then([&] { return device_resident(c, y.span, y.align); })
        .then([&] { return resident(c, {scales, out_scales}, 4); })
        .then([&] { return device_resident(c, workspace, kWorkspaceAlign); });
    return r.status();
}

strix_status describe_call(strix_context c, const strix_amd_fp8_linear_desc* d, bool place, stx::Fp8Call& call,
                           uint64_t& need) {
    need = 0;
    Rules r;
    r.then([&] { return versioned(d); });
    if (!r.held()) return r.status();
    r.need(d->weights && d->weights->owner == c && !d->weights->layer.pair && std::isfinite(d->alpha) &&
               std::isfinite(d->beta),
           STRIX_ERROR_INVALID_ARGUMENT);
    if (!r.held()) return r.status();
    call.alpha = d->alpha;
    call.beta = d->beta;
    return describe_rows(c, d, false, strix_amd_buffer{}, place, call, need);
}

strix_status describe_call(strix_context c, const strix_amd_fp8_gated_desc* d, bool place, stx::Fp8Call& call,
                           uint64_t& need) {
    need = 0;
    Rules r;
    r.then([&] { return versioned(d); });
    if (!r.held()) return r.status();
    r.need(d->weights && d->weights->owner == c && d->weights->layer.pair && !d->flags, STRIX_ERROR_INVALID_ARGUMENT)
        .need(d->activation <= STRIX_AMD_GATED_GELU, STRIX_ERROR_UNSUPPORTED_FORMAT);
    if (!r.held()) return r.status();
    call.activation = d->activation;
    return describe_rows(c, d, true, d->output_scales, place, call, need);
}

struct Fp8CallPlan final : strix_amd_op_plan_impl {
    strix_amd_fp8_weights weights = nullptr;
    stx::Fp8Call call{};
    template <class Desc>
    strix_status describe(strix_context c, const Desc* d) {
        uint64_t need = 0;
        const strix_status s = describe_call(c, d, true, call, need);
        if (s != STRIX_SUCCESS) return s;
        weights = d->weights;
        retained = &weights->plans;
        return STRIX_SUCCESS;
    }
    hipError_t launch() const override {
        return call.rows ? stx::launch_fp8(weights->layer, call, stream) : hipSuccess;
    }
};

}  // namespace

extern "C" {

strix_status strix_amd_fp8_weights_prepare(strix_context c, const strix_amd_fp8_weights_desc* d,
                                           const strix_stream* stream, strix_amd_fp8_weights* out) {
    if (!out) return STRIX_ERROR_INVALID_ARGUMENT;
    *out = nullptr;
    hipStream_t hs{};
    Rules r;
    r.then([&] { return on_context_device(c); })
        .then([&] { return borrowed_stream(c, stream, hs); })
        .then([&] { return versioned(d); });
    if (!r.held()) return r.status();
    const bool pair = !absent(d->up);
    Matrix m[2];
    r.then([&] { return read_matrix(d->weights, d->scales, d->bias, m[0]); });
    if (pair) {
        r.then([&] { return read_matrix(d->up, d->up_scales, d->up_bias, m[1]); })
            .need(m[0].w.rows == m[1].w.rows && m[0].w.width == m[1].w.width && m[0].w.at.type == m[1].w.at.type,
                  STRIX_ERROR_UNSUPPORTED_FORMAT)
            .need(!m[0].bias.size == !m[1].bias.size, STRIX_ERROR_INVALID_ARGUMENT);
    } else {
        r.need(!d->up_scales.data && !d->up_scales.bytes && !d->up_bias.data && !d->up_bias.bytes,
               STRIX_ERROR_INVALID_ARGUMENT);
    }
    for (const Matrix& x : m)
        r.then([&] { return device_resident(c, x.w.span, x.w.align); })
            .then([&] { return resident(c, {x.scales, x.bias}, 4); });
    if (!r.held()) return r.status();
    auto* impl = new (std::nothrow) strix_amd_fp8_weights_impl;
    if (!impl) return STRIX_ERROR_OUT_OF_MEMORY;
    hipError_t e = stx::fp8_allow_lds();
    if (e != hipSuccess) {
        delete impl;
        return status_of(e);
    }
    const uint32_t input = uint32_t(m[0].w.width), output = uint32_t(m[0].w.rows), parts = pair ? 2 : 1;
    const uint64_t blocks = stx::fp8_block_bytes(output, input) * parts;
    const uint64_t scales = blocks_of(output) * blocks_of(input), padded = stx::fp8_row_blocks(output) * 16;
    impl->bytes = blocks + ((scales * parts + 3) / 4 * 4 + (m[0].bias.size ? padded * parts : 0)) * 4;
    e = hipMalloc(&impl->base, impl->bytes);
    if (e != hipSuccess) {
        delete impl;
        return status_of(e);
    }
    auto* base = static_cast<uint8_t*>(impl->base);
    auto* t = reinterpret_cast<float*>(base + blocks);
    float* b = m[0].bias.size ? t + (scales * parts + 3) / 4 * 4 : nullptr;
    for (uint32_t i = 0; i < parts && e == hipSuccess; ++i) {
        e = stx::launch_fp8_weights(m[i].w.at, output, input, at<const float>(m[i].scales),
                                    base + i * 2 * uint64_t(stx::fp8_k_blocks(input)) * 2048, parts, t + i * scales, hs);
        if (e == hipSuccess && b) e = stx::launch_copy_f32(at<const float>(m[i].bias), b + i * padded, output, hs);
    }
    const hipError_t drained = hipStreamSynchronize(hs);
    if (e == hipSuccess) e = drained;
    if (e != hipSuccess) {
        (void)hipFree(impl->base);
        delete impl;
        return status_of(e);
    }
    impl->owner = c;
    impl->layer = {base, t, b, input, output, pair};
    ++c->weights_live;
    *out = impl;
    return STRIX_SUCCESS;
}

strix_status strix_amd_fp8_weights_destroy(strix_amd_fp8_weights w) {
    if (!w || w->plans) return STRIX_ERROR_INVALID_ARGUMENT;
    const strix_status device = on_context_device(w->owner);
    if (device != STRIX_SUCCESS) return device;
    const hipError_t e = hipFree(w->base);
    if (e != hipSuccess) return status_of(e);
    --w->owner->weights_live;
    delete w;
    return STRIX_SUCCESS;
}

strix_status strix_amd_fp8_linear_workspace_bytes(strix_context c, const strix_amd_fp8_linear_desc* d, uint64_t* out) {
    stx::Fp8Call call;
    return query(c, out, [&](uint64_t& need) { return describe_call(c, d, false, call, need); });
}

strix_status strix_amd_fp8_linear(strix_context c, const strix_amd_fp8_linear_desc* d, const strix_stream* stream) {
    return direct<Fp8CallPlan>(c, d, stream);
}

strix_status strix_amd_fp8_linear_plan_create(strix_context c, const strix_amd_fp8_linear_desc* d,
                                              const strix_stream* stream, strix_amd_op_plan* out) {
    return create<Fp8CallPlan>(c, d, stream, out);
}

strix_status strix_amd_fp8_gated_workspace_bytes(strix_context c, const strix_amd_fp8_gated_desc* d, uint64_t* out) {
    stx::Fp8Call call;
    return query(c, out, [&](uint64_t& need) { return describe_call(c, d, false, call, need); });
}

strix_status strix_amd_fp8_gated(strix_context c, const strix_amd_fp8_gated_desc* d, const strix_stream* stream) {
    return direct<Fp8CallPlan>(c, d, stream);
}

strix_status strix_amd_fp8_gated_plan_create(strix_context c, const strix_amd_fp8_gated_desc* d,
                                             const strix_stream* stream, strix_amd_op_plan* out) {
    return create<Fp8CallPlan>(c, d, stream, out);
}

}  // extern "C"
