// Parts that the C layers of the operators around the trellis layers share:
// views and buffers of a descriptor, and prepared operators.
//
// Each operator is described by one function, which checks the descriptor and
// the device residence of every buffer and leaves the kernels' arguments; a
// direct call launches with them, a plan keeps them.  The order of the checks
// is the linear calls': device, stream, descriptor, shapes and types,
// overlaps, residence.
#pragma once
#include <climits>
#include <cmath>
#include <new>

#include "api_internal.hpp"
#include "fp8.hpp"
#include "ops.hpp"
#include "strix_trellis_ops.h"

// A plan counts among its context's live handles (strix_context_impl::weights_live)
// and, where it has weights, among their plans.
struct strix_amd_op_plan_impl {
    strix_context owner = nullptr;
    hipStream_t stream{};
    uint64_t* retained = nullptr;   // its weights' count of plans
    virtual hipError_t launch() const = 0;
    virtual ~strix_amd_op_plan_impl() = default;
};

namespace stx_ops {

using namespace stx_api;

inline uint64_t size_of(uint32_t type) {
    return type == stx::kF32 ? 4 : type == stx::kF16 || type == stx::kBF16 ? 2 : type == stx::kI8 || type == stx::kE4M3 ? 1 : 0;
}
inline bool is_float(uint32_t type) { return type == stx::kF32 || type == stx::kF16 || type == stx::kBF16; }

// A view of the descriptor and the bytes it covers; e4m3: of an operator that takes that type.
struct Rows {
    bool given = false;
    uint64_t rows = 0, width = 0;
    stx::OpRows at{};
    Span span;
    uint64_t align = 1;
};

inline bool absent(const strix_amd_view& v) {
    static const strix_amd_view none{};
    return std::memcmp(&v, &none, sizeof(v)) == 0;
}

inline strix_status read_view(const strix_amd_view& v, bool optional, Rows& out, bool e4m3 = false) {
    out = {};
    if (optional && absent(v)) return STRIX_SUCCESS;
    const uint64_t size = size_of(v.dtype);
    uint64_t last = 0, elements = 0, bytes = 0;
    Rules r;
    r.then([&] { return versioned(&v); })
        .need(!v.flags, STRIX_ERROR_INVALID_ARGUMENT)
        .need(size && (e4m3 || v.dtype != stx::kE4M3) && v.rows <= INT_MAX && v.width >= 1 && v.width <= INT_MAX, STRIX_ERROR_UNSUPPORTED_FORMAT);
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
inline strix_status read_buffer(const strix_amd_buffer& b, bool optional, uint64_t count, Span& out) {
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

inline strix_status read_workspace(const strix_amd_buffer& b, uint64_t need, Span& out) {
    out = Span(b.data, b.bytes);
    Rules r;
    r.need(b.bytes >= need, STRIX_ERROR_INSUFFICIENT_BUFFER)
        .need(out.addressable() && (!b.bytes || (b.data && out.aligned(kWorkspaceAlign))),
              STRIX_ERROR_INVALID_ARGUMENT);
    return r.status();
}

inline bool apart(std::initializer_list<Span> written, std::initializer_list<Span> read) {
    for (auto w = written.begin(); w != written.end(); ++w) {
        for (auto v = w + 1; v != written.end(); ++v)
            if (w->meets(*v)) return false;
        for (const Span& v : read)
            if (w->meets(v)) return false;
    }
    return true;
}

inline strix_status resident(strix_context c, std::initializer_list<Span> spans, uint64_t align) {
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

// Plan: an operator's kind of plan, with describe(context, descriptor) that leaves
// its arguments and launch().
template <class Plan, class Desc>
strix_status direct(strix_context c, const Desc* d, const strix_stream* stream) {
    Plan p;
    Rules r;
    r.then([&] { return on_context_device(c); })
        .then([&] { return borrowed_stream(c, stream, p.stream); })
        .then([&] { return p.describe(c, d); })
        .then([&] { return status_of(p.launch()); });
    return r.status();
}

template <class Plan, class Desc>
strix_status create(strix_context c, const Desc* d, const strix_stream* stream, strix_amd_op_plan* out) {
    if (!out) return STRIX_ERROR_INVALID_ARGUMENT;
    *out = nullptr;
    Plan p;
    Rules r;
    r.then([&] { return on_context_device(c); })
        .then([&] { return borrowed_stream(c, stream, p.stream); })
        .then([&] { return p.describe(c, d); });
    if (!r.held()) return r.status();
    p.owner = c;
    auto* plan = new (std::nothrow) Plan(p);
    if (!plan) return STRIX_ERROR_OUT_OF_MEMORY;
    if (plan->retained) ++*plan->retained;
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

}  // namespace stx_ops
