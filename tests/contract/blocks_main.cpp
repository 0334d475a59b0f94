// Contract of the e4m3 layers (include/strix_trellis_fp8.h) and of the beam operators
// (include/strix_trellis_beam.h) over a fake HIP runtime: argument checks, failure mapping,
// leaks, plans that only launch, and the sizing rules.
#include "beam.hpp"
#include "fake.hpp"
#include "fp8.hpp"
#include "strix_trellis_beam.h"
#include "strix_trellis_fp8.h"

#include <climits>
#include <cstdio>
#include <cstdlib>
#include <limits>

static int checks = 0;
#define CHECK(cond)                                                                       \
    do {                                                                                  \
        ++checks;                                                                         \
        if (!(cond)) {                                                                    \
            std::fprintf(stderr, "%s:%d: CHECK failed: %s\n", __FILE__, __LINE__, #cond); \
            std::exit(1);                                                                 \
        }                                                                                 \
    } while (0)

constexpr strix_status kOk = STRIX_SUCCESS, kArg = STRIX_ERROR_INVALID_ARGUMENT, kAbi = STRIX_ERROR_ABI_MISMATCH,
                       kFormat = STRIX_ERROR_UNSUPPORTED_FORMAT, kShort = STRIX_ERROR_INSUFFICIENT_BUFFER,
                       kMemory = STRIX_ERROR_OUT_OF_MEMORY, kBackend = STRIX_ERROR_BACKEND;
constexpr uint32_t BF16 = STRIX_DTYPE_BF16, F32 = STRIX_DTYPE_F32, I8 = STRIX_AMD_DTYPE_I8, E4M3 = STRIX_AMD_DTYPE_E4M3;
constexpr float kInf = std::numeric_limits<float>::infinity(), kNan = std::numeric_limits<float>::quiet_NaN();

template <class T>
static T header() {
    T d{};
    d.struct_size = sizeof(T);
    d.abi_version = STRIX_TRELLIS_ABI_VERSION;
    return d;
}
static void* device(size_t bytes) {
    void* p = nullptr;
    CHECK(hipMalloc(&p, bytes) == hipSuccess);
    return p;
}
static uint64_t size_of(uint32_t type) { return type == F32 ? 4 : type == I8 || type == E4M3 ? 1 : 2; }
static strix_amd_view view(void* p, uint32_t type, uint64_t rows, uint64_t width, uint64_t stride = 0) {
    auto v = header<strix_amd_view>();
    v.data = p;
    v.dtype = type;
    v.rows = rows;
    v.width = width;
    v.row_stride = stride ? stride : width;
    v.buffer_bytes = rows ? ((rows - 1) * v.row_stride + width) * size_of(type) : 0;
    return v;
}
static strix_amd_buffer buffer(void* p, uint64_t count) { return {p, count * 4}; }

struct Env {
    strix_context c = nullptr;
    hipStream_t hs{};
    strix_stream s{};
};

// A plan only launches; its handle keeps the context alive.
template <class Create>
static void plan_contract(Env& e, const char* name, Create create) {
    strix_amd_op_plan p = nullptr;
    CHECK(create(&p) == kOk && p);
    CHECK(strix_context_destroy(e.c) == kArg);
    const fake::Counters before = fake::n;
    fake::launches.clear();
    for (int i = 0; i < 3; ++i) CHECK(strix_amd_op_plan_submit(p) == kOk);
    CHECK(fake::launches.size() == 3 && fake::launches[0].name == name && fake::launches[0].stream == e.hs);
    CHECK(fake::n.mallocs == before.mallocs && fake::n.frees == before.frees && fake::n.copies == before.copies);
    CHECK(fake::n.syncs == before.syncs && fake::n.pointer_queries == before.pointer_queries);
    CHECK(fake::n.range_queries == before.range_queries && fake::n.stream_queries == before.stream_queries);
    fake::launch_fail_at = 0;
    CHECK(strix_amd_op_plan_submit(p) == kBackend);
    fake::current_device = 1;
    CHECK(strix_amd_op_plan_submit(p) == kArg);
    strix_amd_op_plan q = p;
    CHECK(create(&q) == kArg && !q);   // another device is current
    fake::current_device = 0;
    CHECK(create(nullptr) == kArg);
    CHECK(strix_amd_op_plan_destroy(p) == kOk);
}

static void weights_contract(Env& e) {
    const uint64_t N = 270, I = 300, scales = 3 * 3;
    void *q = device(N * I), *u = device(N * I), *t = device(scales * 4), *ut = device(scales * 4), *b = device(N * 4),
         *ub = device(N * 4), *wf = device(N * I * 4);
    auto d = header<strix_amd_fp8_weights_desc>();
    d.weights = view(q, E4M3, N, I);
    d.scales = buffer(t, scales);
    d.bias = buffer(b, N);
    auto pair = d;
    pair.up = view(u, E4M3, N, I);
    pair.up_scales = buffer(ut, scales);
    pair.up_bias = buffer(ub, N);
    const uint64_t live = fake::live.size();
    auto prepare = [&](strix_amd_fp8_weights_desc x) {
        strix_amd_fp8_weights w = reinterpret_cast<strix_amd_fp8_weights>(1);
        const strix_status s = strix_amd_fp8_weights_prepare(e.c, &x, &e.s, &w);
        CHECK((s == kOk) == (w != nullptr));
        if (w) CHECK(strix_amd_fp8_weights_destroy(w) == kOk);
        CHECK(fake::live.size() == live);
        return s;
    };
    CHECK(prepare(d) == kOk && prepare(pair) == kOk);
    for (const auto& good : {d, pair}) {
        auto x = good;
        x.struct_size -= 1;
        CHECK(prepare(x) == kAbi);
        x = good;
        x.reserved[3] = 1;
        CHECK(prepare(x) == kArg);
        x = good;
        x.weights.flags = 1;
        CHECK(prepare(x) == kArg);
        x = good;
        x.scales = {};
        CHECK(prepare(x) == kShort);
        x = good;
        x.scales.bytes -= 4;
        CHECK(prepare(x) == kShort);
        x = good;
        x.scales.data = static_cast<char*>(t) + 2;
        CHECK(prepare(x) == kArg);
        x = good;
        x.bias.bytes -= 1;
        CHECK(prepare(x) == kShort);
        x = good;
        x.weights = view(q, I8, N, I);
        CHECK(prepare(x) == kFormat);
        x = good;
        x.weights.rows = 0;
        CHECK(prepare(x) == kFormat);
        x = good;
        x.weights.width = 0;
        CHECK(prepare(x) == kFormat);
        x = good;
        x.weights.row_stride = I - 1;
        CHECK(prepare(x) == kFormat);
        x = good;
        x.weights.buffer_bytes -= 1;
        CHECK(prepare(x) == kShort);
        x = good;
        x.weights.data = &x;   // host memory
        CHECK(prepare(x) == kArg);
        // every step that can fail leaves nothing behind
        const int launches = good.up.data ? 5 : 3;   // LDS, and a matrix and a bias each
        for (int at = 0; at < launches; ++at) {
            fake::launch_fail_at = at;
            CHECK(prepare(good) == kBackend);
        }
        fake::sync_fail_at = 0;
        CHECK(prepare(good) == kBackend);
        fake::malloc_fail_at = 0;
        CHECK(prepare(good) == kMemory);
        fake::reset_failures();
    }
    auto x = d;
    x.weights.width = uint64_t(STRIX_AMD_FP8_MAX_INPUT) + 1;
    x.weights.rows = 1;
    x.weights.buffer_bytes = uint64_t(1) << 20;
    CHECK(prepare(x) == kFormat);
    x = d;
    x.up_bias = buffer(ub, N);
    CHECK(prepare(x) == kArg);
    x = d;
    x.up_scales = buffer(ut, scales);
    CHECK(prepare(x) == kArg);
    x = pair;
    x.up.rows -= 1;
    x.up.buffer_bytes -= I;
    CHECK(prepare(x) == kFormat);
    x = pair;
    x.up = view(wf, F32, N, I);
    x.up_scales = {};
    CHECK(prepare(x) == kFormat);   // matrices of two types
    x = pair;
    x.up_bias = {};
    CHECK(prepare(x) == kArg);
    x = pair;
    x.up_scales = {};
    CHECK(prepare(x) == kShort);
    x = d;
    x.weights = view(wf, F32, N, I);
    CHECK(prepare(x) == kArg);   // scales of float weights
    x.scales = {};
    CHECK(prepare(x) == kOk);
    CHECK(strix_amd_fp8_weights_prepare(e.c, &d, &e.s, nullptr) == kArg);
    CHECK(strix_amd_fp8_weights_prepare(e.c, nullptr, &e.s, reinterpret_cast<strix_amd_fp8_weights*>(&x)) == kArg);
    CHECK(strix_amd_fp8_weights_destroy(nullptr) == kArg);
    for (void* v : {q, u, t, ut, b, ub, wf}) CHECK(hipFree(v) == hipSuccess);
}

static void fp8_contract(Env& e) {
    const uint64_t N = 200, I = 300, rows = 40, kbs = 3, nbs = 2;
    void *q = device(N * I), *t = device(kbs * nbs * 4);
    auto wd = header<strix_amd_fp8_weights_desc>();
    wd.weights = view(q, E4M3, N, I);
    wd.scales = buffer(t, kbs * nbs);
    strix_amd_fp8_weights w = nullptr, pair = nullptr;
    CHECK(strix_amd_fp8_weights_prepare(e.c, &wd, &e.s, &w) == kOk);
    wd.up = view(q, E4M3, N, I);
    wd.up_scales = buffer(t, kbs * nbs);
    CHECK(strix_amd_fp8_weights_prepare(e.c, &wd, &e.s, &pair) == kOk);
    void *in = device(rows * I * 4), *out = device(rows * N * 4), *sc = device(rows * kbs * 4), *os = device(rows * nbs * 4);

    auto c = header<strix_amd_fp8_linear_desc>();
    c.weights = w;
    c.input = view(in, F32, rows, I);
    c.output = view(out, BF16, rows, N);
    c.alpha = 1;
    auto g = header<strix_amd_fp8_gated_desc>();
    g.weights = pair;
    g.input = view(in, E4M3, rows, I);
    g.input_scales = buffer(sc, rows * kbs);
    g.output = view(out, E4M3, rows, N);
    g.output_scales = buffer(os, rows * nbs);
    uint64_t need = 1, gated_need = 1;
    CHECK(strix_amd_fp8_linear_workspace_bytes(e.c, &c, &need) == kOk);
    CHECK(need == stx::fp8_workspace_bytes(rows, I, N, false, false, false));
    CHECK(strix_amd_fp8_gated_workspace_bytes(e.c, &g, &gated_need) == kOk);
    CHECK(gated_need == stx::fp8_workspace_bytes(rows, I, N, true, true, true));
    CHECK(strix_amd_fp8_linear_workspace_bytes(e.c, &c, nullptr) == kArg);
    void* ws = device(gated_need > need ? gated_need : need);
    c.workspace = {ws, need};
    g.workspace = {ws, gated_need};
    auto call = [&](const strix_amd_fp8_linear_desc& y) {
        fake::launches.clear();
        const strix_status s = strix_amd_fp8_linear(e.c, &y, &e.s);
        CHECK(fake::launches.empty() == (s != kOk || !y.input.rows));
        return s;
    };
    auto gate = [&](const strix_amd_fp8_gated_desc& y) {
        fake::launches.clear();
        const strix_status s = strix_amd_fp8_gated(e.c, &y, &e.s);
        CHECK(fake::launches.empty() == (s != kOk || !y.input.rows));
        return s;
    };
    CHECK(call(c) == kOk && gate(g) == kOk);
    auto y = c;
    y.weights = nullptr;
    CHECK(call(y) == kArg);
    y.weights = pair;
    CHECK(call(y) == kArg);
    auto h = g;
    h.weights = w;
    CHECK(gate(h) == kArg);
    for (float bad : {kInf, kNan}) {
        y = c;
        y.alpha = bad;
        CHECK(call(y) == kArg);
        y = c;
        y.beta = bad;
        CHECK(call(y) == kArg);
    }
    y = c;
    y.struct_size += 8;
    CHECK(call(y) == kAbi);
    y = c;
    y.reserved[0] = 1;
    CHECK(call(y) == kArg);
    y = c;
    y.input = view(in, I8, rows, I);
    CHECK(call(y) == kFormat);
    y = c;
    y.output = view(out, E4M3, rows, N);   // of the gated call alone
    CHECK(call(y) == kFormat);
    y = c;
    y.input.width -= 1;
    CHECK(call(y) == kFormat);
    y = c;
    y.output.rows -= 1;
    CHECK(call(y) == kFormat);
    y = c;
    y.input_scales = buffer(sc, rows * kbs);
    CHECK(call(y) == kArg);
    y.input = view(in, E4M3, rows, I);
    CHECK(call(y) == kOk);
    y.input_scales.bytes -= 4;
    CHECK(call(y) == kShort);
    y.input_scales = {};
    CHECK(call(y) == kShort);
    y = c;
    y.workspace.bytes -= 1;
    CHECK(call(y) == kShort);
    y = c;
    y.workspace.data = static_cast<char*>(ws) + 4;
    CHECK(call(y) == kArg);
    y = c;
    y.output.data = in;   // over the input
    CHECK(call(y) == kArg);
    y = c;
    y.workspace = {out, rows * N * 4};
    CHECK(call(y) == kArg);
    y = c;
    y.output.data = static_cast<char*>(out) + 1;
    CHECK(call(y) == kArg);
    y = c;
    y.input.data = &y;
    CHECK(call(y) == kArg);
    y = c;
    y.input.rows = y.output.rows = 0;
    y.workspace = {};
    CHECK(call(y) == kOk);
    h = g;
    h.output_scales = {};
    CHECK(gate(h) == kShort);
    h = g;
    h.output_scales = buffer(sc, rows * nbs);   // over the input's
    CHECK(gate(h) == kArg);
    h = g;
    h.output = view(out, F32, rows, N);
    CHECK(gate(h) == kArg);   // scales of a float output
    h.output_scales = {};
    CHECK(gate(h) == kOk);
    h = g;
    h.activation = 2;
    CHECK(gate(h) == kFormat);
    h = g;
    h.flags = 1;
    CHECK(gate(h) == kArg);
    fake::launch_fail_at = 0;
    CHECK(strix_amd_fp8_linear(e.c, &c, &e.s) == kBackend);
    fake::reset_failures();
    CHECK(strix_amd_fp8_linear(e.c, &c, nullptr) == kArg && strix_amd_fp8_linear(nullptr, &c, &e.s) == kArg);
    plan_contract(e, "fp8_linear", [&](strix_amd_op_plan* p) { return strix_amd_fp8_linear_plan_create(e.c, &c, &e.s, p); });
    plan_contract(e, "fp8_gated", [&](strix_amd_op_plan* p) { return strix_amd_fp8_gated_plan_create(e.c, &g, &e.s, p); });
    strix_amd_op_plan p = nullptr;
    CHECK(strix_amd_fp8_linear_plan_create(e.c, &c, &e.s, &p) == kOk);
    CHECK(strix_amd_fp8_weights_destroy(w) == kArg);   // a plan holds it
    CHECK(strix_amd_op_plan_destroy(p) == kOk);
    fake::free_fail_at = 0;
    CHECK(strix_amd_fp8_weights_destroy(w) == kBackend);   // the handle stays
    CHECK(strix_amd_fp8_weights_destroy(w) == kOk && strix_amd_fp8_weights_destroy(pair) == kOk);
    for (void* v : {q, t, in, out, sc, os, ws}) CHECK(hipFree(v) == hipSuccess);
}

static void select_contract(Env& e) {
    const uint64_t beams = 4, prompts = 3, rows = beams * prompts, vocab = 20000, keep = 8;
    void *x = device(rows * vocab * 4), *s = device(rows * 4), *f = device(rows * 4), *ns = device(prompts * keep * 4),
         *pa = device(prompts * keep * 4), *to = device(prompts * keep * 4);
    auto d = header<strix_amd_beam_select_desc>();
    d.logits = view(x, F32, rows, vocab);
    d.scores = buffer(s, rows);
    d.finished = buffer(f, rows);
    d.next_scores = buffer(ns, prompts * keep);
    d.parents = buffer(pa, prompts * keep);
    d.tokens = buffer(to, prompts * keep);
    d.beams = beams;
    d.keep = keep;
    d.scale = 1;
    uint64_t need = 0;
    CHECK(strix_amd_beam_select_workspace_bytes(e.c, &d, &need) == kOk);
    CHECK(need == stx::beam_select_workspace_bytes(rows, vocab, F32, keep) && need);
    void* ws = device(need);
    d.workspace = {ws, need};
    auto call = [&](const strix_amd_beam_select_desc& y) {
        fake::launches.clear();
        const strix_status r = strix_amd_beam_select(e.c, &y, &e.s);
        CHECK(fake::launches.empty() == (r != kOk || !y.logits.rows));
        return r;
    };
    CHECK(call(d) == kOk);
    auto y = d;
    y.finished = {};
    CHECK(call(y) == kOk);
    for (uint32_t bad : {0u, 5u, 65u}) {
        y = d;
        y.beams = bad;
        CHECK(call(y) == kFormat);
    }
    for (uint32_t bad : {0u, 65u}) {
        y = d;
        y.keep = bad;
        CHECK(call(y) == kFormat);
    }
    for (float bad : {0.0f, -1.0f, kInf, kNan, 0x1p17f}) {
        y = d;
        y.scale = bad;
        CHECK(call(y) == kArg);
    }
    y = d;
    y.logits = view(x, I8, rows, vocab);
    CHECK(call(y) == kFormat);
    y = d;
    y.logits = view(x, E4M3, rows, vocab);
    CHECK(call(y) == kFormat);
    for (auto m : {&strix_amd_beam_select_desc::scores, &strix_amd_beam_select_desc::next_scores,
                   &strix_amd_beam_select_desc::parents, &strix_amd_beam_select_desc::tokens}) {
        y = d;
        y.*m = {};
        CHECK(call(y) == kShort);
        y = d;
        (y.*m).bytes -= 1;
        CHECK(call(y) == kShort);
    }
    y = d;
    y.parents = d.tokens;
    CHECK(call(y) == kArg);
    y = d;
    y.next_scores.data = s;
    y.next_scores.bytes = prompts * keep * 4;
    CHECK(call(y) == kArg);
    y = d;
    y.workspace.bytes -= 1;
    CHECK(call(y) == kShort);
    y = d;
    y.reserved[1] = 1;
    CHECK(call(y) == kArg);
    y = d;
    y.logits.rows = 0;
    CHECK(call(y) == kOk);
    plan_contract(e, "beam_select", [&](strix_amd_op_plan* p) { return strix_amd_beam_select_plan_create(e.c, &d, &e.s, p); });
    for (void* v : {x, s, f, ns, pa, to, ws}) CHECK(hipFree(v) == hipSuccess);
}

static void reorder_contract(Env& e) {
    const uint64_t outer = 2, prompts = 3, beams = 4, inner = 5, bytes = 96, room = 128, rows = prompts * beams;
    const uint64_t all = outer * rows * inner * room;
    void *pa = device(rows * 4), *a = device(all), *b = device(all);
    auto d = header<strix_amd_beam_reorder_desc>();
    d.parents = buffer(pa, rows);
    d.source = {a, all, {rows * inner * room, inner * room, room}};
    d.target = {b, all, {rows * inner * room, inner * room, room}};
    d.prompts = prompts;
    d.outer = outer;
    d.inner = inner;
    d.bytes = bytes;
    d.beams = beams;
    auto call = [&](const strix_amd_beam_reorder_desc& y) {
        fake::launches.clear();
        return strix_amd_beam_reorder(e.c, &y, &e.s);
    };
    CHECK(call(d) == kOk && fake::launches.size() == 1);
    auto y = d;
    y.target = y.source;
    CHECK(call(y) == kOk && fake::launches.size() == 1);
    y.target.strides[1] = room;   // the same memory in another order
    y.target.strides[2] = rows * room;
    CHECK(call(y) == kArg);
    y = d;
    y.target.strides[0] = inner * room;   // pieces over each other
    CHECK(call(y) == kFormat);
    y = d;
    y.target.strides[2] = bytes - 1;
    CHECK(call(y) == kFormat);
    y = d;
    y.source.strides[1] = 0;   // every row the same state
    CHECK(call(y) == kOk);
    y = d;
    y.target.data = static_cast<char*>(a) + room;
    y.target.buffer_bytes = all - room;
    y.outer = 1;
    CHECK(call(y) == kArg);
    for (uint32_t bad : {0u, 65u}) {
        y = d;
        y.beams = bad;
        CHECK(call(y) == kFormat);
    }
    y = d;
    y.flags = 1;
    CHECK(call(y) == kArg);
    y = d;
    y.parents = {};
    CHECK(call(y) == kShort);
    y = d;
    y.parents.bytes -= 1;
    CHECK(call(y) == kShort);
    y = d;
    y.source.buffer_bytes = (outer - 1) * d.source.strides[0] + (rows - 1) * d.source.strides[1] + (inner - 1) * room + bytes;
    CHECK(call(y) == kOk);
    y.source.buffer_bytes -= 1;
    CHECK(call(y) == kShort);
    y = d;
    y.target.data = nullptr;
    CHECK(call(y) == kArg);
    y = d;
    y.source.strides[0] = UINT64_MAX / 2;
    CHECK(call(y) == kArg || call(y) == kShort);
    y = d;
    y.prompts = uint64_t(1) << 60;
    CHECK(call(y) == kFormat);
    y = d;
    y.parents.data = b;   // what is written holds the parents
    CHECK(call(y) == kArg);
    for (auto m : {&strix_amd_beam_reorder_desc::prompts, &strix_amd_beam_reorder_desc::outer,
                   &strix_amd_beam_reorder_desc::inner, &strix_amd_beam_reorder_desc::bytes}) {
        y = d;
        y.*m = 0;
        CHECK(call(y) == kOk && fake::launches.empty());
    }
    plan_contract(e, "beam_reorder", [&](strix_amd_op_plan* p) { return strix_amd_beam_reorder_plan_create(e.c, &d, &e.s, p); });
    for (void* v : {pa, a, b}) CHECK(hipFree(v) == hipSuccess);
}

// Passes and tiles cover every row and channel within the kernels' limits.
static void sizing() {
    // channels (of weights' rows) and rows of a tile, by core
    const uint64_t shape[][2] = {{0, 0},   {16, 16}, {16, 32},   {32, 16},   {32, 32},
                                {32, 64}, {64, 64}, {128, 128}, {256, 128}, {256, 256}};
    for (uint64_t rows : {1ull, 2ull, 3ull, 4ull, 5ull, 8ull, 9ull, 16ull, 17ull, 32ull, 33ull, 64ull, 65ull, 255ull, 333ull, 2048ull, 65536ull})
        for (uint32_t I : {1u, 128u, 2048u, 2049u, 5120u, 8192u, 40000u, 131072u})
            for (uint32_t N : {1u, 16u, 512u, 5120u, 12288u, 129280u})
                for (int kind = 0; kind < 5; ++kind) {
                    const bool pair = kind & 1, exact = kind >= 2, rounded = kind == 3;
                    const stx::Fp8Plan p = stx::fp8_plan(rows, I, N, pair, exact, rounded);
                    const uint64_t kbs = stx::fp8_k_blocks(I);
                    if (p.core == stx::kFp8Decode) {
                        CHECK(rows <= 2 || (rows <= 4 && I <= 8192) || (rows <= 8 && I <= 2048));
                        CHECK(p.bytes == (rounded ? (rows * N * 4 + 255) / 256 * 256 : 0) && !p.hidden_at);
                        continue;
                    }
                    CHECK(p.scales_at == stx::fp8_block_bytes(rows, I));
                    CHECK(p.bytes >= p.scales_at + kbs * stx::fp8_padded_rows(rows) * 4);
                    CHECK(!p.hidden || rounded);
                    CHECK(p.core != stx::kFp8Wide256x256 || !exact);
                    if (p.hidden) CHECK(p.hidden_at % 256 == 0 && p.bytes >= p.hidden_at + rows * N * 4);
                    const uint64_t weights = pair ? (uint64_t(N) + 31) / 32 * 64 : N;
                    CHECK(p.n_tiles == (weights + shape[p.core][0] - 1) / shape[p.core][0]);
                    CHECK(p.m_tiles == (rows + shape[p.core][1] - 1) / shape[p.core][1]);
                    CHECK(!pair || shape[p.core][0] >= 32);
                    if (stx::fp8_pass_rows(rows, N) == rows) CHECK(stx::fp8_workspace_bytes(rows, I, N, pair, exact, rounded) == p.bytes);
                }
    for (uint64_t rows : {1ull, 9ull, 127ull, 128ull, 5000ull, 1ull << 20, 1ull << 31})
        for (uint32_t N : {1u, 128u, 4096u, 129280u, 16777216u}) {
            const uint64_t pass = stx::fp8_pass_rows(rows, N);
            CHECK(pass >= 1 && pass <= rows && (pass == rows || pass % 128 == 0));
            CHECK(pass <= 65536);   // 16-row blocks in a side of a grid
            for (uint32_t I : {1u, 4096u, 131072u})
                for (int kind = 0; kind < 4; ++kind)
                    for (uint64_t part = 1; part <= pass; part = part < pass ? (part * 2 < pass ? part * 2 : pass) : pass + 1) {
                        const stx::Fp8Plan p = stx::fp8_plan(part, I, N, kind & 1, kind & 2, false);
                        const uint64_t spread = uint64_t(p.n_tiles + 7) / 8 * 8 * p.m_tiles;
                        CHECK(spread * 512 < uint64_t(1) << 32);
                    }
        }
    // no tile is there for nothing: every kind of layer takes each that it can
    bool taken[2][2][10] = {};
    for (int kind = 0; kind < 4; ++kind)
        for (uint64_t rows : {1, 5, 9, 33, 65, 130, 257, 333, 513, 1500, 2048, 4096})
            for (uint32_t I : {128, 130, 300, 500, 1000, 2048, 4096, 6933, 8192})
                for (uint32_t N : {16, 17, 130, 300, 2307, 4100, 5125, 8192, 12288})
                    taken[kind & 1][kind / 2][stx::fp8_plan(rows, I, N, kind & 1, kind & 2, false).core] = true;
    for (int kind = 0; kind < 4; ++kind)
        for (uint32_t core = 0; core < 10; ++core) {
            const bool narrow = core == stx::kFp8Split16x16 || core == stx::kFp8Split16x32;
            CHECK(taken[kind & 1][kind / 2][core] ==
                  !((kind & 1 && narrow) || (kind & 2 && core == stx::kFp8Wide256x256)));
        }
    for (uint64_t rows : {1ull, 4ull, 64ull, 511ull, 512ull, 100000ull})
        for (uint32_t vocab : {1u, 2048u, 8192u, 8193u, 129280u, 2147483647u})
            for (uint32_t type : {F32, BF16}) {
                const stx::BeamSplits s = stx::beam_splits(rows, vocab, type);
                CHECK(s.each == 16 || s.each == (type == F32 ? 4 : 8));
                CHECK(s.length % (512 * s.each) == 0 && (s.splits == 1 || s.splits * rows <= 512));
                CHECK(uint64_t(s.splits - 1) * s.length < vocab && uint64_t(s.splits) * s.length >= vocab);
                CHECK(stx::beam_select_workspace_bytes(rows, vocab, type, 64) >=
                      rows * s.splits * (8 + (vocab < 64 ? vocab : 64) * 8));
            }
}

int main() {
    Env e;
    auto cd = header<strix_context_desc>();
    CHECK(strix_context_create(&cd, &e.c) == kOk);
    const uint64_t live0 = fake::live.size();
    e.hs = fake::make_stream(0);
    e.s = header<strix_stream>();
    e.s.hip_stream = e.hs;
    weights_contract(e);
    fp8_contract(e);
    select_contract(e);
    reorder_contract(e);
    sizing();
    CHECK(strix_context_destroy(e.c) == kOk);
    CHECK(fake::live.size() == live0);
    fake::destroy_streams();
    std::printf("%d checks passed\n", checks);
    return 0;
}
