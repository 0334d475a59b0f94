// Contract of the operators around the trellis layers (include/strix_trellis_ops.h)
// over a fake HIP runtime: argument checks, failure mapping, leaks, plans that
// only launch, and the sizing rules.
#include "fake.hpp"
#include "ops.hpp"
#include "strix_trellis_ops.h"

#include <climits>
#include <cstdio>
#include <cstdlib>
#include <cstring>
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
constexpr uint32_t F16 = STRIX_DTYPE_F16, BF16 = STRIX_DTYPE_BF16, F32 = STRIX_DTYPE_F32, I8 = STRIX_AMD_DTYPE_I8;
constexpr float kInf = std::numeric_limits<float>::infinity(), kNan = std::numeric_limits<float>::quiet_NaN();

template <class T>
static T header() {
    T d{};
    d.struct_size = sizeof(T);
    d.abi_version = STRIX_TRELLIS_ABI_VERSION;
    return d;
}
static strix_stream stream_of(hipStream_t s) {
    auto d = header<strix_stream>();
    d.hip_stream = s;
    return d;
}
static void* device(size_t bytes) {
    void* p = nullptr;
    CHECK(hipMalloc(&p, bytes) == hipSuccess);
    return p;
}
static uint64_t size_of(uint32_t type) { return type == F32 ? 4 : type == I8 ? 1 : 2; }
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

// A plan only launches; its handle keeps the context (and `weights`) alive.
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
    CHECK(create(nullptr) == kArg);
    strix_amd_op_plan q = p;
    CHECK(create(&q) == kArg && !q);   // another device is current
    fake::current_device = 0;
    CHECK(strix_amd_op_plan_destroy(p) == kOk);
}

static void int8_contract(Env& e) {
    const uint64_t live0 = fake::live.size();
    const uint64_t N = 70, I = 300, rows = 9;
    void *q = device(N * I), *t = device(N * 4), *b = device(N * 4), *wf = device(N * I * 4);
    auto d = header<strix_amd_int8_weights_desc>();
    d.weights = view(q, I8, N, I);
    d.scales = buffer(t, N);
    d.bias = buffer(b, N);
    auto prepare = [&](strix_amd_int8_weights_desc x) {
        strix_amd_int8_weights w = reinterpret_cast<strix_amd_int8_weights>(1);
        const strix_status s = strix_amd_int8_weights_prepare(e.c, &x, &e.s, &w);
        CHECK((s == kOk) == (w != nullptr));
        if (w) CHECK(strix_amd_int8_weights_destroy(w) == kOk);
        return s;
    };
    const uint64_t live1 = fake::live.size();
    CHECK(prepare(d) == kOk);
    auto x = d;
    x.struct_size -= 1;
    CHECK(prepare(x) == kAbi);
    x = d;
    x.reserved[3] = 1;
    CHECK(prepare(x) == kArg);
    x = d;
    x.weights.abi_version = 2;
    CHECK(prepare(x) == kAbi);
    x = d;
    x.weights.flags = 1;
    CHECK(prepare(x) == kArg);
    x = d;
    x.scales = {};
    CHECK(prepare(x) == kShort);
    x.scales = {nullptr, N * 4};
    CHECK(prepare(x) == kArg);
    x = d;
    x.scales.bytes -= 4;
    CHECK(prepare(x) == kShort);
    x = d;
    x.bias.bytes -= 1;
    CHECK(prepare(x) == kShort);
    x = d;
    x.weights = view(wf, F32, N, I);
    CHECK(prepare(x) == kArg);   // scales of float weights
    x.scales = {};
    CHECK(prepare(x) == kOk);
    x.weights.dtype = 7;
    CHECK(prepare(x) == kFormat);
    x = d;
    x.weights.rows = 0;
    CHECK(prepare(x) == kFormat);
    x = d;
    x.weights.width = 0;
    CHECK(prepare(x) == kFormat);
    x.weights.width = uint64_t(STRIX_AMD_INT8_MAX_INPUT) + 1;
    x.weights.rows = 1;
    x.weights.buffer_bytes = uint64_t(1) << 20;
    CHECK(prepare(x) == kFormat);
    x = d;
    x.weights.row_stride = I - 1;
    CHECK(prepare(x) == kFormat);
    x = d;
    x.weights.buffer_bytes -= 1;
    CHECK(prepare(x) == kShort);
    x = d;
    x.weights.rows += 1;   // beyond the allocation
    x.weights.buffer_bytes += I;
    x.scales = buffer(wf, N + 1);
    x.bias = {};
    CHECK(prepare(x) == kShort);
    x = d;
    x.weights.data = &x;   // host memory
    CHECK(prepare(x) == kArg);
    for (int at = 0; at < 3; ++at) {
        fake::launch_fail_at = at;
        CHECK(prepare(d) == kBackend && fake::live.size() == live1);
    }
    fake::sync_fail_at = 0;
    CHECK(prepare(d) == kBackend && fake::live.size() == live1);
    fake::malloc_fail_at = 0;
    CHECK(prepare(d) == kMemory && fake::live.size() == live1);
    fake::reset_failures();
    CHECK(strix_amd_int8_weights_prepare(e.c, &d, &e.s, nullptr) == kArg);
    CHECK(strix_amd_int8_weights_destroy(nullptr) == kArg);

    strix_amd_int8_weights w = nullptr;
    CHECK(strix_amd_int8_weights_prepare(e.c, &d, &e.s, &w) == kOk);
    fake::free_fail_at = 0;
    CHECK(strix_amd_int8_weights_destroy(w) == kBackend);   // the handle stays
    void *in = device(rows * I * 4), *out = device(rows * N * 4), *sc = device(rows * 4);
    auto c = header<strix_amd_int8_linear_desc>();
    c.weights = w;
    c.input = view(in, F32, rows, I);
    c.output = view(out, BF16, rows, N);
    c.alpha = 1;
    uint64_t need = 1;
    CHECK(strix_amd_int8_linear_workspace_bytes(e.c, &c, &need) == kOk);
    CHECK(need == stx::int8_workspace_bytes(rows, I, N));
    void* ws = device(need);
    c.workspace = {ws, need};
    auto call = [&](const strix_amd_int8_linear_desc& y) {
        fake::launches.clear();
        const strix_status s = strix_amd_int8_linear(e.c, &y, &e.s);
        CHECK(fake::launches.empty() == (s != kOk || !y.input.rows));
        return s;
    };
    CHECK(call(c) == kOk);
    auto y = c;
    y.weights = nullptr;
    CHECK(call(y) == kArg);
    for (float bad : {kInf, kNan}) {
        y = c;
        y.alpha = bad;
        CHECK(call(y) == kArg);
        y = c;
        y.beta = bad;
        CHECK(call(y) == kArg);
    }
    y = c;
    y.input.width -= 1;
    CHECK(call(y) == kFormat);
    y = c;
    y.output.rows -= 1;
    CHECK(call(y) == kFormat);
    y = c;
    y.output.dtype = I8;
    CHECK(call(y) == kFormat);
    y = c;
    y.input_scales = buffer(sc, rows);
    CHECK(call(y) == kArg);
    y.input = view(in, I8, rows, I);
    CHECK(call(y) == kOk);
    y.input_scales.bytes -= 4;
    CHECK(call(y) == kShort);
    y = c;
    y.workspace.bytes -= 1;
    CHECK(call(y) == kShort);
    y = c;
    y.workspace.data = static_cast<char*>(ws) + 4;
    CHECK(call(y) == kArg);
    y = c;
    y.output = view(in, F32, rows, N);
    CHECK(call(y) == kArg);   // overlaps the input
    y = c;
    y.input.row_stride = UINT64_MAX / 2;
    CHECK(call(y) == kArg);   // the extent overflows
    y = c;
    y.input.data = static_cast<char*>(in) + 1;
    CHECK(call(y) == kArg);
    y = c;
    y.input.rows = y.output.rows = uint64_t(INT_MAX) + 1;
    CHECK(call(y) == kFormat);
    y = c;
    y.input = view(nullptr, F32, 0, I);
    y.output = view(nullptr, F32, 0, N);
    y.workspace = {};
    CHECK(call(y) == kOk);
    y = c;
    y.input.rows = y.output.rows = 1;   // one row: the stride does not count
    y.input.row_stride = 0;
    CHECK(call(y) == kOk);
    plan_contract(e, "int8_linear",
                  [&](strix_amd_op_plan* p) { return strix_amd_int8_linear_plan_create(e.c, &c, &e.s, p); });
    strix_amd_op_plan p = nullptr;
    CHECK(strix_amd_int8_linear_plan_create(e.c, &c, &e.s, &p) == kOk);
    CHECK(strix_amd_int8_weights_destroy(w) == kArg);   // held by the plan
    CHECK(strix_amd_op_plan_destroy(p) == kOk);
    CHECK(strix_amd_int8_weights_destroy(w) == kOk);
    for (void* v : {q, t, b, wf, in, out, sc, ws}) CHECK(hipFree(v) == hipSuccess);
    CHECK(fake::live.size() == live0);
}

static void norm_contract(Env& e) {
    const uint64_t rows = 3, width = 40, n = rows * width;
    void *a = device(n * 4), *b = device(n * 4), *h = device(n * 4), *m = device(n * 4), *g = device(n * 4),
         *w = device(width * 4);
    auto d = header<strix_amd_block_norm_desc>();
    d.block = view(a, F32, rows, width);
    d.residual = view(b, F32, rows, width);
    d.gate = view(g, F32, rows, width);
    d.hidden = view(h, F32, rows, width);
    d.normed = view(m, F32, rows, width);
    d.post_weight = d.pre_weight = buffer(w, width);
    d.eps = 1e-6f;
    d.residual_scale = d.block_scale = 1;
    auto call = [&](const strix_amd_block_norm_desc& y) {
        fake::launches.clear();
        const strix_status s = strix_amd_block_norm(e.c, &y, &e.s);
        CHECK(fake::launches.size() <= (s == kOk ? 1u : 0u));
        return s;
    };
    CHECK(call(d) == kOk && fake::launches.size() == 1);
    auto y = d;
    for (uint64_t r : {uint64_t(1), rows})
        for (uint64_t c : {uint64_t(1), width}) {
            y.gate = view(g, F32, r, c);
            CHECK(call(y) == kOk);
        }
    y.gate = view(g, F32, 2, width);
    CHECK(call(y) == kFormat);
    y.gate = view(g, F32, rows, 2);
    CHECK(call(y) == kFormat);
    y.gate = view(g, F16, rows, width);
    CHECK(call(y) == kFormat);
    y = d;
    y.gate = {};
    CHECK(call(y) == kOk);
    y.gate_activation = STRIX_AMD_GATE_SIGMOID;   // of no gate
    CHECK(call(y) == kArg);
    y = d;
    y.gate_activation = 2;
    CHECK(call(y) == kFormat);
    y = d;
    y.norm = 2;
    CHECK(call(y) == kFormat);
    for (float bad : {0.0f, -1.0f, kInf, kNan}) {
        y = d;
        y.eps = bad;
        CHECK(call(y) == kArg);
    }
    y = d;
    y.block_scale = kNan;
    CHECK(call(y) == kArg);
    y = d;
    y.hidden = y.normed = {};
    CHECK(call(y) == kArg);
    y = d;
    y.normed = {};
    CHECK(call(y) == kArg);   // pre_weight without normed
    y.pre_weight = {};
    CHECK(call(y) == kOk);
    y.pre_bias = buffer(w, width);
    CHECK(call(y) == kArg);
    y = d;
    y.block = {};
    CHECK(call(y) == kArg);   // a gate of nothing
    y.gate = {};
    y.post_weight = {};
    CHECK(call(y) == kOk);
    y.residual = {};
    CHECK(call(y) == kArg);
    // in place: exactly block or residual
    y = d;
    y.hidden = d.residual;
    y.normed = d.block;
    CHECK(call(y) == kOk);
    y.normed = d.residual;
    CHECK(call(y) == kArg);   // both outputs in one place
    y = d;
    y.hidden = view(static_cast<float*>(a) + 1, F32, rows, width - 1, width);
    CHECK(call(y) == kFormat);
    y = d;
    y.residual = y.hidden = view(a, F32, rows, width);
    CHECK(call(y) == kOk);   // block and residual are one tensor, hidden takes its place
    y = d;
    y.hidden = view(g, F32, rows, width);
    CHECK(call(y) == kArg);
    y = d;
    y.hidden = view(w, F32, 1, width);
    CHECK(call(y) == kFormat);
    y = d;
    y.post_weight = buffer(h, width);
    CHECK(call(y) == kArg);   // a vector in an output
    y = d;
    y.post_weight.bytes -= 4;
    CHECK(call(y) == kShort);
    y = d;
    y.block.dtype = y.residual.dtype = y.gate.dtype = y.hidden.dtype = y.normed.dtype = I8;
    CHECK(call(y) == kFormat);
    y = d;
    for (auto* v : {&y.block, &y.residual, &y.gate, &y.hidden, &y.normed}) v->rows = 0;
    CHECK(call(y) == kOk && fake::launches.empty());
    plan_contract(e, "block_norm",
                  [&](strix_amd_op_plan* p) { return strix_amd_block_norm_plan_create(e.c, &d, &e.s, p); });
    for (void* v : {a, b, h, m, g, w}) CHECK(hipFree(v) == hipSuccess);
}

static void logprobs_contract(Env& e) {
    const uint64_t rows = 3, vocab = 20000;
    void *x = device(rows * vocab * 4), *ids = device(rows * 4), *lp = device(rows * 4), *rk = device(rows * 4),
         *en = device(rows * 4), *ti = device(rows * 64 * 4), *tl = device(rows * 64 * 4);
    auto d = header<strix_amd_token_logprobs_desc>();
    d.logits = view(x, F32, rows, vocab);
    d.tokens = buffer(ids, rows);
    d.logprobs = buffer(lp, rows);
    d.ranks = buffer(rk, rows);
    d.entropy = buffer(en, rows);
    d.top = 64;
    d.top_ids = buffer(ti, rows * 64);
    d.top_logprobs = buffer(tl, rows * 64);
    d.scale = 1;
    uint64_t need = 0;
    CHECK(strix_amd_token_logprobs_workspace_bytes(e.c, &d, &need) == kOk);
    CHECK(need && need == stx::logprobs_workspace_bytes(rows, vocab, 64));
    void* ws = device(need);
    d.workspace = {ws, need};
    auto call = [&](const strix_amd_token_logprobs_desc& y) {
        fake::launches.clear();
        const strix_status s = strix_amd_token_logprobs(e.c, &y, &e.s);
        CHECK(fake::launches.size() <= (s == kOk ? 1u : 0u));
        return s;
    };
    CHECK(call(d) == kOk && fake::launches.size() == 1);
    auto y = d;
    y.top = 65;
    CHECK(call(y) == kFormat);
    y = d;
    y.logits = view(x, F32, rows, 63);
    CHECK(call(y) == kFormat);   // more tokens asked for than there are
    y = d;
    y.logits = view(x, I8, rows, vocab);
    CHECK(call(y) == kFormat);
    for (float bad : {0.0f, -1.0f, 1e-6f, 1e6f, kInf, kNan}) {
        y = d;
        y.scale = bad;
        CHECK(call(y) == kArg);
    }
    y = d;
    y.tokens = {};
    CHECK(call(y) == kArg);
    y.logprobs = {};
    CHECK(call(y) == kArg);
    y.ranks = {};
    CHECK(call(y) == kOk);
    y.top = 0;
    CHECK(call(y) == kArg);
    y.top_ids = y.top_logprobs = {};
    CHECK(call(y) == kOk);
    y.entropy = {};
    CHECK(call(y) == kArg);
    y = d;
    y.top_ids.bytes -= 1;
    CHECK(call(y) == kShort);
    y = d;
    y.entropy = y.logprobs;
    CHECK(call(y) == kArg);
    y = d;
    y.top_logprobs = buffer(x, rows * 64);
    CHECK(call(y) == kArg);
    y = d;
    y.workspace.bytes -= 256;
    CHECK(call(y) == kShort);
    y = d;
    y.logits.rows = 0;
    CHECK(call(y) == kOk && fake::launches.empty());
    plan_contract(e, "token_logprobs",
                  [&](strix_amd_op_plan* p) { return strix_amd_token_logprobs_plan_create(e.c, &d, &e.s, p); });
    for (void* v : {x, ids, lp, rk, en, ti, tl, ws}) CHECK(hipFree(v) == hipSuccess);
}

// Passes and splits cover every row and token within the kernels' limits.
static void sizing() {
    // every row and channel lies in a tile, and a pass's workspace serves every smaller one
    for (uint64_t rows : {1ull, 2ull, 4ull, 5ull, 8ull, 9ull, 16ull, 17ull, 32ull, 33ull, 64ull, 65ull, 333ull, 2048ull, 65536ull})
        for (uint32_t I : {1u, 1536u, 1537u, 5120u, 40000u, 131071u})
            for (uint32_t N : {1u, 16u, 512u, 5120u, 12288u, 129280u}) {
                const stx::Int8Plan p = stx::int8_plan(rows, I, N);
                const uint64_t shape[][2] = {{0, 0}, {16, 16}, {32, 32}, {32, 64}, {64, 64}, {128, 128}, {256, 128}};
                if (p.core == stx::kInt8Decode) {
                    CHECK(rows <= 8 && rows * (stx::int8_k_blocks(I) * 64 + 64) <= stx::kInt8DecodeLds && !p.bytes);
                    continue;
                }
                CHECK(p.n_tiles == (N + shape[p.core][0] - 1) / shape[p.core][0]);
                CHECK(p.m_tiles == (rows + shape[p.core][1] - 1) / shape[p.core][1]);
                CHECK(p.core != stx::kInt8Rows16 || p.m_tiles == 1);
                CHECK(p.scales_at == stx::int8_block_bytes(rows, I) && p.bytes >= p.scales_at + rows * 4);
                CHECK(stx::int8_workspace_bytes(rows, I, N) >= stx::int8_workspace_bytes(rows - 1, I, N));
            }
    for (uint64_t rows : {1ull, 9ull, 127ull, 128ull, 5000ull, 1ull << 20, 1ull << 31})
        for (uint32_t N : {1u, 128u, 4096u, 129280u, 16777216u}) {
            const uint64_t pass = stx::int8_pass_rows(rows, N);
            CHECK(pass >= 1 && pass <= rows && (pass == rows || pass % 128 == 0));
            CHECK((pass + 127) / 128 * ((uint64_t(N) + 127) / 128) * 256 < uint64_t(1) << 32);
            CHECK(stx::int8_row_blocks(pass) * 4 * 256 < uint64_t(1) << 32);
            // a launch of any core the plan picks for any part of a pass holds fewer than 2^32 threads
            for (uint32_t I : {1u, 64u, 4096u, 40000u, 131071u})
                for (uint64_t part = 1; part <= pass; part = part < pass ? (part * 2 < pass ? part * 2 : pass) : pass + 1) {
                    const stx::Int8Plan p = stx::int8_plan(part, I, N);
                    const uint64_t spread = uint64_t(p.n_tiles + 7) / 8 * 8 * p.m_tiles;
                    CHECK(p.core == stx::kInt8Decode || spread * 512 < uint64_t(1) << 32);
                }
        }
    for (uint64_t rows : {1ull, 2ull, 7ull, 511ull, 512ull, 1ull << 30})
        for (uint32_t vocab : {1u, 8192u, 8193u, 129280u, 1000000u, 2147483647u}) {
            const uint64_t s = stx::logprobs_splits(rows, vocab), batches = (uint64_t(vocab) + 8191) / 8192;
            const uint64_t length = (batches + s - 1) / s * 8192;
            CHECK(s >= 1 && (s - 1) * length < vocab && s * length >= vocab);
            CHECK(s == 1 || s * rows <= 512);
        }
}

int main() {
    Env e;
    auto cd = header<strix_context_desc>();
    CHECK(strix_context_create(&cd, &e.c) == kOk);
    const uint64_t live0 = fake::live.size();
    e.hs = fake::make_stream(0);
    e.s = stream_of(e.hs);
    int8_contract(e);
    norm_contract(e);
    logprobs_contract(e);
    sizing();
    CHECK(strix_amd_op_plan_submit(nullptr) == kArg && strix_amd_op_plan_destroy(nullptr) == kArg);
    CHECK(strix_context_destroy(e.c) == kOk);
    CHECK(fake::live.size() == live0);
    fake::destroy_streams();
    std::printf("%d checks passed\n", checks);
    return 0;
}
