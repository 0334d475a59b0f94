// Decoding with several beams: the selection of continuations and the reordering of states.
//
// Selection.  The first launch leaves, per row of logits and split of its
// vocabulary, the softmax statistics and the `keep` first tokens in order
// (launch_logprobs_parts).  The second has one workgroup per prompt: it joins the
// beams' statistics, and merges the sorted lists of all beams and splits.
#include "beam.hpp"
#include "logprobs_device.hpp"

namespace stx {

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr uint32_t kList = 1024, kMaxBeams = 64;

struct Candidate {
    double c;
    uint64_t id;   // beam over token
};
__device__ __forceinline__ bool ahead_of(const Candidate& a, const Candidate& b) {
    return a.c > b.c || (a.c == b.c && a.id < b.id);
}

struct SelectArgs {
    const float* scores;
    const int32_t* finished;
    const float* part;           // [rows][splits][8]
    const uint64_t* keys;        // [rows][splits][top]
    float* next_scores;
    int32_t *parents, *tokens;
    uint32_t beams, keep, top, splits, last;   // last: tokens of a row's last split
    int32_t pad;
    float c;
    double scale, slope;         // slope: (scale log2 e - c) / c ln 2
};

__global__ __launch_bounds__(kThreads) void beam_join_kernel(SelectArgs a) {
    __shared__ Candidate list[kList];
    __shared__ double beam_at[kMaxBeams];    // a candidate's value is beam_at + scale * (logit - beam_m)
    __shared__ float beam_m[kMaxBeams];
    __shared__ uint32_t beam_kind[kMaxBeams];   // 0 offers nothing, 1 its tokens, 2 the pad token
    __shared__ uint32_t list_end;
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint64_t row0 = uint64_t(blockIdx.x) * a.beams;
    if (tid == 0) list_end = 0;
    for (uint32_t b = w; b < a.beams; b += kWaves) {
        const float score = ld_global(a.scores + row0 + b);
        const bool over = a.finished && ld_global(a.finished + row0 + b) != 0;
        uint32_t kind = 0;
        double at = score;
        float m = 0.0f;
        if (fabsf(score) < kInf) {
            kind = 2;
            if (!over) {
                Stats t = kNothing;
                for (uint32_t i = lane; i < a.splits; i += 64) {
                    const f32x4 o = ld_global(reinterpret_cast<const f32x4*>(a.part + ((row0 + b) * a.splits + i) * 8));
                    join(t, {o[0], o[1], o[2], o[3]}, a.c);
                }
                t = join_lanes(t, a.c);
                kind = t.n > 0.0f && t.m < kInf && t.s == t.s ? 1 : 0;
                // The statistics were taken at c, scale log2 e rounded to FP32: the first
                // order of the log sum in the difference, whose square is below 1e-14.
                const double sum = double(t.n) + double(t.s);
                at = double(score) - (log(sum) + a.slope * double(t.h) / sum);
                m = t.m;
            }
        }
        if (lane == 0) {
            beam_kind[b] = kind;
            beam_at[b] = at;
            beam_m[b] = m;
        }
    }
    __syncthreads();

    // The lists, first keys first: rounds of about 128 keys that enter if they beat
    // the last of the best so far.  The lists are sorted, so a round of which
    // none enters is the last.
    const uint32_t lists = a.beams * a.splits, depth = lists >= 128 ? 1 : 128 / lists;
    uint32_t count = 0;
    Candidate bound{-double(kInf), ~uint64_t(0)};
    for (uint32_t d0 = 0; d0 < a.top; d0 += depth) {
        auto enter = [&](const Candidate& k) {
            if (k.c == -double(kInf) || (count == a.keep && !ahead_of(k, bound))) return;
            list[atomicAdd(&list_end, 1u)] = k;   // 64 kept, 64 finished and 512 others at most
        };
        if (d0 == 0 && tid < a.beams && beam_kind[tid] == 2)
            enter({beam_at[tid], uint64_t(tid) << 32 | uint32_t(a.pad)});
        for (uint32_t i = tid; i < lists * depth; i += kThreads) {
            const uint32_t l = i % lists, d = d0 + i / lists, b = l / a.splits, split = l % a.splits;
            const uint32_t length = split + 1 < a.splits || a.last > a.top ? a.top : a.last;
            if (d >= length || beam_kind[b] != 1) continue;
            const uint64_t key = ld_global(a.keys + ((row0 + b) * a.splits + split) * a.top + d);
            const double x = value_of(key);
            enter({beam_at[b] + a.scale * (x - double(beam_m[b])), uint64_t(b) << 32 | id_of(key)});
        }
        __syncthreads();
        const uint32_t n = list_end;
        if (n == count && d0) break;
        Candidate mine[2];
        uint32_t rank[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 2; ++j) mine[j] = tid + j * kThreads < n ? list[tid + j * kThreads] : Candidate{0.0, 0};
        if (uint32_t(__builtin_amdgcn_readfirstlane(tid)) < n) {   // the wave holds candidates
            for (uint32_t i = 0; i < n; ++i) {
                const Candidate k = list[i];
#pragma unroll
                for (int j = 0; j < 2; ++j) rank[j] += ahead_of(k, mine[j]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (tid + j * kThreads < n && rank[j] < a.keep) list[rank[j]] = mine[j];
        count = n < a.keep ? n : a.keep;
        if (tid == 0) list_end = count;
        __syncthreads();
        if (count == a.keep) bound = list[count - 1];
    }
    for (uint32_t j = tid; j < a.keep; j += kThreads) {
        const uint64_t to = uint64_t(blockIdx.x) * a.keep + j;
        const Candidate k = j < count ? list[j] : Candidate{-double(kInf), ~uint64_t(0)};
        st_global(a.next_scores + to, float(k.c));
        st_global(a.parents + to, int32_t(k.id >> 32));
        st_global(a.tokens + to, int32_t(uint32_t(k.id)));
    }
}

// ---- reordering ----
struct ReorderArgs {
    const int32_t* parents;
    const uint8_t* source;
    uint8_t* target;
    uint64_t bytes;
    uint64_t source_strides[3], target_strides[3];
    uint32_t beams, inner;
    uint64_t chunk, piece, prompt;   // the launch's first
};

// N bytes at any alignment, and the registers that hold them.
template <int N>
struct Unit {
    typedef uint32_t type __attribute__((ext_vector_type(N / 4), aligned(1)));
    typedef uint32_t held __attribute__((ext_vector_type(N / 4)));
};
template <>
struct Unit<4> {
    typedef uint32_t type __attribute__((aligned(1)));
    typedef uint32_t held;
};
template <>
struct Unit<1> {
    typedef uint8_t type;
    typedef uint32_t held;
};

// One unit of every beam, all of them read before one is written.  (A variable for each
// beam: an array would be kept as one vector, copied whole at every branch.)
template <int N, int B, class Parent, class... V>
__device__ __forceinline__ void move(const uint8_t* from, uint64_t from_row, uint8_t* to, uint64_t to_row, uint32_t k,
                                     const Parent& parent, V&... v) {
    using T = typename Unit<N>::type;
    constexpr int b = sizeof...(V);
    if constexpr (b < B) {
        typename Unit<N>::held x{};
        const uint32_t p = parent(b);   // ~0: the beam stays
        if (p != ~0u) x = *(const __attribute__((address_space(1))) T*)(from + p * from_row + k);
        move<N, B>(from, from_row, to, to_row, k, parent, v..., x);
    } else {
        // Every read arrives here.  Left to where a value is used, behind a branch, the waits
        // would be for the stores ahead of it too: they share a counter.
        auto arrive = [](auto& x) __attribute__((always_inline)) { asm volatile("" : "+v"(x)); };
        (arrive(v), ...);
        int i = 0;
        auto store = [&](const auto& x) __attribute__((always_inline)) {
            if (parent(i) != ~0u) *(__attribute__((address_space(1))) T*)(to + i * to_row + k) = x;
            ++i;
        };
        (store(v), ...);
    }
}

// A thread moves one unit of N bytes of every beam of a prompt: it reads all of them
// before it writes one, so that source and target may be one.  B: beams at most.
template <int B, int N, bool IN_PLACE>
__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderArgs a) {
    const uint64_t piece = a.piece + blockIdx.y, prompt = a.prompt + blockIdx.z;
    uint64_t outer = piece, inner = 0;
    if (a.inner > 1) {   // fewer than 2^32 of them, or 64-bit arithmetic
        outer = piece >> 32 ? piece / a.inner : uint32_t(piece) / a.inner;
        inner = piece - outer * a.inner;
    }
    const uint64_t row0 = prompt * a.beams, chunk = a.chunk + blockIdx.x;
    const uint64_t at = chunk * 256 * N, left = a.bytes - at;
    const uint8_t* from =
        a.source + outer * a.source_strides[0] + row0 * a.source_strides[1] + inner * a.source_strides[2] + at;
    uint8_t* to = a.target + outer * a.target_strides[0] + row0 * a.target_strides[1] + inner * a.target_strides[2] + at;
    // lane b has beam b's parent
    const uint32_t lane = threadIdx.x & 63;
    uint32_t mine = ~0u;
    if (lane < a.beams) {
        const uint32_t p = ld_global(a.parents + row0 + lane), own = IN_PLACE ? ~0u : lane;
        mine = p >= a.beams || p == lane ? own : p;
    }
    auto parent = [&](int b) { return uint32_t(__builtin_amdgcn_readlane(mine, b)); };
    const uint32_t units = left < 256 * N ? uint32_t(left) / N : 256, tail = left < 256 * N ? uint32_t(left) % N : 0;
    if (threadIdx.x < units)
        move<N, B>(from, a.source_strides[1], to, a.target_strides[1], threadIdx.x * N, parent);
    if (threadIdx.x < tail)
        move<1, B>(from, a.source_strides[1], to, a.target_strides[1], units * N + threadIdx.x, parent);
}

template <int B, int N>
hipError_t reorder(const BeamReorderCall& call, hipStream_t stream) {
    ReorderArgs a{};
    a.parents = call.parents;
    a.source = call.source;
    a.target = call.target;
    a.bytes = call.bytes;
    for (int i = 0; i < 3; ++i) {
        a.source_strides[i] = call.source_strides[i];
        a.target_strides[i] = call.target_strides[i];
    }
    a.beams = call.beams;
    a.inner = uint32_t(call.inner);
    // a launch holds fewer than 2^32 threads, and its grid 2^16 - 1 workgroups in y and z
    const uint64_t chunks = (call.bytes + 256 * N - 1) / (256 * N), pieces = call.outer * call.inner;
    constexpr uint64_t kMost = 1u << 23, kSide = 32768;
    auto part = [](uint64_t left, uint64_t most) { return uint32_t(left < most ? left : most); };
    const uint32_t x = part(chunks, kMost), y = part(pieces, part(kMost / x, kSide));
    const uint32_t z = part(call.prompts, part(kMost / x / y, kSide));
    for (a.prompt = 0; a.prompt < call.prompts; a.prompt += z)
        for (a.piece = 0; a.piece < pieces; a.piece += y)
            for (a.chunk = 0; a.chunk < chunks; a.chunk += x) {
                const dim3 grid(part(chunks - a.chunk, x), part(pieces - a.piece, y), part(call.prompts - a.prompt, z));
                if (call.in_place)
                    hipLaunchKernelGGL((beam_reorder_kernel<B, N, true>), grid, dim3(256), 0, stream, a);
                else
                    hipLaunchKernelGGL((beam_reorder_kernel<B, N, false>), grid, dim3(256), 0, stream, a);
                const hipError_t e = hipGetLastError();
                if (e != hipSuccess) return e;
            }
    return hipSuccess;
}

}  // namespace

hipError_t launch_beam_select(const BeamSelectCall& call, hipStream_t stream) {
    SelectArgs a{};
    a.scores = call.scores;
    a.finished = call.finished;
    a.next_scores = call.next_scores;
    a.parents = call.parents;
    a.tokens = call.tokens;
    a.beams = call.beams;
    a.keep = call.keep;
    a.top = call.keep < call.vocab ? call.keep : call.vocab;
    a.splits = logprobs_splits(call.rows, call.vocab);
    a.last = call.vocab - (a.splits - 1) * logprobs_split_length(a.splits, call.vocab);
    a.pad = call.pad;
    a.c = logprobs_exponent(call.scale);
    const double c = double(call.scale) * 1.4426950408889634074;
    a.scale = call.scale;
    a.slope = (c - double(a.c)) / double(a.c) * 0.69314718055994530942;
    a.part = static_cast<const float*>(call.workspace);
    a.keys = reinterpret_cast<const uint64_t*>(a.part + call.rows * a.splits * 8);
    const hipError_t e = launch_logprobs_parts(call.logits, call.rows, call.vocab, a.top, call.scale, call.scores,
                                               call.finished, call.workspace, stream);
    if (e != hipSuccess) return e;
    const uint64_t prompts = call.rows / call.beams;
    constexpr uint64_t kPrompts = 1u << 22;   // a launch holds fewer than 2^32 threads
    for (uint64_t p = 0; p < prompts; p += kPrompts) {
        const uint64_t n = prompts - p < kPrompts ? prompts - p : kPrompts;
        hipLaunchKernelGGL(beam_join_kernel, dim3(uint32_t(n)), dim3(kThreads), 0, stream, a);
        const hipError_t joined = hipGetLastError();
        if (joined != hipSuccess) return joined;
        a.scores += n * a.beams;
        if (a.finished) a.finished += n * a.beams;
        a.part += n * a.beams * a.splits * 8;
        a.keys += n * a.beams * a.splits * a.top;
        a.next_scores += n * a.keep;
        a.parents += n * a.keep;
        a.tokens += n * a.keep;
    }
    return hipSuccess;
}

hipError_t launch_beam_reorder(const BeamReorderCall& call, hipStream_t stream) {
    if (call.beams <= 4) return reorder<4, 16>(call, stream);
    if (call.beams <= 8) return reorder<8, 16>(call, stream);
    if (call.beams <= 16) return reorder<16, 16>(call, stream);
    if (call.beams <= 32) return reorder<32, 8>(call, stream);
    return reorder<64, 4>(call, stream);
}

}  // namespace stx
