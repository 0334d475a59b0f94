// Decoding with several beams: the selection of continuations and the reordering of states.
//
// Selection.  Two launches: the first reads the logits once, and leaves for each row and
// split of its vocabulary the softmax statistics and the `keep` first tokens in order; the second has
// one workgroup per prompt, which joins its beams' statistics and picks among their
// tokens.
//
// Statistics.  With m the largest logit of a wave so far, the wave's lanes hold
//   s = sum e^(scale (x - m))
// in FP32; the half steps of scale log2 e and of its product move a sum by 2^-24 (m - x) scale at most,
// 7e-7 where all of a vocabulary of 2^17 is as likely.  A batch whose largest logit stays below m
// needs no rescaling.  The splits' sums
// are joined in FP64, in which the candidates' values are compared too.
//
// Tokens.  A token's place in the order of its row is one 64-bit key: the logit's bits,
// made monotonic, over the inverted id.  The workgroup keeps a list of candidates in LDS and
// a bound that at least `top` keys reach.  The first batch takes its bound from the
// threads' largest logits (the k-th largest of each wave, with k * waves >= top).  Behind 1, 4,
// 16, .. batches the list is cut to the first `top` keys, the last of which is the new bound: about
// 1.4 `top` tokens enter between two cuts, and the waves meet only there.  A list that
// overflowed in between is filled again from memory, with a higher bound.
//
// 64 x 8 beams of 129280 BF16, 16 kept: the pass 37 us (3.2 TB/s of the rows it reads; its vector steps take half the cycles,
// and two batches on their way for three took 3 us more), the join 5 us.  4 beams of 129280 F32: 5.5 and 5.2,
// a chain of round trips each.
#include <type_traits>

#include "beam.hpp"
#include "logprobs_device.hpp"

namespace stx {

namespace {

constexpr int kThreads = kScanThreads, kWaves = kThreads / 64;
constexpr uint32_t kMaxBeams = 64;
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct ScanArgs {
    const void* logits;
    uint64_t stride;
    const float* scores;         // rows with a score that is not finite are not read,
    const int32_t* finished;     // nor finished ones
    float* part;                 // [rows][splits]{m, s}
    uint64_t* keys;              // [rows][splits][top]
    uint32_t vocab, top, splits, split_length;
    float c;                     // scale log2 e
};

// The k-th largest of a wave's values, -inf where there are fewer; k >= 1.
__device__ __forceinline__ float kth_of_wave(float v, uint32_t k) {
    float kth = -kInf;
    for (;;) {
        kth = wave_max(v);
        if (--k == 0) return kth;
        const uint64_t at = __ballot(v == kth);
        if (at && (threadIdx.x & 63) == uint32_t(__builtin_ctzll(at))) v = -kInf;
    }
}

template <class T, int EACH>
__global__ __launch_bounds__(kThreads, 4) void beam_scan_kernel(ScanArgs a) {
    using B = Batch<T, EACH>;
    constexpr uint32_t kBatch = B::kBatch, kList = kScanList;
    // batches on their way: a round trip to memory takes longer than a batch
    constexpr int kAhead = sizeof(T) == 4 && EACH == 16 ? 2 : 3;
    __shared__ __align__(16) uint64_t list[kList];
    __shared__ float wave_bound[kWaves], wave_sums[kWaves];
    __shared__ uint32_t list_end;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint64_t row = blockIdx.x / a.splits;
    if (!(fabsf(ld_global(a.scores + row)) < kInf) || (a.finished && ld_global(a.finished + row))) return;
    const uint32_t split = blockIdx.x % a.splits, v0 = split * a.split_length;
    const uint32_t v1 = a.vocab - v0 < a.split_length ? a.vocab : v0 + a.split_length;
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    B batch[kAhead + 1];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (v0 + i * kBatch < v1) batch[i].load(x, v0 + i * kBatch, v1);
    float m = kLowest, s = 0.0f;   // m is the wave's
    uint64_t bound = 0;            // keys below it do not enter the list
    float reach = -kInf;           // its logit
    uint32_t count = 0;            // keys in the list behind the last cut
    float peak = -kInf;            // the thread's largest logit since then
    uint32_t since = v0, cut_at = v0;   // the first batch since then, the batch behind which the next cut comes
    if (tid == 0) list_end = 0;

    auto weight = [&](float d) { return __builtin_amdgcn_exp2f(d * a.c); };
    auto enter = [&](uint32_t b0, const float (&v)[EACH]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            if (!__any(v[e] >= reach)) continue;
            const uint32_t id = B::id(b0, v1, e);
            const uint64_t k = key_of(v[e], id);
            if (v[e] >= reach && k >= bound && id != ~0u) {
                const uint32_t slot = atomicAdd(&list_end, 1u);
                if (slot < kList) list[slot] = k;
            }
        }
    };
    // A logit that at least `top` of the tokens since `since` reach, or -inf: the
    // k-th largest peak of each wave of which every lane has tokens, the least
    // of them.  Ends with a barrier.
    auto reach_of_peaks = [&] {
        const uint32_t tokens = v1 - since, of_wave = tokens / (64 * B::kGroup);
        const uint32_t waves = of_wave < 1 ? 1 : of_wave < kWaves ? of_wave : kWaves;
        const float kth = kth_of_wave(peak, (a.top + waves - 1) / waves);
        if (lane == 0) wave_bound[w] = uint32_t(w) < waves ? kth : kInf;
        __syncthreads();
        float least = wave_bound[0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) least = fminf(least, wave_bound[i]);
        __syncthreads();
        return least;
    };

    for (uint32_t b0 = v0; b0 < v1; b0 += kBatch) {
        if (v1 - b0 > kAhead * kBatch) batch[kAhead].load(x, b0 + kAhead * kBatch, v1);
        float v[EACH];
        batch[0].values(b0, v1, v);

        // ---- statistics ----
        float most = v[0];   // NaN if one is among them
#pragma unroll
        for (int e = 1; e < EACH; ++e) most = __builtin_elementwise_maximum(most, v[e]);
        const float wave_most = wave_max(most);
        if (wave_most > m) {   // the wave as one
            s *= weight(m - wave_most);
            m = wave_most;
        }
        float e2[EACH];
#pragma unroll
        for (int e = 0; e < EACH; ++e) e2[e] = weight(v[e] - m);
#pragma unroll
        for (int by = EACH / 2; by; by /= 2)   // pairwise
#pragma unroll
            for (int e = 0; e < by; ++e) e2[e] += e2[e + by];
        s += e2[0];

        // ---- tokens ----
        peak = fmaxf(peak, most);
        if (b0 == v0) {
            reach = reach_of_peaks();
            bound = uint64_t(key_of(reach, 0) >> 32) << 32;   // every id of that logit
        }
        if (__any(most >= reach)) enter(b0, v);
        const bool last = v1 - b0 <= kBatch;
        if (b0 == cut_at || last) {
            __syncthreads();
            while (list_end > kList) {
                // More tokens than the list holds.  The peaks or, with many
                // equal logits, the keys that got in give a higher bound; the
                // batches since the last cut enter again behind its keys.  By
                // the list's own bound at least kList - 2 top keys fewer do
                // each time.
                const uint64_t kept = uint32_t(tid) < count ? list[tid] : 0;
                const float higher = reach_of_peaks();
                cut(list, kList, a.top);
                const uint64_t of_list = list[a.top - 1], of_peaks = uint64_t(key_of(higher, 0) >> 32) << 32;
                bound = of_list > of_peaks ? of_list : of_peaks;
                reach = value_of(bound);
                __syncthreads();
                if (uint32_t(tid) < count) list[tid] = kept;
                if (tid == 0) list_end = count;
                __syncthreads();
                for (uint32_t b = since; b <= b0; b += kBatch) {
                    B again;
                    again.load(x, b, v1);
                    float u[EACH];
                    again.values(b, v1, u);
                    enter(b, u);
                }
                __syncthreads();
            }
            count = cut(list, list_end, a.top);
            if (!last) {
                if (count == a.top) {
                    bound = list[a.top - 1];
                    reach = value_of(bound);
                }
                if (tid == 0) list_end = count;
                since = b0 + kBatch;
                cut_at += 3 * (cut_at - v0 + kBatch);   // behind 1, 4, 16, .. batches
                peak = -kInf;
                __syncthreads();
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) batch[i] = batch[i + 1];
    }
    // the waves' statistics as one (their peaks' place is free behind the last cut)
    const uint64_t p = row * a.splits + split;
    s = wave_sum(s);
    if (lane == 0) {
        wave_bound[w] = m;
        wave_sums[w] = s;
    }
    __syncthreads();
    if (tid < kWaves) {
        const float of = wave_bound[tid];
        float most = wave_bound[0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) most = fmaxf(most, wave_bound[i]);
        float sum = wave_sums[tid] * weight(of - most);
        sum += __shfl_xor(sum, 1);
        sum += __shfl_xor(sum, 2);
        sum += __shfl_xor(sum, 4);
        if (tid == 0) st_global(reinterpret_cast<f32x2*>(a.part) + p, f32x2{most, sum});
    }
    // only the last split can be shorter than `top`: its keys end the row's
    if (uint32_t(tid) < count) st_global(a.keys + p * a.top + tid, list[tid]);
}

struct Candidate {
    double c;
    uint64_t id;   // beam over token
};
__device__ __forceinline__ bool ahead_of(const Candidate& a, const Candidate& b) {
    return a.c > b.c || (a.c == b.c && a.id < b.id);
}

struct JoinArgs {
    const float* scores;
    const int32_t* finished;
    const float* part;
    const uint64_t* keys;
    float* next_scores;
    int32_t *parents, *tokens;
    uint32_t beams, keep, top, splits, last;   // last: tokens of a row's last split
    int32_t pad;
    double scale;
};

// The beams' lists of keys, first keys first, are taken 1024 at a time (nearly always all of them at
// once); what reaches a bound that `keep` of them reach enters a list in LDS, whose first `keep` are
// found by counting who is ahead of whom.  The lists are sorted, so behind a round of which none
// enters there is nothing.  Keys dealt list by list to the waves would leave a wave with the lowest beam
// alone, whose keys then bound nothing (22 us for 5 with eight beams).
__global__ __launch_bounds__(kThreads) void beam_join_kernel(JoinArgs a) {
    constexpr uint32_t kRound = 2 * kThreads, kList = kRound + 2 * kMaxBeams;   // + kept ones and pad tokens
    __shared__ Candidate list[kList];
    __shared__ double beam_at[kMaxBeams];       // a candidate's value is beam_at + scale * (logit - beam_m)
    __shared__ float beam_m[kMaxBeams];
    __shared__ uint32_t beam_kind[kMaxBeams];   // 0 offers nothing, 1 its tokens, 2 the pad token
    __shared__ float wave_bound[kWaves];
    __shared__ uint32_t list_end;
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint64_t row0 = uint64_t(blockIdx.x) * a.beams;
    const uint32_t lists = a.beams * a.splits, all = lists * a.top;
    // A round's items by depth in their lists, dealt out to the waves in turn, another one first each time:
    // the waves' bounds are as high as their first keys are evenly spread.
    auto key_at = [&](uint32_t i) -> uint64_t {
        const uint32_t d = i / lists, l = i - d * lists, split = l % a.splits;
        const uint32_t length = split + 1 < a.splits || a.last > a.top ? a.top : a.last;
        return i < all && d < length ? ld_global(a.keys + (row0 * a.splits + l) * a.top + d) : 0;
    };
    // of rows that were not read they hold anything, and are not used
    uint64_t key[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) key[j] = key_at(j * kThreads + lane * kWaves + ((w + lane) % kWaves));
    if (tid == 0) list_end = 0;
    for (uint32_t b = w; b < a.beams; b += kWaves) {
        const f32x2* from = reinterpret_cast<const f32x2*>(a.part) + (row0 + b) * a.splits;
        const f32x2 none = {kLowest, 0.0f}, first = lane < a.splits ? ld_global(from + lane) : none;
        const float score = ld_global(a.scores + row0 + b);
        const bool over = a.finished && ld_global(a.finished + row0 + b) != 0;
        uint32_t kind = 0;
        double at = score;
        float m = first[0];
        if (fabsf(score) < kInf) {
            kind = 2;
            if (!over) {
                for (uint32_t i = lane + 64; i < a.splits; i += 64) m = fmaxf(m, ld_global(from + i)[0]);
                m = wave_max(m);
                // a split that had no logit above -inf has a sum of 0
                auto joined = [&](f32x2 o) {
                    return o[1] == 0.0f ? 0.0 : double(o[1]) * exp(a.scale * (double(o[0]) - double(m)));
                };
                double sum = joined(first);
                for (uint32_t i = lane + 64; i < a.splits; i += 64) sum += joined(ld_global(from + i));
#pragma unroll
                for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
                kind = sum > 0.0 && m < kInf ? 1 : 0;   // neither where it is NaN
                at = double(score) - log(sum);
            }
        }
        if (lane == 0) {
            beam_kind[b] = kind;
            beam_at[b] = at;
            beam_m[b] = m;
        }
    }
    __syncthreads();

    uint32_t count = 0;
    Candidate bound{-double(kInf), ~uint64_t(0)};   // the last of the kept ones
    for (uint32_t i0 = 0; i0 < all; i0 += kRound) {
        Candidate mine[3];
        float most = -kInf;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t i = i0 + j * kThreads + lane * kWaves + ((w + lane) % kWaves), l = i % lists, b = l / a.splits;
            if (i0) key[j] = key_at(i);
            mine[j].c = -double(kInf);
            if (key[j] && beam_kind[b] == 1)
                mine[j] = {beam_at[b] + a.scale * (double(value_of(key[j])) - double(beam_m[b])),
                           uint64_t(b) << 32 | id_of(key[j])};
            most = fmaxf(most, float(mine[j].c));
        }
        mine[2].c = -double(kInf);
        if (i0 == 0 && tid < a.beams && beam_kind[tid] == 2) mine[2] = {beam_at[tid], uint64_t(tid) << 32 | uint32_t(a.pad)};
        // the least of the waves' k-th largest, with k * waves >= keep (FP32 keeps the order)
        float reach = -kInf;
        if (i0 == 0) {
            const float kth = kth_of_wave(most, (a.keep + kWaves - 1) / kWaves);
            if (lane == 0) wave_bound[w] = kth;
            __syncthreads();
            reach = wave_bound[0];
#pragma unroll
            for (int j = 1; j < kWaves; ++j) reach = fminf(reach, wave_bound[j]);
        }
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            const Candidate& k = mine[j];
            const float c = float(k.c);   // what leaves: a value below FP32's range is -inf, and no candidate
            if (c == -kInf || c < reach || (count == a.keep && !ahead_of(k, bound))) continue;
            list[atomicAdd(&list_end, 1u)] = k;
        }
        __syncthreads();
        const uint32_t n = list_end;
        if (n == count && i0) break;
        // who is ahead of whom: as many threads to a candidate as there are (64 kept of 8 beams of
        // 8192 BF16, 64 prompts, about 130 candidates: 27.9 us for the call with one thread each, 18.2 so)
        auto rank = [&](auto threads) __attribute__((always_inline)) {
            constexpr uint32_t G = decltype(threads)::value;
            const uint32_t i = tid / G, part = tid % G;
            const Candidate mine = list[i < n ? i : 0];
            uint32_t ahead = 0;
            for (uint32_t j = part; j < n; j += 4 * G) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint32_t at = j + u * G;
                    ahead += at < n && ahead_of(list[at < n ? at : 0], mine);
                }
            }
            if (G >= 2) ahead += __builtin_amdgcn_update_dpp(0, ahead, 0xB1, 0xf, 0xf, true);    // quad_perm 1,0,3,2
            if (G >= 4) ahead += __builtin_amdgcn_update_dpp(0, ahead, 0x4E, 0xf, 0xf, true);    // quad_perm 2,3,0,1
            if (G >= 8) ahead += __builtin_amdgcn_update_dpp(0, ahead, 0x141, 0xf, 0xf, true);   // row_half_mirror
            __syncthreads();
            if (part == 0 && i < n && ahead < a.keep) list[ahead] = mine;
        };
        using std::integral_constant;
        if (n <= kThreads / 8) {
            rank(integral_constant<uint32_t, 8>{});
        } else if (n <= kThreads / 4) {
            rank(integral_constant<uint32_t, 4>{});
        } else if (n <= kThreads / 2) {
            rank(integral_constant<uint32_t, 2>{});
        } else {
            constexpr int kEach = (kList + kThreads - 1) / kThreads;
            Candidate k[kEach];
            uint32_t ahead[kEach] = {};
#pragma unroll
            for (int j = 0; j < kEach; ++j)
                if (tid + j * kThreads < n) k[j] = list[tid + j * kThreads];
            for (uint32_t i = 0; i < n; ++i) {
                const Candidate o = list[i];
#pragma unroll
                for (int j = 0; j < kEach; ++j) ahead[j] += ahead_of(o, k[j]);
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < kEach; ++j)
                if (tid + j * kThreads < n && ahead[j] < a.keep) list[ahead[j]] = k[j];
        }
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

template <class T>
hipError_t scan(const ScanArgs& a, const BeamSplits& splits, uint64_t rows, hipStream_t stream) {
    constexpr int kSmall = 16 / sizeof(T);
    const dim3 grid(a.splits * uint32_t(rows));
    if (splits.each == 16) hipLaunchKernelGGL((beam_scan_kernel<T, 16>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((beam_scan_kernel<T, kSmall>), grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
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
// Bytes: half of 64 rows' 8 MiB in place 92 us, 5.3 TB/s read and written.
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
    const BeamSplits splits = beam_splits(call.rows, call.vocab, call.logits.type);
    const uint32_t top = call.keep < call.vocab ? call.keep : call.vocab;
    auto* part = static_cast<float*>(call.workspace);
    auto* keys = reinterpret_cast<uint64_t*>(part + call.rows * splits.splits * 2);
    ScanArgs a{};
    a.logits = call.logits.data;
    a.stride = call.logits.stride;
    a.scores = call.scores;
    a.finished = call.finished;
    a.part = part;
    a.keys = keys;
    a.vocab = call.vocab;
    a.top = top;
    a.splits = splits.splits;
    a.split_length = splits.length;
    a.c = float(double(call.scale) * 1.4426950408889634074);
    JoinArgs j{};
    j.scores = call.scores;
    j.finished = call.finished;
    j.part = part;
    j.keys = keys;
    j.next_scores = call.next_scores;
    j.parents = call.parents;
    j.tokens = call.tokens;
    j.beams = call.beams;
    j.keep = call.keep;
    j.top = top;
    j.splits = splits.splits;
    j.last = call.vocab - (splits.splits - 1) * splits.length;
    j.pad = call.pad;
    j.scale = call.scale;
    // a launch holds fewer than 2^32 threads (rows in such numbers take one split)
    constexpr uint64_t kRows = 1u << 20;
    for (uint64_t left = call.rows; left;) {
        const uint64_t n = left < kRows ? left : kRows;
        hipError_t e = hipErrorInvalidValue;
        switch (call.logits.type) {
            case kF32: e = scan<float>(a, splits, n, stream); break;
            case kF16: e = scan<_Float16>(a, splits, n, stream); break;
            case kBF16: e = scan<__bf16>(a, splits, n, stream); break;
        }
        if (e != hipSuccess) return e;
        left -= n;
        a.logits = static_cast<const char*>(a.logits) + n * a.stride * (call.logits.type == kF32 ? 4 : 2);
        a.scores += n;
        if (a.finished) a.finished += n;
        a.part += n * splits.splits * 2;
        a.keys += n * splits.splits * top;
    }
    const uint64_t prompts = call.rows / call.beams;
    constexpr uint64_t kPrompts = 1u << 22;
    for (uint64_t p = 0; p < prompts; p += kPrompts) {
        const uint64_t n = prompts - p < kPrompts ? prompts - p : kPrompts;
        hipLaunchKernelGGL(beam_join_kernel, dim3(uint32_t(n)), dim3(kThreads), 0, stream, j);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        j.scores += n * j.beams;
        if (j.finished) j.finished += n * j.beams;
        j.part += n * j.beams * splits.splits * 2;
        j.keys += n * j.beams * splits.splits * top;
        j.next_scores += n * j.keep;
        j.parents += n * j.keep;
        j.tokens += n * j.keep;
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
