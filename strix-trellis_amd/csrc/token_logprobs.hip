// Log probabilities behind the output head: for each row of logits the log
// probability and rank of a given token, the entropy, and the most likely
// tokens, in one pass over the logits.
//
// Running statistics.  With m the largest logit so far, c = scale, a thread
// holds n = the count of logits equal to m, and over the others
//   s = sum e^(c (x - m))      h = sum e^(c (x - m)) c (x - m)
// so that log sum = log n + log1p(s / n) and entropy = log sum - h / (n + s)
// keep their relative precision where one token takes nearly everything.  h is
// held in units of log2 e.  Logits of -inf add nothing: m starts at the
// lowest finite float.
//
// Most likely tokens.  A token's place in the order is one 64-bit key: the
// logit's bits, made monotonic, over the inverted id, so larger keys come
// first and equal logits go by the lower id.  The workgroup keeps a list of
// candidates in LDS and a bound that at least `top` keys reach; a token
// enters the list if it reaches the bound.  The first batch takes its bound
// from the threads' largest tokens (the k-th largest of each wave, with k * waves
// >= top), and whenever the list has grown it is cut to the first `top` keys,
// the last of which is the new bound.  Only a few dozen of 10^5 tokens ever
// enter.
#include "ops_device.hpp"

namespace stx {

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kEach = 16;                               // logits per thread and batch
constexpr uint32_t kBatch = kThreads * kEach;
static_assert(kBatch == kLogprobsBatch);
constexpr uint32_t kList = 1024;                        // candidate capacity, above the most `top`
constexpr uint32_t kCut = 256;                          // list length that is cut at the end of a batch
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLowest = -3.40282346638528859812e38f;

__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);   // -0 counts as 0
    return uint64_t(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | uint32_t(~id);
}
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t b = uint32_t(key >> 32);
    return __builtin_bit_cast(float, b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}
__device__ __forceinline__ uint32_t id_of(uint64_t key) { return ~uint32_t(key); }

struct Stats {
    float m, n, s, h;
};
constexpr Stats kNothing = {kLowest, 0.0f, 0.0f, 0.0f};

// c as a sum of two floats times log2 e: exponents of 2 without a rounding that
// grows with the distance.
struct Scale {
    float hi, lo;
};
// Distances past 2^24 have no weight at any admitted scale (2^24 times 2^-16
// log2 e is over 300); kept finite, a weight of 0 times one is 0.  NaN stays NaN.
__device__ __forceinline__ float power(float d, Scale c) {
    d = __builtin_elementwise_maximum(d, -0x1p24f);
    return __builtin_fmaf(d, c.hi, d * c.lo);
}

// Joins b into a.
__device__ __forceinline__ void join(Stats& a, const Stats& b, Scale c) {
    const float m = fmaxf(a.m, b.m);
    auto part = [&](const Stats& p) {
        Stats q = p;
        if (p.m == m) return q;
        const float d = power(p.m - m, c), f = exp2f(d), t = p.n + p.s;
        q.n = 0.0f;
        q.s = f * t;
        q.h = f * __builtin_fmaf(t, d, p.h);
        return q;
    };
    const Stats x = part(a), y = part(b);
    a = {m, x.n + y.n, x.s + y.s, x.h + y.h};
}

// What the statistics of a whole row say; invalid rows give NaN.
struct Answer {
    bool valid;
    float log_sum, entropy;   // log sum of e^(c (x - m))
};
__device__ __forceinline__ Answer answer_of(const Stats& t) {
    Answer a;
    a.valid = t.n > 0.0f && t.m < __builtin_inff() && t.s == t.s;
    a.log_sum = logf(t.n) + log1pf(t.s / t.n);
    a.entropy = a.log_sum - t.h * kLn2 / (t.n + t.s);
    return a;
}

struct Args {
    const void* logits;
    uint64_t stride;
    const int32_t* tokens;
    float* logprobs;
    int32_t* ranks;
    float* entropy;
    int32_t* top_ids;
    float* top_logprobs;
    uint32_t vocab, top, splits, split_length;
    float scale;
    Scale c;
    // splits > 1: per row and split the statistics and the tokens ahead
    // ([rows][splits][8] words), then the keys ([rows][splits][top]).
    float* part;
    uint64_t* part_keys;
};

// Sorts the first `top` of list[0..count) to its front (largest first) and
// returns how many there are.  All threads call it; ends with a barrier.
// Ranks by counting: every key is distinct.
__device__ __forceinline__ uint32_t cut(uint64_t* list, uint32_t count, uint32_t top) {
    constexpr int kMine = kList / kThreads;
    uint64_t mine[kMine];
    uint32_t ahead[kMine] = {};
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
        const uint32_t i = threadIdx.x + j * kThreads;
        mine[j] = i < count ? list[i] : 0;
    }
    if (threadIdx.x < count) {
        for (uint32_t i = 0; i < count; ++i) {
            const uint64_t k = list[i];
#pragma unroll
            for (int j = 0; j < kMine; ++j) ahead[j] += k > mine[j];
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMine; ++j)
        if (threadIdx.x + j * kThreads < count && ahead[j] < top) list[ahead[j]] = mine[j];
    __syncthreads();
    return count < top ? count : top;
}

// Writes the row's results from its statistics, the tokens ahead of the given
// one, and the sorted list of its first tokens.
template <class T>
__device__ __forceinline__ void finish(const Args& a, uint64_t row, const Stats& t, uint32_t ahead,
                                       const uint64_t* list) {
    const Answer r = answer_of(t);
    const float nan = __builtin_nanf("");
    auto log_p = [&](float x) { return a.scale * (x - t.m) - r.log_sum; };
    if (threadIdx.x == 0) {
        if (a.entropy) st_global(a.entropy + row, r.valid ? r.entropy : nan);
        if (a.tokens) {
            const int32_t id = ld_global(a.tokens + row);
            const bool fine = r.valid && uint32_t(id) < a.vocab;
            if (a.ranks) st_global(a.ranks + row, fine ? int32_t(ahead) : -1);
            if (a.logprobs) {
                const float x = fine ? float(ld_global(static_cast<const T*>(a.logits) + row * a.stride + id)) : 0.0f;
                st_global(a.logprobs + row, fine ? log_p(x) : nan);
            }
        }
    }
    for (uint32_t j = threadIdx.x; j < a.top; j += kThreads) {
        const uint64_t k = list[j];
        if (a.top_ids) st_global(a.top_ids + row * a.top + j, r.valid ? int32_t(id_of(k)) : -1);
        if (a.top_logprobs) st_global(a.top_logprobs + row * a.top + j, r.valid ? log_p(value_of(k)) : nan);
    }
}

template <class T>
__global__ __launch_bounds__(kThreads) void token_logprobs_kernel(Args a) {
    __shared__ uint64_t list[kList];
    __shared__ uint64_t wave_key[kWaves];
    __shared__ Stats wave_stats[kWaves];
    __shared__ uint32_t wave_ahead[kWaves];
    __shared__ uint32_t list_count;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const uint64_t row = blockIdx.x / a.splits;
    const uint32_t split = blockIdx.x % a.splits, v0 = split * a.split_length;
    const uint32_t v1 = a.vocab - v0 < a.split_length ? a.vocab : v0 + a.split_length;
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    int32_t token = a.tokens ? ld_global(a.tokens + row) : -1;
    const bool have_token = uint32_t(token) < a.vocab;
    const float given = have_token ? float(ld_global(x + token)) : __builtin_inff();
    Stats t = kNothing;
    uint32_t ahead = 0;
    uint64_t bound = 0;        // keys below it do not enter the list
    uint32_t count = 0;        // length of the list, the same in every thread
    if (tid == 0) list_count = 0;

    for (uint32_t b0 = v0; b0 < v1; b0 += kBatch) {
        // logits 4 j .. 4 j + 3 of the thread's four groups, 4 kThreads apart
        float v[kEach];
#pragma unroll
        for (int j = 0; j < kEach / 4; ++j) {
            float q[4];
            load_row<4>(x, b0 + (j * kThreads + tid) * 4, v1, -__builtin_inff(), q);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * j + i] = q[i];
        }
        auto id_at = [&](int e) { return b0 + ((e >> 2) * kThreads + tid) * 4 + (e & 3); };

        // ---- statistics ----
        float most = t.m;
#pragma unroll
        for (int e = 0; e < kEach; ++e) most = fmaxf(most, v[e]);
        if (most > t.m) {
            const float d = power(t.m - most, a.c), f = exp2f(d), all = t.n + t.s;
            t = {most, 0.0f, f * all, f * __builtin_fmaf(all, d, t.h)};
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const float d = power(v[e] - t.m, a.c);
            const float p = v[e] == t.m ? 0.0f : exp2f(d);
            t.n += v[e] == t.m ? 1.0f : 0.0f;
            t.s += p;
            t.h = __builtin_fmaf(p, d, t.h);
        }
        if (have_token) {
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                ahead += v[e] > given || (v[e] == given && id_at(e) < uint32_t(token));
        }
        if (!a.top) continue;

        // ---- candidates ----
        if (b0 == v0) {
            // The bound of the first batch: every wave's k-th largest thread
            // key, the least of them.  A thread without a token has key 0.
            uint64_t best = 0;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const uint64_t k = id_at(e) < v1 ? key_of(v[e], id_at(e)) : 0;
                best = k > best ? k : best;
            }
            const uint32_t kth = (a.top + kWaves - 1) / kWaves - 1;
            uint32_t before = 0;   // keys of the wave ahead of this one (equal zero keys: by lane)
            for (int l = 0; l < 64; ++l) {
                const uint64_t o = __shfl(best, l);
                before += o > best || (o == best && l < lane);
            }
            if (before == kth) wave_key[w] = best;
            __syncthreads();
            uint64_t least = wave_key[0];
#pragma unroll
            for (int i = 1; i < kWaves; ++i) least = wave_key[i] < least ? wave_key[i] : least;
            bound = least;
        }
        for (;;) {
            const float reach = bound ? value_of(bound) : -__builtin_inff();
            uint32_t enter = 0;
#pragma unroll
            for (int e = 0; e < kEach; ++e) enter |= uint32_t(v[e] >= reach) << e;
            if (enter) {
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    if (!(enter >> e & 1) || id_at(e) >= v1) continue;
                    const uint64_t k = key_of(v[e], id_at(e));
                    if (k < bound) continue;
                    const uint32_t slot = atomicAdd(&list_count, 1u);
                    if (slot < kList) list[slot] = k;
                }
            }
            __syncthreads();
            const uint32_t entered = list_count;
            __syncthreads();
            if (entered <= kList) {
                count = entered;
                break;
            }
            // More tokens than the list holds (many equal ones): the keys that
            // got in give a higher bound; the list goes back to the earlier
            // batches' keys, which all stay within the first `top` slots, and
            // the batch enters again.  Each time at least kList - top fewer do.
            uint64_t kept = tid < int(count) ? list[tid] : 0;   // count <= kCut < kThreads here
            __syncthreads();
            cut(list, kList, a.top);
            bound = list[a.top - 1];
            __syncthreads();
            if (tid < int(count)) list[tid] = kept;
            if (tid == 0) list_count = count;
            __syncthreads();
        }
        if (count > kCut && b0 + kBatch < v1) {
            count = cut(list, count, a.top);
            if (count == a.top) bound = list[a.top - 1];
            if (tid == 0) list_count = count;
            __syncthreads();
        }
    }

    // ---- the row's or the split's results ----
    // a +inf or NaN row: m is +inf or s NaN, whichever thread saw it
#pragma unroll
    for (int s = 32; s; s >>= 1) {
        const Stats o = {__shfl_xor(t.m, s), __shfl_xor(t.n, s), __shfl_xor(t.s, s), __shfl_xor(t.h, s)};
        join(t, o, a.c);
        ahead += __shfl_xor(ahead, s);
    }
    if (lane == 0) {
        wave_stats[w] = t;
        wave_ahead[w] = ahead;
    }
    __syncthreads();
    t = wave_stats[0];
    ahead = wave_ahead[0];
    for (int i = 1; i < kWaves; ++i) {
        join(t, wave_stats[i], a.c);
        ahead += wave_ahead[i];
    }
    if (a.top) count = cut(list, count, a.top);
    if (a.splits == 1) {
        finish<T>(a, row, t, ahead, list);
        return;
    }
    const uint64_t p = row * a.splits + split;
    if (tid == 0) {
        float* to = a.part + p * 8;
        st_global(to, t.m);
        st_global(to + 1, t.n);
        st_global(to + 2, t.s);
        st_global(to + 3, t.h);
        st_global(reinterpret_cast<uint32_t*>(to + 4), ahead);
    }
    // only the last split can be shorter than `top`: its keys end the row's
    if (uint32_t(tid) < count) st_global(a.part_keys + p * a.top + tid, list[tid]);
}

// Joins the splits of a row.
template <class T>
__global__ __launch_bounds__(kThreads) void token_logprobs_join_kernel(Args a) {
    __shared__ uint64_t list[kList];
    const uint64_t row = blockIdx.x, p = row * a.splits;
    Stats t = kNothing;
    uint32_t ahead = 0;
    for (uint32_t i = 0; i < a.splits; ++i) {
        const float* from = a.part + (p + i) * 8;
        const Stats o = {ld_global(from), ld_global(from + 1), ld_global(from + 2), ld_global(from + 3)};
        join(t, o, a.c);
        ahead += ld_global(reinterpret_cast<const uint32_t*>(from + 4));
    }
    if (a.top) {
        // the list in rounds, as many splits at a time as it holds
        uint32_t count = 0;
        const uint32_t last = a.vocab - (a.splits - 1) * a.split_length;
        const uint32_t keys = (a.splits - 1) * a.top + (last < a.top ? last : a.top);
        for (uint32_t i = 0; i < keys;) {
            const uint32_t n = keys - i < kList - count ? keys - i : kList - count;
            for (uint32_t j = threadIdx.x; j < n; j += kThreads) list[count + j] = ld_global(a.part_keys + p * a.top + i + j);
            __syncthreads();
            count = cut(list, count + n, a.top);
            i += n;
        }
    }
    finish<T>(a, row, t, ahead, list);
}

template <class T>
hipError_t dispatch(const Args& a, uint64_t rows, hipStream_t stream) {
    hipLaunchKernelGGL(token_logprobs_kernel<T>, dim3(a.splits * uint32_t(rows)), dim3(kThreads), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    hipLaunchKernelGGL(token_logprobs_join_kernel<T>, dim3(uint32_t(rows)), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_token_logprobs(const LogprobsCall& call, hipStream_t stream) {
    Args a{};
    a.logits = call.logits.data;
    a.stride = call.logits.stride;
    a.tokens = call.logprobs || call.ranks ? call.tokens : nullptr;
    a.logprobs = call.logprobs;
    a.ranks = call.ranks;
    a.entropy = call.entropy;
    a.top_ids = call.top_ids;
    a.top_logprobs = call.top_logprobs;
    a.vocab = call.vocab;
    a.top = call.top;
    a.scale = call.scale;
    const double c = double(call.scale) * 1.4426950408889634074;
    a.c.hi = float(c);
    a.c.lo = float(c - double(a.c.hi));
    const uint64_t batches = (uint64_t(call.vocab) + kBatch - 1) / kBatch;
    a.splits = logprobs_splits(call.rows, call.vocab);
    a.split_length = uint32_t((batches + a.splits - 1) / a.splits) * kBatch;
    a.part = static_cast<float*>(call.workspace);
    a.part_keys = reinterpret_cast<uint64_t*>(a.part + call.rows * a.splits * 8);
    // a launch holds fewer than 2^32 threads (more rows than that take one split)
    constexpr uint64_t kRows = 1u << 20;
    for (uint64_t left = call.rows; left;) {
        const uint64_t rows = left < kRows ? left : kRows;
        hipError_t e = hipErrorInvalidValue;
        switch (call.logits.type) {
            case kF32: e = dispatch<float>(a, rows, stream); break;
            case kF16: e = dispatch<_Float16>(a, rows, stream); break;
            case kBF16: e = dispatch<__bf16>(a, rows, stream); break;
        }
        if (e != hipSuccess) return e;
        left -= rows;
        a.logits = static_cast<const char*>(a.logits) + rows * a.stride * (call.logits.type == kF32 ? 4 : 2);
        auto step = [&](auto*& p, uint64_t each) {
            if (p) p += rows * each;
        };
        step(a.tokens, 1);
        step(a.logprobs, 1);
        step(a.ranks, 1);
        step(a.entropy, 1);
        step(a.top_ids, a.top);
        step(a.top_logprobs, a.top);
    }
    return hipSuccess;
}

}  // namespace stx
