// Log probabilities behind the output head: for each row of logits the log
// probability and rank of a given token, the entropy, and the most likely
// tokens, in one pass over the logits.
//
// Running statistics.  With m the largest logit so far, c = scale, a wave holds
// n = the count of logits equal to m, and over the others
//   s = sum e^(c (x - m))      h = sum e^(c (x - m)) c (x - m)
// so that log sum = log n + log1p(s / n) and entropy = log sum - h / (n + s)
// keep their relative precision where one token takes nearly everything.  h is
// held in units of log2 e.  Logits of -inf add nothing: m starts at the
// lowest finite float.  m is the wave's, so a batch whose largest logit stays
// below it (nearly all of them) needs neither a rescaling nor a count.
//
// Rank.  Tokens ahead of the given one are those of at least its logit before
// it and of more than its logit behind it: one comparison per logit, with a
// bound that changes once.
//
// Most likely tokens.  A token's place in the order is one 64-bit key: the
// logit's bits, made monotonic, over the inverted id, so larger keys come
// first and equal logits go by the lower id.  The workgroup keeps a list of
// candidates in LDS and a bound that at least `top` keys reach; a token
// enters the list if it reaches the bound.  The first batch takes its bound
// from the threads' largest logits (the k-th largest of each wave, with k * waves
// >= top).  Behind batches 1, 2, 4, 8, .. the list is cut to the first `top`
// keys, the last of which is the new bound: about `top` tokens enter between two
// cuts, and the waves meet only there.  A list that overflowed in between
// (rising or equal logits) is filled again from memory, with a higher bound.
//
// Many rows are bound by their bytes and by what a logit costs: 512 x 129280 F32
// 55.5 us with 8 tokens, rank and entropy, 4.8 TB/s; entropy alone 50 us, all with 20
// tokens 57; in BF16, half the bytes, 31 and 49 (an exponential and six other
// operations for each logit; the entropy's sum is always taken).  From 257 to 512 rows a
// row is one workgroup, 512 of which the chip holds at once, so 257 / 400 / 512 rows take
// 45 / 50 / 56 us and 513, with a second round, 78.  Few rows take two launches, up to 512
// workgroups of whole batches and a join: one row 12.8 us (the splits 8, the join 4; 6.9
// with the entropy alone), 33 rows of 100277 BF16, half masked, 13.7, with 98 % masked 21
// (few threads hold a finite logit, so there is no first bound and the list overflows).
// A last-arrival join in one launch would save the second launch, but needs a coherent
// round trip and counters that are zero at the start, which a caller's workspace is not;
// it was not built.
#include "ops_device.hpp"

namespace stx {

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kEach = 16;                               // logits per thread and batch
constexpr uint32_t kBatch = kThreads * kEach;
static_assert(kBatch == kLogprobsBatch);
constexpr uint32_t kList = 1024;                        // candidate capacity
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLowest = -3.40282346638528859812e38f, kInf = __builtin_inff();

__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);   // -0 counts as 0
    return uint64_t(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | uint32_t(~id);
}
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t b = uint32_t(key >> 32);
    return __builtin_bit_cast(float, b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}
__device__ __forceinline__ uint32_t id_of(uint64_t key) { return ~uint32_t(key); }

// The next float above x (x not NaN or +inf).
__device__ __forceinline__ float above(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return __builtin_bit_cast(float, b & 0x80000000u ? b - 1 : b + 1);
}

struct Stats {
    float m, n, s, h;
};
constexpr Stats kNothing = {kLowest, 0.0f, 0.0f, 0.0f};

// Distances past 2^24 have no weight at any admitted scale (2^24 times 2^-16
// log2 e is over 300); kept finite, a weight of 0 times one is 0.
__device__ __forceinline__ float power(float d, float c) { return fmaxf(d, -0x1p24f) * c; }

// Statistics p against the larger maximum m.
__device__ __forceinline__ Stats against(const Stats& p, float m, float c) {
    const float d = power(p.m - m, c), f = __builtin_amdgcn_exp2f(d), t = p.n + p.s;
    return p.m == m ? p : Stats{m, 0.0f, f * t, f * __builtin_fmaf(t, d, p.h)};
}
__device__ __forceinline__ void join(Stats& a, const Stats& b, float c) {
    const float m = fmaxf(a.m, b.m);
    const Stats x = against(a, m, c), y = against(b, m, c);
    a = {m, x.n + y.n, x.s + y.s, x.h + y.h};
}
// Joins the lanes' statistics; every lane gets the result.
__device__ __forceinline__ Stats join_lanes(const Stats& mine, float c) {
    const float m = wave_max(mine.m);
    const Stats x = against(mine, m, c);
    return {m, wave_sum(x.n), wave_sum(x.s), wave_sum(x.h)};
}

// What the statistics of a whole row say; invalid rows give NaN.
struct Answer {
    bool valid;
    float log_sum, entropy;   // log sum of e^(c (x - m))
};
__device__ __forceinline__ Answer answer_of(const Stats& t) {
    Answer a;
    a.valid = t.n > 0.0f && t.m < kInf && t.s == t.s;
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
    float scale, c;           // c = scale log2 e
    // splits > 1: per row and split the statistics and the tokens ahead
    // ([rows][splits][8] words), then the keys ([rows][splits][top]).
    float* part;
    uint64_t* part_keys;
};

// Sorts the first `top` of list[0..count) to its front (largest first) and
// returns how many there are.  All threads call it; ends with a barrier.
// Ranks by counting (every key is distinct).  Up to 64 keys, the usual cut of a
// few tokens, are spread over all threads and take one LDS round trip (512 x
// 129280 BF16, 20 tokens, 42.0 -> 40.1 us; 33 x 100277, 5 tokens, 12.7 -> 11.9: tokens and
// entropy of the same normal logits each time, from the last-level cache); more go a key
// or two to a thread, eight of the list in flight per step, and keys past the count are
// 0, which is ahead of none.
__device__ __forceinline__ uint32_t cut(uint64_t* list, uint32_t count, uint32_t top) {
    typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
    if (count <= kThreads / 8) {   // eight threads to a key, eight keys each
        const uint32_t i = threadIdx.x >> 3, part = threadIdx.x & 7;
        __syncthreads();
        const uint64_t mine = list[i];
        uint64_t k[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) k[j] = list[part + 8 * j];
        uint32_t ahead = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) ahead += part + 8 * j < count && k[j] > mine;
        ahead += __builtin_amdgcn_update_dpp(0, ahead, 0xB1, 0xf, 0xf, true);    // quad_perm 1,0,3,2
        ahead += __builtin_amdgcn_update_dpp(0, ahead, 0x4E, 0xf, 0xf, true);    // quad_perm 2,3,0,1
        ahead += __builtin_amdgcn_update_dpp(0, ahead, 0x141, 0xf, 0xf, true);   // row_half_mirror
        __syncthreads();
        if (part == 0 && i < count && ahead < top) list[ahead] = mine;
        __syncthreads();
        return count < top ? count : top;
    }
    const uint32_t i0 = threadIdx.x, i1 = threadIdx.x + kThreads, padded = (count + 7) & ~7u;
    if (count + i0 < padded) list[count + i0] = 0;
    __syncthreads();
    const uint64_t k0 = i0 < count ? list[i0] : 0, k1 = i1 < count ? list[i1] : 0;
    uint32_t a0 = 0, a1 = 0;
    if (uint32_t(__builtin_amdgcn_readfirstlane(i0)) < count) {   // the wave holds keys
        for (uint32_t i = 0; i < padded; i += 8) {
            u64x2 k[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const u64x2*>(list + i + 2 * j);
#pragma unroll
            for (int j = 0; j < 4; ++j) a0 += (k[j][0] > k0) + (k[j][1] > k0);
            if (count > kThreads) {
#pragma unroll
                for (int j = 0; j < 4; ++j) a1 += (k[j][0] > k1) + (k[j][1] > k1);
            }
        }
    }
    __syncthreads();
    if (i0 < count && a0 < top) list[a0] = k0;
    if (i1 < count && a1 < top) list[a1] = k1;
    __syncthreads();
    return count < top ? count : top;
}

// Writes the row's results from its statistics, the tokens ahead of the given
// one, and the sorted list of its first tokens.
__device__ __forceinline__ void finish(const Args& a, uint64_t row, const Stats& t, uint32_t token, float given,
                                       uint32_t ahead, const uint64_t* list) {
    const Answer r = answer_of(t);
    const float nan = __builtin_nanf("");
    // half the distance: finite logits may be farther apart than FP32 holds, and a
    // small scale brings that back into its range (the halves round nothing that counts)
    const float two = 2.0f * a.scale, half_m = 0.5f * t.m;
    auto log_p = [&](float x) { return two * __builtin_fmaf(0.5f, x, -half_m) - r.log_sum; };
    if (threadIdx.x == 0) {
        if (a.entropy) st_global(a.entropy + row, r.valid ? r.entropy : nan);
        const bool fine = r.valid && token < a.vocab;
        if (a.ranks) st_global(a.ranks + row, fine ? int32_t(ahead) : -1);
        if (a.logprobs) st_global(a.logprobs + row, fine ? log_p(given) : nan);
    }
    for (uint32_t j = threadIdx.x; j < a.top; j += kThreads) {
        const uint64_t k = list[j];
        if (a.top_ids) st_global(a.top_ids + row * a.top + j, r.valid ? int32_t(id_of(k)) : -1);
        if (a.top_logprobs) st_global(a.top_logprobs + row * a.top + j, r.valid ? log_p(value_of(k)) : nan);
    }
}

// A thread's logits of a batch as loaded: groups of 16 bytes, the workgroup's
// groups side by side.
template <class T>
struct Batch {
    static constexpr int kGroup = 16 / sizeof(T), kGroups = kEach / kGroup;
    typename Packed<T, kGroup>::type raw[kGroups];

    static __device__ __forceinline__ uint32_t first(int g) { return (g * kThreads + threadIdx.x) * kGroup; }
    // A group that would reach past v1 is loaded where it ends at v1: its first
    // logits are another group's, and drop out by `id`.
    static __device__ __forceinline__ uint32_t place(uint32_t b0, uint32_t v1, int g) {
        const uint32_t k = b0 + first(g);
        return k < v1 - kGroup ? k : v1 - kGroup;
    }
    __device__ __forceinline__ void load(const T* x, uint32_t b0, uint32_t v1) {
        if (b0 + kBatch <= v1) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) raw[g] = ld_packed<kGroup>(x + b0 + first(g));
        } else if (v1 >= uint32_t(kGroup)) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) raw[g] = ld_packed<kGroup>(x + place(b0, v1, g));
        } else {
#pragma unroll
            for (int i = 0; i < kGroup; ++i) raw[0][i] = uint32_t(i) < v1 ? ld_global(x + i) : T(-kInf);
        }
    }
    // Token of element e, ~0 where another element is that token or there is none.
    static __device__ __forceinline__ uint32_t id(uint32_t b0, uint32_t v1, int e) {
        const uint32_t k = b0 + first(e / kGroup);
        if (b0 + kBatch <= v1) return k + e % kGroup;
        if (v1 < uint32_t(kGroup)) return k + e % kGroup < v1 ? k + e % kGroup : ~0u;
        const uint32_t i = place(b0, v1, e / kGroup) + e % kGroup;
        return i >= k ? i : ~0u;
    }
    // The logits, -inf where `id` gives none.
    __device__ __forceinline__ void values(uint32_t b0, uint32_t v1, float (&v)[kEach]) const {
#pragma unroll
        for (int e = 0; e < kEach; ++e) v[e] = float(raw[e / kGroup][e % kGroup]);
        if (b0 + kBatch > v1) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) v[e] = id(b0, v1, e) != ~0u ? v[e] : -kInf;
        }
    }
};

template <class T>
__global__ __launch_bounds__(kThreads, 4) void token_logprobs_kernel(Args a) {
    __shared__ __align__(16) uint64_t list[kList];
    __shared__ float wave_bound[kWaves];
    __shared__ Stats wave_stats[kWaves];
    __shared__ uint32_t wave_ahead[kWaves];
    __shared__ uint32_t list_end;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint64_t row = blockIdx.x / a.splits;
    const uint32_t split = blockIdx.x % a.splits, v0 = split * a.split_length;
    const uint32_t v1 = a.vocab - v0 < a.split_length ? a.vocab : v0 + a.split_length;
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    using B = Batch<T>;
    const uint32_t token = a.tokens ? uint32_t(ld_global(a.tokens + row)) : ~0u;   // first: its logit's address
    B batch, next, later;   // two batches ahead: a round trip to memory takes longer than a batch
    batch.load(x, v0, v1);
    if (v0 + kBatch < v1) next.load(x, v0 + kBatch, v1);
    const float given = token < a.vocab ? float(ld_global(x + token)) : kInf;
    Stats t = kNothing;        // m is the wave's
    uint32_t ahead = 0;        // the wave's
    bool bad = false;          // a NaN
    uint64_t bound = 0;        // keys below it do not enter the list
    float reach = -kInf;       // its logit
    uint32_t count = 0;        // keys in the list behind the last cut
    float peak = -kInf;        // the thread's largest logit since then
    uint32_t since = v0, cut_at = v0;   // the first batch since then, the batch behind which the next cut comes
    if (tid == 0) list_end = 0;

    auto enter = [&](uint32_t b0, const float (&v)[kEach]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
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
        float left = peak, kth = -kInf;
        for (uint32_t k = (a.top + waves - 1) / waves; k; --k) {
            kth = wave_max(left);
            const uint64_t at = __ballot(left == kth);
            if (at && lane == __builtin_ctzll(at)) left = -kInf;
        }
        if (lane == 0) wave_bound[w] = uint32_t(w) < waves ? kth : kInf;
        __syncthreads();
        float least = wave_bound[0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) least = fminf(least, wave_bound[i]);
        __syncthreads();
        return least;
    };

    for (uint32_t b0 = v0; b0 < v1; b0 += kBatch) {
        if (v1 - b0 > 2 * kBatch) later.load(x, b0 + 2 * kBatch, v1);
        float v[kEach];
        batch.values(b0, v1, v);

        // ---- statistics ----
        float most = v[0];   // NaN if one is among them
#pragma unroll
        for (int e = 1; e < kEach; ++e) most = __builtin_elementwise_maximum(most, v[e]);
        bad |= most != most;
        const float wave_most = wave_max(most);
        if (wave_most >= t.m) {   // the wave as one
            t = against(t, wave_most, a.c);
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const float d = power(v[e] - t.m, a.c), p = v[e] == t.m ? 0.0f : __builtin_amdgcn_exp2f(d);
                t.n += v[e] == t.m ? 1.0f : 0.0f;
                t.s += p;
                t.h = __builtin_fmaf(p, d, t.h);
            }
        } else {
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const float d = power(v[e] - t.m, a.c), p = __builtin_amdgcn_exp2f(d);
                t.s += p;
                t.h = __builtin_fmaf(p, d, t.h);
            }
        }
        // ---- rank ----
        if (token < a.vocab) {
            if (token - b0 < kBatch) {
#pragma unroll
                for (int e = 0; e < kEach; ++e)
                    ahead += __popcll(__ballot(v[e] > given || (v[e] == given && B::id(b0, v1, e) < token)));
            } else {
                const float least = b0 < token ? given : above(given);
#pragma unroll
                for (int e = 0; e < kEach; ++e) ahead += __popcll(__ballot(v[e] >= least));
            }
        }
        // ---- candidates ----
        if (a.top) {
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
                        float u[kEach];
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
                    cut_at += cut_at - v0 + kBatch;   // behind batch 0, 1, 3, 7, ..
                    peak = -kInf;
                    __syncthreads();
                }
            }
        }
        batch = next;
        next = later;
    }

    // ---- the row's or the split's results ----
    if (bad) t.s = __builtin_nanf("");
    t.n = wave_sum(t.n);
    t.s = wave_sum(t.s);
    t.h = wave_sum(t.h);
    if (lane == 0) {
        wave_stats[w] = t;
        wave_ahead[w] = ahead;
    }
    __syncthreads();
    t = join_lanes(lane < kWaves ? wave_stats[lane & (kWaves - 1)] : kNothing, a.c);
    ahead = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) ahead += wave_ahead[i];
    if (a.splits == 1) {
        finish(a, row, t, token, given, ahead, list);
        return;
    }
    const uint64_t p = row * a.splits + split;
    if (tid == 0) {
        float* to = a.part + p * 8;
        st_global(reinterpret_cast<f32x4*>(to), f32x4{t.m, t.n, t.s, t.h});
        st_global(reinterpret_cast<uint32_t*>(to + 4), ahead);
    }
    // only the last split can be shorter than `top`: its keys end the row's
    if (uint32_t(tid) < count) st_global(a.part_keys + p * a.top + tid, list[tid]);
}

// Joins the splits of a row.
template <class T>
__global__ __launch_bounds__(kThreads) void token_logprobs_join_kernel(Args a) {
    __shared__ __align__(16) uint64_t list[kList];
    const uint64_t row = blockIdx.x, p = row * a.splits;
    __shared__ uint32_t list_end;
    const uint32_t tid = threadIdx.x, lane = tid & 63, last = a.vocab - (a.splits - 1) * a.split_length;
    const uint32_t keys = a.top ? (a.splits - 1) * a.top + (last < a.top ? last : a.top) : 0;
    const uint64_t* from = a.part_keys + p * a.top;
    if (tid == 0) list_end = 0;
    const uint32_t token = a.tokens ? uint32_t(ld_global(a.tokens + row)) : ~0u;
    // the thread's keys and the statistics on their way together
    constexpr int kMine = 2;
    uint64_t mine[kMine];
#pragma unroll
    for (int j = 0; j < kMine; ++j) mine[j] = tid + j * kThreads < keys ? ld_global(from + tid + j * kThreads) : 0;
    const float given =
        token < a.vocab ? float(ld_global(static_cast<const T*>(a.logits) + row * a.stride + token)) : 0.0f;
    // At least `top` keys reach the last key of any whole split, and the least of
    // the whole splits' k-th keys where k of each make `top`.
    uint64_t most_last = 0, least_kth = ~uint64_t(0);
    const uint32_t kth = a.top ? (a.top + a.splits - 2) / (a.splits - 1) - 1 : 0;
    Stats t = kNothing;
    float ahead = 0;   // whole numbers of a row's tokens: two halves, each exact in a float sum
    float ahead_high = 0;
    for (uint32_t i = lane; i < a.splits; i += 64) {
        const f32x4 o = ld_global(reinterpret_cast<const f32x4*>(a.part + (p + i) * 8));
        const uint32_t n = ld_global(reinterpret_cast<const uint32_t*>(a.part + (p + i) * 8 + 4));
        if (a.top && i + 1 < a.splits) {
            const uint64_t u = ld_global(from + i * a.top + a.top - 1), v = ld_global(from + i * a.top + kth);
            most_last = u > most_last ? u : most_last;
            least_kth = v < least_kth ? v : least_kth;
        }
        join(t, {o[0], o[1], o[2], o[3]}, a.c);
        ahead += float(n & 0x3FFFu);
        ahead_high += float(n >> 14);
    }
    t = join_lanes(t, a.c);
    const uint32_t total = uint32_t(wave_sum(ahead)) + (uint32_t(wave_sum(ahead_high)) << 14);
    if (a.top) {
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            const uint64_t u = __shfl_xor(most_last, o), v = __shfl_xor(least_kth, o);
            most_last = u > most_last ? u : most_last;
            least_kth = v < least_kth ? v : least_kth;
        }
        const uint64_t bound = most_last > least_kth ? most_last : least_kth;
        __syncthreads();
        auto enter = [&](uint64_t k) {
            if (k < bound) return;
            const uint32_t slot = atomicAdd(&list_end, 1u);
            if (slot < kList) list[slot] = k;
        };
#pragma unroll
        for (int j = 0; j < kMine; ++j)
            if (tid + j * kThreads < keys) enter(mine[j]);
        for (uint32_t i = tid + kMine * kThreads; i < keys; i += kThreads) enter(ld_global(from + i));
        __syncthreads();
        uint32_t count = list_end, taken = keys;
        if (count > kList) {   // the list in rounds, as many keys at a time as it holds
            __syncthreads();
            count = taken = kList;
            for (uint32_t i = tid; i < kList; i += kThreads) list[i] = ld_global(from + i);
            __syncthreads();
        }
        count = cut(list, count, a.top);
        while (taken < keys) {
            const uint32_t n = keys - taken < kList - count ? keys - taken : kList - count;
            for (uint32_t i = tid; i < n; i += kThreads) list[count + i] = ld_global(from + taken + i);
            __syncthreads();
            count = cut(list, count + n, a.top);
            taken += n;
        }
    }
    finish(a, row, t, token, given, total, list);
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
    a.c = float(double(call.scale) * 1.4426950408889634074);
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
