// What the kernels behind the output head share: a token's place in the order of
// its row as one key, logits in batches, and the sorted front of a list of keys.
#pragma once
#include "ops_device.hpp"

namespace stx {

namespace {

constexpr int kScanThreads = 512;
constexpr uint32_t kScanList = 1024;   // keys of a list in LDS
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
    if (count <= kScanThreads / 8) {   // eight threads to a key, eight keys each
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
    const uint32_t i0 = threadIdx.x, i1 = threadIdx.x + kScanThreads, padded = (count + 7) & ~7u;
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
            if (count > kScanThreads) {
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

// A thread's logits of a batch as loaded: groups of 16 bytes, the workgroup's
// groups side by side.
template <class T, int EACH>
struct Batch {
    static constexpr int kGroup = 16 / sizeof(T), kGroups = EACH / kGroup;
    static constexpr uint32_t kBatch = kScanThreads * EACH;
    typename Packed<T, kGroup>::type raw[kGroups];

    static __device__ __forceinline__ uint32_t first(int g) { return (g * kScanThreads + threadIdx.x) * kGroup; }
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
    __device__ __forceinline__ void values(uint32_t b0, uint32_t v1, float (&v)[EACH]) const {
#pragma unroll
        for (int e = 0; e < EACH; ++e) v[e] = float(raw[e / kGroup][e % kGroup]);
        if (b0 + kBatch > v1) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) v[e] = id(b0, v1, e) != ~0u ? v[e] : -kInf;
        }
    }
};

}  // namespace

}  // namespace stx
