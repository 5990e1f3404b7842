// Counter-based random bits of the dropout passes: Philox4x32 with 7 rounds (Salmon, Moraes,
// Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011, who find 7 rounds
// the fewest that pass all of BigCrush; a mask needs no margin beyond that).
//
// One call gives 128 bits, 16 for each of eight consecutive elements: element i of a tensor takes
// half i % 2 (low half first) of word (i % 8) / 2 at counter (i / 8, offset) under key `seed`,
// each a pair of 32-bit words, low word first. The element is kept where its 16 bits are below
// the threshold. Sixteen bits an element halve the multiplies of 32 (at 32 the pass would be
// bound by them, not by memory); they make p a multiple of 2^-16.
#pragma once

#include "common.h"

namespace dsalt {

struct DropoutParams {
    uint64_t seed, offset;
    const int64_t *seed_ptr;  // the seed on the device (NULL: `seed`)
    uint32_t threshold;       // kept where bits < threshold, 0 .. 65536
    float scale;              // 65536 / threshold, 0 for threshold 0
};

__device__ __forceinline__ uint64_t dropout_seed(const DropoutParams &p) {
    return p.seed_ptr ? (uint64_t)*p.seed_ptr : p.seed;
}

__device__ __forceinline__ uint4 philox7(uint64_t ctr, uint64_t offset, uint64_t seed) {
    uint32_t c0 = (uint32_t)ctr, c1 = (uint32_t)(ctr >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// Bit e set: element e of the eight is kept. LEAN: the round keys are formed anew on every call
// (scalar additions) instead of being held in 14 scalar registers across a caller's loop.
template <bool LEAN = false>
__device__ __forceinline__ uint32_t keep8(uint64_t group, const DropoutParams &p, uint64_t seed) {
    if constexpr (LEAN) {
        uint32_t lo = (uint32_t)seed, hi = (uint32_t)(seed >> 32);
        asm volatile("" : "+s"(lo), "+s"(hi));
        seed = ((uint64_t)hi << 32) | lo;
    }
    const uint4 r = philox7(group, p.offset, seed);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        m |= (w[e] & 0xffffu) < p.threshold ? 1u << (2 * e) : 0u;
        m |= (w[e] >> 16) < p.threshold ? 2u << (2 * e) : 0u;
    }
    return m;
}

// v * scale where kept, else 0, whatever a dropped element holds.
__device__ __forceinline__ void apply_keep(uint32_t m, float scale, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (m >> e) & 1u ? v[e] * scale : 0.f;
}

// Threshold, scale, seed and offset as an argument struct holds them.
inline DropoutParams dropout_params(int threshold, int64_t seed, const int64_t *seed_ptr, int64_t offset) {
    return {(uint64_t)seed, (uint64_t)offset, seed_ptr, (uint32_t)threshold,
            threshold ? (float)(65536.0 / threshold) : 0.f};
}

}  // namespace dsalt
