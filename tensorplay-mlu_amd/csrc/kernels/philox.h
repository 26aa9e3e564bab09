// The counter-based generator of Salmon, Moraes, Dror and Shaw, "Parallel
// random numbers: as easy as 1, 2, 3" (SC 2011): ten rounds of two 32 x 32
// -> 64-bit multiplies on a 4-word counter under a 2-word key bumped by the
// Weyl constants after each round.  Element e of a tensor takes word e % 4
// of the block for counter (low word of e / 4, its high word, offset_lo,
// offset_hi) under the key (seed_lo, seed_hi); its uniform is (word >> 8) * 2^-24
// in [0, 1), and it is kept when the uniform is >= p, decided exactly as
// word >> 8 >= ceil(p 2^24).
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

namespace tp_amd {

struct Philox {
    uint32_t c[4];
};

// a ^ b ^ c in one instruction (the truth table of three bits' sum).
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }

__device__ __forceinline__ Philox philox4x32_10(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3,
                                                uint32_t k0, uint32_t k1) {
    constexpr uint32_t M0 = 0xD2511F53u, M1 = 0xCD9E8D57u, W0 = 0x9E3779B9u, W1 = 0xBB67AE85u;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = static_cast<uint64_t>(M0) * c0;
        const uint64_t p1 = static_cast<uint64_t>(M1) * c2;
        const uint32_t hi0 = static_cast<uint32_t>(p0 >> 32), lo0 = static_cast<uint32_t>(p0);
        const uint32_t hi1 = static_cast<uint32_t>(p1 >> 32), lo1 = static_cast<uint32_t>(p1);
        const uint32_t n0 = xor3(hi1, c1, k0), n1 = lo1, n2 = xor3(hi0, c3, k1), n3 = lo0;
        c0 = n0;
        c1 = n1;
        c2 = n2;
        c3 = n3;
        k0 += W0;
        k1 += W1;
    }
    return Philox{{c0, c1, c2, c3}};
}

// What a kernel draws its keep bits with.
struct DropArgs {
    uint64_t seed;
    const int64_t* seed_at;  // device memory that holds the seed instead, or null
    uint64_t offset;
    uint32_t threshold;  // ceil(p 2^24): at most 2^24, which keeps nothing
    float scale;         // 1 / (1 - p)
};

// p 2^24 is exact in double; a 24-bit uniform u 2^-24 is >= p exactly when
// u >= ceil(p 2^24).
inline uint32_t keep_threshold(double p) { return static_cast<uint32_t>(std::ceil(std::ldexp(p, 24))); }

struct DropKey {
    uint32_t k0, k1, off0, off1;
    uint32_t least;  // of a word that is kept: threshold 2^8
    uint32_t any;    // bits of elements that can be kept: none where the threshold is 2^24
    __device__ __forceinline__ explicit DropKey(const DropArgs& a) {
        const uint64_t s = a.seed_at != nullptr ? static_cast<uint64_t>(*a.seed_at) : a.seed;
        k0 = static_cast<uint32_t>(s);
        k1 = static_cast<uint32_t>(s >> 32);
        off0 = static_cast<uint32_t>(a.offset);
        off1 = static_cast<uint32_t>(a.offset >> 32);
        least = a.threshold << 8;
        any = a.threshold >> 24 ? 0u : ~0u;
    }
};

// Bit j of the result: is element 4 (high 2^32 + low) + j kept, for NB blocks.
// (word >> 8 >= threshold is word >= threshold 2^8, the word's low bits being
// the threshold's zeros.)  `high` is best a scalar: two of the first rounds'
// products are then the same for a wave.
template <int NB>
__device__ __forceinline__ uint32_t keep_blocks(const DropKey& d, uint32_t low, uint32_t high) {
    uint32_t bits = 0;
#pragma unroll
    for (int b = NB - 1; b >= 0; --b) {
        const Philox r = philox4x32_10(low + b, high, d.off0, d.off1, d.k0, d.k1);
#pragma unroll
        for (int j = 3; j >= 0; --j) bits = bits + bits + (r.c[j] >= d.least ? 1u : 0u);
    }
    return bits & d.any;
}

// Bit j: is element first + j kept, for N elements that start anywhere; LOW:
// all blocks' numbers lie below 2^32.
template <int N, bool LOW>
__device__ __forceinline__ uint32_t keep_bits_at(const DropKey& d, uint64_t first) {
    constexpr int NB = (N + 3) / 4;
    const uint32_t phase = static_cast<uint32_t>(first) & 3u;
    const uint64_t block = first >> 2;
    if constexpr (LOW) {
        const uint32_t low = static_cast<uint32_t>(block);
        if (N == 1) return keep_blocks<1>(d, low, 0) >> phase;
        if (phase == 0) return keep_blocks<NB>(d, low, 0);
        return keep_blocks<NB + 1>(d, low, 0) >> phase;
    } else {
        // block by block: their numbers may pass 2^32 between two of them
        uint32_t bits = 0;
        for (int b = 0; b <= (N == 1 ? 0 : NB); ++b) {
            bits |= keep_blocks<1>(d, static_cast<uint32_t>(block + b), static_cast<uint32_t>((block + b) >> 32)) << (4 * b);
        }
        return bits >> phase;
    }
}

// v where bit j of `keep` is set, else 0.
__device__ __forceinline__ float kept(float v, uint32_t keep, int j) {
    return __uint_as_float(__float_as_uint(v) & static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(keep), j, 1)));
}

}  // namespace tp_amd
