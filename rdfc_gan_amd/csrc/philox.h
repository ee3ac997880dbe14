// philox.h -- the counter-based generator behind dropout: Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011).  A mask is a pure function of (seed, offset, element), so a backward pass draws the forward's mask again
// instead of reading it: nothing is stored.
//
// Element e of a map (its index in the dense [N][H][W][C] order, whatever the strides) takes the 16-bit half e % 8 of the four words of
// counter (e / 8, offset).  16 bits, not 32: eight elements -- one 16-byte vector of a 16-bit map -- per call, and the twenty wide
// multiplications of a call are what bounds a dropout pass once the map streams.  The price is that the drop probability is
// a multiple of 2^-16; the survivors are scaled by 1 / (1 - T / 65536), the probability that is really drawn, so the mean is exact.
#pragma once
#include "common.h"

// host side of a dropout: T of 65536 elements are dropped
struct DropArgs {
    unsigned threshold;              // drop where word16 < threshold (0: nothing is dropped, 65536: everything)
    float inv;                       // 1 / (1 - threshold / 65536)
    unsigned long long seed, offset;
    const unsigned long long *key;   // device memory {seed, offset}, read in place of the two above; NULL: none
};
static inline bool drop_args(DropArgs &d, int threshold, uint64_t seed, uint64_t offset, const uint64_t *key) {
    d.threshold = (unsigned)threshold;
    d.inv = threshold >= 65536 ? 0.f : (float)(1.0 / (1.0 - threshold / 65536.0));
    d.seed = seed;
    d.offset = offset;
    d.key = reinterpret_cast<const unsigned long long *>(key);
    return threshold >= 0 && threshold <= 65536;
}

__device__ __forceinline__ void philox_round(unsigned (&c)[4], unsigned k0, unsigned k1) {
    const unsigned long long a = (unsigned long long)c[0] * 0xD2511F53u, b = (unsigned long long)c[2] * 0xCD9E8D57u;
    c[0] = (unsigned)(b >> 32) ^ c[1] ^ k0;
    c[1] = (unsigned)b;
    c[2] = (unsigned)(a >> 32) ^ c[3] ^ k1;
    c[3] = (unsigned)a;
}
// the four words of counter (q, offset)
__device__ __forceinline__ u32x4 philox(unsigned long long q, unsigned long long seed, unsigned long long offset) {
    unsigned c[4] = {(unsigned)q, (unsigned)(q >> 32), (unsigned)offset, (unsigned)(offset >> 32)};
    unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        philox_round(c, k0, k1);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u32x4{c[0], c[1], c[2], c[3]};
}
__device__ __forceinline__ unsigned word16(const u32x4 &w, int i) { return i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu; }

// bit i of the result: element e0 + i is kept (i = 0 .. 7).  WHOLE: e0 is a multiple of 8; else two calls where it is not
template <bool WHOLE = false> __device__ __forceinline__ unsigned keep8(unsigned long long e0, unsigned threshold, unsigned long long seed, unsigned long long offset) {
    auto bits = [&](unsigned long long q) {
        const u32x4 w = philox(q, seed, offset);
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m |= (word16(w, i) >= threshold ? 1u : 0u) << i;
        return m;
    };
    unsigned m = bits(e0 >> 3);
    if constexpr (!WHOLE) {
        const int s = (int)(e0 & 7);
        if (s) m = (m | bits((e0 >> 3) + 1) << 8) >> s;
    }
    return m;
}
