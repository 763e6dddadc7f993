// Dropout whose mask is a function of seed, step and place, so that nobody has to keep it: what the forward pass left out the backward
// pass finds out again.
//
// Bits come from Philox4x32 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) with seven rounds,
// the fewest that its authors report to pass BigCrush. One evaluation gives 128 bits, 16 for each of eight elements: a probability is a
// multiple of 2^-16.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cmath>

namespace vetrast
{
__device__ __forceinline__ uint32_t exclusive_or(uint32_t a, uint32_t b, uint32_t c)  // of three, in one instruction
{
    uint32_t x;
    asm("v_bitop3_b32 %0, %1, %2, %3 bitop3:0x96" : "=v"(x) : "v"(a), "v"(b), "v"(c));
    return x;
}

struct DropoutBits
{
    uint32_t key[2];             // the seed
    uint64_t step;
    const int64_t* device_step;  // added to the step, or null
    uint32_t threshold;          // an element whose 16 bits are below it is left out; 0: none is, 65536: all are
};

inline uint32_t dropout_threshold(double p) { return (uint32_t)std::floor(p * 65536.0 + 0.5); }
inline DropoutBits dropout_bits(double p, uint64_t seed, uint64_t step, const int64_t* device_step)
{
    return {{(uint32_t)seed, (uint32_t)(seed >> 32)}, step, device_step, dropout_threshold(p)};
}

__device__ __forceinline__ uint64_t dropout_step(const DropoutBits& d)
{
    return d.step + (d.device_step ? (uint64_t)*d.device_step : 0ull);
}

// The bits of elements 8 * block .. 8 * block + 7, two to a word.
__device__ __forceinline__ uint4 dropout_words(const DropoutBits& d, uint64_t step, uint64_t block)
{
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)step, c3 = (uint32_t)(step >> 32);
    uint32_t k0 = d.key[0], k1 = d.key[1];
#pragma unroll
    for (int r = 0; r < 7; ++r)
    {
        const uint64_t p = (uint64_t)c0 * 0xD2511F53u, q = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = exclusive_or((uint32_t)(q >> 32), c1, k0);
        c2 = exclusive_or((uint32_t)(p >> 32), c3, k1);
        c1 = (uint32_t)q, c3 = (uint32_t)p;
        k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// Whether element `at` is left out, for callers whose elements are no neighbours.
__device__ __forceinline__ bool dropped_out(const DropoutBits& d, uint64_t step, uint64_t at)
{
    const uint4 w         = dropout_words(d, step, at >> 3);
    const uint32_t pair   = (at & 4) ? ((at & 2) ? w.w : w.z) : ((at & 2) ? w.y : w.x);
    const uint32_t bits   = (at & 1) ? pair >> 16 : pair & 0xFFFFu;
    return bits < d.threshold;
}
}  // namespace vetrast
