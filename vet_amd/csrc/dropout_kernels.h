// Dropout whose mask is a function of seed, step and place, so that nobody has to keep it: what the forward pass left out the backward
// pass finds out again.
//
// Bits come from Philox4x32 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) with seven rounds,
// the fewest that its authors report to pass BigCrush. One evaluation gives 128 bits, 16 for each of eight elements: a probability is a
// multiple of 2^-16.
#pragma once
#include <cmath>

#include "common.h"
#include "elements.h"

namespace vetrast
{
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

struct DropoutPass
{
    const void* x;
    const void* residual;  // or null
    void* y;
    uint64_t n;
    uint64_t first_block;  // of eight elements
    float scale;
    DropoutBits bits;
};

// y = scale * x where x is kept, else 0, plus the residual: one rounding to the type. What is left out is not looked at, so that an
// infinity or a NaN there leaves nothing behind. A thread takes eight elements.
template <int TYPE, bool RESIDUAL>
__global__ void __launch_bounds__(kBlock) dropout_kernel(DropoutPass a)
{
    constexpr int kBytes = TYPE == VETRAST_F32 ? 4 : 2;
    const uint64_t start = (uint64_t)blockIdx.x * kOptimChunk;
    const char* x        = (const char*)a.x + start * kBytes;
    const char* residual = (const char*)a.residual + start * kBytes;
    char* y              = (char*)a.y + start * kBytes;
    const bool whole     = start + kOptimChunk <= a.n;
    const uint32_t left  = whole ? kOptimChunk : (uint32_t)(a.n - start), count = count_of(0, left);
    if (count == 0) return;
    const RawEight rx = load_any(x, TYPE, 0, count, whole);
    RawEight rr;
    if constexpr (RESIDUAL) rr = load_any(residual, TYPE, 0, count, whole);
    const uint4 words   = dropout_words(a.bits, dropout_step(a.bits), a.first_block + start / 8 + threadIdx.x);
    const uint32_t w[4] = {words.x, words.y, words.z, words.w};
    float v[8], r[8];
    to_floats(rx, TYPE, v);
    if constexpr (RESIDUAL) to_floats(rr, TYPE, r);
#pragma unroll
    for (int j = 0; j < 8; ++j)
    {
        const uint32_t bits = j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xFFFFu;
        v[j]                = bits < a.bits.threshold ? 0.f : v[j] * a.scale;
        if constexpr (RESIDUAL) v[j] += r[j];
    }
    store_any(y, TYPE, 0, count, whole, from_floats(v, TYPE));
}
}  // namespace vetrast
