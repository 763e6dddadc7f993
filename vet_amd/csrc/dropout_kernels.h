// Dropout over a tensor's elements (dropout_bits.h has where the mask comes from).
#pragma once
#include "common.h"
#include "elements.h"

namespace vetrast
{
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
// infinity or a NaN there leaves nothing behind.
//
// A thread takes the eight elements of one evaluation of the generator, one load of 16 bytes for types of 16 bits; the evaluation lies
// between the loads and the first use of what they bring. Memory bounds it: 66 M float16 with a residual take 69 us, 5.8 TB/s, 16.8 M bf16 18
// with a residual and 13.4 without. Below about 1 M elements a call is its launch, 4 us.
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
