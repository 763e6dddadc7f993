// Tables of tensors in a launch's arguments, and elements of tensors of float32, bfloat16 and float16, eight to a thread.
#pragma once
#include "common.h"

namespace vetrast
{
constexpr uint32_t kOptimChunk = 8 * kBlock;  // elements of a workgroup

// Tables hold up to 64 * GROUPS entries: lane k of a wave knows which chunk of the launch is the first of entries k, k + 64, ...
template <int GROUPS>
struct ChunkFinder
{
    uint32_t begins[GROUPS];
    template <class Launch>
    __device__ __forceinline__ explicit ChunkFinder(const Launch& a)
    {
#pragma unroll
        for (int q = 0; q < GROUPS; ++q)
        {
            const uint32_t k = q * kWave + threadIdx.x % kWave;
            begins[q]        = k < a.entries ? a.e[k].begins() : 0xFFFFFFFFu;
        }
    }
    // The entry of a chunk; all lanes of the wave take part.
    __device__ __forceinline__ uint32_t operator()(uint32_t chunk) const
    {
        uint32_t k = 0;
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) k += (uint32_t)__popcll(__ballot(begins[q] <= chunk));
        return k - 1u;
    }
};
constexpr int finder_groups(int entries) { return (entries + kWave - 1) / kWave; }

// As they lie in memory, 32 bytes or (16-bit types) 16. Loads of several arrays are under way before the first is looked at.
struct RawEight
{
    uint4 a, b;
};

// Loads and stores of many bytes at addresses that are multiples of an element's size only: the same instructions as at multiples of 16,
// a little slower where they straddle lines (parameter and gradient one element on: 10 M float32 53.4 us and 53.6, with 8-bit moments 27.7
// and 28.3; 16 M bf16 66.9 and 66.8, with 8-bit moments 27.9 and 32.2).
typedef uint32_t LooseFour __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t LooseTwo __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ uint4 load_four(const char* p)
{
    const LooseFour x = *(const LooseFour*)p;
    return make_uint4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ uint2 load_two(const char* p)
{
    const LooseTwo x = *(const LooseTwo*)p;
    return make_uint2(x[0], x[1]);
}
__device__ __forceinline__ void store_four(char* p, const uint4& x) { *(LooseFour*)p = (LooseFour){x.x, x.y, x.z, x.w}; }
__device__ __forceinline__ void store_two(char* p, uint32_t x, uint32_t y) { *(LooseTwo*)p = (LooseTwo){x, y}; }

// A thread's eight elements of a chunk that begins at element `start` of a tensor: the eight from 8 * threadIdx.x on, or (halves) the four
// from 4 * threadIdx.x on and the four HALF elements behind these, with which a wave's access to float32 has no gaps. Writes gain by
// that, in what the last-level cache holds: 10 M first and second moments written 24.9 us, in halves 18.8; a step of 4 M elements with
// masters 20.3 us, in halves 18.5. Beyond it a step does not (27.5 M float32: 142 us either way).
// Addresses are one scalar for the workgroup and 32 bits for the thread. Registers that a load does not fill are left alone: to clear
// them would wait for what is under way.
template <int BYTES, uint32_t HALF = 0>
__device__ __forceinline__ RawEight load_eight(const void* p, uint32_t start)
{
    const char* base = (const char*)p + (size_t)start * BYTES;
    RawEight r;
    if constexpr (HALF != 0)
    {
        constexpr uint32_t half = HALF * BYTES;
        const uint32_t here     = threadIdx.x * 4u * BYTES;
        if constexpr (BYTES == 4)
        {
            r.a = load_four(base + here);
            r.b = load_four(base + here + half);
        }
        else
        {
            const uint2 x = load_two(base + here), y = load_two(base + here + half);
            r.a = make_uint4(x.x, x.y, y.x, y.y);
        }
    }
    else
    {
        const uint32_t here = threadIdx.x * 8u * BYTES;
        r.a                 = load_four(base + here);
        if constexpr (BYTES == 4) r.b = load_four(base + here + 16);
    }
    return r;
}
template <int BYTES, uint32_t HALF = 0>
__device__ __forceinline__ void store_eight(void* p, uint32_t start, const RawEight& r)
{
    char* base = (char*)p + (size_t)start * BYTES;
    if constexpr (HALF != 0)
    {
        constexpr uint32_t half = HALF * BYTES;
        const uint32_t here     = threadIdx.x * 4u * BYTES;
        if constexpr (BYTES == 4)
        {
            store_four(base + here, r.a);
            store_four(base + here + half, r.b);
        }
        else
        {
            store_two(base + here, r.a.x, r.a.y);
            store_two(base + here + half, r.a.z, r.a.w);
        }
    }
    else
    {
        const uint32_t here = threadIdx.x * 8u * BYTES;
        store_four(base + here, r.a);
        if constexpr (BYTES == 4) store_four(base + here + 16, r.b);
    }
}

// The first `count` of them; the others read as zeros and are not written.
template <int BYTES>
__device__ __forceinline__ RawEight load_some(const void* p, uint32_t start, uint32_t count)
{
    RawEight r;
    r.a = r.b = make_uint4(0, 0, 0, 0);
    if (count)
    {
        const char* base    = (const char*)p + (size_t)start * BYTES;
        const uint32_t here = threadIdx.x * 8u * BYTES;
        uint32_t w[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
        {
            const char* x = base + here + min(j, count - 1) * BYTES;
            if constexpr (BYTES == 4) w[j] = *(const uint32_t*)x;
            else w[j] = *(const uint16_t*)x;
        }
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) w[j] = j < count ? w[j] : 0u;
        if constexpr (BYTES == 4)
        {
            r.a = make_uint4(w[0], w[1], w[2], w[3]);
            r.b = make_uint4(w[4], w[5], w[6], w[7]);
        }
        else r.a = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    }
    return r;
}
template <int BYTES>
__device__ __forceinline__ void store_some(void* p, uint32_t start, uint32_t count, const RawEight& r)
{
    char* base          = (char*)p + (size_t)start * BYTES;
    const uint32_t here = threadIdx.x * 8u * BYTES;
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j)
        if (j < count)
        {
            if constexpr (BYTES == 4) *(uint32_t*)(base + here + j * 4) = w[j];
            else *(uint16_t*)(base + here + j * 2) = (uint16_t)(w[j / 2] >> 16 * (j % 2));
        }
}

// Of a type known at run time, `whole` where all threads have their eight.
__device__ __forceinline__ RawEight load_any(const void* p, uint32_t type, uint32_t start, uint32_t count, bool whole)
{
    if (type == VETRAST_F32) return whole ? load_eight<4>(p, start) : load_some<4>(p, start, count);
    return whole ? load_eight<2>(p, start) : load_some<2>(p, start, count);
}
__device__ __forceinline__ void store_any(void* p, uint32_t type, uint32_t start, uint32_t count, bool whole, const RawEight& r)
{
    if (type == VETRAST_F32)
    {
        if (whole) store_eight<4>(p, start, r);
        else store_some<4>(p, start, count, r);
    }
    else if (whole) store_eight<2>(p, start, r);
    else store_some<2>(p, start, count, r);
}
__device__ __forceinline__ uint32_t count_of(uint32_t start, uint32_t n)
{
    const uint32_t i = start + threadIdx.x * 8u;
    return i < n ? min(n - i, 8u) : 0u;
}

__device__ __forceinline__ void to_floats(const RawEight& r, uint32_t type, float* x)
{
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    if (type == VETRAST_F32)
    {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(w[j]);
    }
    else if (type == VETRAST_BF16)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            x[2 * j]     = __uint_as_float(w[j] << 16);
            x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        }
    }
    else
    {
        typedef _Float16 Half2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            const Half2 h = __builtin_bit_cast(Half2, w[j]);
            x[2 * j]      = (float)h[0];
            x[2 * j + 1]  = (float)h[1];
        }
    }
}

// Rounded to nearest.
__device__ __forceinline__ RawEight from_floats(const float* x, uint32_t type)
{
    RawEight r;
    if (type == VETRAST_F32)
    {
        r.a = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
        r.b = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
        return r;
    }
    uint32_t w[4];
    if (type == VETRAST_BF16)
    {
        typedef __bf16 Pair __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __builtin_bit_cast(uint32_t, (Pair){(__bf16)x[2 * j], (__bf16)x[2 * j + 1]});
    }
    else
    {
        typedef _Float16 Pair __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __builtin_bit_cast(uint32_t, (Pair){(_Float16)x[2 * j], (_Float16)x[2 * j + 1]});
    }
    r.a = make_uint4(w[0], w[1], w[2], w[3]);
    return r;
}
}  // namespace vetrast
