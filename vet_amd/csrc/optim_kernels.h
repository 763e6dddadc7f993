// Optimiser kernels over lists of tensors: AdamW with moments in 32 or 8 bits, the norm of all gradients, moments to 8 bits and back.
#pragma once
#include "common.h"

namespace vetrast
{
constexpr uint32_t kOptimChunk   = 8 * kBlock;  // elements a workgroup takes at a time: 8 a thread
constexpr int kAdamWEntries      = 60;          // tensors of one launch: what 4 KB of kernel arguments hold
constexpr int kAdamWGroups       = 8;           // ... and of how many groups
constexpr int kNormEntries       = 160;
constexpr int kMomentEntries     = 80;
constexpr int kMomentBlock       = VETRAST_MOMENT_BLOCK;
constexpr uint32_t kMomentMargin = 0x100100;    // see code_base
static_assert(kOptimChunk % kMomentBlock == 0 && kMomentBlock == 16 * 8, "16 lanes of 8 elements hold a block");

enum { kAligned = 1u << 6, kHasCopy = 1u << 7 };  // bits of AdamWEntry::types, above param | grad << 2 | copy << 4; group << 8

struct AdamWEntry
{
    void* param;
    void* grad;
    void* copy;
    void* m;
    void* v;
    uint8_t* scale;
    uint32_t n;
    uint32_t first;  // chunk of the launch that is this entry's first
    uint32_t types;
    uint32_t pair;   // number of the entry's first pair of elements in the stream of random bits
};

struct AdamWGroup
{
    float step_size;     // lr / (1 - beta1^step)
    float keep;          // 1 - lr * weight_decay
    float inv_sqrt_bc2;  // 1 / sqrt(1 - beta2^step)
    uint32_t key;        // of this step's random bits
};

struct AdamWDevice  // vetrast_adamw_device_state and what adamw_begin_kernel leaves for the step's launches
{
    vetrast_adamw_device_state state;
    AdamWGroup group[1];
};

struct AdamWLaunch
{
    AdamWEntry e[kAdamWEntries];
    AdamWGroup g[kAdamWGroups];
    const float* grad_scale;
    const AdamWDevice* device;  // where set, g[].key are places in device->group
    uint32_t entries, chunks;
    float beta1, one_minus_beta1, beta2, one_minus_beta2, eps;
    int zero_grad, stochastic;
};
static_assert(sizeof(AdamWLaunch) <= 4096, "kernel arguments");

// A step's key of the random bits: two rounds of a 64-bit mixing function (the finalizer of splitmix64) over seed and step.
__host__ __device__ inline uint64_t mix64(uint64_t z)
{
    z += 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}
__host__ __device__ inline uint32_t step_key(uint64_t seed, int64_t step)
{
    return (uint32_t)mix64(mix64(seed) + (uint64_t)step);
}

// 32 random bits for a pair of elements. The lower 20 are the first element's, the upper 20 the second's.
__device__ __forceinline__ uint32_t pair_bits(uint32_t pair, uint32_t key)
{
    uint32_t x = pair * 0x9E3779B1u;
    x ^= x >> 15;
    x ^= key;
    x *= 0xBB67AE85u;
    x ^= x >> 15;
    x *= 0xA54FF53Bu;
    return x ^ (x >> 15);
}

// The largest of 16 lanes' values, in all of them (a row of a wave).
__device__ __forceinline__ uint32_t row_max(uint32_t v)
{
    v = max(v, dpp_move<0x128>(v));  // row_ror:8
    v = max(v, dpp_move<0x124>(v));
    v = max(v, dpp_move<0x122>(v));
    return max(v, dpp_move<0x121>(v));
}

// Scale byte D of a block whose largest magnitude has the float bits `largest`: its exponent less the binades that codes span, one
// more where rounding may carry (bits + 2^20 - 1 from rounding, and 2^8 from the offset 2^(D-127) at 15 binades). 255: not finite, or
// so large that a code next to it would be infinite.
template <int BINADES>
__device__ __forceinline__ uint32_t code_base(uint32_t largest)
{
    const int exponent = (int)((largest + kMomentMargin) >> 23);
    return exponent >= 255 ? 255u : (uint32_t)max(exponent - BINADES, 1);
}

// Code of magnitude x, `r` in [0, 2^20): x + 2^(D-127) is a float whose bits less those of 2^(D-127) are the code, 20 bits below it
// decide between it and the next. Evenly spaced values between two codes, so random r leaves the mean as it is.
__device__ __forceinline__ uint32_t magnitude_code(float x, uint32_t base_bits, uint32_t r)
{
    return (__float_as_uint(x + __uint_as_float(base_bits)) + r - base_bits) >> 20;
}
__device__ __forceinline__ float code_value(uint32_t code, uint32_t base_bits)
{
    return __uint_as_float((code << 20) + base_bits) - __uint_as_float(base_bits);
}

// Eight codes of both moments as two pairs of words, from the values and their random bits.
__device__ __forceinline__ void encode_moments(const float* m, const float* v, const uint32_t* rm, const uint32_t* rv, uint2& mc, uint2& vc, uint32_t& scale)
{
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
    {
        top_m = max(top_m, __float_as_uint(m[j]) & 0x7FFFFFFFu);
        top_v = max(top_v, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    }
    const uint32_t dm = code_base<15>(row_max(top_m)), dv = code_base<31>(row_max(top_v));
    const uint32_t bm = dm << 23, bv = dv << 23;
    uint32_t a[2] = {0, 0}, b[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
    {
        const uint32_t bits = __float_as_uint(m[j]);
        const uint32_t cm   = magnitude_code(fabsf(m[j]), bm, rm[j]) | ((bits >> 31) << 7);
        const uint32_t cv   = max(magnitude_code(v[j], bv, rv[j]), min(__float_as_uint(v[j]), 1u));
        a[j / 4] |= cm << (8 * (j % 4));
        b[j / 4] |= cv << (8 * (j % 4));
    }
    mc    = dm == 255 ? make_uint2(0, 0) : make_uint2(a[0], a[1]);  // code 0 at D = 255: infinity less infinity
    vc    = dv == 255 ? make_uint2(0, 0) : make_uint2(b[0], b[1]);
    scale = dm | (dv << 8);
}

__device__ __forceinline__ void decode_moments(uint2 mc, uint2 vc, uint32_t scale, float* m, float* v)
{
    const uint32_t bm = (scale & 255u) << 23, bv = ((scale >> 8) & 255u) << 23;
#pragma unroll
    for (int j = 0; j < 8; ++j)
    {
        const uint32_t wm = j < 4 ? mc.x : mc.y, wv = j < 4 ? vc.x : vc.y;
        const uint32_t cm = (wm >> (8 * (j % 4))) & 255u, cv = (wv >> (8 * (j % 4))) & 255u;
        m[j] = copysignf(code_value(cm & 127u, bm), __uint_as_float(cm << 24));
        v[j] = code_value(cv, bv);
    }
}

// Elements of the three types as floats and back, eight at a time or one.
template <int T>
struct Element;
template <>
struct Element<VETRAST_F32>
{
    using type = float;
    static __device__ __forceinline__ float get(float x) { return x; }
    static __device__ __forceinline__ float put(float x) { return x; }
};
template <>
struct Element<VETRAST_BF16>
{
    using type = __bf16;
    static __device__ __forceinline__ float get(__bf16 x) { return (float)x; }
    static __device__ __forceinline__ __bf16 put(float x) { return (__bf16)x; }
};
template <>
struct Element<VETRAST_F16>
{
    using type = _Float16;
    static __device__ __forceinline__ float get(_Float16 x) { return (float)x; }
    static __device__ __forceinline__ _Float16 put(float x) { return (_Float16)x; }
};

// `count` of the 8 elements from p + i on (the others read as zero); `whole`: all eight, and 16-byte aligned.
template <int T>
__device__ __forceinline__ void load_eight(const void* p_, uint32_t i, uint32_t count, bool whole, float* x)
{
    using E    = typename Element<T>::type;
    const E* p = (const E*)p_ + i;
    if (whole)
    {
        typedef E Vec __attribute__((ext_vector_type(16 / sizeof(E))));
        constexpr int W = 16 / sizeof(E);
#pragma unroll
        for (int q = 0; q < 8 / W; ++q)
        {
            const Vec w = ((const Vec*)p)[q];
#pragma unroll
            for (int j = 0; j < W; ++j) x[q * W + j] = Element<T>::get(w[j]);
        }
    }
    else
    {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) x[j] = j < count ? Element<T>::get(p[j]) : 0.f;
    }
}

template <int T>
__device__ __forceinline__ void store_eight(void* p_, uint32_t i, uint32_t count, bool whole, const float* x)
{
    using E = typename Element<T>::type;
    E* p    = (E*)p_ + i;
    if (whole)
    {
        typedef E Vec __attribute__((ext_vector_type(16 / sizeof(E))));
        constexpr int W = 16 / sizeof(E);
#pragma unroll
        for (int q = 0; q < 8 / W; ++q)
        {
            Vec w;
#pragma unroll
            for (int j = 0; j < W; ++j) w[j] = Element<T>::put(x[q * W + j]);
            ((Vec*)p)[q] = w;
        }
    }
    else
    {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            if (j < count) p[j] = Element<T>::put(x[j]);
    }
}

// Step count, learning rates and keys of a step whose count lies on the device; one thread a group.
struct AdamWBeginGroup
{
    double lr, weight_decay;
};
constexpr int kBeginGroups = 128;
struct AdamWBegin
{
    AdamWBeginGroup g[kBeginGroups];
    AdamWDevice* device;
    const float* grad_scale;
    double beta1, beta2;
    uint64_t seed;
    int first, groups, last;
};

// The groups' constants of step `state.step + 1`, or of the step before where gradients overflowed (nothing is read of them then). The
// launch with the last groups writes the new count; each launch reads the old one, so it is a kernel of one workgroup that waits in
// between.
__global__ void __launch_bounds__(kBeginGroups) adamw_begin_kernel(const AdamWBegin a)
{
    const bool counts  = !a.grad_scale || isfinite(*a.grad_scale);
    const int64_t step = a.device->state.step + 1;
    const float factor = a.device->state.lr_factor;
    __syncthreads();
    const int k = (int)threadIdx.x;
    if (k < a.groups)
    {
        const double lr  = a.g[k].lr * (double)factor;
        const double bc1 = 1.0 - pow(a.beta1, (double)step), bc2 = 1.0 - pow(a.beta2, (double)step);
        AdamWGroup g;
        g.step_size    = (float)(lr / bc1);
        g.keep         = (float)(1.0 - lr * a.g[k].weight_decay);
        g.inv_sqrt_bc2 = (float)(1.0 / sqrt(bc2));
        g.key          = step_key(a.seed, step);
        a.device->group[a.first + k] = g;
    }
    if (a.last && counts && k == 0) a.device->state.step = step;
}

template <int BITS, int P, int G>
__device__ __forceinline__ void adamw_eight(const AdamWLaunch& a, const AdamWEntry& e, const AdamWGroup& g, float grad_scale, bool leave, uint32_t i)
{
    const uint32_t n     = e.n;
    const uint32_t count = i < n ? min(n - i, 8u) : 0u;
    const bool whole     = count == 8u && (e.types & kAligned);
    const bool codes     = i < (n + kMomentBlock - 1) / kMomentBlock * kMomentBlock;
    float gr[8], p[8], m[8], v[8];
    if (leave)
    {
        const float zero[8] = {};
        if (a.zero_grad) store_eight<G>(e.grad, i, count, whole, zero);
        return;
    }
    load_eight<G>(e.grad, i, count, whole, gr);
    load_eight<P>(e.param, i, count, whole, p);
    if constexpr (BITS == 32)
    {
        load_eight<VETRAST_F32>(e.m, i, count, whole, m);
        load_eight<VETRAST_F32>(e.v, i, count, whole, v);
    }
    else
    {
        uint2 mc = make_uint2(0, 0), vc = make_uint2(0, 0);
        uint32_t scale = 0;
        if (codes)
        {
            mc    = *(const uint2*)((const uint8_t*)e.m + i);
            vc    = *(const uint2*)((const uint8_t*)e.v + i);
            scale = ((const uint16_t*)e.scale)[i / kMomentBlock];
        }
        decode_moments(mc, vc, scale, m, v);
    }
    uint32_t rm[8];
    if (BITS == 8 || (P == VETRAST_BF16 && a.stochastic))
    {
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            const uint32_t r = pair_bits(e.pair + i / 2 + j, g.key);
            rm[2 * j]        = r & 0xFFFFFu;
            rm[2 * j + 1]    = r >> 12;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
    {
        const float x = gr[j] * grad_scale;
        m[j]          = m[j] * a.beta1 + x * a.one_minus_beta1;
        v[j]          = v[j] * a.beta2 + (x * a.one_minus_beta2) * x;
        const float d = sqrtf(v[j]) * g.inv_sqrt_bc2 + a.eps;
        p[j]          = p[j] * g.keep - g.step_size * (m[j] / d);
    }
    if (e.types & kHasCopy)
    {
        if ((e.types >> 4 & 3) == VETRAST_BF16) store_eight<VETRAST_BF16>(e.copy, i, count, whole, p);
        else store_eight<VETRAST_F16>(e.copy, i, count, whole, p);
    }
    if (P == VETRAST_BF16 && a.stochastic)
    {
#pragma unroll
        for (int j = 0; j < 8; ++j)
        {
            const uint32_t bits = __float_as_uint(p[j]);
            const uint32_t r    = (rm[j] * 0xE2Bu) >> 4 & 0xFFFFu;
            if ((bits & 0x7F800000u) != 0x7F800000u) p[j] = __uint_as_float((bits + r) & 0xFFFF0000u);
        }
    }
    store_eight<P>(e.param, i, count, whole, p);
    if constexpr (BITS == 32)
    {
        store_eight<VETRAST_F32>(e.m, i, count, whole, m);
        store_eight<VETRAST_F32>(e.v, i, count, whole, v);
    }
    else
    {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            if (j >= count) m[j] = v[j] = 0.f;
        uint32_t rv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) rv[j] = rm[j] * 0x5D3u & 0xFFFFFu;
        uint2 mc, vc;
        uint32_t scale;
        encode_moments(m, v, rm, rv, mc, vc, scale);
        if (codes)
        {
            *(uint2*)((uint8_t*)e.m + i) = mc;
            *(uint2*)((uint8_t*)e.v + i) = vc;
            if (i % kMomentBlock == 0) ((uint16_t*)e.scale)[i / kMomentBlock] = (uint16_t)scale;
        }
    }
    if (a.zero_grad)
    {
        const float zero[8] = {};
        store_eight<G>(e.grad, i, count, whole, zero);
    }
}

// The entry a chunk belongs to: lane k holds where entry k begins.
__device__ __forceinline__ uint32_t entry_of(uint32_t begins, uint32_t chunk)
{
    return (uint32_t)__popcll(__ballot(begins <= chunk)) - 1u;
}

template <int BITS>
__global__ void __launch_bounds__(kBlock) adamw_step_kernel(const AdamWLaunch a)
{
    const uint32_t lane   = threadIdx.x % kWave;
    const uint32_t begins = lane < a.entries ? a.e[lane].first : 0xFFFFFFFFu;
    const float scale     = a.grad_scale ? *a.grad_scale : 1.f;
    const bool leave      = !isfinite(scale);
    for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x)
    {
        const uint32_t k    = entry_of(begins, chunk);
        const AdamWEntry& e = a.e[k];
        const uint32_t slot = e.types >> 8;
        AdamWGroup g        = a.g[slot];
        if (a.device) g = a.device->group[g.key];
        const uint32_t i = (chunk - e.first) * kOptimChunk + threadIdx.x * 8u;
        switch (e.types & 15u)
        {
#define VET_ADAMW(P, G) \
    case P | G << 2: adamw_eight<BITS, P, G>(a, e, g, scale, leave, i); break;
            VET_ADAMW(VETRAST_F32, VETRAST_F32)
            VET_ADAMW(VETRAST_F32, VETRAST_BF16)
            VET_ADAMW(VETRAST_F32, VETRAST_F16)
            VET_ADAMW(VETRAST_BF16, VETRAST_F32)
            VET_ADAMW(VETRAST_BF16, VETRAST_BF16)
            VET_ADAMW(VETRAST_BF16, VETRAST_F16)
            VET_ADAMW(VETRAST_F16, VETRAST_F32)
            VET_ADAMW(VETRAST_F16, VETRAST_BF16)
            VET_ADAMW(VETRAST_F16, VETRAST_F16)
#undef VET_ADAMW
        }
    }
}

struct NormEntry
{
    const void* grad;
    uint32_t n, first, type, aligned;
};
struct NormLaunch
{
    NormEntry e[kNormEntries];
    double* partial;  // of this launch, one a workgroup
    uint32_t entries, chunks;
};
static_assert(sizeof(NormLaunch) <= 4096, "kernel arguments");

__device__ __forceinline__ double wave_sum(double x)
{
    for (int d = kWave / 2; d > 0; d >>= 1) x += __shfl_down(x, d);
    return x;
}
// Sum over a workgroup of kBlock threads, in thread 0.
__device__ __forceinline__ double block_sum(double x)
{
    __shared__ double part[kBlock / kWave];
    x = wave_sum(x);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = x;
    __syncthreads();
    x = 0;
    for (int w = 0; w < kBlock / kWave; ++w) x += part[w];
    return x;
}

template <int T>
__device__ __forceinline__ double squares_of_eight(const NormEntry& e, uint32_t i)
{
    const uint32_t count = i < e.n ? min(e.n - i, 8u) : 0u;
    float x[8];
    load_eight<T>(e.grad, i, count, count == 8u && e.aligned, x);
    double s = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += (double)x[j] * (double)x[j];
    return s;
}

__global__ void __launch_bounds__(kBlock) gradient_squares_kernel(const NormLaunch a)
{
    double sum = 0;
    uint32_t k = 0;
    for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x)
    {
        while (k + 1 < a.entries && a.e[k + 1].first <= chunk) ++k;
        const NormEntry& e = a.e[k];
        const uint32_t i   = (chunk - e.first) * kOptimChunk + threadIdx.x * 8u;
        if (e.type == VETRAST_F32) sum += squares_of_eight<VETRAST_F32>(e, i);
        else if (e.type == VETRAST_BF16) sum += squares_of_eight<VETRAST_BF16>(e, i);
        else sum += squares_of_eight<VETRAST_F16>(e, i);
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = sum;
}

// Norm and factor from the workgroups' sums, added in an order of their own number.
__global__ void __launch_bounds__(kBlock) gradient_norm_kernel(const double* __restrict__ partial, uint32_t count, double max_norm, double scale, float* __restrict__ out)
{
    double sum = 0;
    for (uint32_t k = threadIdx.x; k < count; k += kBlock) sum += partial[k];
    sum = block_sum(sum);
    if (threadIdx.x == 0)
    {
        const double norm = fabs(scale) * sqrt(sum);
        const float told  = (float)norm;
        out[0]            = told;
        out[1]            = !isfinite(told) ? __builtin_nanf("") : (float)(max_norm > 0 && norm > max_norm ? scale * (max_norm / norm) : scale);
    }
}

struct MomentEntry
{
    float *m, *v;
    uint8_t *mc, *vc, *scale;
    uint32_t n, first;
};
struct MomentLaunch
{
    MomentEntry e[kMomentEntries];
    uint32_t entries, chunks;
};
static_assert(sizeof(MomentLaunch) <= 4096, "kernel arguments");

template <bool PACK>
__global__ void __launch_bounds__(kBlock) convert_moments_kernel(const MomentLaunch a)
{
    uint32_t k = 0;
    for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x)
    {
        while (k + 1 < a.entries && a.e[k + 1].first <= chunk) ++k;
        const MomentEntry& e = a.e[k];
        const uint32_t i     = (chunk - e.first) * kOptimChunk + threadIdx.x * 8u;
        const uint32_t count = i < e.n ? min(e.n - i, 8u) : 0u;
        const bool whole     = count == 8u && (((uintptr_t)e.m | (uintptr_t)e.v) & 15) == 0;
        const bool codes     = i < (e.n + kMomentBlock - 1) / kMomentBlock * kMomentBlock;
        float m[8], v[8];
        uint2 mc = make_uint2(0, 0), vc = make_uint2(0, 0);
        uint32_t scale = 0;
        if constexpr (PACK)
        {
            load_eight<VETRAST_F32>(e.m, i, count, whole, m);
            load_eight<VETRAST_F32>(e.v, i, count, whole, v);
            uint32_t half[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
            {
                v[j]    = fabsf(v[j]);
                half[j] = 1u << 19;
            }
            encode_moments(m, v, half, half, mc, vc, scale);
            if (codes)
            {
                *(uint2*)(e.mc + i) = mc;
                *(uint2*)(e.vc + i) = vc;
                if (i % kMomentBlock == 0) ((uint16_t*)e.scale)[i / kMomentBlock] = (uint16_t)scale;
            }
        }
        else
        {
            if (codes)
            {
                mc    = *(const uint2*)(e.mc + i);
                vc    = *(const uint2*)(e.vc + i);
                scale = ((const uint16_t*)e.scale)[i / kMomentBlock];
            }
            decode_moments(mc, vc, scale, m, v);
            store_eight<VETRAST_F32>(e.m, i, count, whole, m);
            store_eight<VETRAST_F32>(e.v, i, count, whole, v);
        }
    }
}
}  // namespace vetrast
