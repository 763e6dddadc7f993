// Optimiser kernels over lists of tensors: AdamW with moments in 32 or 8 bits, the norm of all gradients, moments to 8 bits and back.
//
// A launch takes a table of tensors in its arguments (no copy to the device, nothing to keep, and what a graph captures is whole). It is
// cut into chunks of kOptimChunk elements, 8 a thread, and every workgroup goes through chunks blockIdx.x, blockIdx.x + gridDim.x, ...
#pragma once
#include "common.h"

namespace vetrast
{
constexpr uint32_t kOptimChunk   = 8 * kBlock;  // elements a workgroup takes at a time: 8 a thread
constexpr int kMomentBlock       = VETRAST_MOMENT_BLOCK;
constexpr uint32_t kMomentMargin = 0x100100;  // see code_base
static_assert(kOptimChunk % kMomentBlock == 0 && kMomentBlock == 16 * 8, "16 lanes of 8 elements hold a block");

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
            begins[q]        = k < a.entries ? a.e[k].first_chunk : 0xFFFFFFFFu;
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

// ---- eight elements of a tensor ----------------------------------------------------------------------------------------

// As they lie in memory, 32 bytes or (16-bit types) 16. Loads of several arrays are under way before the first is looked at.
struct RawEight
{
    uint4 a, b;
};

// Elements i ... i + 7 of p, those from `count` on as zeros. whole: all eight are there and p + i is 16-byte aligned.
__device__ __forceinline__ RawEight load_raw(const void* p, uint32_t type, uint32_t i, uint32_t count, bool whole)
{
    RawEight r;
    r.a = r.b = make_uint4(0, 0, 0, 0);
    if (type == VETRAST_F32)
    {
        const uint32_t* x = (const uint32_t*)p + i;
        if (whole)
        {
            r.a = ((const uint4*)x)[0];
            r.b = ((const uint4*)x)[1];
        }
        else if (count)
        {
            uint32_t w[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) w[j] = x[min(j, count - 1)];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) w[j] = j < count ? w[j] : 0u;
            r.a = make_uint4(w[0], w[1], w[2], w[3]);
            r.b = make_uint4(w[4], w[5], w[6], w[7]);
        }
    }
    else
    {
        const uint16_t* x = (const uint16_t*)p + i;
        if (whole) r.a = *(const uint4*)x;
        else if (count)
        {
            uint32_t w[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) w[j] = x[min(j, count - 1)];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) w[j] = j < count ? w[j] : 0u;
            r.a = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
        }
    }
    return r;
}

__device__ __forceinline__ void store_raw(void* p, uint32_t type, uint32_t i, uint32_t count, bool whole, const RawEight& r)
{
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    if (type == VETRAST_F32)
    {
        uint32_t* x = (uint32_t*)p + i;
        if (whole)
        {
            ((uint4*)x)[0] = r.a;
            ((uint4*)x)[1] = r.b;
        }
        else
        {
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j)
                if (j < count) x[j] = w[j];
        }
    }
    else
    {
        uint16_t* x = (uint16_t*)p + i;
        if (whole) *(uint4*)x = r.a;
        else
        {
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j)
                if (j < count) x[j] = (uint16_t)(w[j / 2] >> 16 * (j % 2));
        }
    }
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
    r.b = make_uint4(0, 0, 0, 0);
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

// ---- random bits -------------------------------------------------------------------------------------------------------

// A step's key: two rounds of a 64-bit mixing function (the finalizer of splitmix64) over seed and step.
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

// 20 random bits for each of 8 elements, the first of which is half of pair number `pair`: 32 bits of a hash serve two elements, the
// lower 20 and the upper 20 of them (products of 32 bits take four times as long as other instructions, and the 8-bit step is
// bound by instructions).
__device__ __forceinline__ void random_eight(uint32_t pair, uint32_t key, uint32_t* r)
{
    const uint32_t start = pair * 0x9E3779B1u;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j)
    {
        uint32_t x = start + j * 0x9E3779B1u;
        x          = x ^ (x >> 15) ^ key;
        x *= 0xBB67AE85u;
        x ^= x >> 15;
        x *= 0xA54FF53Bu;
        x ^= x >> 15;
        r[2 * j]     = x & 0xFFFFFu;
        r[2 * j + 1] = x >> 12;
    }
}

// Odd factors make of an element's bits others that go with them without correlation to speak of (measured over 2^20 elements).
__device__ __forceinline__ uint32_t second_bits(uint32_t r) { return __umul24(r, 0x5D3u) & 0xFFFFFu; }
__device__ __forceinline__ uint32_t parameter_bits(uint32_t r) { return __umul24(r, 0xE2Bu) >> 4 & 0xFFFFu; }

// ---- moments in 8 bits -------------------------------------------------------------------------------------------------

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

// A code stands for float(bits = (code << 20) + base) - float(base). Magnitude x gets it from x + float(base), whose bits less those of
// the base are the code, with 20 bits below it that decide between it and the next: values between two codes are evenly
// spaced, so r in [0, 2^20) that is random leaves the mean as it is.
__device__ __forceinline__ uint32_t offset_bits(float x, uint32_t base, uint32_t r)
{
    return __float_as_uint(fabsf(x) + __uint_as_float(base)) + r - base;
}

__device__ __forceinline__ float code_value(uint32_t code, uint32_t base)
{
    return __uint_as_float((code << 20) + base) - __uint_as_float(base);
}

// The middle one of three.
__device__ __forceinline__ uint32_t middle(uint32_t a, uint32_t b, uint32_t c)
{
    return max(min(a, b), min(max(a, b), c));
}

struct Codes
{
    uint2 m, v;      // eight each
    uint32_t scale;  // of the block: D of the first moment, of the second above it
};

// m, v: of this lane's eight elements, a block is a row of 16 lanes. rm, rv: their random bits. v >= 0.
// Maxima of floats pass over NaN, and of integers do not. The second moment is looked at as integers; where the first is not finite
// after a step, the second is not either, as it has its square, or the block was lost before. lost: the block's first moment is not
// finite, whatever the second says.
__device__ __forceinline__ Codes encode_moments(const float* m, const float* v, const uint32_t* rm, const uint32_t* rv, bool lost)
{
    float top_m    = 0.f;
    uint32_t top_v = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
    {
        top_m = fmaxf(top_m, fabsf(m[j]));
        top_v = max(top_v, __float_as_uint(v[j]));
    }
    const uint32_t dv = code_base<31>(row_max(top_v));
    uint32_t dm       = code_base<15>(row_max(__float_as_uint(top_m)));
    if (dv == 255u)
    {
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(m[j]) & 0x7FFFFFFFu);
        dm = code_base<15>(row_max(top));
    }
    if (lost) dm = 255u;
    const uint32_t bm = dm << 23, bv = dv << 23;
    uint32_t a[8], b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
    {
        // seven bits of code to the top, below the sign
        a[j] = (offset_bits(m[j], bm, rm[j]) << 4 & 0x7FFFFFFFu) | (__float_as_uint(m[j]) & 0x80000000u);
        // above zero is at least code 1: a code is never above a value's own bits, so the middle one says so
        b[j] = middle(__float_as_uint(v[j]), 1u, offset_bits(v[j], bv, rv[j]) >> 20);
    }
    Codes c;
    uint32_t w[2], x[2];
#pragma unroll
    for (int q = 0; q < 2; ++q)
    {
        const uint32_t low  = __builtin_amdgcn_perm(a[4 * q + 1], a[4 * q], 0x0C0C0703);  // top bytes
        const uint32_t high = __builtin_amdgcn_perm(a[4 * q + 3], a[4 * q + 2], 0x07030C0C);
        w[q]                = low | high;
        x[q]                = b[4 * q] | b[4 * q + 1] << 8 | b[4 * q + 2] << 16 | b[4 * q + 3] << 24;
    }
    c.m     = dm == 255u ? make_uint2(0, 0) : make_uint2(w[0], w[1]);  // code 0 at D = 255: infinity less infinity
    c.v     = dv == 255u ? make_uint2(0, 0) : make_uint2(x[0], x[1]);
    c.scale = dm | dv << 8;
    return c;
}

__device__ __forceinline__ void decode_moments(const Codes& c, float* m, float* v)
{
    const uint32_t bm = (c.scale & 255u) << 23, bv = c.scale >> 8 << 23;
#pragma unroll
    for (int j = 0; j < 8; ++j)
    {
        const uint32_t wm = j < 4 ? c.m.x : c.m.y, wv = j < 4 ? c.v.x : c.v.y;
        m[j] = copysignf(code_value(wm >> 8 * (j % 4) & 127u, bm), __uint_as_float(wm << (24 - 8 * (j % 4))));
        v[j] = code_value(wv >> 8 * (j % 4) & 255u, bv);
    }
}

// ---- AdamW -------------------------------------------------------------------------------------------------------------

struct AdamWEntry
{
    void* param;
    void* grad;
    uint32_t n;
    uint32_t first_chunk;  // of the launch
    uint32_t block;        // place in the flat arrays
    uint32_t flags;        // kAdamW..., slot of the group from bit 8 on
};
enum
{
    kAdamWParam   = 3,       // type
    kAdamWGrad    = 3 << 2,  // type
    kAdamWAligned = 1 << 4,  // param and grad to 16 bytes
    kAdamWMaster  = 1 << 5
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

constexpr int kAdamWEntries = 120;  // what 4 KB of kernel arguments hold
constexpr int kAdamWFew     = 8;    // ... and a launch whose arguments are 400 bytes
constexpr int kAdamWGroups  = 8;
struct AdamWCommon
{
    AdamWGroup g[kAdamWGroups];
    void* m;
    void* v;
    uint16_t* scale;
    float* master;
    const float* grad_scale;
    const AdamWDevice* device;  // where set, g[].key are places in device->group
    uint32_t entries, chunks;
    float beta1, one_minus_beta1, beta2, one_minus_beta2, eps;
    int zero_grad, stochastic, exact_root;
};
template <int ENTRIES>
struct AdamWLaunch : AdamWCommon
{
    AdamWEntry e[ENTRIES];
};
static_assert(sizeof(AdamWLaunch<kAdamWEntries>) <= 4096, "kernel arguments");

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

// The groups' constants of step `state.step + 1`. The launch with the last groups writes the new count, unless gradients overflowed: then
// nothing is read of the constants.
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

template <int BITS, class Launch>
__global__ void __launch_bounds__(kBlock) adamw_step_kernel(const Launch a)
{
    const ChunkFinder<finder_groups(sizeof(a.e) / sizeof(a.e[0]))> find(a);
    const float grad_scale = a.grad_scale ? *a.grad_scale : 1.f;
    const bool leave       = !isfinite(grad_scale);
    for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x)
    {
        const AdamWEntry& e  = a.e[find(chunk)];
        const uint32_t flags = e.flags, n = e.n;
        const uint32_t p_type = flags & kAdamWParam, g_type = (flags & kAdamWGrad) >> 2;
        const uint32_t i      = (chunk - e.first_chunk) * kOptimChunk + threadIdx.x * 8u;
        const uint32_t count  = i < n ? min(n - i, 8u) : 0u;
        const bool whole      = count == 8u && (flags & kAdamWAligned);
        const uint32_t block  = e.block + i / kMomentBlock;
        const size_t at       = (size_t)block * kMomentBlock + i % kMomentBlock;  // in the flat arrays
        const bool inside     = i < (n + kMomentBlock - 1) / kMomentBlock * kMomentBlock;
        const RawEight zero   = {};
        if (leave)
        {
            if (a.zero_grad) store_raw(e.grad, g_type, i, count, whole, zero);
            continue;
        }
        const bool master = flags & kAdamWMaster;
        RawEight rg, rp = zero, r1 = zero, r2 = zero;
        Codes codes     = {};
        rg              = load_raw(e.grad, g_type, i, count, whole);
        if (!master) rp = load_raw(e.param, p_type, i, count, whole);
        if (inside)
        {
            if (master) rp = {((const uint4*)(a.master + at))[0], ((const uint4*)(a.master + at))[1]};
            if constexpr (BITS == 32)
            {
                r1 = {((const uint4*)((float*)a.m + at))[0], ((const uint4*)((float*)a.m + at))[1]};
                r2 = {((const uint4*)((float*)a.v + at))[0], ((const uint4*)((float*)a.v + at))[1]};
            }
            else
            {
                codes.m     = *(const uint2*)((const uint8_t*)a.m + at);
                codes.v     = *(const uint2*)((const uint8_t*)a.v + at);
                codes.scale = a.scale[block];
            }
        }
        AdamWGroup g = a.g[flags >> 8];
        if (a.device) g = a.device->group[g.key];
        const bool random = a.stochastic && p_type == VETRAST_BF16 && !master;
        uint32_t r[8];
        if (BITS == 8 || random) random_eight((uint32_t)(at / 2), g.key, r);

        float x[8], p[8], m[8], v[8];
        to_floats(rg, g_type, x);
        to_floats(rp, master ? VETRAST_F32 : p_type, p);
        if constexpr (BITS == 32)
        {
            to_floats(r1, VETRAST_F32, m);
            to_floats(r2, VETRAST_F32, v);
        }
        else decode_moments(codes, m, v);
        // Rounded after every operation: both kinds of state, and whoever steps them elsewhere, get the same bits.
#pragma unroll
        for (int j = 0; j < 8; ++j)
        {
            x[j] *= grad_scale;
            m[j] = m[j] * a.beta1 + x[j] * a.one_minus_beta1;
            v[j] = v[j] * a.beta2 + (x[j] * a.one_minus_beta2) * x[j];
        }
        // With 8-bit moments root and quotient are the instructions for them, good to 1.54 half steps of float32 each, as the step is
        // bound by instructions; with 32-bit ones it waits for memory and they are rounded to nearest. The root instruction takes
        // values below 2^-126 for zero: eps makes up for that unless it is tiny itself.
        if (BITS == 32 || a.exact_root)
        {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = sqrtf(v[j]);
        }
        else
        {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_sqrtf(v[j]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
        {
            const float d = fmaf(x[j], g.inv_sqrt_bc2, a.eps);
            const float q = BITS == 32 ? m[j] / d : m[j] * __builtin_amdgcn_rcpf(d);
            p[j]          = fmaf(-g.step_size, q, p[j] * g.keep);
        }

        if (master)
        {
            const RawEight out = from_floats(p, VETRAST_F32);
            if (inside)
            {
                ((uint4*)(a.master + at))[0] = out.a;
                ((uint4*)(a.master + at))[1] = out.b;
            }
        }
        RawEight out;
        if (random)
        {
            out.b = make_uint4(0, 0, 0, 0);
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
            {
                const bool finite = __builtin_isfinite(p[j]);
                w[j]              = __float_as_uint(p[j]) + (finite ? parameter_bits(r[j]) : 0u);
            }
            out.a = make_uint4(__builtin_amdgcn_perm(w[1], w[0], 0x07060302), __builtin_amdgcn_perm(w[3], w[2], 0x07060302),
                               __builtin_amdgcn_perm(w[5], w[4], 0x07060302), __builtin_amdgcn_perm(w[7], w[6], 0x07060302));
        }
        else out = from_floats(p, p_type);
        store_raw(e.param, p_type, i, count, whole, out);
        if constexpr (BITS == 32)
        {
            const RawEight o1 = from_floats(m, VETRAST_F32), o2 = from_floats(v, VETRAST_F32);
            if (inside)
            {
                ((uint4*)((float*)a.m + at))[0] = o1.a;
                ((uint4*)((float*)a.m + at))[1] = o1.b;
                ((uint4*)((float*)a.v + at))[0] = o2.a;
                ((uint4*)((float*)a.v + at))[1] = o2.b;
            }
        }
        else
        {
            uint32_t rv[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) rv[j] = second_bits(r[j]);
            const Codes c = encode_moments(m, v, r, rv, (codes.scale & 255u) == 255u);
            if (inside)
            {
                *(uint2*)((uint8_t*)a.m + at) = c.m;
                *(uint2*)((uint8_t*)a.v + at) = c.v;
                if (i % kMomentBlock == 0) a.scale[block] = (uint16_t)c.scale;
            }
        }
        if (a.zero_grad) store_raw(e.grad, g_type, i, count, whole, zero);
    }
}

// ---- norms -------------------------------------------------------------------------------------------------------------

constexpr int kNormEntries = 250;
struct NormEntry
{
    const void* grad;
    uint32_t n_type;  // n << 2 | type
    uint32_t first_chunk;
};
struct NormLaunch
{
    double* partial;  // of this launch, one a workgroup
    uint32_t entries, chunks;
    NormEntry e[kNormEntries];
};
static_assert(sizeof(NormLaunch) <= 4096, "kernel arguments");

// Sum over a workgroup of kBlock threads, in all of them.
__device__ __forceinline__ double block_sum(double x)
{
    __shared__ double part[kBlock / kWave];
    for (int d = kWave / 2; d > 0; d >>= 1) x += __shfl_down(x, d);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = x;
    __syncthreads();
    x = 0;
    for (int w = 0; w < kBlock / kWave; ++w) x += part[w];
    return x;
}

// In 64 bits throughout: no square overflows or vanishes, and a sum of any length is good to the last bit of a float.
__global__ void __launch_bounds__(kBlock) gradient_squares_kernel(const NormLaunch a)
{
    const ChunkFinder<finder_groups(kNormEntries)> find(a);
    double sum = 0;
    for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x)
    {
        const NormEntry& e   = a.e[find(chunk)];
        const uint32_t n     = e.n_type >> 2, type = e.n_type & 3u;
        const uint32_t i     = (chunk - e.first_chunk) * kOptimChunk + threadIdx.x * 8u;
        const uint32_t count = i < n ? min(n - i, 8u) : 0u;
        float x[8];
        to_floats(load_raw(e.grad, type, i, count, count == 8u && (uintptr_t)e.grad % 16 == 0), type, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fma((double)x[j], (double)x[j], sum);
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

// ---- moments to 8 bits and back ----------------------------------------------------------------------------------------

constexpr int kMomentEntries = 120;
struct MomentEntry
{
    float *m, *v;
    uint32_t n, first_chunk, block, reserved;
};
struct MomentLaunch
{
    uint8_t *m, *v;
    uint16_t* scale;
    uint32_t entries, chunks;
    MomentEntry e[kMomentEntries];
};
static_assert(sizeof(MomentLaunch) <= 4096, "kernel arguments");

template <bool PACK>
__global__ void __launch_bounds__(kBlock) convert_moments_kernel(const MomentLaunch a)
{
    const ChunkFinder<finder_groups(kMomentEntries)> find(a);
    for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x)
    {
        const MomentEntry& e = a.e[find(chunk)];
        const uint32_t i     = (chunk - e.first_chunk) * kOptimChunk + threadIdx.x * 8u;
        const uint32_t count = i < e.n ? min(e.n - i, 8u) : 0u;
        const bool whole     = count == 8u && (((uintptr_t)e.m | (uintptr_t)e.v) & 15) == 0;
        const uint32_t block = e.block + i / kMomentBlock;
        const size_t at      = (size_t)block * kMomentBlock + i % kMomentBlock;
        const bool inside    = i < (e.n + kMomentBlock - 1) / kMomentBlock * kMomentBlock;
        float m[8], v[8];
        if constexpr (PACK)
        {
            const RawEight r1 = load_raw(e.m, VETRAST_F32, i, count, whole), r2 = load_raw(e.v, VETRAST_F32, i, count, whole);
            to_floats(r1, VETRAST_F32, m);
            to_floats(r2, VETRAST_F32, v);
            uint32_t half[8], lost = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
            {
                v[j]    = fabsf(v[j]);
                half[j] = 1u << 19;
                lost |= __builtin_isfinite(m[j]) ? 0u : 1u;
            }
            const Codes c = encode_moments(m, v, half, half, row_max(lost) != 0);
            if (inside)
            {
                *(uint2*)(a.m + at) = c.m;
                *(uint2*)(a.v + at) = c.v;
                if (i % kMomentBlock == 0) a.scale[block] = (uint16_t)c.scale;
            }
        }
        else
        {
            Codes c = {};
            if (inside)
            {
                c.m     = *(const uint2*)(a.m + at);
                c.v     = *(const uint2*)(a.v + at);
                c.scale = a.scale[block];
            }
            decode_moments(c, m, v);
            store_raw(e.m, VETRAST_F32, i, count, whole, from_floats(m, VETRAST_F32));
            store_raw(e.v, VETRAST_F32, i, count, whole, from_floats(v, VETRAST_F32));
        }
    }
}
}  // namespace vetrast
