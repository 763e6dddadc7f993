// Optimiser kernels over lists of tensors: AdamW with moments in 32 or 8 bits, the norm of all gradients, moments to 8 bits and back.
//
// A launch takes a table of tensors in its arguments (no copy to the device, nothing to keep, and what a graph captures is whole). The
// tensors are cut into chunks of 8 elements a thread, one for each workgroup (27.5 M float32 elements: 142 us; workgroups of a
// grid of 2048 that go on to further chunks 154 us), but for norms, where a workgroup leaves a sum.
#pragma once
#include "common.h"
#include "elements.h"

namespace vetrast
{
constexpr uint32_t kWaveChunk    = 8 * kWave;   // ... of a workgroup of one wave
constexpr int kMomentBlock       = VETRAST_MOMENT_BLOCK;
constexpr uint32_t kMomentMargin = 0x100100;  // see code_base
static_assert(kWaveChunk % kMomentBlock == 0 && kMomentBlock == 16 * 8, "16 lanes of 8 elements hold a block");

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

// 20 random bits for each of a thread's eight elements; `pair`: number of the chunk's first pair of elements. 32 bits of a hash serve two
// elements, the lower 20 and the upper 20 of them: products of 32 bits take four times as long as other instructions, and the 8-bit
// step is bound by instructions.
template <uint32_t HALF>
__device__ __forceinline__ void random_eight(uint32_t pair, uint32_t key, uint32_t* r)
{
    const uint32_t start = pair * 0x9E3779B1u + threadIdx.x * ((HALF != 0 ? 2u : 4u) * 0x9E3779B1u);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j)
    {
        const uint32_t k = HALF != 0 && j >= 2 ? HALF / 2 + j - 2 : j;
        uint32_t x       = start + k * 0x9E3779B1u;
        x                = exclusive_or(x, x >> 15, key);
        x *= 0xBB67AE85u;
        x ^= x >> 15;
        x *= 0xA54FF53Bu;
        x ^= x >> 15;
        r[2 * j]     = x & 0xFFFFFu;
        r[2 * j + 1] = x >> 12;
    }
}

// Odd factors make of an element's bits others that go with them without correlation to speak of (measured over 2^20 elements). The
// instruction is named: for products of which only the lower bits are used the compiler takes the one of 32 bits, four times as long.
template <uint32_t FACTOR>
__device__ __forceinline__ uint32_t times(uint32_t r)
{
    uint32_t x;
    asm("v_mul_u32_u24 %0, %1, %2" : "=v"(x) : "s"(FACTOR), "v"(r));
    return x;
}
__device__ __forceinline__ uint32_t second_bits(uint32_t r) { return times<0x5D3>(r) & 0xFFFFFu; }
__device__ __forceinline__ uint32_t parameter_bits(uint32_t r) { return times<0xE2B>(r) >> 4 & 0xFFFFu; }

// ---- moments in 8 bits -------------------------------------------------------------------------------------------------

// The largest of 16 lanes' values, in all of them (a row of a wave).
__device__ __forceinline__ uint32_t row_max(uint32_t v)
{
    v = max(v, dpp_move<0x128>(v));  // row_ror:8
    v = max(v, dpp_move<0x124>(v));
    v = max(v, dpp_move<0x122>(v));
    return max(v, dpp_move<0x121>(v));
}

// Scale byte D of a block whose largest magnitude has the float bits `largest`, without a sign: its exponent less the binades that codes span, one
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
__device__ __forceinline__ uint32_t offset_bits(float x, float base, uint32_t minus_base, uint32_t r)
{
    uint32_t d;  // a sum of three, which the compiler makes two of
    asm("v_add3_u32 %0, %1, %2, %3" : "=v"(d) : "v"(__float_as_uint(fabsf(x) + base)), "v"(r), "v"(minus_base));
    return d;
}

// `BITS` bits of w from bit AT on, as a number that the compiler does not take apart: with the shift and sum behind it two
// instructions, and not three.
template <int AT, int BITS>
__device__ __forceinline__ uint32_t field(uint32_t w)
{
    uint32_t x;
    asm("v_bfe_u32 %0, %1, %2, %3" : "=v"(x) : "v"(w), "i"(AT), "i"(BITS));
    return x;
}
__device__ __forceinline__ float code_value(uint32_t code, uint32_t base)
{
    return __uint_as_float((code << 20) + base) - __uint_as_float(base);
}

// The middle one of three: one instruction, which the compiler does not find for unsigned variables.
__device__ __forceinline__ uint32_t middle(uint32_t a, uint32_t b, uint32_t c)
{
    uint32_t x;
    asm("v_med3_u32 %0, %1, %2, %3" : "=v"(x) : "v"(a), "v"(b), "v"(c));
    return x;
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
    const uint32_t dv = code_base<31>(row_max(top_v) & 0x7FFFFFFFu);  // a NaN may have the sign set, which is above all, and wraps there
    uint32_t dm       = code_base<15>(row_max(__float_as_uint(top_m)));
    if (dv == 255u)
    {
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(m[j]) & 0x7FFFFFFFu);
        dm = code_base<15>(row_max(top));
    }
    if (lost) dm = 255u;
    const float bm = __uint_as_float(dm << 23), bv = __uint_as_float(dv << 23);
    const uint32_t minus_m = 0u - (dm << 23), minus_v = 0u - (dv << 23);
    uint32_t a[8], b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
    {
        // seven bits of code to the top, below the sign
        a[j] = __float_as_uint(copysignf(__uint_as_float(offset_bits(m[j], bm, minus_m, rm[j]) << 4), m[j]));
        // above zero is at least code 1: a code is never above a value's own bits, so the middle one says so
        b[j] = middle(__float_as_uint(v[j]), 1u, offset_bits(v[j], bv, minus_v, rv[j]) >> 20);
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

template <int AT>
__device__ __forceinline__ void decode_one(uint32_t wm, uint32_t wv, uint32_t bm, uint32_t bv, float& m, float& v)
{
    m = copysignf(code_value(field<AT, 7>(wm), bm), __uint_as_float(wm << (24 - AT)));
    v = code_value(field<AT, 8>(wv), bv);
}
__device__ __forceinline__ void decode_four(uint32_t wm, uint32_t wv, uint32_t scale, float* m, float* v)
{
    const uint32_t bm = (scale & 255u) << 23, bv = scale >> 8 << 23;
    decode_one<0>(wm, wv, bm, bv, m[0], v[0]);
    decode_one<8>(wm, wv, bm, bv, m[1], v[1]);
    decode_one<16>(wm, wv, bm, bv, m[2], v[2]);
    decode_one<24>(wm, wv, bm, bv, m[3], v[3]);
}

// ---- AdamW -------------------------------------------------------------------------------------------------------------

// 24 bytes, so that a launch takes 160 of them: a further launch costs a list 4 us.
struct AdamWEntry
{
    uint32_t param_low, grad_low;
    uint16_t param_high, grad_high;  // of addresses of 48 bits
    uint32_t n_slot;                 // n << 3 | slot of the group
    uint32_t block;                  // place in the flat arrays
    uint32_t chunk_types;            // first chunk of the launch << 4 | type of the gradient << 2 | type of the parameter
    __device__ __forceinline__ uint32_t begins() const { return chunk_types >> 4; }
    // Known to lie in global memory: else the compiler takes flat instructions, which wait for each other and for scalar loads.
    typedef __attribute__((address_space(1))) void Global;
    __device__ __forceinline__ void* param() const { return (void*)(Global*)((uint64_t)param_high << 32 | param_low); }
    __device__ __forceinline__ void* grad() const { return (void*)(Global*)((uint64_t)grad_high << 32 | grad_low); }
};

struct AdamWGroup
{
    float root;    // with s = lr / (1 - beta1^step): the parameter changes by m / (root * sqrt(v) + floor), root is
    float floor;   // 1 / (s sqrt(1 - beta2^step)) and floor eps / s
    float keep;    // 1 - lr * weight_decay
    uint32_t key;  // of this step's random bits
};

__host__ __device__ inline AdamWGroup adamw_group(double lr, double weight_decay, double eps, double bc1, double bc2, uint32_t key)
{
    const double s = lr / bc1;
    AdamWGroup g;
    g.root  = (float)(1.0 / (s * sqrt(bc2)));
    g.floor = (float)(eps / s);
    if (!(fabsf(g.root) <= 3e38f) || !(fabsf(g.floor) <= 3e38f)) g.root = 0.f, g.floor = __builtin_inff();  // no step to speak of
    if (fabsf(g.floor) < 1.17549435e-38f) g.floor = copysignf(1.17549435e-38f, g.floor);  // a reciprocal's smallest argument
    g.keep = (float)(1.0 - lr * weight_decay);
    g.key  = key;
    return g;
}

struct alignas(16) AdamWDevice  // vetrast_adamw_device_state and what adamw_begin_kernel leaves for the step's launches
{
    vetrast_adamw_device_state state;
    AdamWGroup group[1];
};

constexpr int kAdamWEntries = 160;  // what 4 KB of kernel arguments hold
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
    float beta1, one_minus_beta1, beta2, one_minus_beta2;
    int zero_grad, stochastic;
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
    double beta1, beta2, eps;
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
        a.device->group[a.first + k] = adamw_group(a.g[k].lr * (double)factor, a.g[k].weight_decay, a.eps, 1.0 - pow(a.beta1, (double)step),
                                                   1.0 - pow(a.beta2, (double)step), step_key(a.seed, step));
    }
    if (a.last && counts && k == 0) a.device->state.step = step;
}

// Both by scalar loads (the device's were written by an earlier launch); left alone the compiler makes one of the two, a flat one, which waits
// for all loads under way before the random bits.
__device__ __forceinline__ AdamWGroup group_of(const AdamWCommon& a, uint32_t slot)
{
    AdamWGroup g = a.g[slot];
    asm("" : "+s"(g.root), "+s"(g.floor), "+s"(g.keep));
    if (a.device)
    {
        typedef uint32_t Four __attribute__((ext_vector_type(4)));
        g = __builtin_bit_cast(AdamWGroup, *(const __attribute__((address_space(4))) Four*)(uintptr_t)&a.device->group[g.key]);
    }
    return g;
}

struct AdamWChunk
{
    void *param, *grad;
    uint32_t n, slot, p_type, g_type;
    uint32_t start;  // the chunk's first element
    uint32_t block;  // of the tensor, in the flat arrays
    bool whole;      // all its elements are there
};

// Chunks of four kinds. In whole ones every thread has its eight elements, parameter and gradient of one width: their loads are straight code, all
// of them under way at once. `kAnyChunk` does for everything else: tails, and gradients of another width, which move their bytes as
// fast (16 M bf16 with float32 gradients 72.5 us, 5.3 TB/s, with 8-bit moments 34.1, 5.7; with bf16 gradients 66.9, 5.3, and 28.0, 5.7).
enum ChunkKind
{
    kFloatChunk,   // float32
    kShortChunk,   // 16 bits
    kMasterChunk,  // 16 bits, with masters
    kAnyChunk
};

template <int BITS, bool EXACT, uint32_t CHUNK, ChunkKind KIND>
__device__ __forceinline__ void adamw_chunk(const AdamWCommon& a, const AdamWChunk& e, float grad_scale)
{
    constexpr bool ANY    = KIND == kAnyChunk;
    constexpr uint32_t HALF = BITS == 32 && !ANY ? CHUNK / 2 : 0;  // blocks of 8-bit moments are eight elements of 16 neighbouring lanes
    constexpr int BYTES   = KIND == kFloatChunk ? 4 : 2;
    const uint32_t p_type = KIND == kFloatChunk ? (uint32_t)VETRAST_F32 : e.p_type;
    const uint32_t g_type = KIND == kFloatChunk ? (uint32_t)VETRAST_F32 : e.g_type;
    const bool master     = ANY ? a.master && p_type != VETRAST_F32 : KIND == kMasterChunk;
    const uint32_t start = e.start, count = ANY ? count_of(start, e.n) : 8u;
    const auto clear      = [&] {
        const RawEight zero = {};
        if constexpr (ANY) store_any(e.grad, g_type, start, count, e.whole, zero);
        else store_eight<BYTES, HALF>(e.grad, start, zero);
    };
    if (!isfinite(grad_scale))
    {
        if (a.zero_grad) clear();
        return;
    }
    // places of the chunk in the flat arrays, and whether this thread's eight belong to a block of the tensor
    const uint32_t block = e.block + start / kMomentBlock;
    const size_t at      = (size_t)block * kMomentBlock;
    const uint32_t mine  = threadIdx.x * 8u;
    const bool inside    = !ANY || start + mine < (e.n + kMomentBlock - 1) / kMomentBlock * kMomentBlock;
    uint8_t *mcs = (uint8_t*)a.m + at, *vcs = (uint8_t*)a.v + at;
    uint16_t* scales = a.scale + block;

    RawEight rg, rp, r1, r2;
    Codes codes;
    if constexpr (ANY) rg = load_any(e.grad, g_type, start, count, e.whole);
    else rg = load_eight<BYTES, HALF>(e.grad, start);
    if constexpr (ANY)
    {
        rp = r1 = r2 = RawEight{};
        codes        = Codes{};
        if (!master) rp = load_any(e.param, p_type, start, count, e.whole);
    }
    if (inside)
    {
        if (master) rp = load_eight<4, HALF>(a.master + at, 0);
        else if constexpr (!ANY) rp = load_eight<BYTES, HALF>(e.param, start);
        if constexpr (BITS == 32)
        {
            r1 = load_eight<4, HALF>((float*)a.m + at, 0);
            r2 = load_eight<4, HALF>((float*)a.v + at, 0);
        }
        else
        {
            codes.m     = *(const uint2*)(mcs + mine);
            codes.v     = *(const uint2*)(vcs + mine);
            codes.scale = scales[mine / kMomentBlock];
        }
    }
    const AdamWGroup g = group_of(a, e.slot);
    const bool random = KIND != kFloatChunk && !master && a.stochastic && p_type == VETRAST_BF16;
    uint32_t r[8];
    if (BITS == 8 || random) random_eight<HALF>((uint32_t)(at / 2), g.key, r);

    float x[8], p[8], m[8], v[8];
    to_floats(rg, g_type, x);
    to_floats(rp, master ? VETRAST_F32 : p_type, p);
    if constexpr (BITS == 32)
    {
        to_floats(r1, VETRAST_F32, m);
        to_floats(r2, VETRAST_F32, v);
    }
    else
    {
        decode_four(codes.m.x, codes.v.x, codes.scale, m, v);
        decode_four(codes.m.y, codes.v.y, codes.scale, m + 4, v + 4);
    }
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
    if constexpr (BITS == 32 || EXACT)
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
        const float d = fmaf(x[j], g.root, g.floor);
        p[j]          = BITS == 32 ? p[j] * g.keep - m[j] / d : fmaf(-m[j], __builtin_amdgcn_rcpf(d), p[j] * g.keep);
    }

    bool lost = true;  // whether one of these eight may not be finite
    if constexpr (BITS == 32)
    {
        if (inside)
        {
            store_eight<4, HALF>((float*)a.m + at, 0, from_floats(m, VETRAST_F32));
            store_eight<4, HALF>((float*)a.v + at, 0, from_floats(v, VETRAST_F32));
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
            *(uint2*)(mcs + mine) = c.m;
            *(uint2*)(vcs + mine) = c.v;
            if (mine % kMomentBlock == 0) scales[mine / kMomentBlock] = (uint16_t)c.scale;
        }
        lost = c.scale >> 8 == 255u;  // a gradient that is not finite shows there; of parameters and first moments that are not,
                                      // the lower bits are zeros
    }
    RawEight out;
    if (random)
    {
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = parameter_bits(r[j]);
        if (lost)
        {
#pragma unroll
            for (int j = 0; j < 8; ++j) r[j] = __builtin_isfinite(p[j]) ? r[j] : 0u;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] += __float_as_uint(p[j]);
        out.a = make_uint4(__builtin_amdgcn_perm(r[1], r[0], 0x07060302), __builtin_amdgcn_perm(r[3], r[2], 0x07060302),
                           __builtin_amdgcn_perm(r[5], r[4], 0x07060302), __builtin_amdgcn_perm(r[7], r[6], 0x07060302));
    }
    else out = from_floats(p, p_type);
    if constexpr (ANY) store_any(e.param, p_type, start, count, e.whole, out);
    else store_eight<BYTES, HALF>(e.param, start, out);
    if (master && inside)
    {
        if constexpr (ANY)  // zeros behind the last element, whatever a lost block makes of them
        {
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) p[j] = j < count ? p[j] : 0.f;
        }
        store_eight<4, HALF>(a.master + at, 0, from_floats(p, VETRAST_F32));
    }
    if (a.zero_grad) clear();
}

// One pass over parameter, gradient and state, each read and written once.
//   32 bits: bound by memory. 27.5 M float32 elements, 28 bytes each: 142 us, 5.4 TB/s.
//   8 bits:  10 M float32 elements, 16 bytes each: 28.0 us, 5.7 TB/s, bound by memory. 40 M bf16 elements, 10 bytes each: one tensor 73 to 76 us,
//            5.3 to 5.5 TB/s, 291 tensors in two launches 49.6 and 34.9; the same loads and stores with nothing in between 74, 48.0 and 33.2.
//            The vector units are at work for 82 to 92 % of the time: 435 instructions for a wave's 512 elements (549 before bits were
//            taken out of words, medians and products by the instructions for them), of which roots, quotients and 32-bit
//            products take four times as long as the others.
// EXACT: eps is so small that roots of values below 2^-126 count.
// THREADS: a workgroup is one wave where the call is small, for then its waves spread over more compute units (100 k float32 elements: 3.8 us,
// with four waves 5.2; 600 k 5.5 and 6.3; 800 k 6.0 and 6.5; 1 M 7.1 and 6.8; 1.5 M 8.9 and 8.6), and with 8-bit moments of 16-bit
// parameters, where compute units that are never idle count (16 M: 29.1 us and 31.0; 40 M 72.7 and 75.4). Else it is four, whose accesses
// lie closer together.
template <int BITS, bool EXACT, int THREADS, class Launch>
__global__ void __launch_bounds__(THREADS) adamw_step_kernel(const Launch a)
{
    constexpr uint32_t CHUNK = 8 * THREADS;
    const ChunkFinder<finder_groups(sizeof(a.e) / sizeof(a.e[0]))> find(a);
    const AdamWEntry& entry = a.e[find(blockIdx.x)];
    const float grad_scale  = a.grad_scale ? *a.grad_scale : 1.f;
    AdamWChunk e;
    e.param  = entry.param();
    e.grad   = entry.grad();
    e.n      = entry.n_slot >> 3;
    e.slot   = entry.n_slot & 7u;
    e.p_type = entry.chunk_types & 3u;
    e.g_type = entry.chunk_types >> 2 & 3u;
    e.start  = (blockIdx.x - entry.begins()) * CHUNK;
    e.block  = entry.block;
    e.whole  = e.n - e.start >= CHUNK;
    if (!e.whole || (e.p_type == VETRAST_F32) != (e.g_type == VETRAST_F32)) adamw_chunk<BITS, EXACT, CHUNK, kAnyChunk>(a, e, grad_scale);
    else if (e.p_type == VETRAST_F32) adamw_chunk<BITS, EXACT, CHUNK, kFloatChunk>(a, e, grad_scale);
    else if (a.master) adamw_chunk<BITS, EXACT, CHUNK, kMasterChunk>(a, e, grad_scale);
    else adamw_chunk<BITS, EXACT, CHUNK, kShortChunk>(a, e, grad_scale);
}

// ---- norms -------------------------------------------------------------------------------------------------------------

constexpr int kNormEntries = 240;  // what 4 KB of kernel arguments hold
constexpr int kNormFew     = 8;    // ... and a launch whose arguments are 176 bytes (100 k elements: 4.8 us a call instead of 5.2)
struct NormEntry
{
    const void* grad;
    uint32_t n_type;  // n << 2 | type
    uint32_t first_chunk;
    __device__ __forceinline__ uint32_t begins() const { return first_chunk; }
};
constexpr uint32_t kNormSlots = 32;
struct NormWorkspace
{
    // Workgroups that have left their sum, by slot, and slots that are complete; zero between calls. A line each: an addition to one place
    // takes 12 ns, and a call has up to a thousand workgroups.
    uint32_t done[kNormSlots + 1][16];
    uint32_t unused[16];
    double partial[1];
};
template <int ENTRIES>
struct NormLaunch
{
    NormWorkspace* workspace;
    float* out;
    double max_norm, scale;
    uint32_t entries, chunks;
    uint32_t first, total;  // this launch's first workgroup among those of the call, and their number
    NormEntry e[ENTRIES];
};
static_assert(sizeof(NormLaunch<kNormEntries>) <= 4096, "kernel arguments");

// Sum over a workgroup of kBlock threads, in all of them.
__device__ __forceinline__ double block_sum(double x)
{
    __shared__ double part[kBlock / kWave];
    for (int d = kWave / 2; d > 0; d >>= 1) x += __shfl_down(x, d);
    __syncthreads();
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = x;
    __syncthreads();
    x = 0;
    for (int w = 0; w < kBlock / kWave; ++w) x += part[w];
    return x;
}

// Leaves a workgroup's sum, and says whether it was the last of the call to do so; one thread of each. The sum goes past the caches of this
// XCD (an atomic store of agent scope) and has arrived when the wait ends, so whoever finds all counts complete may read all sums. A
// release would write back the whole L2 for it: 1024 workgroups 54 us instead of 31, in one slot.
__device__ __forceinline__ bool leave_sum(NormWorkspace* w, uint32_t number, uint32_t total, double sum)
{
    const auto add = [](uint32_t* p) { return __hip_atomic_fetch_add(p, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u; };
    __hip_atomic_store(&w->partial[number], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const uint32_t slots = total <= 2 * kNormSlots ? 1u : kNormSlots;  // a second count takes 1 us
    const uint32_t slot  = number % slots;
    if (add(&w->done[slot][0]) != (total - slot + slots - 1) / slots) return false;
    __hip_atomic_store(&w->done[slot][0], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (slots == 1) return true;
    if (add(&w->done[kNormSlots][0]) != slots) return false;
    __hip_atomic_store(&w->done[kNormSlots][0], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}

// In 64 bits throughout: no square overflows or vanishes, and a sum of any length is good to the last bit of a float. The workgroup that is
// the last of the call to leave its sum adds all of them, in the order of their numbers: one launch instead of two, 4 us of a host's time.
// 27.5 M float32: 20.8 us, 5.3 TB/s. 100 k: 4.1 us, what a launch, a sum's way to memory, the count and the sums' way back take.
template <int ENTRIES>
__global__ void __launch_bounds__(kBlock) gradient_norm_kernel(const NormLaunch<ENTRIES> a)
{
    const ChunkFinder<finder_groups(ENTRIES)> find(a);
    double sum = 0;
    for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x)
    {
        const NormEntry& e   = a.e[find(chunk)];
        const uint32_t n     = e.n_type >> 2, type = e.n_type & 3u;
        const uint32_t start = (chunk - e.first_chunk) * kOptimChunk;
        RawEight r;
        if (n - start >= kOptimChunk)
        {
            if (type == VETRAST_F32) r = load_eight<4, kOptimChunk / 2>(e.grad, start);
            else r = load_eight<2>(e.grad, start);
        }
        else r = load_any(e.grad, type, start, count_of(start, n), false);
        float x[8];
        to_floats(r, type, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fma((double)x[j], (double)x[j], sum);
    }
    sum = block_sum(sum);
    __shared__ bool last;
    if (threadIdx.x == 0) last = leave_sum(a.workspace, a.first + blockIdx.x, a.total, sum);
    __syncthreads();
    if (!last) return;
    sum = 0;
    for (uint32_t k = threadIdx.x; k < a.total; k += kBlock)
        sum += __hip_atomic_load(&a.workspace->partial[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sum = block_sum(sum);
    if (threadIdx.x == 0)
    {
        const double norm = fabs(a.scale) * sqrt(sum);
        const float told  = (float)norm;
        a.out[0]          = told;
        a.out[1]          = !isfinite(told) ? __builtin_nanf("") : (float)(a.max_norm > 0 && norm > a.max_norm ? a.scale * (a.max_norm / norm) : a.scale);
    }
}

// ---- moments to 8 bits and back ----------------------------------------------------------------------------------------

constexpr int kMomentEntries = 120;
struct MomentEntry
{
    float *m, *v;
    uint32_t n, first_chunk, block, reserved;
    __device__ __forceinline__ uint32_t begins() const { return first_chunk; }
};
struct MomentLaunch
{
    uint8_t *m, *v;
    uint16_t* scale;
    uint32_t entries, chunks;
    MomentEntry e[kMomentEntries];
};
static_assert(sizeof(MomentLaunch) <= 4096, "kernel arguments");

// 10 M elements: 16.1 us, 6.2 TB/s, bound by memory.
__device__ __forceinline__ void pack_chunk(const MomentLaunch& a, const MomentEntry& e, uint32_t start, bool whole)
{
    const uint32_t block = e.block + start / kMomentBlock;
    const size_t at      = (size_t)block * kMomentBlock;
    const uint32_t mine  = threadIdx.x * 8u, count = count_of(start, e.n);
    const RawEight r1 = load_any(e.m, VETRAST_F32, start, count, whole), r2 = load_any(e.v, VETRAST_F32, start, count, whole);
    float m[8], v[8];
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
    if (start + mine < (e.n + kMomentBlock - 1) / kMomentBlock * kMomentBlock)
    {
        *(uint2*)(a.m + at + mine) = c.m;
        *(uint2*)(a.v + at + mine) = c.v;
        if (mine % kMomentBlock == 0) a.scale[block + mine / kMomentBlock] = (uint16_t)c.scale;
    }
}

// Four elements' codes at a time, so that a wave's writes have no gaps, and past the L2, which holds none of what they write for long: 10 M
// elements 24.9 us with eight a lane, 18.9 with four, 15.8 past the L2. `whole`: all of them are there.
__device__ __forceinline__ void unpack_chunk(const MomentLaunch& a, const MomentEntry& e, uint32_t start, bool whole)
{
    const uint32_t block = e.block + start / kMomentBlock;
    const size_t at      = (size_t)block * kMomentBlock;
    uint32_t wm[2], wv[2], scale[2];
#pragma unroll
    for (uint32_t q = 0; q < 2; ++q)
    {
        const uint32_t i = q * (kOptimChunk / 2) + threadIdx.x * 4u;
        wm[q] = wv[q] = scale[q] = 0;
        if (whole || start + i < e.n)
        {
            wm[q]    = *(const uint32_t*)(a.m + at + i);
            wv[q]    = *(const uint32_t*)(a.v + at + i);
            scale[q] = a.scale[block + i / kMomentBlock];
        }
    }
#pragma unroll
    for (uint32_t q = 0; q < 2; ++q)
    {
        const uint32_t i = q * (kOptimChunk / 2) + threadIdx.x * 4u;
        float m[4], v[4];
        decode_four(wm[q], wv[q], scale[q], m, v);
        float *pm = e.m + start, *pv = e.v + start;
        if (whole)
        {
            typedef float Four __attribute__((ext_vector_type(4), aligned(4)));
            __builtin_nontemporal_store((Four){m[0], m[1], m[2], m[3]}, (Four*)(pm + i));
            __builtin_nontemporal_store((Four){v[0], v[1], v[2], v[3]}, (Four*)(pv + i));
        }
        else
        {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                if (start + i + j < e.n)
                {
                    pm[i + j] = m[j];
                    pv[i + j] = v[j];
                }
        }
    }
}

template <bool PACK>
__global__ void __launch_bounds__(kBlock) convert_moments_kernel(const MomentLaunch a)
{
    const ChunkFinder<finder_groups(kMomentEntries)> find(a);
    const MomentEntry& e = a.e[find(blockIdx.x)];
    const uint32_t start = (blockIdx.x - e.first_chunk) * kOptimChunk;
    const bool whole     = e.n - start >= kOptimChunk;
    if constexpr (PACK) pack_chunk(a, e, start, whole);
    else unpack_chunk(a, e, start, whole);
}
}  // namespace vetrast
