// What every point gave to the pixels of a render: the sum of its fragments' weights in the blend, T * alpha each. A pixel's sum over its
// list is attention with the points as entries and those as its weights; accumulated over renders they say which entries to evict.
//
// Two passes, as for the gradients: fragments leave what stands in front of them, T, at a place of their own (layer, corner, point), and
// points multiply it with their alpha and add up in a fixed order, so that results do not depend on the order of atomics. A fragment is one
// scattered store; its alpha the point has at hand.
//
// These stores bound it, at 117 to 127 G a second: 1920x1080 with 2 M points has 4.6 M fragments, 37 us, beside 6.7 to clear the slots and 11 for
// the points; four 512x512 crops of the 2x2 splat have 9.0 M, 77 us, and the points 68, of which 27 to find out that no view sees a point. (A
// point's four corners in one store, if they met on the chip, would take 22 us off the crops before the work of letting them meet. 20 k points:
// two launches, 8 us.)
#pragma once
#include "weight_pass.h"

namespace vetrast
{
// Cleared slots hold what no fragment leaves, a NaN with all bits set: a zero there would be multiplied by the confidence of a point that nobody sees, which
// may be infinite or a NaN. A fragment whose T is that NaN leaves another one.
constexpr uint32_t kNoFragment = 0xFFFFFFFFu;
__device__ __forceinline__ bool has_fragment(float slot) { return __float_as_uint(slot) != kNoFragment; }
__device__ __forceinline__ float for_slot(float x) { return has_fragment(x) ? x : __uint_as_float(0x7FC00000u); }

__global__ void __launch_bounds__(kBlock) clear_slots_kernel(WeightPass a, size_t n)
{
    uint4* slots = reinterpret_cast<uint4*>(a.view[blockIdx.y].slots);
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (size_t)gridDim.x * kBlock) slots[i] = make_uint4(kNoFragment, kNoFragment, kNoFragment, kNoFragment);
}

// A wave takes the 256 pixels of a tile, whose lists are one stretch of the fragments: a lane takes a fragment, whichever pixel's it is. Tiles
// with long lists are shared by several waves, each of which takes every `parts`-th 128 fragments. Where a list was not blended to its
// end, a bit in LDS is turned over where a pixel's blended fragments begin and where they end: a fragment was blended if an odd number of bits
// up to its own is set. Neighbouring tiles of a layer go to one XCD: their fragments are of the same blocks of points, whose slots then come
// together in one L2, and are not driven out by lists that are read once (loaded the ordinary way 1080p takes 1.5 us more). (To find a
// fragment's pixel by a search over the lanes took 14 lane exchanges for 64 fragments.)
template <int HITS>
__global__ void __launch_bounds__(kBlock) fragment_weights_kernel(WeightPass a)
{
    // fragments of a lane under way at once (four crops 146.8 us of the call, with 1 147.3, with 4 151, with 8 162; 1080p 53.4, 54.0, 53.7)
    constexpr uint32_t kEach = 2, kWindow = kEach * kWave;
    __shared__ uint32_t turns[kBlock / kWave][kWindow / 32];
    const uint32_t xcd = blockIdx.x % kXcds, group = blockIdx.x / kXcds, lane = threadIdx.x % kWave;
    int l = 0;
    while (l + 1 < a.ly.L && group >= a.share_base[l + 1]) ++l;
    const uint32_t place = __builtin_amdgcn_readfirstlane((xcd * a.shares[l] + group - a.share_base[l]) * (kBlock / kWave) + threadIdx.x / kWave);
    const WeightView& v  = a.view[blockIdx.y];
    const uint32_t parts = a.parts[l], tile = place / parts, part = place - tile * parts;
    if (tile >= a.ly.tile_base[l + 1] - a.ly.tile_base[l]) return;
    const uint32_t pixel   = (a.ly.tile_base[l] + tile) * kTilePixels + 4 * lane;
    const uint4 start      = *reinterpret_cast<const uint4*>(v.offsets + pixel);
    const uint32_t next    = v.offsets[pixel + 4];
    const uint32_t starts[5] = {start.x, start.y, start.z, start.w, next};
    uint32_t keep[4];
    bool cut = false;
    if constexpr (HITS == 1)
    {
#pragma unroll
        for (int k = 0; k < 4; ++k) keep[k] = a.K > 0 ? min(starts[k + 1] - starts[k], (uint32_t)a.K) : starts[k + 1] - starts[k];
    }
    else
    {
        const uint4 kept = *reinterpret_cast<const uint4*>(v.kept + pixel);
        keep[0] = kept.x, keep[1] = kept.y, keep[2] = kept.z, keep[3] = kept.w;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) cut = cut || keep[k] < starts[k + 1] - starts[k];
    const bool any_cut   = __ballot(cut) != 0ull;
    const uint32_t begin = (uint32_t)__builtin_amdgcn_readlane((int)start.x, 0), end = (uint32_t)__builtin_amdgcn_readlane((int)next, kWave - 1);
    uint32_t* const bits = turns[threadIdx.x / kWave];
    for (uint32_t base = begin + part * kWindow; base < end; base += parts * kWindow)
    {
        bool blended[kEach];
#pragma unroll
        for (uint32_t k = 0; k < kEach; ++k) blended[k] = base + k * kWave + lane < end;
        if (any_cut)
        {
            if (lane < kWindow / 32) bits[lane] = 0u;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int k = 0; k < 4; ++k)
            {
                const uint32_t from = max(starts[k], base), to = min(starts[k] + keep[k], base + kWindow);
                if (from >= to) continue;
                atomicXor(&bits[(from - base) / 32], 1u << (from - base) % 32);
                if (to < base + kWindow) atomicXor(&bits[(to - base) / 32], 1u << (to - base) % 32);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            uint32_t odd = 0;
#pragma unroll
            for (uint32_t k = 0; k < kEach; ++k)
            {
                const uint32_t m0 = __builtin_amdgcn_readfirstlane(bits[2 * k]), m1 = __builtin_amdgcn_readfirstlane(bits[2 * k + 1]);
                const uint32_t own = (lane < 32 ? m0 >> lane : m1 >> (lane - 32)) & 1u;
                blended[k]         = blended[k] && ((__builtin_amdgcn_mbcnt_hi(m1, __builtin_amdgcn_mbcnt_lo(m0, 0u)) + own + odd) & 1u);
                odd += (uint32_t)(__popc(m0) + __popc(m1));
            }
            __builtin_amdgcn_wave_barrier();
        }
        uint32_t low[kEach];
        float T[kEach];
#pragma unroll
        for (uint32_t k = 0; k < kEach; ++k)
            if (blended[k])
            {
                low[k] = (uint32_t)__builtin_nontemporal_load(v.fragments + base + k * kWave + lane);
                T[k]   = __builtin_nontemporal_load(v.transmittance + base + k * kWave + lane);
            }
#pragma unroll
        for (uint32_t k = 0; k < kEach; ++k)
        {
            if (!blended[k]) continue;
            const uint32_t id = HITS == 1 ? low[k] : low[k] >> 2;
            if (id < (uint32_t)a.N) v.slots[((size_t)l * a.N + id) * HITS + (HITS == 1 ? 0u : low[k] & 3u)] = HITS == 1 ? for_slot(T[k]) : T[k];
        }
    }
}

// FUZZY_BLEND: a thread walks a pixel's list as the blend does, and leaves weights. The fragments of the nearest bucket share what their mean
// confidence gives; behind it a fragment is blended by itself.
__global__ void __launch_bounds__(kBlock) fragment_weights_fuzzy_kernel(WeightPass a)
{
    int l = 0;
    while (l + 1 < a.ly.L && blockIdx.x >= a.ly.tile_base[l + 1]) ++l;
    const WeightView& v  = a.view[blockIdx.y];
    const uint32_t pixel = blockIdx.x * kTilePixels + threadIdx.x;
    const uint32_t start = v.offsets[pixel], count = v.offsets[pixel + 1] - start;
    const uint32_t keep  = a.K > 0 ? min(count, (uint32_t)a.K) : count;
    if (keep == 0) return;
    const auto depth = [&](uint32_t k) { return __uint_as_float((uint32_t)(v.fragments[start + k] >> 32)); };
    const auto point = [&](uint32_t k) { return (int)(uint32_t)v.fragments[start + k]; };
    const auto conf  = [&](int id) {
        const int row = texture_row(a.index, id, a.N);
        if (row < 0) return 0.f;
        const float c = a.confidence[row];
        return a.confidence_activation ? sigmoid_canon(a.confidence_scale * c) : c;
    };
    const auto store = [&](int id, float w) {
        if ((uint32_t)id < (uint32_t)a.N) v.slots[(size_t)l * a.N + id] = for_slot(w);
    };
    uint32_t m  = 0;
    float sum   = 0.f;
    const float nearest = depth(0);
    while (m < keep && depth(m) - nearest < a.depth_accept) sum += conf(point(m++));
    const float mean = sum / (float)m, share = mean / (float)m;
    for (uint32_t k = 0; k < m; ++k) store(point(k), share);
    float T = 1.f - mean;
    for (uint32_t k = m; k < keep; ++k)
    {
        const int id  = point(k);
        const float c = conf(id);
        store(id, T * c);
        T = (1.f - c) * T;
    }
}

__device__ __forceinline__ float confidence_of(const ViewPass& vp, int i)
{
    const int row = texture_row(vp.index, i, vp.N);
    if (row < 0) return 0.f;
    const float c = vp.confidence[row];
    return vp.confidence_activation ? sigmoid_canon(vp.confidence_scale * c) : c;
}
__device__ __forceinline__ void add_weight(const PointWeightPass& a, int i, float sum)
{
    if (a.accumulate) a.sum[i] += sum;
    else a.sum[i] = (a.decay != 0.f ? a.decay * a.sum[i] : 0.f) + sum;
}

// Slots of points without a fragment say so.
__global__ void __launch_bounds__(kBlock) point_weights_cleared_kernel(PointWeightPass a)
{
    const int i = blockIdx.x * kBlock + threadIdx.x, N = a.vp.N, L = a.vp.ly.L;
    if (i >= N) return;
    const float alpha = a.fuzzy ? 1.f : confidence_of(a.vp, i);
    float sum         = 0.f;
    for (int view = 0; view < a.view_count; ++view)
    {
        float T[VETRAST_MAX_LAYERS];
#pragma unroll
        for (int l = 0; l < VETRAST_MAX_LAYERS; ++l) T[l] = l < L ? a.slots[(size_t)view * a.slots_stride + (size_t)l * N + i] : __uint_as_float(kNoFragment);
#pragma unroll
        for (int l = 0; l < VETRAST_MAX_LAYERS; ++l) sum += has_fragment(T[l]) ? alpha * T[l] : 0.f;
    }
    add_weight(a, i, sum);
}

// Slots are not cleared (slots_are_cleared): a thread finds its point's pixels again, and out whether its fragments there were blended, in the way of the
// gradients' pass. (With the 2x2 splat zeroed slots would be 64 bytes a point and view, most of which a crop does not see.)
template <int HITS>
__global__ void __launch_bounds__(kBlock) point_weights_kernel(PointWeightPass a)
{
    const int i = blockIdx.x * kBlock + threadIdx.x, N = a.vp.N;
    if (i >= N) return;
    const LayerTable& ly = a.vp.ly;
    const float4 wp      = a.vp.position[i];
    const float reach    = (float)(1 << (ly.L - 1)) + 1.f;
    const bool never     = point_is_skipped_in_all_views(a.vp, i);
    const float conf     = confidence_of(a.vp, i);
    float sum            = 0.f;
    for (int view = 0; view < a.view_count && !never; ++view)
    {
        const DeviceView& cam = a.vp.view[view];
        const uint8_t* is_cut = a.list_is_cut + (size_t)view * a.flags_stride;
        const uint64_t* last  = a.last_key + (size_t)view * a.last_key_stride;
        const float* slots    = a.slots + (size_t)view * a.slots_stride;
        Projected p;
        if (surely_outside(cam, (float)ly.w[0], (float)ly.h[0], reach, wp) || point_is_dropped(a.vp, view, i) || !project_point(cam, wp, p)) continue;
        if (!(p.ipx >= -reach && p.ipx <= (float)ly.w[0] + reach && p.ipy >= -reach && p.ipy <= (float)ly.h[0] + reach)) continue;
        const uint64_t key = (uint64_t)__float_as_uint(p.z) << 32 | (HITS == 1 ? (uint32_t)i : (uint32_t)i << 2);
        for (int l = 0; l < ly.L; ++l, p.ipx *= 0.5f, p.ipy *= 0.5f, p.radius *= 0.5f)
        {
            if (a.vp.drop_by_radius && p.radius < a.vp.radius_threshold) break;
            if constexpr (HITS == 1)
            {
                const float fx   = rintf(p.ipx), fy = rintf(p.ipy);
                const bool in    = fx >= 0.f && fx < (float)ly.w[l] && fy >= 0.f && fy < (float)ly.h[l];
                const uint32_t x = in ? (uint32_t)(int)fx : 0u, y = in ? (uint32_t)(int)fy : 0u;
                const uint32_t q = ly.base[l] + (y / kTile * (uint32_t)ly.tiles_x[l] + x / kTile) * kTilePixels + y % kTile * kTile + x % kTile;
                const bool cut   = is_cut[q] != 0;
                const float T    = slots[(size_t)l * N + i];
                if (in && (!cut || key <= last[q])) sum += a.fuzzy ? T : conf * T;
                continue;
            }
            // pixel number = part of its column + part of its row (tile_pixel)
            const float fx = floorf(p.ipx), fy = floorf(p.ipy), sx = p.ipx - fx, sy = p.ipy - fy;
            const int x = (int)fx, y = (int)fy, w = ly.w[l], h = ly.h[l];
            bool in_x[2], in_y[2];
            uint32_t of_x[2], of_y[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
            {
                in_x[k]          = (uint32_t)(x + k) < (uint32_t)w;
                in_y[k]          = (uint32_t)(y + k) < (uint32_t)h;
                const uint32_t u = in_x[k] ? x + k : 0, v = in_y[k] ? y + k : 0;
                of_x[k]          = u / kTile * kTilePixels + u % kTile;
                of_y[k]          = ly.base[l] + v / kTile * (uint32_t)ly.tiles_x[l] * kTilePixels + v % kTile * kTile;
            }
            // the corners' flags, then what they ask for, side by side
            bool kept[4], cut[4];
#pragma unroll
            for (int c = 0; c < 4; ++c)
            {
                kept[c] = in_x[c & 1] && in_y[c >> 1];
                cut[c]  = is_cut[of_x[c & 1] + of_y[c >> 1]] != 0;
            }
            const float4 slot = reinterpret_cast<const float4*>(slots)[(size_t)l * N + i];
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (kept[c] && cut[c]) kept[c] = (key | (uint32_t)c) <= last[of_x[c & 1] + of_y[c >> 1]];
            const float T[4] = {slot.x, slot.y, slot.z, slot.w};
#pragma unroll
            for (int c = 0; c < 4; ++c)
            {
                const float weight = ((c & 1) ? sx : 1.f - sx) * ((c & 2) ? sy : 1.f - sy);  // as bilinear_weight has it
                if (kept[c]) sum += T[c] * (weight * conf);
            }
        }
    }
    add_weight(a, i, sum);
}
}  // namespace vetrast
