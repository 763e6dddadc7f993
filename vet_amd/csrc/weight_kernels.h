// What every point gave to the pixels of a render: the sum of its fragments' weights in the blend, T * alpha each. A pixel's sum over its
// list is attention with the points as entries and those as its weights; accumulated over renders they say which entries to evict.
//
// Two passes, as for the gradients: fragments leave their weights at a place of their own (layer, corner, point), and points add theirs up
// in a fixed order, so that results do not depend on the order of atomics.
#pragma once
#include "weight_pass.h"

namespace vetrast
{
__device__ __forceinline__ float confidence_of(const WeightPass& a, int row)
{
    const float c = a.confidence[row];
    return a.confidence_activation ? sigmoid_canon(a.confidence_scale * c) : c;
}

// A workgroup takes a tile, each of its waves 64 consecutive pixels, whose lists are one stretch of the fragments: a lane takes a fragment,
// whichever pixel's it is. Only where a list was not blended to its end a lane has to find its pixel. Tiles with long lists are shared by several
// workgroups, each of which takes every `parts`-th 64 fragments.
template <int HITS>
__global__ void __launch_bounds__(kBlock) fragment_weights_kernel(WeightPass a)
{
    int l = 0;
    while (l + 1 < a.ly.L && blockIdx.x >= a.group_base[l + 1]) ++l;
    const WeightView& v    = a.view[blockIdx.y];
    const uint32_t group   = blockIdx.x - a.group_base[l], tile = group / a.parts[l], part = group - tile * a.parts[l];
    const uint32_t lane    = threadIdx.x % kWave;
    const uint32_t pixel   = (a.ly.tile_base[l] + tile) * kTilePixels + threadIdx.x;
    const uint32_t start   = v.offsets[pixel], next = v.offsets[pixel + 1];
    const uint32_t count   = next - start;
    const uint32_t keep    = HITS == 1 ? (a.K > 0 ? min(count, (uint32_t)a.K) : count) : v.kept[pixel];
    const bool any_cut     = __ballot(keep < count) != 0ull;
    const uint32_t begin   = (uint32_t)__builtin_amdgcn_readlane((int)start, 0), end = (uint32_t)__builtin_amdgcn_readlane((int)next, kWave - 1);
    for (uint32_t base = begin + part * kWave; base < end; base += a.parts[l] * kWave)
    {
        const uint32_t at = base + lane;
        bool blended      = at < end;
        if (any_cut)
        {
            // the last pixel that starts at or in front of the fragment
            uint32_t owner = 0;
#pragma unroll
            for (uint32_t step = kWave / 2; step > 0; step /= 2)
                if ((uint32_t)__shfl((int)start, (int)(owner + step), kWave) <= at) owner += step;
            const uint32_t first = (uint32_t)__shfl((int)start, (int)owner, kWave), some = (uint32_t)__shfl((int)keep, (int)owner, kWave);
            blended              = blended && at - first < some;
        }
        if (!blended) continue;
        const uint32_t low = (uint32_t)v.fragments[at];
        const float T      = v.transmittance[at];
        const int id       = HITS == 1 ? (int)low : (int)(low >> 2);
        if ((uint32_t)id >= (uint32_t)a.N) continue;
        const int row = texture_row(a.index, id, a.N);
        float alpha   = row < 0 ? 0.f : confidence_of(a, row);
        if constexpr (HITS != 1)
        {
            float2 position = v.projected[id];
            for (int k = 0; k < l; ++k) position.x *= 0.5f, position.y *= 0.5f;
            alpha = bilinear_weight(position.x, position.y, (int)(low & 3u)) * alpha;
        }
        v.weights[gradient_record(a.point_major, a.N, a.ly.L, l, id) * HITS + (HITS == 1 ? 0u : low & 3u)] = T * alpha;
    }
}

// FUZZY_BLEND: a thread walks a pixel's list as the blend does. The fragments of the nearest bucket share what their mean confidence
// gives; behind it a fragment is blended by itself.
__global__ void __launch_bounds__(kBlock) fragment_weights_fuzzy_kernel(WeightPass a)
{
    int l = 0;
    while (l + 1 < a.ly.L && blockIdx.x >= a.group_base[l + 1]) ++l;
    const WeightView& v  = a.view[blockIdx.y];
    const uint32_t pixel = (a.ly.tile_base[l] + (blockIdx.x - a.group_base[l])) * kTilePixels + threadIdx.x;
    const uint32_t start = v.offsets[pixel], count = v.offsets[pixel + 1] - start;
    const uint32_t keep  = a.K > 0 ? min(count, (uint32_t)a.K) : count;
    if (keep == 0) return;
    const auto depth = [&](uint32_t k) { return __uint_as_float((uint32_t)(v.fragments[start + k] >> 32)); };
    const auto point = [&](uint32_t k) { return (int)(uint32_t)v.fragments[start + k]; };
    const auto conf  = [&](int id) {
        const int row = texture_row(a.index, id, a.N);
        return row < 0 ? 0.f : confidence_of(a, row);
    };
    const auto store = [&](int id, float w) {
        if ((uint32_t)id < (uint32_t)a.N) v.weights[gradient_record(a.point_major, a.N, a.ly.L, l, id)] = w;
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

// A thread finds its point's pixels again, and out whether its fragments there were blended, in the way of the gradients' pass.
template <int HITS>
__global__ void __launch_bounds__(kBlock) point_weights_kernel(PointWeightPass a)
{
    const int i = blockIdx.x * kBlock + threadIdx.x, N = a.vp.N;
    if (i >= N) return;
    const LayerTable& ly = a.vp.ly;
    const float4 wp      = a.vp.position[i];
    const float reach    = (float)(1 << (ly.L - 1)) + 1.f;
    const bool never     = point_is_skipped_in_all_views(a.vp, i);
    float sum            = 0.f;
    for (int view = 0; view < a.view_count && !never; ++view)
    {
        const DeviceView& cam  = a.vp.view[view];
        const uint8_t* is_cut  = a.list_is_cut + (size_t)view * a.flags_stride;
        const uint64_t* last   = a.last_key + (size_t)view * a.last_key_stride;
        const float* weights   = a.weights + (size_t)view * a.weights_stride;
        Projected p;
        if (point_is_dropped(a.vp, view, i) || !project_point(cam, wp, p)) continue;
        if (!(p.ipx >= -reach && p.ipx <= (float)ly.w[0] + reach && p.ipy >= -reach && p.ipy <= (float)ly.h[0] + reach)) continue;
        const uint64_t depth_key = (uint64_t)__float_as_uint(p.z) << 32;
        for (int l = 0; l < ly.L; ++l, p.ipx *= 0.5f, p.ipy *= 0.5f, p.radius *= 0.5f)
        {
            if (a.vp.drop_by_radius && p.radius < a.vp.radius_threshold) break;
#pragma unroll
            for (int h = 0; h < HITS; ++h)
            {
                uint32_t tile, in_tile;
                if (!layer_hit<HITS>(ly, l, p.ipx, p.ipy, h, tile, in_tile)) continue;
                const uint32_t q   = tile * kTilePixels + in_tile;
                const uint64_t key = depth_key | (HITS == 1 ? (uint32_t)i : (((uint32_t)i << 2) | (uint32_t)h));
                if (is_cut[q] && (HITS != 1 || a.K > 0) && key > last[q]) continue;
                sum += weights[gradient_record(a.point_major, N, ly.L, l, i) * HITS + h];
            }
        }
    }
    if (a.accumulate) a.sum[i] += sum;
    else a.sum[i] = (a.decay != 0.f ? a.decay * a.sum[i] : 0.f) + sum;
}
}  // namespace vetrast
