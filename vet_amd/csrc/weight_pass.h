// What a render's points gave to its pixels (weight_kernels.h): arguments and launches.
#pragma once
#include <algorithm>
#include <cmath>

#include "common.h"

namespace vetrast
{
// One view's lists.
struct WeightView
{
    const uint32_t* offsets;  // [P + 1]
    const uint32_t* kept;     // [P], 2x2 splat: fragments that were blended
    const uint64_t* fragments;
    const float* transmittance;
    // [layer][point][corner], also for views that see little of the cloud: point after point the stores are spread over more lines (1080p 37 -> 69 us,
    // four 512x512 crops of the 2x2 splat 88 -> 116)
    float* slots;
};
struct WeightPass
{
    WeightView view[kViewLanes];
    LayerTable ly;
    const int32_t* index;
    const float* confidence;
    int confidence_activation;
    float confidence_scale;
    int N, K;
    float depth_accept;                          // FUZZY_BLEND
    uint32_t parts[VETRAST_MAX_LAYERS];           // waves of a tile of the layer
    uint32_t shares[VETRAST_MAX_LAYERS];          // workgroups of the layer on one XCD
    uint32_t share_base[VETRAST_MAX_LAYERS + 1];  // ... of the layers in front of it
};
struct PointWeightPass
{
    ViewPass vp;                 // of the round's first view, as for the gradients
    const uint8_t* list_is_cut;
    const uint64_t* last_key;
    const float* slots;          // of the first lane
    size_t flags_stride, last_key_stride, slots_stride;
    int view_count;
    int fuzzy;                   // slots hold weights, else transmittances
    float decay;
    int accumulate;              // the call's further rounds add
    float* sum;                  // [N]
};

// Waves that share a tile of a layer, from an upper bound of its fragments (every point lands in the layer). A wave then has 128 at most with one hit
// per layer, all of them under way at once, for the waves of the fullest tiles are the last (1080p: 500 k points 22.3 us of the call, with 256 25.3,
// with 1024 50.5; 2 M 53.4, 53.1 and 77), and 1024 with the 2x2 splat, with which mostly crops are rendered, that see a part of the points (four
// 512x512 crops: 147 us, with 256 and four times as many waves, most of them without a fragment, 155, with 4096 155).
inline uint32_t weight_parts(double fragments, uint32_t tiles, int hits)
{
    return (uint32_t)std::min(std::max(std::ceil(fragments / tiles / (hits == 1 ? 128.0 : 1024.0)), 1.0), 64.0);
}

// Whether slots are cleared for points without a fragment, and points read them without looking where they are. With one hit per layer, and where there are
// many points: 2 M at 1080p 54.8 us (finding pixels again 65), 200 k 18.1 (18.8), 400 k in one layer of 256x256 13.7 (15.2); for few ones it
// is a launch too many, 100 k 12.8 us (12.4), 20 k 9.6 (8.2).
inline bool slots_are_cleared(int hits, int points) { return hits == 1 && points > 131072; }

// entries.hip
void launch_fragment_weights(const WeightPass& pass, int hits, bool fuzzy, int views, hipStream_t stream);
void launch_point_weights(const PointWeightPass& pass, int hits, hipStream_t stream);
}  // namespace vetrast
