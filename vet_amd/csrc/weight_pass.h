// What a render's points gave to its pixels (weight_kernels.h): arguments and launches.
#pragma once
#include <algorithm>

#include "common.h"

namespace vetrast
{
// One view's lists.
struct WeightView
{
    const uint32_t* offsets;     // [P + 1]
    const uint32_t* kept;        // [P], 2x2 splat: fragments that were blended
    const uint64_t* fragments;
    const float* transmittance;
    const float2* projected;     // 2x2 splat
    float* weights;              // [layer][point][corner], or point by point (gradient_record)
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
    int point_major;
    float depth_accept;                          // FUZZY_BLEND
    uint32_t parts[VETRAST_MAX_LAYERS];          // workgroups of a tile of the layer
    uint32_t group_base[VETRAST_MAX_LAYERS + 1];  // first workgroup of the layer
};

struct PointWeightPass
{
    ViewPass vp;                 // of the round's first view, as for the gradients
    const uint8_t* list_is_cut;
    const uint64_t* last_key;
    const float* weights;        // of the first lane
    size_t flags_stride, last_key_stride, weights_stride;
    int view_count, K, point_major;
    float decay;
    int accumulate;              // the call's further rounds add
    float* sum;                  // [N]
};

// Workgroups that share a tile of a layer, from an upper bound of its fragments (every point lands in the layer): a wave then has about
// four times its 64 at most.
inline uint32_t weight_parts(double fragments, uint32_t tiles)
{
    const double each = fragments / tiles / (4.0 * kBlock);
    return (uint32_t)std::min(std::max(std::ceil(each), 1.0), 64.0);
}

// entries.hip
void launch_fragment_weights(const WeightPass& pass, int hits, bool fuzzy, int views, hipStream_t stream);
void launch_point_weights(const PointWeightPass& pass, int hits, hipStream_t stream);
}  // namespace vetrast
