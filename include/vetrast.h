/*
 * vetrast — C ABI of the MI355X (gfx950) blending point rasterizer.
 *
 * This header is the whole drop-in boundary: plain pointers, sizes and PODs, no torch or HIP types.
 * All `device` pointers are hipMalloc'ed (or torch-allocated) memory on the GPU the context was created
 * on; all `host` pointers are ordinary host memory that only has to stay valid for the duration of the call.
 * Every entry point returns 0 on success or a negative vetrast_status, never aborts, never allocates device
 * memory behind the caller's back (the caller owns inputs, outputs and the workspace) and, unless stated
 * otherwise, only enqueues work on the given stream (pass the hipStream_t as `void*`, NULL = default stream).
 * A context serves one host thread at a time.
 *
 * The reference has no C ABI; its seam is the libtorch function
 *   std::vector<torch::Tensor> BlendPointCloud(NeuralRenderInfo*)          src/lib/rendering/PointRenderer.h:53
 *   torch::autograd::PointRender::forward / ::backward                      src/lib/rendering/PointRenderer.h:39-47
 * implemented by BlendPointCloudForward / BlendPointCloudBackward            src/lib/rendering/PointRenderer.cu:657,1111
 * The entry points below are what a libtorch shim with that signature binds (see vet_amd/torch_ext).
 */
#ifndef VETRAST_H
#define VETRAST_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define VETRAST_MAX_LAYERS 5   /* max_layers, src/lib/rendering/RenderConstants.h:33 */
#define VETRAST_MAX_CHANNELS 4 /* CUDA_KERNEL_ASSERT(num_texture_channels <= 4), src/lib/rendering/RenderForward.cu:1322 */

typedef enum vetrast_status
{
    VETRAST_OK                  = 0,
    VETRAST_ERR_INVALID_ARG     = -1, /* null pointer, size out of range, misaligned workspace */
    VETRAST_ERR_WORKSPACE_SMALL = -2, /* workspace_bytes below vetrast_forward_workspace_bytes() */
    VETRAST_ERR_HIP             = -3, /* a HIP runtime call failed; see vetrast_last_hip_error() */
    VETRAST_ERR_UNSUPPORTED     = -4, /* a reference feature outside the blending path (OCam, normals, ...) */
    VETRAST_ERR_BAD_INPUT_DATA  = -5, /* device-side check failed (non-zero distortion that was not allowed), from
                                         vetrast_query_device_flags */
    VETRAST_ERR_TOO_LARGE       = -6  /* size beyond the fixed maximum of an entry point that allocates nothing */
} vetrast_status;

/* Camera model tag of a view. Mirrors enum CameraModel, src/lib/data/SceneData.h:30-35.
 * Only PINHOLE_DISTORTION is implemented; non-zero distortion coefficients need vetrast_params.allow_distortion. */
#define VETRAST_CAMERA_PINHOLE_DISTORTION 0
#define VETRAST_CAMERA_OCAM 1
#define VETRAST_CAMERA_SPHERICAL 2

/* One view of the batch. Mirrors struct ReducedImageInfo, src/lib/data/SceneData.h:39-50, field by field
 * (the Eigen members are spelled out as floats). The reference passes it by value as a kernel argument
 * (CountingPrepassMulti, src/lib/rendering/RenderForward.cu:807); so does this library. */
typedef struct vetrast_view
{
    int32_t w, h;              /* full-resolution size of layer 0; must be equal for all views of a call */
    int32_t image_index;       /* row of poses_se3 / pose gradient */
    int32_t camera_index;      /* row of intrinsics / intrinsics gradient */
    int32_t camera_model_type; /* VETRAST_CAMERA_* */
    float crop_transform[5];   /* fx, fy, cx, cy, s of IntrinsicsPinholef crop_transform */
    float crop_rotation[4];    /* r00, r01, r10, r11 (row-major; Eigen stores the 2x2 column-major) */
} vetrast_view;

/* Scalar parameters of the path. Mirrors the RenderParams fields the blending path reads
 * (src/lib/data/Settings.h:19-93, copied into DeviceRenderParams at src/lib/rendering/RenderConstants.h:105-126). */
typedef struct vetrast_params
{
    int32_t num_texture_channels;         /* C, 1..4 */
    int32_t num_layers;                   /* L, 1..5  (NeuralRenderInfo::num_layers) */
    int32_t debug_max_list_length;        /* K; <= 0 means no cut (reference default -1) */
    int32_t use_environment_map;          /* 0: the background colour is blended behind the last fragment */
    int32_t need_point_gradient;          /* backward: compute the position gradient */
    int32_t viewer_only;                  /* with it, points with confidence < stability_cutoff_value are skipped */
    float stability_cutoff_value;
    int32_t drop_out_points_by_radius;    /* stop descending layers once the splat radius falls below the threshold */
    float drop_out_radius_threshold;
    int32_t output_background_mask;       /* forward also writes out_mask = (weight == 0 ? mask_value : 1) */
    float output_background_mask_value;
    int32_t check_normal;                 /* must be 0 (needs saiga's UnpackNormal10Bit) */
    /* Two switches for behaviours of the reference that are accidents of its implementation: */
    int32_t quirk_background_confidence_leak; /* 1: the background pseudo-fragment also adds its alpha gradient to
                                                 grad_confidence[0], as src/lib/rendering/RenderBackward.cu:1157 does */
    int32_t point_gradient_normalization;     /* 0: leave sums and counts; 1: row i / count i;
                                                 2: literal reference (vec3 stride over the [N,4] buffer,
                                                 src/lib/rendering/PointRenderer.cu:1278-1279) */
    /* Pose / intrinsics gradients (only computed when the matching buffers of vetrast_backward_args are given): */
    float K_gradient_factor;                  /* RenderParams::K_gradient_factor, src/lib/data/Settings.h:55 */
    int32_t camera_gradient_normalization;    /* 0: leave sums and counts; 1: divide each pose / intrinsics row by its
                                                 count as src/lib/rendering/PointRenderer.cu:1253-1308 does (the count
                                                 grows by 1/1024 per fragment, so this is 1024 x the mean) */
    int32_t render_mode;                      /* RenderParams::render_mode, src/lib/data/Settings.h: 1 = FULL_BLEND
                                                 (a point lands in the pixel it rounds to), 3 = BILINEAR_BLEND (a point
                                                 lands in the 2x2 pixels around it, alpha = bilinear weight x confidence,
                                                 blending stops once the transmittance falls below 0.001), 2 =
                                                 FUZZY_BLEND (FULL_BLEND lists; the nearest fragments of a pixel that
                                                 lie within depth_accept_blend of the first one are averaged before
                                                 they are blended). Other values (0 = FUZZY_DT, the
                                                 depth-test mode, included) are refused. */
    /* The steps VET runs on the optimised tensors right before the rasterizer, fused into it
     * (NeuralPointTextureImpl::PrepareConfidence / PrepareTexture, src/lib/models/NeuralTexture.h:38-55; called from
     * src/lib/models/Pipeline.cpp:113-124). With them on, `confidence`, `texture` and `background` are the RAW tensors
     * and the gradients vetrast_backward returns are those of the raw tensors. */
    int32_t confidence_activation;            /* 0: confidence is used as given; 1: sigmoid(confidence_scale * confidence) */
    float confidence_scale;                   /* 10 + sigmoid_narrowing_factor * epoch in VET */
    int32_t texture_abs;                      /* 1: |texture| and |background| (PipelineParams::non_subzero_texture) */
    float depth_accept_blend;                 /* FUZZY_BLEND: depth range of a bucket, RenderParams::depth_accept_blend
                                                 (src/lib/data/Settings.h:42, default 0.01); must lie in (0, 1e4) */
    /* A hint for speed only; results do not depend on it. The pixels of a layer are cut into bins sized so that a bin
     * is expected to hold about a thousand fragments if EVERY point lands in the layer. A view that sees a part of the
     * cloud (VET trains on 512x512 crops, configs/config.ini:27) or drops points by radius at the coarse layers then
     * gets bins far too small. expected_fragments[l] > 0 says how many fragments ONE view is expected to leave in layer
     * l (e.g. what the previous call left there: offsets[layer_pixel_base[l + 1]] - offsets[layer_pixel_base[l]]); the
     * bins of that layer are sized for it. 0: every point. No counterpart in the reference. */
    float expected_fragments[VETRAST_MAX_LAYERS];
    /* Lens distortion. The reference distorts the normalised image point with saiga's distortNormalizedPoint
     * (src/lib/rendering/PointRendererHelper.h:207,348), which is not part of its source tree; cameras with non-zero
     * coefficients are therefore refused (VETRAST_ERR_BAD_INPUT_DATA through vetrast_query_device_flags) unless
     * allow_distortion is set. With it, columns 5..12 of `intrinsics` are taken as k1 k2 k3 k4 k5 k6 p1 p2 (the order
     * of src/lib/data/SceneData.cpp:464-478) of the rational model
     *   x' = x (1 + k1 r^2 + k2 r^4 + k3 r^6) / (1 + k4 r^2 + k5 r^4 + k6 r^6) + 2 p1 x y + p2 (r^2 + 2 x^2)
     *   y' = y (   same ratio   )                                              + p1 (r^2 + 2 y^2) + 2 p2 x y
     * and the backward pass returns their gradient scaled as src/lib/rendering/RenderBackward.cu:1440-1455 scales it
     * (k3 x 0.25, k4..k6 and p1, p2 x 0.1, everything x distortion_gradient_factor). PARITY WITH THE REFERENCE IS
     * UNPINNED for such cameras: the formula is the published one the coefficient layout implies, not saiga's code,
     * and RenderParams::dist_cutoff (points beyond the radius where the polynomial stops being monotonic are culled
     * by saiga) is not applied. */
    int32_t allow_distortion;
    float distortion_gradient_factor;         /* RenderParams::distortion_gradient_factor, src/lib/data/Settings.h:54 */
} vetrast_params;

#define VETRAST_RENDER_FULL_BLEND 1
#define VETRAST_RENDER_FUZZY_BLEND 2
#define VETRAST_RENDER_BILINEAR_BLEND 3

typedef struct vetrast_ctx vetrast_ctx;

/* Per-kernel timing scopes, named after the reference's CudaTimerSystem scopes
 * (src/lib/rendering/PointRenderer.cu:249,770,791,843,872,886,1222,1252). */
typedef enum vetrast_scope
{
    VETRAST_SCOPE_PREPARE = 0,      /* "Build Cache": zero-fill, view preparation */
    VETRAST_SCOPE_PACK,             /* "Build Cache": descriptor interleave; it rides along with the COUNT kernel of the
                                       first view, so this scope reports no launches of its own */
    VETRAST_SCOPE_COUNT,            /* "CountingPass": fragments per bin (a 16x16 pixel tile or a piece of one) and, in
                                       the same pass over the points, the fragment records written to their bins */
    VETRAST_SCOPE_SCAN,             /* "CreateAndAllocateBuffers" (prefix scan over the bins; no allocation here) */
    VETRAST_SCOPE_FILL,             /* "CollectionPass", first half: the records that did not fit their bin's own room
                                       are filed behind the scan (an almost empty kernel as a rule) */
    VETRAST_SCOPE_BUILD,            /* "CollectionPass" second half + "SortingPass" + "BlendingPass": one pass per bin */
    VETRAST_SCOPE_BACKWARD_PREPARE, /* "Prepare Backward": zero-fill of gradient buffers */
    VETRAST_SCOPE_BACKWARD_BLEND,   /* "BlendBackwards", per-pixel part */
    VETRAST_SCOPE_BACKWARD_GATHER,  /* "BlendBackwards", per-point sum of the stored fragment gradients */
    VETRAST_SCOPE_BACKWARD_POST,    /* "Post Process Gradient" (a launch of its own while profiling; else a call with camera
                                       gradients does it beside them) */
    VETRAST_SCOPE_LIFT_ERROR,       /* vetrast_lift_error (the reference times FillSceneGridWithLoss in no scope) */
    VETRAST_SCOPE_COUNT_
} vetrast_scope;

/* Byte offsets of the arrays inside the forward workspace, so that a caller (or a test) can read the
 * per-pixel fragment lists. Pixels are numbered tile by tile: every layer is cut into 16x16 pixel tiles (the last
 * column / row of tiles may hang over the image; those pixels exist in the numbering and have empty lists), and
 *   q = 256 * (layer_tile_base[l] + (y / 16) * layer_tiles_x[l] + x / 16) + 16 * (y % 16) + x % 16. */
typedef struct vetrast_workspace_layout
{
    int32_t layer_w[VETRAST_MAX_LAYERS];
    int32_t layer_h[VETRAST_MAX_LAYERS];
    int32_t layer_tiles_x[VETRAST_MAX_LAYERS];        /* tiles per row of the layer = ceil(w_l / 16) */
    int32_t reserved0;
    int64_t layer_tile_base[VETRAST_MAX_LAYERS + 1];  /* first tile of the layer; [L] = number of tiles T */
    int64_t layer_pixel_base[VETRAST_MAX_LAYERS + 1]; /* 256 * layer_tile_base; [L] = pixel numbers P of one view */
    int64_t fragment_capacity;                        /* N * L * hits_per_layer, the per-view upper bound on fragments */
    int32_t hits_per_layer;                           /* 1 (FULL_BLEND) or 4 (BILINEAR_BLEND): fragments of a point per layer */
    int32_t reserved1;
    size_t total_bytes;
    /* per-view arrays: offset of view b = base + b * stride */
    size_t offsets_base, offsets_stride;     /* uint32 [P+1]: exclusive scan of per-pixel counts; [P] = fragments of the view */
    size_t fragments_base, fragments_stride; /* uint64 [N*L]: (depth_bits << 32) | point_id, per pixel ascending; only the
                                                first min(count, K) entries of a pixel's list are sorted and meaningful */
    size_t transmittance_base, transmittance_stride; /* float [N*L]: transmittance in front of each kept fragment */
    size_t weight_base, weight_stride;       /* float [P]: final transmittance per pixel (the reference's `weight` image) */
    size_t kept_base, kept_stride;           /* uint32 [P], BILINEAR_BLEND only: fragments of the pixel's list that took part in
                                                the blend (FULL_BLEND: min(count, K), not stored) */
    size_t cut_flags_base, cut_flags_stride; /* uint8 [P]: 1 where some fragments of the pixel's list did not (top-K cut, saturation) */
    /* shared by all views */
    size_t packed_base;    /* float [N][8]: descriptor (4, zero padded), confidence, 3 pad */
    size_t slots_base;     /* uint32, shaped like the log: rank inside its bin of every logged record (scratch) */
    size_t views_base;     /* prepared per-view camera constants */
    size_t scan_partials_base; /* per lane: partial sums of the scan, behind them the list of the bins that a workgroup builds */
    int64_t num_bins;      /* bins of one view: runs of 256 / 64 / 16 / 4 consecutive pixel numbers, chosen per layer from N */
    size_t bin_counts_base, bin_counts_stride; /* per view, uint32 [2][num_bins+1 padded]: fragments per bin, and their
                                                  exclusive scan (in place of the counts where a view has more than
                                                  15 360 bins) */
    size_t binned_base;    /* uint32 [N*L*hits][4]: compact array of fragment records (key low, key high, pixel in bin, 0),
                              only used for the records beyond a bin's own room; scratch. In FULL_BLEND / FUZZY_BLEND with
                              N <= 2^24 a record is uint32 [2]: (depth bits, point id << 8 | pixel in bin) */
    size_t flags_base;     /* uint32 [4] device status flags, then at +64 bytes float [4]: the background as it is blended */
    size_t forward_only_bytes; /* a forward call with save_for_backward = 0 needs only this much */
    size_t partial_base;   /* float [L][N][8]: backward scratch, gradient record of the fragment of point i in layer l (with
                              the 2x2 splat float [L][N][4][2], behind which follows float [P][4], the upstream gradient
                              with its channels side by side) */
    size_t background_partial_base; /* float [workgroups][8]: backward scratch, per-workgroup background-gradient sums */
    size_t camera_partial_base;     /* double [ceil(N/256)][12]: backward scratch, per-workgroup pose / intrinsics sums */
    /* scratch shared by all views: the scatter pass writes the records of a bin to the bin's own room while their rank
     * is below the room's size (2048 records where about a thousand are expected per bin, 1024 where at most 512 are);
     * records beyond that go to a log of 256 segments (record + bin, rank in the slots array) and are filed into the
     * compact array after the scan. log_cursor: per view, 256 uint32 64 bytes apart, entries in every segment.
     * The log and the slots array only live inside a forward call: partial_base == log_base, the scratch of the
     * backward call lies on top of them (forward_only_bytes covers the log, total_bytes both). */
    size_t primary_base;   /* the rooms, layer after layer, bin after bin: 16-byte records, or 8-byte ones (see binned_base) */
    size_t log_base;       /* uint32 [256][ceil(ceil(N/256)/256)*256*L*hits][4] */
    size_t log_cursor_base;
    size_t last_key_base, last_key_stride;   /* per view, uint64 [P]: where cut_flags is 1, the key of the last fragment of
                                                the pixel's list that took part in the blend (0 if none did) */
    size_t projected_base, projected_stride; /* per view, float [N][2], BILINEAR_BLEND only (stride 0 otherwise): image
                                                position of every visible point at layer 0, from which the blend and its
                                                backward pass form the bilinear weights */
    /* A call with several views takes them view_lanes = min(num_views, 4) at a time: every kernel of the call is one
     * launch for the views of such a round (view b of the call on lane b % view_lanes), so the scratch that one view
     * needs exists once per lane: lane k's copy of binned, primary and scan_partials lies k * the stride behind the
     * base, its copy of the log / slots / partial / background_partial block k * lane_scratch_stride behind theirs. */
    int32_t view_lanes;
    int32_t reserved2;
    size_t binned_stride, primary_stride, scan_partials_stride, lane_scratch_stride;
} vetrast_workspace_layout;

/* Arguments of the forward pass. Replaces the inputs PointRender::forward receives
 * (src/lib/rendering/RenderInfo.cpp:25-29,34-43) plus what it reads through info->scene. */
typedef struct vetrast_forward_args
{
    int32_t num_points; /* N */
    int32_t num_views;  /* B = info->images.size() */
    int32_t num_poses;  /* F, rows of poses_se3 */
    int32_t num_cameras;
    const float* position;    /* device [N,4] x,y,z,drop-out radius (t_position, src/lib/rendering/NeuralPointCloudCuda.h:193-224) */
    const int32_t* index;     /* device [N] texture index of a point (t_index) or NULL for the identity */
    const float* texture;     /* device [C,N] planar descriptors */
    const float* confidence;  /* device [N] (the reference's [1,N]) already in (0,1) */
    const float* background;  /* device [C] */
    const float* dropout;     /* device [B,N], a point is skipped in view b where the value == 1; NULL = none */
    const double* poses_se3;  /* device [F,8] world->camera: unit quaternion x,y,z,w, translation, 1 pad
                                 (src/lib/data/NeuralStructure.cpp:15-28) */
    const float* intrinsics;  /* device [num_cameras,13]: fx,fy,cx,cy,s,k1..k6,p1,p2 (src/lib/data/NeuralStructure.cpp:65-99) */
    const vetrast_view* views; /* host [B] */
    vetrast_params params;
    int32_t save_for_backward; /* also store the per-fragment transmittance the backward pass reads */
    float* out[VETRAST_MAX_LAYERS];      /* device, layer l: [B,C,h_l,w_l] contiguous NCHW; fully overwritten */
    float* out_mask[VETRAST_MAX_LAYERS]; /* device, layer l: [B,1,h_l,w_l]; only with output_background_mask */
    void* workspace;                     /* device, 256-byte aligned */
    size_t workspace_bytes;
    /* Optional, layer l: device [B,1,h_l,w_l], the transmittance left behind the last blended fragment of every pixel
     * (1 where no point landed): the `weight` tensor of the reference's layer cache
     * (src/lib/rendering/RenderForward.cu:1355-1356), which PointRenderModuleImpl::forward hands to the environment map
     * (src/lib/rendering/RenderModule.cpp:132-196). NULL = not wanted. */
    float* out_weight[VETRAST_MAX_LAYERS];
    /* Optional, device [N]: a permutation of 0..N-1, the order in which the binning pass walks the points (thread i
     * takes point point_order[i]). Results do not depend on it, bit for bit; the time of the binning pass does: it
     * groups the points of a wave by bin before it touches global counters, so it wants neighbours in the array to be
     * neighbours in space. A cloud in the order of VET's preprocessing (src/lib/data/SceneData.cpp:105-108) needs none;
     * one that has grown since (NeuralScene::AddNewPoints appends, src/lib/data/NeuralScene.cpp:1013) or comes in
     * file order does. Point ids everywhere else (index, gradients, dropout) stay the caller's. NULL = array order.
     * No counterpart in the reference. */
    const int32_t* point_order;
    /* Optional, device float [N][8], 32-byte aligned: the descriptor records vetrast_pack_descriptors wrote from THIS
     * texture and confidence under THESE params (num_texture_channels, confidence_activation, confidence_scale,
     * texture_abs). The call then reads a fragment's descriptor and confidence from it and leaves out the interleave
     * it otherwise does on the side in every call: for callers that render a scene more than once between changes of
     * its texture (a viewer; evaluation). The caller vouches that the records are current; vetrast_backward reads the
     * same array. NULL = the call interleaves for itself, into the workspace. No counterpart in the reference, which
     * reads the planar tensors per channel (src/lib/rendering/RenderForward.cu:1338-1342). */
    const float* packed_descriptors;
    /* Optional: drop-out of points without a mask in memory, instead of `dropout` (which must be NULL then). Point i is skipped in view b
     * where vetrast_dropout would leave out element b * num_points + i, with p = point_dropout, seed = dropout_seed and step =
     * dropout_step (+ *dropout_device_step, device, where it isn't NULL: for calls that are captured in a graph). What a backward
     * pass is handed has to be what the forward pass had, *dropout_device_step included. 0: none. */
    double point_dropout;
    uint64_t dropout_seed, dropout_step;
    const int64_t* dropout_device_step;
} vetrast_forward_args;

/* Arguments of the backward pass. Replaces BlendPointCloudBackward's inputs and its seven returned tensors
 * (src/lib/rendering/PointRenderer.cu:1111-1323). The workspace and `out` must be those of the matching forward call
 * (made with save_for_backward = 1) and unchanged since; this is the saved state of
 * src/lib/rendering/PointRenderer.cu:1027-1059. fwd.out_mask is not used and may be left NULL. */
typedef struct vetrast_backward_args
{
    vetrast_forward_args fwd;                      /* same values as passed to vetrast_forward */
    const float* grad_out[VETRAST_MAX_LAYERS];     /* device, layer l: [B,C,h_l,w_l] upstream gradient */
    float* grad_texture;     /* device [C,N]; overwritten */
    float* grad_confidence;  /* device [N]; overwritten */
    float* grad_background;  /* device [C]; overwritten */
    float* grad_points;      /* device [N,4] or NULL (points do not require grad); xyz sums (w stays 0); overwritten */
    float* grad_point_count; /* device [N]; number of fragments that contributed to a point; required with grad_points */
    /* Optional camera gradients, accumulated over every fragment that gets a position gradient
     * (src/lib/rendering/RenderBackward.cu:1418-1459). NULL = not wanted. */
    double* grad_pose;           /* device [F,6]: d/d(se3 tangent: translation, rotation) of pose row image_index; overwritten */
    float* grad_pose_count;      /* device [F]: fragments / 1024 per pose row; required with grad_pose */
    float* grad_intrinsics;      /* device [num_cameras,13]: fx,fy,cx,cy scaled by K_gradient_factor; the skew column is
                                    zeroed as in the reference; the 8 distortion columns are filled where
                                    vetrast_params.allow_distortion is set, else stay 0; overwritten */
    float* grad_intrinsics_count; /* device [num_cameras]: fragments / 1024 per camera row; required with grad_intrinsics */
} vetrast_backward_args;

/* What every point gave to the pixels of a render: weight[i] = decay * weight[i] + the sum, over the views, layers and pixels in which a
 * fragment of point i was blended, of its weight there, the transmittance in front of it times its alpha (its confidence; with the 2x2
 * splat times the corner's weight; in FUZZY_BLEND its share of the bucket's). That is the derivative of the sum of all pixels of one
 * channel by the point's descriptor; a point without a fragment adds nothing, whatever its confidence. Accumulated over renders it says which points a budget should keep (vetrast_select_kept).
 * Sums are formed in float32 in a fixed order, without atomics, and kept so from call to call. No counterpart in the reference, which removes points by their
 * confidence alone (src/apps/train.cpp:727-741). */
typedef struct vetrast_point_weights_args
{
    vetrast_forward_args fwd; /* same values as passed to vetrast_forward, with save_for_backward = 1; workspace and inputs unchanged
                                 since. The backward scratch of the workspace is written: not between or during other calls on it */
    float* weight;            /* device [N] */
    float decay;              /* finite, >= 0; 0: the old values are not read */
    int32_t reserved;
} vetrast_point_weights_args;
int vetrast_point_weights(vetrast_ctx* ctx, const vetrast_point_weights_args* args, void* stream);

/* Create / destroy a context bound to the current HIP device. The context owns only a few HIP events. */
int vetrast_create(vetrast_ctx** out_ctx);
void vetrast_destroy(vetrast_ctx* ctx);

/* Layer pyramid by repeated integer halving (src/lib/rendering/PointRenderer.cu:351-381). Pure host arithmetic. */
int vetrast_layer_sizes(int32_t w, int32_t h, int32_t num_layers, int32_t* layer_w, int32_t* layer_h);

/* Size and layout of the workspace a forward call with these dimensions needs. Pure host arithmetic. The reference
 * sizes its fragment buffers from a device->host read of the scan total (src/lib/rendering/PointRenderer.cu:811-821);
 * here the buffer has the upper bound N*L entries per view instead, so no read-back is needed. */
int vetrast_workspace_layout_for(int32_t num_points, int32_t num_views, int32_t num_layers, int32_t w, int32_t h,
                                 vetrast_workspace_layout* layout);
/* The same for a given render mode (BILINEAR_BLEND needs room for four fragments per point and layer);
 * vetrast_workspace_layout_for and vetrast_forward_workspace_bytes are the FULL_BLEND case. */
int vetrast_workspace_layout_for_mode(int32_t num_points, int32_t num_views, int32_t num_layers, int32_t w, int32_t h,
                                      int32_t render_mode, vetrast_workspace_layout* layout);
size_t vetrast_forward_workspace_bytes(int32_t num_points, int32_t num_views, int32_t num_layers, int32_t w, int32_t h);

/* Forward: project, count, scan, fill, per-pixel sort by (depth bits, point id), top-K cut, front-to-back blend.
 * Replaces BlendPointCloudForward in FULL_BLEND mode (src/lib/rendering/PointRenderer.cu:657-1069). */
int vetrast_forward(vetrast_ctx* ctx, const vetrast_forward_args* args, void* stream);

/* Backward: gradients to descriptors, confidence, background and point positions.
 * Replaces BlendPointCloudBackward in FULL_BLEND mode (src/lib/rendering/PointRenderer.cu:1111-1323). */
int vetrast_backward(vetrast_ctx* ctx, const vetrast_backward_args* args, void* stream);

/* Blocking: waits for the stream, then reads the device flag word of the workspace. Returns VETRAST_OK or
 * VETRAST_ERR_BAD_INPUT_DATA (a camera with non-zero distortion coefficients was used; the reference's saiga
 * distortion model is not available, so such input is flagged instead of guessed). */
int vetrast_query_device_flags(vetrast_ctx* ctx, const void* workspace, const vetrast_workspace_layout* layout,
                               void* stream);

/* Writes the descriptor records of vetrast_forward_args.packed_descriptors: row i = texture[0..C-1][i] (|.| with
 * texture_abs), then confidence[i] (sigmoid(confidence_scale * .) with confidence_activation), then zeros; the steps
 * of NeuralPointTextureImpl::PrepareTexture / PrepareConfidence (src/lib/models/NeuralTexture.h:38-55) and the
 * interleave in one pass. Of `params` only those four members are read. One streaming kernel, 52 bytes per point. */
typedef struct vetrast_pack_args
{
    int32_t num_points;
    const float* texture;    /* device [C,N] */
    const float* confidence; /* device [N] */
    vetrast_params params;
    float* packed;           /* device [N][8], 32-byte aligned; fully overwritten */
} vetrast_pack_args;
size_t vetrast_packed_descriptor_bytes(int32_t num_points);
int vetrast_pack_descriptors(vetrast_ctx* ctx, const vetrast_pack_args* args, void* stream);

/* One Adam step on a flat float tensor, the update MyAdam::step applies to texture_raw, confidence_raw and
 * background_color_raw after every batch (src/lib/models/my_adam.cpp:25-104 = torch's Adam without amsgrad; options as
 * in src/lib/data/NeuralScene.cpp:238-281): one kernel instead of the ~10 elementwise launches of the tensor-op form.
 *   g = grad + weight_decay * param;  m = beta1 * m + (1 - beta1) * g;  v = beta2 * v + (1 - beta2) * g * g;
 *   param -= lr / (1 - beta1^step) * m / (sqrt(v) / sqrt(1 - beta2^step) + eps)
 * `step` is the state's step count after the increment (1 on the first call). With zero_grad the gradient is cleared
 * in the same pass (texture_optimizer->zero_grad(), src/lib/data/NeuralScene.cpp:1247-1248). */
typedef struct vetrast_adam_args
{
    float* param;      /* device [n] */
    float* grad;       /* device [n] */
    float* exp_avg;    /* device [n], zero before the first step */
    float* exp_avg_sq; /* device [n], zero before the first step */
    int64_t n;
    int64_t step;
    double lr, beta1, beta2, eps, weight_decay; /* doubles as in torch's AdamOptions: 1 - beta2 must not be formed in float */
    int32_t zero_grad;
} vetrast_adam_args;
int vetrast_adam_step(vetrast_ctx* ctx, const vetrast_adam_args* args, void* stream);

/* ---- AdamW over lists of tensors ----------------------------------------------------------------------------------
 * The optimiser of everything a training step has gradients for, descriptors and render network alike, in as few launches
 * as the list needs (one for up to 160 tensors). Per element, with t the group's step:
 *   g = grad * *grad_scale;  m = beta1 * m + (1 - beta1) * g;  v = beta2 * v + ((1 - beta2) * g) * g
 *   param = (1 - lr * weight_decay) * param - lr / (1 - beta1^t) * (m / (sqrt(v) * (1 / sqrt(1 - beta2^t)) + eps))
 * in 32 bits; the moments are rounded after every operation, in this order. The reference steps its network with torch's
 * Adam, one tensor at a time; with weight_decay 0 this is the same update.
 *
 * State. The moments of all tensors lie in flat arrays that the caller owns, and so do float32 masters of 16-bit parameters
 * where wanted. Tensor k has the elements from `first` on, a multiple of VETRAST_MOMENT_BLOCK, and the arrays hold whole
 * blocks: VETRAST_MOMENT_BLOCK * ceil(n / VETRAST_MOMENT_BLOCK) elements a tensor, zero behind its last one (the step keeps
 * them zero). Zeroed memory is the state before the first step.
 *
 * Moments in 8 bits. A block has two scale bytes, D of the first and of the second moment, and a code c stands for
 *   float(bits = (c << 20) + (D << 23)) - 2^(D - 127)
 * i.e. a float with three mantissa bits, moved so that zero is a code and the values next to it are evenly spaced. The first
 * moment's code is 7 such bits below a sign bit and spans 15 binades below the block's largest value, the second's is 8 bits
 * and spans 31. Codes are rounded up or down by random bits (unbiased), since beta2 = 0.999 moves the second moment by less
 * than half a step of 8 bits at a time: rounded to nearest it settles at a quarter of its value. A second moment above zero
 * stays above zero. A block that meets a value that is not finite, or above 3.19e38, has D = 255 and reads as NaN from then
 * on, all of it. */
#define VETRAST_MOMENT_BLOCK 128

typedef enum vetrast_dtype
{
    VETRAST_F32  = 0,
    VETRAST_BF16 = 1,
    VETRAST_F16  = 2
} vetrast_dtype;

typedef struct vetrast_adamw_tensor
{
    void* param;   /* device [n] of param_type, contiguous, aligned to its element; updated in place */
    void* grad;    /* device [n] of grad_type, the same; cleared with zero_grad */
    int64_t n;     /* >= 0, at most 2^38 */
    int64_t first; /* below 2^38: its place in the flat arrays and, modulo 2^33, in the stream of random bits */
    int32_t param_type, grad_type; /* vetrast_dtype */
    int32_t group;
    int32_t reserved;
} vetrast_adamw_tensor;

typedef struct vetrast_adamw_group
{
    double lr, weight_decay;
    int64_t step; /* count after the increment (1 on the first call); unused with device_state */
} vetrast_adamw_group;

/* Step count and learning rate factor on the device, for steps that are captured in a graph: the count goes up with every
 * replay, and a caller may write either between replays. vetrast_adamw_device_state_bytes(num_groups) bytes, 16-byte
 * aligned, begun with this struct, the rest is scratch. One step at a time may use it. */
typedef struct vetrast_adamw_device_state
{
    int64_t step;    /* steps done so far; a step that is left out is not counted */
    float lr_factor; /* every group's lr is multiplied by it */
    float reserved;
} vetrast_adamw_device_state;
size_t vetrast_adamw_device_state_bytes(int32_t num_groups);

typedef struct vetrast_adamw_args
{
    const vetrast_adamw_tensor* tensors; /* host [num_tensors] */
    const vetrast_adamw_group* groups;   /* host [num_groups] */
    int32_t num_tensors, num_groups;     /* num_groups <= VETRAST_ADAMW_MAX_GROUPS */
    void* exp_avg;        /* device float [], or uint8 [] with moment_bits = 8; 16-byte aligned like all flat arrays */
    void* exp_avg_sq;     /* the same */
    uint8_t* block_scale; /* with moment_bits = 8: device [elements / VETRAST_MOMENT_BLOCK][2] */
    float* master;        /* optional, device: 16-bit parameters are stepped here, and receive the result rounded to nearest */
    double beta1, beta2, eps;    /* eps >= FLT_MIN: a second moment of zero divides by it */
    int32_t moment_bits;         /* 32 or 8 */
    int32_t stochastic_rounding; /* BF16 parameters without master are rounded by random bits instead of to nearest */
    uint64_t seed;               /* of the random bits; they are a function of seed, step and place */
    int32_t zero_grad;           /* gradients are cleared in the same pass */
    int32_t reserved;
    const float* grad_scale; /* optional, device: gradients are multiplied by it. Where it is not finite the step is left
                                out: nothing but zero_grad happens (vetrast_gradient_norm writes NaN for gradients that
                                overflowed) */
    void* device_state;      /* optional, device; see above */
} vetrast_adamw_args;
#define VETRAST_ADAMW_MAX_GROUPS 1024
/* Tensors of a call must not overlap in memory or in the flat arrays. Enqueues kernels only; allocates nothing. */
int vetrast_adamw_step(vetrast_ctx* ctx, const vetrast_adamw_args* args, void* stream);

/* The 2-norm of all gradients together and the factor that clips it:
 *   out[0] = |scale| * sqrt(sum of squares);  out[1] = scale * min(1, max_norm / out[0])   (max_norm <= 0: out[1] = scale)
 * Squares are summed in 64 bits in an order that depends on the sizes alone. With scale = 1 / loss scale, out[0] is the norm
 * of the true gradients and out + 1 what vetrast_adamw_args.grad_scale takes. If out[0] is not finite, out[1] is NaN. */
typedef struct vetrast_gradient
{
    const void* grad; /* device [n], contiguous, aligned to its element */
    int64_t n;        /* >= 0, at most 2^38 */
    int32_t type; /* vetrast_dtype */
    int32_t reserved;
} vetrast_gradient;
typedef struct vetrast_gradient_norm_args
{
    const vetrast_gradient* gradients; /* host [num_gradients] */
    int32_t num_gradients;
    int32_t reserved;
    double max_norm, scale;
    float* out;      /* device [2] */
    void* workspace; /* device, 16-byte aligned. Zeroed before the first call that uses it, and left alone between calls.
                        Not shared by calls that may overlap, replays of graphs among them */
    size_t workspace_bytes;
} vetrast_gradient_norm_args;
size_t vetrast_gradient_norm_workspace_bytes(const vetrast_gradient* gradients, int32_t num_gradients);
int vetrast_gradient_norm(vetrast_ctx* ctx, const vetrast_gradient_norm_args* args, void* stream);

/* Moments to 8 bits, rounded to nearest (ties away from zero), and back: a run with moments in 32 bits is continued in 8 and
 * the other way round. Packing writes whole blocks, zeros behind a tensor's last element. */
typedef struct vetrast_moment_tensor
{
    float* exp_avg;    /* device [n], contiguous, aligned to 4 bytes */
    float* exp_avg_sq; /* the same; its magnitudes are taken */
    int64_t n;         /* >= 0, at most 2^38 */
    int64_t first;     /* below 2^38: place in the flat arrays, a multiple of VETRAST_MOMENT_BLOCK */
} vetrast_moment_tensor;
typedef struct vetrast_moments_args
{
    const vetrast_moment_tensor* tensors; /* host [num_tensors] */
    int32_t num_tensors;
    int32_t reserved;
    uint8_t* exp_avg; /* the flat arrays of vetrast_adamw_args with moment_bits = 8 */
    uint8_t* exp_avg_sq;
    uint8_t* block_scale;
} vetrast_moments_args;
int vetrast_pack_moments(vetrast_ctx* ctx, const vetrast_moments_args* args, void* stream);
int vetrast_unpack_moments(vetrast_ctx* ctx, const vetrast_moments_args* args, void* stream);

/* ---- Dropout without a stored mask ---------------------------------------------------------------------------------
 *   y[i] = (left out(i) ? 0 : x[i] * 65536 / (65536 - t)) + residual[i],   t = floor(65536 p + 1/2)
 * in 32 bits, rounded once. Element i is left out where its 16 random bits are below t. They are those of Philox4x32 with
 * seven rounds (Salmon et al., 2011) at the counter (i / 8, step), 64 bits each, under the key `seed`: of the four words that
 * gives, word (i % 8) / 2, its lower half for even i. The backward pass is the same call on the upstream gradient, without a
 * residual: nothing is kept between the two. p below 2^-17 leaves out nothing, from 1 - 2^-17 on everything is left out; what is left out is
 * not looked at (a NaN there becomes 0). The same element of two calls with the same seed and step has the same bits: give
 * every layer of a network a seed of its own and count steps. */
typedef struct vetrast_dropout_args
{
    const void* x;        /* device [n], contiguous, aligned to its element */
    const void* residual; /* the same, or NULL */
    void* y;              /* the same; may be x or residual itself, and must not overlap them otherwise */
    int64_t n;            /* >= 0, at most 2^38 */
    int32_t type;         /* vetrast_dtype of all three */
    int32_t reserved;
    double p;             /* 0 .. 1 */
    uint64_t seed, step;
    const int64_t* device_step; /* optional, device: added to the step. For calls that are captured in a graph, whose replays
                                   then differ as the caller counts on (vetrast_adamw_device_state.step does by itself) */
} vetrast_dropout_args;
int vetrast_dropout(vetrast_ctx* ctx, const vetrast_dropout_args* args, void* stream);

/* ---- Eviction ------------------------------------------------------------------------------------------------------
 * A scene (or a cache) that may hold `budget` entries keeps those that gave most. vetrast_select_kept says which ones, from
 * the weights they have accumulated; vetrast_keep_rows takes the rows of a list of tensors along.
 *
 * Of a row's first length[row] entries the last `recent` ones stay whatever their scores (points that were added a moment
 * ago have had no time to gather weight), and of those in front of them the budget - recent with the highest scores, of
 * equal ones those with the lowest numbers. +0 and -0 are equal, a NaN is below everything. A row of at most `budget` entries
 * keeps them all. The entries that are kept are given in ascending order, the order of a cloud in memory, and behind them
 * -1. Only the first length[row] scores of a row are read. */
typedef struct vetrast_select_args
{
    const float* score;    /* device [rows][n], a row every row_stride elements */
    int64_t row_stride;    /* >= n */
    const int32_t* length; /* optional, device [rows]: entries of a row, taken as 0 below 0 and as n above n. NULL: n */
    int32_t* index;        /* device [rows][budget]; overwritten */
    int32_t* count;        /* device [rows]: entries kept, min(length, budget); overwritten */
    int32_t rows, n;       /* >= 0; n at most 2^30 */
    int32_t budget;        /* 0 .. 2^30; may be more than n */
    int32_t recent;        /* 0 .. budget */
    void* workspace;       /* device, 16-byte aligned; its contents before and after the call do not matter */
    size_t workspace_bytes;
} vetrast_select_args;
size_t vetrast_select_kept_workspace_bytes(int32_t rows, int32_t n); /* 0 for rows that one workgroup takes */
int vetrast_select_kept(vetrast_ctx* ctx, const vetrast_select_args* args, void* stream);

/* dst[o][k] = src[o][index[r][k]] for a list of tensors, entries being rows of row_bytes bytes of any kind; o counts what
 * lies outside the dimension of the entries (the channels of a planar texture [C,N]; heads), and the outers of a tensor share
 * the rows of indices evenly: r = o / (outers / index_rows). An index that is negative or not below n leaves zeros. dst is
 * contiguous and must overlap neither a source nor another dst. Few launches whatever the length of the list (one for up to
 * 32 tensors). */
typedef struct vetrast_keep_tensor
{
    const void* src;
    void* dst;               /* [outers][kept][row_bytes] */
    int64_t outers;          /* a multiple of index_rows; at most 2^31 - 1 */
    int64_t n;               /* entries of an outer, at most 2^31 - 1 */
    int64_t row_bytes;       /* 1 .. 2^30 */
    int64_t src_outer_bytes; /* from one outer to the next, and from one entry to the next; >= 0 */
    int64_t src_row_bytes;
} vetrast_keep_tensor;
typedef struct vetrast_keep_args
{
    const vetrast_keep_tensor* tensors; /* host [num_tensors] */
    int32_t num_tensors;
    int32_t index_rows;      /* >= 1 */
    int32_t kept;            /* >= 0, indices of a row */
    int32_t reserved;
    int64_t index_row_stride; /* elements, >= kept */
    const int32_t* index;     /* device [index_rows][kept] */
} vetrast_keep_args;
int vetrast_keep_rows(vetrast_ctx* ctx, const vetrast_keep_args* args, void* stream);

/* Error lifting: adds the per-pixel error of one rendered view to every cell of the scene grid whose projection covers
 * the pixel. Replaces PointRendererCache::FillSceneGridWithLoss and its kernel FillSceneGridWithLossRasterize
 * (src/lib/rendering/RenderForward.cu:605-632,639-791; called once per view of a batch in the epoch before points are
 * added, src/apps/train.cpp:1069-1078; cell tensors: src/lib/rendering/NeuralPointCloudCuda.h:100-106,166-191,
 * built by UpdateCellStructureForPointOptim, src/lib/rendering/NeuralPointCloudCuda.cpp:95-147).
 *
 * For every cell: the 8 corners bb_min + bb_length * {000,100,010,001,110,101,011,111} are projected like points
 * (pinhole, zero distortion, crop transform and rotation of `view`); a cell with a corner at or behind the camera
 * plane is skipped; the pixel box of the 8 projections is cut to the image minus a border of `border_pixels`
 * (VETRAST_LIFT_BORDER_PIXELS in the reference); every integer pixel of the box that lies in one of the 12 projected
 * face triangles adds sum_c |loss_image[c][y][x]| to cell_value and 1 to cell_access_count.
 *
 * The reference adds the float terms with atomics in arrival order; here the terms of a cell are summed in double (also
 * in arrival order, row by row) and added to cell_value with one rounding: two calls give the same float unless a sum lies
 * within its last double bits of halfway between two floats. cell_value and cell_access_count are
 * accumulated into, not cleared (ResetCellValues / NormalizeBBCellValue stay with the caller,
 * src/lib/rendering/NeuralPointCloudCuda.h:42-52). */
#define VETRAST_LIFT_BORDER_PIXELS 32
/* Byte offset inside the workspace of a uint32 that is 1 after the call if the camera row holds non-zero distortion
 * coefficients (they are ignored, as in vetrast_forward), else 0. */
#define VETRAST_LIFT_FLAGS_OFFSET 192
/* Byte offset inside the workspace of a uint32 that holds, after the call, how many cells have a box of more than 4096
 * pixels on screen (a diagnostic; nothing has to read it). */
#define VETRAST_LIFT_QUEUE_LENGTH_OFFSET 176
typedef struct vetrast_lift_args
{
    int64_t num_cells;
    const float* cell_bb_min;    /* device [num_cells,3] (t_cell_bb_min) */
    const float* cell_bb_length; /* device [num_cells,3] (t_cell_bb_length) */
    float* cell_value;           /* device [num_cells] (t_cell_value, [num_cells,1]); accumulated into */
    int32_t* cell_access_count;  /* device [num_cells] (t_cell_access_count); accumulated into */
    int32_t num_poses;           /* rows of poses_se3 */
    int32_t num_cameras;
    const double* poses_se3;     /* device [num_poses,8], as in vetrast_forward_args */
    const float* intrinsics;     /* device [num_cameras,13], as in vetrast_forward_args */
    vetrast_view view;           /* the view the error image belongs to (images[batch]); w / 2, h / 2 is the crop rotation centre */
    const float* loss_image;     /* device [channels,height,width], e.g. |target - output| of that view */
    int32_t channels, height, width;
    int32_t border_pixels;       /* >= 0; the reference's constant is VETRAST_LIFT_BORDER_PIXELS */
    void* workspace;             /* device, 256-byte aligned, vetrast_lift_workspace_bytes_for_image(num_cells, width,
                                  * height) bytes or more */
    size_t workspace_bytes;
} vetrast_lift_args;
/* Bytes for an image of that size (20 per cell, 8 per pixel and row, at most 33.6 MB of the latter), and bytes that do for
 * an image of any size. */
size_t vetrast_lift_workspace_bytes_for_image(int64_t num_cells, int32_t width, int32_t height);
size_t vetrast_lift_workspace_bytes(int64_t num_cells);
int vetrast_lift_error(vetrast_ctx* ctx, const vetrast_lift_args* args, void* stream);

/* vetrast_lift_error for callers that cannot allocate device memory (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc). It has no counterpart in the reference. Same arguments, same kernels and
 * same results as vetrast_lift_error, but `workspace` / `workspace_bytes` are ignored: the scratch is an array inside
 * the library (about 27 MB of device memory per GPU, held until the process ends), whose address on the context's
 * device vetrast_create looks up once. The call itself allocates and frees nothing, creates no events (it reports no
 * timing scope) and only launches kernels.
 *   - num_cells > VETRAST_LIFT_STATIC_MAX_CELLS is refused with VETRAST_ERR_TOO_LARGE.
 *   - The context's device must be the current device, else VETRAST_ERR_INVALID_ARG.
 *   - All calls on one GPU share that GPU's array (every call rewrites what it reads, nothing has to be cleared in
 *     between): calls that overlap on one GPU, on different streams or from different contexts, race. Calls on one
 *     stream are safe.
 *   - The distortion flag word of vetrast_lift_error lives in the scratch and cannot be read back here; check the
 *     intrinsics beforehand. */
#define VETRAST_LIFT_STATIC_MAX_CELLS (1 << 19)
int vetrast_lift_error_static(vetrast_ctx* ctx, const vetrast_lift_args* args, void* stream);

/* Per-kernel timing, the counterpart of NeuralRenderInfo::timer_system (src/lib/rendering/PointRenderer.h:32).
 * With profiling enabled every launch is bracketed by HIP events on the call's stream; vetrast_scope_times
 * synchronises on them and returns, per scope, the summed kernel time in milliseconds and the number of launches
 * since the last vetrast_reset_scope_times. */
int vetrast_set_profiling(vetrast_ctx* ctx, int32_t enabled);
int vetrast_reset_scope_times(vetrast_ctx* ctx);
int vetrast_scope_times(vetrast_ctx* ctx, float* ms /* [VETRAST_SCOPE_COUNT_] */,
                        int32_t* launches /* [VETRAST_SCOPE_COUNT_] */);
const char* vetrast_scope_name(int32_t scope);

const char* vetrast_status_string(int status);
/* hipError_t value of the last failed HIP call of this context (0 if none). */
int vetrast_last_hip_error(const vetrast_ctx* ctx);

#ifdef __cplusplus
}
#endif
#endif /* VETRAST_H */
