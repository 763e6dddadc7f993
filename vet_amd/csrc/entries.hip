// C ABI of the operators that leave entries out: argument checks and launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <limits>

#include "common.h"
#include "context.h"
#include "dropout_kernels.h"
#include "evict_kernels.h"
#include "weight_kernels.h"

using namespace vetrast;

namespace vetrast
{
void launch_fragment_weights(const WeightPass& pass, int hits, bool fuzzy, int views, hipStream_t stream)
{
    const dim3 block(kBlock);
    if (slots_are_cleared(hits, pass.N))
    {
        const size_t n = ((size_t)pass.N * pass.ly.L + 3) / 4;
        hipLaunchKernelGGL(clear_slots_kernel, dim3((uint32_t)std::min<size_t>((n + kBlock - 1) / kBlock, 8192), (uint32_t)views), block, 0, stream, pass, n);
    }
    if (fuzzy)
    {
        hipLaunchKernelGGL(fragment_weights_fuzzy_kernel, dim3(pass.ly.tile_base[pass.ly.L], (uint32_t)views), block, 0, stream, pass);
        return;
    }
    const dim3 grid(pass.share_base[pass.ly.L] * kXcds, (uint32_t)views);
    if (hits == 1) hipLaunchKernelGGL((fragment_weights_kernel<1>), grid, block, 0, stream, pass);
    else hipLaunchKernelGGL((fragment_weights_kernel<4>), grid, block, 0, stream, pass);
}
void launch_point_weights(const PointWeightPass& pass, int hits, hipStream_t stream)
{
    const dim3 grid((uint32_t)((pass.vp.N + kBlock - 1) / kBlock)), block(kBlock);
    if (slots_are_cleared(hits, pass.vp.N)) hipLaunchKernelGGL(point_weights_cleared_kernel, grid, block, 0, stream, pass);
    else if (hits == 1) hipLaunchKernelGGL((point_weights_kernel<1>), grid, block, 0, stream, pass);
    else hipLaunchKernelGGL((point_weights_kernel<4>), grid, block, 0, stream, pass);
}
}  // namespace vetrast

namespace
{
constexpr int64_t kDropoutAtOnce = (int64_t)1 << 33;  // elements of a launch: its threads are counted in 32 bits

template <int TYPE>
void launch_dropout(DropoutPass& l, hipStream_t stream)
{
    const dim3 grid((uint32_t)((l.n + kOptimChunk - 1) / kOptimChunk));
    if (l.residual) hipLaunchKernelGGL((dropout_kernel<TYPE, true>), grid, dim3(kBlock), 0, stream, l);
    else hipLaunchKernelGGL((dropout_kernel<TYPE, false>), grid, dim3(kBlock), 0, stream, l);
}

// Whether two stretches of memory share some of it without being the same one.
inline bool overlap(const void* a, const void* b, size_t bytes)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x != y && (x < y ? y - x : x - y) < bytes;
}
// Rows of more entries than a workgroup holds are shared by several: a piece of 12 entries a thread each, or more where there are many.
constexpr int kSelectGroups   = 1024;     // workgroups of a row at most
constexpr int kDigitGroups    = 256;      // ... where digits are counted (5.5 M entries 45.5 us, with 512 47.6, with 128 50.6)
constexpr int kSelectGridRows = 32768;    // rows of a launch
constexpr int kSelectRows     = 1 << 21;  // ... where each is one workgroup: a launch's threads are counted in 32 bits
constexpr int kSelectMost     = 1 << 30;  // scores of a row, and a budget: places stay within 32 bits with a piece behind them
inline int select_share(int n)
{
    const int64_t pieces = ((int64_t)n + kSharePiece - 1) / kSharePiece;
    return (int)((pieces + kSelectGroups - 1) / kSelectGroups) * kSharePiece;
}
inline int select_groups(int n) { return (int)(((int64_t)n + select_share(n) - 1) / select_share(n)); }
inline size_t select_words(int n) { return kDigits * (size_t)kBins + 2 + 2 * kDigits + 2 * (size_t)select_groups(n); }  // of a row

// Threads and keys a thread by the length of a row. Rows just within a bound, with what stands here and with the next variant: 1024 rows of 1000 8.3 and
// 17.5 us, 64 rows of 4000 5.6 and 6.5, 64 rows of 12 000 9.2 and 12.2; the last bound: one row of 32 768 18.7 and with several workgroups 20.0, of
// 20 000 14.7 and 19.1, 256 rows of 32 768 25 and 53.
void launch_select_row(SelectPass p, hipStream_t stream)
{
    const SelectPass all = p;
    for (int64_t from = 0; from < all.rows; from += kSelectRows)
    {
        p.rows   = (int)std::min<int64_t>(all.rows - from, kSelectRows);
        p.score  = all.score + from * all.row_stride;
        p.length = all.length ? all.length + from : nullptr;
        p.index  = all.index + from * all.budget;
        p.count  = all.count + from;
        const dim3 grid((uint32_t)p.rows);
        if (p.n <= 4 * kBlock) hipLaunchKernelGGL((select_row_kernel<kBlock, 1>), grid, dim3(kBlock), 0, stream, p);
        else if (p.n <= 4 * kSelectThreads) hipLaunchKernelGGL((select_row_kernel<kSelectThreads, 1>), grid, dim3(kSelectThreads), 0, stream, p);
        else if (p.n <= 12 * kSelectThreads) hipLaunchKernelGGL((select_row_kernel<kSelectThreads, 3>), grid, dim3(kSelectThreads), 0, stream, p);
        else hipLaunchKernelGGL((select_row_kernel<kSelectThreads, 8>), grid, dim3(kSelectThreads), 0, stream, p);
    }
}

void launch_select_rows(SelectPass p, char* workspace, hipStream_t stream)
{
    p.share  = select_share(p.n);
    p.groups = select_groups(p.n);
    p.shares = (p.groups + kDigitGroups - 1) / kDigitGroups;
    const int rows        = p.rows;
    const SelectPass all  = p;
    for (int64_t from = 0; from < rows; from += kSelectGridRows)
    {
        p           = all;
        p.rows      = (int)std::min<int64_t>(rows - from, kSelectGridRows);
        p.score     = all.score + from * all.row_stride;
        p.length    = all.length ? all.length + from : nullptr;
        p.index     = all.index + from * all.budget;
        p.count     = all.count + from;
        p.histogram = reinterpret_cast<uint32_t*>(workspace) + (size_t)from * select_words(p.n);
        p.zeros     = p.histogram + (size_t)p.rows * kDigits * kBins;
        p.known     = reinterpret_cast<uint2*>(p.zeros + 2 * (size_t)p.rows);
        p.counts    = p.known + (size_t)p.rows * kDigits;
        const size_t words = (size_t)p.rows * (kDigits * kBins + 1);  // histograms and zeros
        const dim3 grid((uint32_t)p.groups, (uint32_t)p.rows), digits((uint32_t)((p.groups + p.shares - 1) / p.shares), (uint32_t)p.rows), block(kShareThreads);
        hipLaunchKernelGGL(select_clear_kernel, dim3((uint32_t)std::min<size_t>((words + kBlock - 1) / kBlock, 2048)), dim3(kBlock), 0, stream, p.histogram, words);
        hipLaunchKernelGGL((select_digit_kernel<0>), digits, block, 0, stream, p);
        hipLaunchKernelGGL((select_digit_kernel<1>), digits, block, 0, stream, p);
        hipLaunchKernelGGL((select_digit_kernel<2>), digits, block, 0, stream, p);
        hipLaunchKernelGGL(select_count_kernel, grid, block, 0, stream, p);
        hipLaunchKernelGGL(select_place_kernel, grid, block, 0, stream, p);
    }
}

// Bytes from a tensor's first to behind its last.
inline uint64_t stretch(int64_t outers, int64_t n, int64_t outer_bytes, int64_t row_bytes, int64_t bytes)
{
    return (uint64_t)(outers - 1) * (uint64_t)outer_bytes + (uint64_t)(n - 1) * (uint64_t)row_bytes + (uint64_t)bytes;
}
constexpr int64_t kKeepMost       = (int64_t)1 << 30;  // units of an entry's outer: places in it are 32 bits
constexpr int64_t kKeepGroupsMost = (int64_t)1 << 22;  // workgroups of an entry, and with those in front twice that: a launch's threads are 32 bits
}  // namespace

extern "C" {

int vetrast_dropout(vetrast_ctx* ctx, const vetrast_dropout_args* a, void* stream_)
{
    if (!ctx || !a) return VETRAST_ERR_INVALID_ARG;
    if (a->n < 0 || a->n > kOptimMaxElements || !is_dtype(a->type) || !(a->p >= 0.0 && a->p <= 1.0)) return VETRAST_ERR_INVALID_ARG;
    if (!aligned_to(a->device_step, 8)) return VETRAST_ERR_INVALID_ARG;
    if (a->n == 0) return VETRAST_OK;
    const size_t each = dtype_bytes(a->type), bytes = (size_t)a->n * each;
    if (!a->x || !a->y || !aligned_to(a->x, each) || !aligned_to(a->y, each) || !aligned_to(a->residual, each)) return VETRAST_ERR_INVALID_ARG;
    if (overlap(a->x, a->y, bytes) || (a->residual && overlap(a->residual, a->y, bytes))) return VETRAST_ERR_INVALID_ARG;
    hipStream_t stream = (hipStream_t)stream_;
    DropoutPass l;
    l.bits  = dropout_bits(a->p, a->seed, a->step, a->device_step);
    l.scale = l.bits.threshold < 65536u ? (float)(65536.0 / (65536.0 - l.bits.threshold)) : 0.f;
    for (int64_t from = 0; from < a->n; from += kDropoutAtOnce)
    {
        l.x           = static_cast<const char*>(a->x) + (size_t)from * each;
        l.residual    = a->residual ? static_cast<const char*>(a->residual) + (size_t)from * each : nullptr;
        l.y           = static_cast<char*>(a->y) + (size_t)from * each;
        l.n           = (uint64_t)std::min(a->n - from, kDropoutAtOnce);
        l.first_block = (uint64_t)from / 8;
        if (a->type == VETRAST_F32) launch_dropout<VETRAST_F32>(l, stream);
        else if (a->type == VETRAST_BF16) launch_dropout<VETRAST_BF16>(l, stream);
        else launch_dropout<VETRAST_F16>(l, stream);
    }
    VET_HIP(ctx, hipGetLastError());
    return VETRAST_OK;
}

size_t vetrast_select_kept_workspace_bytes(int32_t rows, int32_t n)
{
    if (rows <= 0 || n <= kSelectRowMost) return 0;
    return (size_t)rows * select_words(n) * sizeof(uint32_t);
}

int vetrast_select_kept(vetrast_ctx* ctx, const vetrast_select_args* a, void* stream_)
{
    if (!ctx || !a) return VETRAST_ERR_INVALID_ARG;
    if (a->rows < 0 || a->n < 0 || a->budget < 0 || a->recent < 0 || a->recent > a->budget || a->row_stride < a->n || a->n > kSelectMost ||
        a->budget > kSelectMost)
        return VETRAST_ERR_INVALID_ARG;
    if (!aligned_to(a->score, 4) || !aligned_to(a->length, 4) || !aligned_to(a->index, 4) || !aligned_to(a->count, 4) || !aligned_to(a->workspace, 16))
        return VETRAST_ERR_INVALID_ARG;
    if (a->rows == 0) return VETRAST_OK;
    if (!a->count || (a->budget > 0 && !a->index) || (a->n > 0 && !a->score)) return VETRAST_ERR_INVALID_ARG;
    const size_t need = vetrast_select_kept_workspace_bytes(a->rows, a->n);
    if (need > 0 && !a->workspace) return VETRAST_ERR_INVALID_ARG;
    if (a->workspace_bytes < need) return VETRAST_ERR_WORKSPACE_SMALL;
    SelectPass p;
    p.score      = a->score;
    p.row_stride = a->row_stride;
    p.length     = a->length;
    p.index      = a->index;
    p.count      = a->count;
    p.rows       = a->rows;
    p.n          = a->n;
    p.budget     = a->budget;
    p.recent     = a->recent;
    p.histogram  = nullptr;
    p.zeros      = nullptr;
    p.known      = nullptr;
    p.counts     = nullptr;
    p.share = p.groups = p.shares = 0;
    hipStream_t stream = (hipStream_t)stream_;
    if (need == 0) launch_select_row(p, stream);
    else launch_select_rows(p, static_cast<char*>(a->workspace), stream);
    VET_HIP(ctx, hipGetLastError());
    return VETRAST_OK;
}

int vetrast_keep_rows(vetrast_ctx* ctx, const vetrast_keep_args* a, void* stream_)
{
    if (!ctx || !a) return VETRAST_ERR_INVALID_ARG;
    if (a->num_tensors < 0 || (a->num_tensors > 0 && !a->tensors) || a->index_rows < 1 || a->kept < 0 || a->index_row_stride < a->kept)
        return VETRAST_ERR_INVALID_ARG;
    if (!aligned_to(a->index, 4) || (a->kept > 0 && !a->index)) return VETRAST_ERR_INVALID_ARG;
    constexpr int64_t kMost = std::numeric_limits<int32_t>::max(), kFar = (int64_t)1 << 47;
    bool any = false;
    for (int k = 0; k < a->num_tensors; ++k)
    {
        const vetrast_keep_tensor& t = a->tensors[k];
        if (t.outers < 0 || t.outers > kMost || t.outers % a->index_rows != 0 || t.n < 0 || t.n > kMost) return VETRAST_ERR_INVALID_ARG;
        if (t.row_bytes < 1 || t.row_bytes > kKeepMost || t.src_outer_bytes < 0 || t.src_row_bytes < 0) return VETRAST_ERR_INVALID_ARG;
        if (t.outers == 0 || a->kept == 0) continue;
        any = true;
        if (!t.dst || (t.n > 0 && !t.src)) return VETRAST_ERR_INVALID_ARG;
        // no memory is as long as this; products below stay within 64 bits
        if ((double)t.outers * a->kept * t.row_bytes > (double)kFar || (double)t.outers * t.src_outer_bytes > (double)kFar ||
            (double)t.n * t.src_row_bytes > (double)kFar)
            return VETRAST_ERR_INVALID_ARG;
        if (t.n == 0) continue;
        const uint64_t from = reinterpret_cast<uintptr_t>(t.src), to = reinterpret_cast<uintptr_t>(t.dst);
        const uint64_t there = stretch(t.outers, t.n, t.src_outer_bytes, t.src_row_bytes, t.row_bytes);
        const uint64_t here  = (uint64_t)t.outers * (uint64_t)a->kept * (uint64_t)t.row_bytes;
        if (from < to + here && to < from + there) return VETRAST_ERR_INVALID_ARG;
    }
    if (!any) return VETRAST_OK;
    hipStream_t stream = (hipStream_t)stream_;
    KeepLaunch l;
    l.entries = l.total = 0;
    const auto launch = [&] {
        if (l.entries > 0) hipLaunchKernelGGL(keep_rows_kernel, dim3(l.total), dim3(kBlock), 0, stream, l);
        l.entries = l.total = 0;
    };
    for (int k = 0; k < a->num_tensors; ++k)
    {
        const vetrast_keep_tensor& t = a->tensors[k];
        if (t.outers == 0 || a->kept == 0) continue;
        uint64_t bits = reinterpret_cast<uintptr_t>(t.src) | reinterpret_cast<uintptr_t>(t.dst) | (uint64_t)t.row_bytes | 16;
        if (t.n > 1) bits |= (uint64_t)t.src_row_bytes;
        if (t.outers > 1) bits |= (uint64_t)t.src_outer_bytes;
        const uint32_t unit_log = (uint32_t)__builtin_ctzll(bits);
        const int64_t units = t.row_bytes >> unit_log, per_index = t.outers / a->index_rows;
        const int64_t rows_at_once = std::max<int64_t>(kKeepMost / units, 1);
        for (int64_t row = 0; row < a->kept; row += rows_at_once)
        {
            const int64_t rows   = std::min<int64_t>(a->kept - row, rows_at_once);
            const int64_t chunk  = unit_log == 2 && units == 1 && t.n > 0 ? kKeepWords : kKeepChunk;
            const int64_t chunks = (rows * units + chunk - 1) / chunk, outers_at_once = std::max<int64_t>(kKeepGroupsMost / chunks, 1);
            for (int64_t outer = 0; outer < t.outers; outer += outers_at_once)
            {
                const int64_t outers = std::min(t.outers - outer, outers_at_once);
                if (l.entries == (uint32_t)kKeepEntries || l.total + outers * chunks > 2 * kKeepGroupsMost) launch();
                KeepEntry& e   = l.e[l.entries++];
                e.src          = static_cast<const char*>(t.src) + outer * t.src_outer_bytes;
                e.dst          = static_cast<char*>(t.dst) + (outer * a->kept + row) * t.row_bytes;
                e.src_outer    = t.src_outer_bytes;
                e.src_row      = t.src_row_bytes;
                e.dst_outer    = a->kept * t.row_bytes;
                e.index        = a->index + (outer / per_index) * a->index_row_stride + row;
                e.index_stride = a->index_row_stride;
                e.per_index    = (uint32_t)per_index;
                e.outer_in_row = (uint32_t)(outer % per_index);
                e.kept         = (uint32_t)rows;
                e.units        = (uint32_t)units;
                e.n            = (uint32_t)t.n;
                e.chunks       = (uint32_t)chunks;
                e.first_chunk  = l.total;
                e.unit_log     = unit_log;
                e.units_log    = (units & (units - 1)) == 0 ? (uint32_t)__builtin_ctzll((uint64_t)units) : 32u;
                l.total += (uint32_t)(outers * chunks);
            }
        }
    }
    launch();
    VET_HIP(ctx, hipGetLastError());
    return VETRAST_OK;
}

}  // extern "C"
