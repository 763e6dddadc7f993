// Eviction: which entries of a row a budget keeps, by the weight they have accumulated, and the rows of tensors that go with them.
//
// The entries that are kept are given in their order (the order of a cloud in memory is worth keeping), so what has to be found is a
// threshold: the key of the last one that is kept, and how many of those that share it are. Keys are found digit by digit from the
// top (11, 11 and 10 bits) with histograms in LDS; then every entry knows by itself whether it stays, and a scan gives it its place.
#pragma once
#include "common.h"
#include "elements.h"

namespace vetrast
{
constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves   = kSelectThreads / kWave;
constexpr int kDigits        = 3;
constexpr uint32_t kBins     = 2048;
constexpr int kSelectRowMost = 32 * kSelectThreads;  // entries of a row that one workgroup holds in registers

// Larger for larger scores. Both zeros are one, a NaN is below everything.
__device__ __forceinline__ uint32_t score_key(float score)
{
    const uint32_t b = __float_as_uint(score + 0.f);
    const uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return score == score ? k : 0u;
}
constexpr uint32_t kZeroKey = 0x80000000u;

__device__ __forceinline__ constexpr int digit_shift(int digit) { return digit == 0 ? 21 : digit == 1 ? 10 : 0; }
__device__ __forceinline__ uint32_t digit_of(uint32_t key, int digit) { return digit == 2 ? key & 1023u : (key >> digit_shift(digit)) & 2047u; }

struct SelectPass
{
    const float* score;
    int64_t row_stride;
    const int32_t* length;  // [rows] or null
    int32_t* index;         // [rows][budget]
    int32_t* count;         // [rows]
    int rows, n, budget, recent;
    // rows of several workgroups
    uint32_t* histogram;  // [rows][kDigits][kBins]
    uint2* counts;        // [rows][groups]: above the threshold, at it
    int share, groups;    // entries of a workgroup (a multiple of kSelectThreads), workgroups of a row
};

// What a row is asked for: `need` of its first `range` entries, and all from there to `length`.
struct RowRange
{
    int length, range, need;
};
__device__ __forceinline__ RowRange row_range(const SelectPass& a, int row)
{
    RowRange r;
    r.length = a.length ? min(max(a.length[row], 0), a.n) : a.n;
    r.range  = max(r.length - a.recent, 0);
    r.need   = a.budget - a.recent;
    if (r.length <= a.budget) r.range = 0, r.need = 0;  // everything stays
    return r;
}

struct SelectRoom
{
    uint32_t bins[kBins];
    uint32_t sums[kSelectWaves];
    uint32_t bin, left;
};

// Inclusive sum over the workgroup's threads; all take part.
__device__ __forceinline__ uint32_t group_inclusive_scan(uint32_t v, uint32_t* sums)
{
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    v = wave_inclusive_scan(v, lane);
    if (lane == kWave - 1) sums[wave] = v;
    __syncthreads();
    uint32_t before = 0;
#pragma unroll
    for (int w = 0; w < kSelectWaves; ++w) before += w < wave ? sums[w] : 0u;
    return v + before;
}

// From the counts of two neighbouring bins a thread, the bin that the need-th largest lies in, and how many of it are needed
// (room.bin, room.left). need is at least 1 and at most the sum of all.
__device__ __forceinline__ void find_bin(SelectRoom& room, uint32_t upper, uint32_t lower, uint32_t need)
{
    const uint32_t sum = group_inclusive_scan(upper + lower, room.sums), before = sum - upper - lower;
    if (before < need && need <= sum)
    {
        const bool first = need <= before + upper;
        room.bin         = kBins - 1 - 2 * threadIdx.x - (first ? 0 : 1);
        room.left        = need - before - (first ? 0 : upper);
    }
    __syncthreads();
}

// Counts one key in the histogram. A third of a cloud may be seen by no view: equal scores of zero would queue up at one address.
__device__ __forceinline__ void count_key(SelectRoom& room, bool there, uint32_t key, int digit)
{
    const bool zero      = there && key == kZeroKey;
    const uint64_t zeros = __ballot(zero);
    if (zeros && threadIdx.x % kWave == 0) atomicAdd(&room.bins[digit_of(kZeroKey, digit)], (uint32_t)__popcll(zeros));
    if (there && !zero) atomicAdd(&room.bins[digit_of(key, digit)], 1u);
}

__device__ __forceinline__ void clear_bins(SelectRoom& room)
{
    room.bins[threadIdx.x] = room.bins[threadIdx.x + kSelectThreads] = 0u;
    __syncthreads();
}

// One workgroup for a row, its keys in registers.
template <int ITEMS>
__global__ void __launch_bounds__(kSelectThreads) select_row_kernel(SelectPass a)
{
    __shared__ SelectRoom room;
    __shared__ uint32_t places[ITEMS * kSelectWaves + 1];
    const int row = blockIdx.x, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const RowRange r   = row_range(a, row);
    const float* score = a.score + (int64_t)row * a.row_stride;
    int32_t* index     = a.index + (int64_t)row * a.budget;
    float raw[ITEMS];
    uint32_t key[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
    {
        const int i = k * kSelectThreads + (int)threadIdx.x;
        raw[k]      = r.range > 0 ? score[min(i, r.range - 1)] : 0.f;  // without branches, so that all are under way before the first is looked at
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) key[k] = score_key(raw[k]);
    uint32_t prefix = 0, mask = 0, left = (uint32_t)r.need;
    if (r.range > 0 && r.need > 0)
    {
        for (int digit = 0; digit < kDigits; ++digit)
        {
            clear_bins(room);
#pragma unroll
            for (int k = 0; k < ITEMS; ++k)
            {
                const int i = k * kSelectThreads + (int)threadIdx.x;
                count_key(room, i < r.range && (key[k] & mask) == prefix, key[k], digit);
            }
            __syncthreads();
            find_bin(room, room.bins[kBins - 1 - 2 * threadIdx.x], room.bins[kBins - 2 - 2 * threadIdx.x], left);
            left = room.left;
            prefix |= room.bin << digit_shift(digit);
            mask |= (digit == 2 ? 1023u : 2047u) << digit_shift(digit);
            __syncthreads();
        }
        // places: entries above the threshold in front of a wave's 64 (lower half), entries at it (upper half)
        uint64_t above[ITEMS], at[ITEMS];
#pragma unroll
        for (int k = 0; k < ITEMS; ++k)
        {
            const int i = k * kSelectThreads + (int)threadIdx.x;
            above[k]    = __ballot(i < r.range && key[k] > prefix);
            at[k]       = __ballot(i < r.range && key[k] == prefix);
            if (lane == 0) places[k * kSelectWaves + wave] = (uint32_t)__popcll(above[k]) | (uint32_t)__popcll(at[k]) << 16;
        }
        __syncthreads();
        const uint32_t mine = threadIdx.x < (uint32_t)(ITEMS * kSelectWaves) ? places[threadIdx.x] : 0u;
        const uint32_t sum  = group_inclusive_scan(mine, room.sums);
        if (threadIdx.x < (uint32_t)(ITEMS * kSelectWaves)) places[threadIdx.x] = sum - mine;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ITEMS; ++k)
        {
            const int i             = k * kSelectThreads + (int)threadIdx.x;
            const uint32_t in_front = places[k * kSelectWaves + wave];
            const auto below = [](uint64_t m) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u)); };
            const uint32_t larger = (in_front & 0xFFFFu) + below(above[k]), equal = (in_front >> 16) + below(at[k]);
            const bool stays      = i < r.range && (key[k] > prefix || (key[k] == prefix && equal < left));
            if (stays) index[larger + min(equal, left)] = i;
        }
    }
    const int selected = min(r.need, r.range), total = selected + r.length - r.range;
    for (int i = (int)threadIdx.x; i < a.budget - selected; i += kSelectThreads) index[selected + i] = i < r.length - r.range ? r.range + i : -1;
    if (threadIdx.x == 0) a.count[row] = total;
}

// ---- rows of several workgroups: a launch for each digit, one that counts and one that gives places ---------------------------

__global__ void __launch_bounds__(kBlock) select_clear_kernel(uint32_t* p, size_t n)
{
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (size_t)gridDim.x * kBlock) p[i] = 0u;
}

// The threshold's digits in front of `digits`, from the histograms that are there, and how many at it are needed.
__device__ __forceinline__ uint32_t known_digits(const SelectPass& a, SelectRoom& room, int row, int digits, uint32_t& left)
{
    uint32_t prefix = 0;
    for (int digit = 0; digit < digits; ++digit)
    {
        const uint2 pair = reinterpret_cast<const uint2*>(a.histogram + ((size_t)row * kDigits + digit) * kBins)[kBins / 2 - 1 - threadIdx.x];
        find_bin(room, pair.y, pair.x, left);
        left = room.left;
        prefix |= room.bin << digit_shift(digit);
        __syncthreads();
    }
    return prefix;
}

template <int DIGIT>
__global__ void __launch_bounds__(kSelectThreads) select_digit_kernel(SelectPass a)
{
    __shared__ SelectRoom room;
    const int row    = blockIdx.y;
    const RowRange r = row_range(a, row);
    const int first = (int)blockIdx.x * a.share, last = min(r.range, first + a.share);
    if (r.need <= 0 || first >= last) return;
    uint32_t left         = (uint32_t)r.need;
    const uint32_t prefix = known_digits(a, room, row, DIGIT, left);
    const uint32_t mask   = DIGIT == 0 ? 0u : ~0u << digit_shift(DIGIT - 1);
    clear_bins(room);
    const float* score = a.score + (int64_t)row * a.row_stride;
    for (int base = first; base < last; base += kSelectThreads)
    {
        const int i        = base + (int)threadIdx.x;
        const uint32_t key = i < last ? score_key(score[i]) : 0u;
        count_key(room, i < last && (key & mask) == prefix, key, DIGIT);
    }
    __syncthreads();
    uint32_t* histogram = a.histogram + ((size_t)row * kDigits + DIGIT) * kBins;
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k)
    {
        const uint32_t bin = threadIdx.x + k * kSelectThreads, v = room.bins[bin];
        if (v) atomicAdd(&histogram[bin], v);
    }
}

__global__ void __launch_bounds__(kSelectThreads) select_count_kernel(SelectPass a)
{
    __shared__ SelectRoom room;
    const int row    = blockIdx.y;
    const RowRange r = row_range(a, row);
    const int first = (int)blockIdx.x * a.share, last = min(r.range, first + a.share);
    uint32_t above = 0, at = 0;
    if (r.need > 0 && first < last)
    {
        uint32_t left         = (uint32_t)r.need;
        const uint32_t prefix = known_digits(a, room, row, kDigits, left);
        const float* score    = a.score + (int64_t)row * a.row_stride;
        for (int i = first + (int)threadIdx.x; i < last; i += kSelectThreads)
        {
            const uint32_t key = score_key(score[i]);
            above += key > prefix;
            at += key == prefix;
        }
    }
    above = group_inclusive_scan(above, room.sums);
    __syncthreads();
    at = group_inclusive_scan(at, room.sums);
    if (threadIdx.x == kSelectThreads - 1) a.counts[(size_t)row * a.groups + blockIdx.x] = make_uint2(above, at);
}

__global__ void __launch_bounds__(kSelectThreads) select_place_kernel(SelectPass a)
{
    __shared__ SelectRoom room;
    __shared__ uint32_t totals[2][kSelectWaves];
    const int row    = blockIdx.y, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const RowRange r = row_range(a, row);
    int32_t* index   = a.index + (int64_t)row * a.budget;
    const int first = (int)blockIdx.x * a.share, last = min(r.range, first + a.share);
    if (r.need > 0 && first < last)
    {
        uint32_t left         = (uint32_t)r.need;
        const uint32_t prefix = known_digits(a, room, row, kDigits, left);
        // what the workgroups in front have
        uint2 sum = make_uint2(0, 0);
        for (int g = (int)threadIdx.x; g < (int)blockIdx.x; g += kSelectThreads)
        {
            const uint2 c = a.counts[(size_t)row * a.groups + g];
            sum.x += c.x, sum.y += c.y;
        }
        sum.x = group_inclusive_scan(sum.x, room.sums);
        __syncthreads();
        sum.y = group_inclusive_scan(sum.y, room.sums);
        if (threadIdx.x == kSelectThreads - 1) room.bin = sum.x, room.left = sum.y;
        __syncthreads();
        uint32_t larger = room.bin, equal = room.left;
        const float* score = a.score + (int64_t)row * a.row_stride;
        for (int base = first; base < last; base += kSelectThreads)
        {
            const int i          = base + (int)threadIdx.x;
            const uint32_t key   = i < last ? score_key(score[i]) : 0u;
            const uint64_t above = __ballot(i < last && key > prefix), at = __ballot(i < last && key == prefix);
            if (lane == 0) totals[0][wave] = (uint32_t)__popcll(above), totals[1][wave] = (uint32_t)__popcll(at);
            __syncthreads();
            uint32_t more = 0, same = 0, all_more = 0, all_same = 0;
#pragma unroll
            for (int w = 0; w < kSelectWaves; ++w)
            {
                more += w < wave ? totals[0][w] : 0u, same += w < wave ? totals[1][w] : 0u;
                all_more += totals[0][w], all_same += totals[1][w];
            }
            const auto below = [](uint64_t m) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u)); };
            const uint32_t before_more = larger + more + below(above), before_same = equal + same + below(at);
            const bool stays           = i < last && (key > prefix || (key == prefix && before_same < left));
            if (stays) index[before_more + min(before_same, left)] = i;
            larger += all_more, equal += all_same;
            __syncthreads();
        }
    }
    // the entries that stay in any case, and what is left of the row
    const int selected = min(r.need, r.range), behind = a.budget - selected;
    for (int64_t i = (int64_t)blockIdx.x * kSelectThreads + threadIdx.x; i < behind; i += (int64_t)gridDim.x * kSelectThreads)
        index[selected + i] = i < r.length - r.range ? r.range + (int)i : -1;
    if (blockIdx.x == 0 && threadIdx.x == 0) a.count[row] = selected + r.length - r.range;
}

// ---- rows of tensors ---------------------------------------------------------------------------------------------------------

constexpr int kKeepEntries     = 32;
constexpr uint32_t kKeepEach   = 4;                    // units of a thread
constexpr uint32_t kKeepChunk  = kKeepEach * kBlock;  // ... of a workgroup

struct KeepEntry
{
    const char* src;
    char* dst;
    int64_t src_outer, src_row;  // bytes from one outer (entry) to the next
    int64_t dst_outer;
    const int32_t* index;        // of the first outer
    int64_t index_stride;        // from a row of indices to the next
    uint32_t per_index;          // outers that share a row of indices
    uint32_t outer_in_row;       // of the first outer, among those
    uint32_t kept, units, n;     // entries here, units of an entry, entries there are
    uint32_t chunks;             // workgroups of an outer
    uint32_t first_chunk;        // of the launch
    uint32_t unit_log;
    __device__ __forceinline__ uint32_t begins() const { return first_chunk; }
};
struct KeepLaunch
{
    KeepEntry e[kKeepEntries];
    uint32_t entries, total;
};

template <class Unit>
__device__ __forceinline__ void keep_units(const KeepEntry& e, uint32_t chunk)
{
    const uint32_t outer = chunk / e.chunks, begin = (chunk - outer * e.chunks) * kKeepChunk, end = e.kept * e.units;
    const uint32_t of_row = (outer + e.outer_in_row) / e.per_index;
    const int32_t* index  = e.index + (int64_t)of_row * e.index_stride;
    const char* src       = e.src + (int64_t)outer * e.src_outer;
    char* dst             = e.dst + (int64_t)outer * e.dst_outer;
    uint32_t unit[kKeepEach];
    int32_t at[kKeepEach];
    Unit v[kKeepEach];
#pragma unroll
    for (uint32_t k = 0; k < kKeepEach; ++k)
    {
        const uint32_t p = begin + k * kBlock + threadIdx.x, j = e.units == 1 ? p : p / e.units;
        unit[k]          = p - j * e.units;
        at[k]            = p < end ? index[j] : -1;
    }
#pragma unroll
    for (uint32_t k = 0; k < kKeepEach; ++k)
    {
        v[k] = Unit{};
        if ((uint32_t)at[k] < e.n) v[k] = *reinterpret_cast<const Unit*>(src + (int64_t)at[k] * e.src_row + (int64_t)unit[k] * (int64_t)sizeof(Unit));
    }
#pragma unroll
    for (uint32_t k = 0; k < kKeepEach; ++k)
    {
        const uint32_t p = begin + k * kBlock + threadIdx.x;
        if (p < end) *reinterpret_cast<Unit*>(dst + (int64_t)p * (int64_t)sizeof(Unit)) = v[k];
    }
}

__global__ void __launch_bounds__(kBlock) keep_rows_kernel(KeepLaunch a)
{
    const ChunkFinder<finder_groups(kKeepEntries)> find(a);
    const uint32_t k   = __builtin_amdgcn_readfirstlane(find(blockIdx.x));
    const KeepEntry& e = a.e[k];
    const uint32_t chunk = blockIdx.x - e.first_chunk;
    if (e.unit_log == 4) keep_units<uint4>(e, chunk);
    else if (e.unit_log == 3) keep_units<uint2>(e, chunk);
    else if (e.unit_log == 2) keep_units<uint32_t>(e, chunk);
    else if (e.unit_log == 1) keep_units<uint16_t>(e, chunk);
    else keep_units<uint8_t>(e, chunk);
}
}  // namespace vetrast
