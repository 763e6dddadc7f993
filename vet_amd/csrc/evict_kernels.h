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
constexpr int kDigits        = 3;
constexpr uint32_t kBins     = 2048;
constexpr int kSelectRowMost = 32 * kSelectThreads;  // entries of a row that one workgroup holds in registers

// Larger for larger scores. Both zeros are one, a NaN is below everything, and below that is what stands for no entry: no more are asked for than there
// are, so that the threshold is above it.
__device__ __forceinline__ uint32_t score_key(float score)
{
    const uint32_t b = __float_as_uint(score + 0.f);
    const uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return score == score ? k : 1u;
}
constexpr uint32_t kNoKey = 0u, kZeroKey = 0x80000000u;

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
    uint32_t* zeros;      // [rows]: scores of zero
    uint2* known;         // [rows][kDigits]: see Known
    uint2* counts;        // [rows][groups]: above the threshold, at it
    int share, groups;    // entries of a workgroup (a multiple of kSharePiece), workgroups of a row
    int shares;           // of a workgroup that counts digits
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

// A thread has groups of four neighbouring entries: entry 4 * (group * THREADS + thread) + k.
template <int THREADS>
struct SelectRoom
{
    uint32_t bins[kBins];
    uint32_t sums[THREADS / kWave];
    uint32_t bin, left;
    uint32_t zeros;  // scores of zero that were counted with the first digit
};

// Inclusive sum over the workgroup's threads; all take part.
template <int THREADS>
__device__ __forceinline__ uint32_t group_inclusive_scan(uint32_t v, uint32_t* sums)
{
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    v = wave_inclusive_scan(v, lane);
    if (lane == kWave - 1) sums[wave] = v;
    __syncthreads();
    uint32_t before = 0;
#pragma unroll
    for (int w = 0; w < THREADS / kWave; ++w) before += w < wave ? sums[w] : 0u;
    return v + before;
}

// The bin that the need-th largest lies in, and how many of it are needed (room.bin, room.left), from the counts in `bins` (room.bins, or those in
// memory). need is at least 1 and at most the sum of all.
template <int THREADS>
__device__ __forceinline__ void find_bin(SelectRoom<THREADS>& room, const uint32_t* bins, uint32_t need)
{
    constexpr uint32_t kEach = kBins / THREADS;
    const uint32_t top       = kBins - kEach * (threadIdx.x + 1);  // the lowest of this thread's bins
    uint32_t counts[kEach], sum = 0;
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) counts[k] = bins[top + k];
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) sum += counts[k];
    const uint32_t end = group_inclusive_scan<THREADS>(sum, room.sums);
    if (end - sum < need && need <= end)
    {
        uint32_t before = end - sum;
#pragma unroll
        for (int k = kEach - 1; k >= 0; --k)
        {
            if (before < need && need <= before + counts[k]) room.bin = top + k, room.left = need - before;
            before += counts[k];
        }
    }
    __syncthreads();
}

template <int THREADS>
__device__ __forceinline__ void clear_bins(SelectRoom<THREADS>& room)
{
#pragma unroll
    for (uint32_t k = 0; k < kBins; k += THREADS) room.bins[k + threadIdx.x] = 0u;
    if (threadIdx.x == 0) room.zeros = 0u;
    __syncthreads();
}

// Scores that a third of a scene's points may share, as no view has seen them, are counted by the thread and not in LDS, where they would queue up at one address.
__device__ __forceinline__ void count_key(uint32_t* bins, uint32_t& zeros, bool matches, uint32_t key, int digit)
{
    zeros += matches && key == kZeroKey;
    if (matches && key != kZeroKey && key != kNoKey) atomicAdd(&bins[digit_of(key, digit)], 1u);
}
template <int THREADS>
__device__ __forceinline__ void count_zeros(SelectRoom<THREADS>& room, uint32_t zeros, int digit)
{
    zeros = wave_inclusive_scan(zeros, 0);
    if (threadIdx.x % kWave != kWave - 1 || zeros == 0) return;
    atomicAdd(&room.bins[digit_of(kZeroKey, digit)], zeros);
    if (digit == 0) atomicAdd(&room.zeros, zeros);
}

// Four neighbouring scores, the first of them entry i, as they lie in memory; those from `end` on are some others of the row (end is at least 1).
__device__ __forceinline__ void load_scores(const float* score, int i, int end, float* raw)
{
    if (i + 4 <= end)
    {
        const uint4 x = load_four(reinterpret_cast<const char*>(score + i));
        raw[0] = __uint_as_float(x.x), raw[1] = __uint_as_float(x.y), raw[2] = __uint_as_float(x.z), raw[3] = __uint_as_float(x.w);
    }
    else
    {
#pragma unroll
        for (int k = 0; k < 4; ++k) raw[k] = score[min(i + k, end - 1)];
    }
}
// Their keys.
__device__ __forceinline__ void keys_of(const float* raw, int i, int end, uint32_t* key)
{
#pragma unroll
    for (int k = 0; k < 4; ++k) key[k] = i + k < end ? score_key(raw[k]) : kNoKey;
}

// Places of the entries that stay, in order. key: GROUPS groups of four a thread, of entries first + ...; threshold and left: as found; larger, equal:
// entries above and at the threshold in front of these, for the last thread afterwards with these; index: of place `base`.
template <int THREADS, int GROUPS>
__device__ __forceinline__ void give_places(const uint32_t (&key)[4 * GROUPS], int first, uint32_t threshold, uint32_t left, uint32_t& larger, uint32_t& equal,
                                            int32_t* index, uint32_t base, uint32_t (&totals)[GROUPS * (THREADS / kWave)])
{
    constexpr int kWaves = THREADS / kWave;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    uint32_t counts[GROUPS], ends[GROUPS];  // of a thread's four: above the threshold in the lower half, at it in the upper
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
    {
        counts[g] = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) counts[g] += key[4 * g + k] > threshold ? 1u : key[4 * g + k] == threshold ? 1u << 16 : 0u;
        ends[g] = wave_inclusive_scan(counts[g], lane);
        if (lane == kWave - 1) totals[g * kWaves + wave] = ends[g];
    }
    __syncthreads();
    // (at most 32768 entries: neither half runs over)
    if (wave == 0)
    {
        uint32_t before = 0;
#pragma unroll
        for (int t = 0; t < GROUPS * kWaves; t += kWave)
        {
            const uint32_t own = t + lane < GROUPS * kWaves ? totals[t + lane] : 0u, end = wave_inclusive_scan(own, lane);
            if (t + lane < GROUPS * kWaves) totals[t + lane] = before + end - own;
            before += (uint32_t)__builtin_amdgcn_readlane((int)end, kWave - 1);
        }
    }
    __syncthreads();
    uint32_t more = 0, same = 0;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
    {
        const int i             = first + 4 * (g * THREADS + (int)threadIdx.x);
        const uint32_t in_front = totals[g * kWaves + wave] + ends[g] - counts[g];
        more = larger + (in_front & 0xFFFFu), same = equal + (in_front >> 16);
#pragma unroll
        for (int k = 0; k < 4; ++k)
        {
            const bool above = key[4 * g + k] > threshold, at = key[4 * g + k] == threshold;
            if (above || (at && same < left)) index[more + min(same, left) - base] = i + k;
            more += above, same += at;
        }
    }
    larger = more, equal = same;
}

// One workgroup for a row, its keys in registers: what it costs is instructions, barriers and atomics in LDS, one after the other. A row of 20 k scores takes
// 14.7 us, 11 where the budget ends among zeros; 64 rows of 8193 7.5.
template <int THREADS, int GROUPS>
__global__ void __launch_bounds__(THREADS) select_row_kernel(SelectPass a)
{
    __shared__ SelectRoom<THREADS> room;
    __shared__ uint32_t totals[GROUPS * (THREADS / kWave)];
    const int row      = blockIdx.x;
    const RowRange r   = row_range(a, row);
    const float* score = a.score + (int64_t)row * a.row_stride;
    int32_t* index     = a.index + (int64_t)row * a.budget;
    if (r.range > 0 && r.need > 0)
    {
        uint32_t key[4 * GROUPS];
        {
            float raw[4 * GROUPS];
            const int mine = 4 * (int)threadIdx.x;
            // (the same branches in all threads)
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
                if (4 * g * THREADS < r.range) load_scores(score, 4 * g * THREADS + mine, r.range, raw + 4 * g);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
            {
                key[4 * g] = key[4 * g + 1] = key[4 * g + 2] = key[4 * g + 3] = kNoKey;
                if (4 * g * THREADS < r.range) keys_of(raw + 4 * g, 4 * g * THREADS + mine, r.range, key + 4 * g);
            }
        }
        uint32_t threshold = 0, mask = 0, left = (uint32_t)r.need;
#pragma unroll
        for (int digit = 0; digit < kDigits; ++digit)
        {
            clear_bins(room);
            uint32_t zeros = 0;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
                if (4 * g * THREADS < r.range)
                {
#pragma unroll
                    for (int k = 0; k < 4; ++k) count_key(room.bins, zeros, (key[4 * g + k] & mask) == threshold, key[4 * g + k], digit);
                }
            count_zeros(room, zeros, digit);
            __syncthreads();
            find_bin(room, room.bins, left);
            left = room.left;
            // where the budget ends among points that nobody has seen, all of the bin are alike: 20 k entries 15.6 -> 11.6 us
            if (digit == 0 && room.bin == digit_of(kZeroKey, 0) && room.bins[room.bin] == room.zeros)
            {
                threshold = kZeroKey;
                break;
            }
            threshold |= room.bin << digit_shift(digit);
            mask |= (digit == 2 ? 1023u : 2047u) << digit_shift(digit);
            __syncthreads();
        }
        uint32_t larger = 0, equal = 0;
        give_places<THREADS, GROUPS>(key, 0, threshold, left, larger, equal, index, 0, totals);
    }
    const int selected = min(r.need, r.range), total = selected + r.length - r.range;
    for (int i = (int)threadIdx.x; i < a.budget - selected; i += THREADS) index[selected + i] = i < r.length - r.range ? r.range + i : -1;
    if (threadIdx.x == 0) a.count[row] = total;
}

// ---- rows of several workgroups: a launch for each digit, one that counts and one that gives places ---------------------------
// A launch is the barrier between workgroups. Five passes over the scores, most of them from the last-level cache: 5.5 M take 34.6 us, of
// which 10 are the first digit, 7 the counts, 11 the places, 2 to clear, and 6 two launches that learn from the ones before that nothing is left to
// count: 2 and 4.4, with the first piece of every workgroup loaded by then, which in the second is the whole row (45 in all where the budget does
// not end among zeros).

// Workgroups of 512: a row of 40 k entries takes 20.0 us of all launches, 64 rows of 131 k 48.5, one of 5.5 M 34.5 (with 1024 threads 23.8, 62 and
// 34.8; with 256 19.9, 48 and 39). Three groups of four of a thread under way at once (5.5 M entries: with 2 7 us more).
constexpr int kShareThreads = 512;
constexpr int kShareGroups  = 3;
constexpr int kSharePiece  = 4 * kShareGroups * kShareThreads;

__global__ void __launch_bounds__(kBlock) select_clear_kernel(uint32_t* p, size_t n)
{
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (size_t)gridDim.x * kBlock) p[i] = 0u;
}

using SharedRoom = SelectRoom<kShareThreads>;

// What is known of a row's threshold: its digits so far, how many entries at it are needed, and whether it is whole (as it is after the first digit
// where the budget ends among scores of zero).
struct Known
{
    uint32_t digits, left;
    bool whole;
};
__device__ __forceinline__ Known unpack_known(uint2 k) { return {k.x, k.y & 0x7FFFFFFFu, (k.y >> 31) != 0u}; }

// The threshold's first DIGITS digits. The last of them comes from the histogram of the launch before, the others this launch finds in memory, and
// leaves what it knows there for the next one.
template <int DIGITS>
__device__ __forceinline__ Known known_digits(const SelectPass& a, SharedRoom& room, int row, int need)
{
    Known known = {0u, (uint32_t)need, false};
    if constexpr (DIGITS > 1) known = unpack_known(a.known[(size_t)row * kDigits + DIGITS - 2]);
    if constexpr (DIGITS > 0)
    {
        if (!known.whole)
        {
            const uint32_t* bins = a.histogram + ((size_t)row * kDigits + DIGITS - 1) * kBins;
            find_bin(room, bins, known.left);
            const uint32_t bin = room.bin;
            known.left         = room.left;
            if (DIGITS == 1 && bin == digit_of(kZeroKey, 0) && bins[bin] == a.zeros[row]) known.digits = kZeroKey, known.whole = true;
            else known.digits |= bin << digit_shift(DIGITS - 1);
        }
        if (blockIdx.x == 0 && threadIdx.x == 0) a.known[(size_t)row * kDigits + DIGITS - 1] = make_uint2(known.digits, known.left | (known.whole ? 0x80000000u : 0u));
        __syncthreads();
    }
    return known;
}

// A piece of a share: kShareGroups groups of four a thread, from entry `base` on. Loads come first.
struct Piece
{
    float raw[4 * kShareGroups];
    __device__ __forceinline__ Piece(const float* score, int base, int last)
    {
#pragma unroll
        for (int g = 0; g < kShareGroups; ++g) load_scores(score, base + 4 * (g * kShareThreads + (int)threadIdx.x), last, raw + 4 * g);
    }
    __device__ __forceinline__ void keys(int base, int last, uint32_t* key) const
    {
#pragma unroll
        for (int g = 0; g < kShareGroups; ++g) keys_of(raw + 4 * g, base + 4 * (g * kShareThreads + (int)threadIdx.x), last, key + 4 * g);
    }
};

// Entries above and at the threshold, of a share.
__device__ __forceinline__ void leave_counts(const SelectPass& a, SharedRoom& room, int row, int share, uint32_t above, uint32_t at)
{
    __syncthreads();
    above = group_inclusive_scan<kShareThreads>(above, room.sums);
    __syncthreads();
    at = group_inclusive_scan<kShareThreads>(at, room.sums);
    if (threadIdx.x == kShareThreads - 1) a.counts[(size_t)row * a.groups + share] = make_uint2(above, at);
}
__device__ __forceinline__ void count_piece(const uint32_t (&key)[4 * kShareGroups], uint32_t threshold, uint32_t& above, uint32_t& at)
{
#pragma unroll
    for (int k = 0; k < 4 * kShareGroups; ++k)
    {
        above += key[k] > threshold;
        at += key[k] == threshold;
    }
}

// Workgroups take several shares, since each adds its histogram to the row's, at addresses that all of them want. Where the threshold is whole after the
// first digit the second launch counts what select_count_kernel otherwise does.
template <int DIGIT>
__global__ void __launch_bounds__(kShareThreads) select_digit_kernel(SelectPass a)
{
    __shared__ SharedRoom room;
    const int row    = blockIdx.y;
    const RowRange r = row_range(a, row);
    const int first = (int)blockIdx.x * a.shares * a.share, last = (int)min((int64_t)r.range, (int64_t)first + (int64_t)a.shares * a.share);
    if (r.need <= 0 || first >= last) return;
    const float* score = a.score + (int64_t)row * a.row_stride;
    uint32_t zeros = 0;
    Known known = {0u, 0u, false};
    constexpr uint32_t kMask = DIGIT == 0 ? 0u : ~0u << digit_shift(DIGIT == 0 ? 0 : DIGIT - 1);
    uint32_t above = 0, at = 0;
    for (int base = first; base < last; base += kSharePiece)
    {
        const Piece piece(score, base, last);
        if (base == first)  // while the loads are under way
        {
            known = known_digits<DIGIT>(a, room, row, r.need);
            if (DIGIT > 1 && known.whole) return;
            if (!known.whole) clear_bins(room);
        }
        uint32_t key[4 * kShareGroups];
        piece.keys(base, last, key);
        if (DIGIT == 1 && known.whole)
        {
            count_piece(key, known.digits, above, at);
            if (base + kSharePiece >= last || (base + kSharePiece - first) % a.share == 0)
            {
                leave_counts(a, room, row, base / a.share, above, at);
                above = at = 0;
            }
            continue;
        }
#pragma unroll
        for (int k = 0; k < 4 * kShareGroups; ++k) count_key(room.bins, zeros, (key[k] & kMask) == known.digits, key[k], DIGIT);
    }
    if (DIGIT == 1 && known.whole) return;
    count_zeros(room, zeros, DIGIT);
    __syncthreads();
    if (DIGIT == 0 && threadIdx.x == 0 && room.zeros) atomicAdd(&a.zeros[row], room.zeros);
    uint32_t* histogram = a.histogram + ((size_t)row * kDigits + DIGIT) * kBins;
#pragma unroll
    for (uint32_t k = 0; k < kBins; k += kShareThreads)
    {
        const uint32_t v = room.bins[k + threadIdx.x];
        if (v) atomicAdd(&histogram[k + threadIdx.x], v);
    }
}

__global__ void __launch_bounds__(kShareThreads) select_count_kernel(SelectPass a)
{
    __shared__ SharedRoom room;
    const int row    = blockIdx.y;
    const RowRange r = row_range(a, row);
    const int first = (int)blockIdx.x * a.share, last = min(r.range, first + a.share);
    if (r.need <= 0 || first >= last) return;
    const float* score = a.score + (int64_t)row * a.row_stride;
    uint32_t threshold = 0, above = 0, at = 0;
    for (int base = first; base < last; base += kSharePiece)
    {
        const Piece piece(score, base, last);
        if (base == first)
        {
            const Known known = known_digits<kDigits>(a, room, row, r.need);
            if (known.whole) return;
            threshold = known.digits;
        }
        uint32_t key[4 * kShareGroups];
        piece.keys(base, last, key);
        count_piece(key, threshold, above, at);
    }
    leave_counts(a, room, row, (int)blockIdx.x, above, at);
}

// A piece's entries are put together in LDS first, so that a wave's stores are neighbours (5.5 M entries, 4.1 M kept: 34.5 us of all launches, not 36.1).
__global__ void __launch_bounds__(kShareThreads) select_place_kernel(SelectPass a)
{
    __shared__ SharedRoom room;
    __shared__ uint32_t totals[kShareGroups * (kShareThreads / kWave)];
    __shared__ int32_t placed[kSharePiece];
    const int row    = blockIdx.y;
    const RowRange r = row_range(a, row);
    int32_t* index   = a.index + (int64_t)row * a.budget;
    const int first = (int)blockIdx.x * a.share, last = min(r.range, first + a.share);
    if (r.need > 0 && first < last)
    {
        const float* score   = a.score + (int64_t)row * a.row_stride;
        const Known known    = unpack_known(a.known[(size_t)row * kDigits + kDigits - 1]);
        const uint32_t left  = known.left;
        uint32_t larger = 0, equal = 0;
        for (int base = first; base < last; base += kSharePiece)
        {
            const Piece piece(score, base, last);
            if (base == first)
            {
                // what the workgroups in front have
                uint2 sum = make_uint2(0, 0);
                for (int g = (int)threadIdx.x; g < (int)blockIdx.x; g += kShareThreads)
                {
                    const uint2 c = a.counts[(size_t)row * a.groups + g];
                    sum.x += c.x, sum.y += c.y;
                }
                sum.x = group_inclusive_scan<kShareThreads>(sum.x, room.sums);
                __syncthreads();
                sum.y = group_inclusive_scan<kShareThreads>(sum.y, room.sums);
                if (threadIdx.x == kShareThreads - 1) room.bin = sum.x, room.left = sum.y;
                __syncthreads();
            }
            larger = room.bin, equal = room.left;
            uint32_t key[4 * kShareGroups];
            piece.keys(base, last, key);
            const uint32_t from = larger + min(equal, left);
            give_places<kShareThreads, kShareGroups>(key, base, known.digits, left, larger, equal, placed, from, totals);
            if (threadIdx.x == kShareThreads - 1) room.bin = larger, room.left = equal;
            __syncthreads();
            const uint32_t to = room.bin + min(room.left, left);
            for (uint32_t i = from + threadIdx.x; i < to; i += kShareThreads) index[i] = placed[i - from];
            // (the next piece's are written behind two barriers)
        }
    }
    // the entries that stay in any case, and what is left of the row
    const int selected = min(r.need, r.range), behind = a.budget - selected;
    for (int64_t i = (int64_t)blockIdx.x * kShareThreads + threadIdx.x; i < behind; i += (int64_t)gridDim.x * kShareThreads)
        index[selected + i] = i < r.length - r.range ? r.range + (int)i : -1;
    if (blockIdx.x == 0 && threadIdx.x == 0) a.count[row] = selected + r.length - r.range;
}

// ---- rows of tensors ---------------------------------------------------------------------------------------------------------

constexpr int kKeepEntries     = 32;
constexpr uint32_t kKeepEach   = 4;                    // units of a thread
constexpr uint32_t kKeepChunk  = kKeepEach * kBlock;  // ... of a workgroup
constexpr uint32_t kKeepQuads  = 4;                    // where an entry is 4 bytes: four entries each (a scene of 2 M points 72 us, with 2 76; 64 heads 26.6 and 25.8)
constexpr uint32_t kKeepWords  = 4 * kKeepQuads * kBlock;

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
    uint32_t unit_log, units_log;  // 32 where units is no power of two
    __device__ __forceinline__ uint32_t begins() const { return first_chunk; }
};
struct KeepLaunch
{
    KeepEntry e[kKeepEntries];
    uint32_t entries, total;
};

__device__ __forceinline__ uint4 nothing(const uint4&) { return make_uint4(0, 0, 0, 0); }
__device__ __forceinline__ uint2 nothing(const uint2&) { return make_uint2(0, 0); }
template <class Unit>
__device__ __forceinline__ Unit nothing(const Unit&)
{
    return 0;
}

// A workgroup goes through kKeepChunk units of an outer, units being the largest that size, strides and addresses allow (16 bytes at most). Loads are made by
// all threads, of an entry that is there, so that none waits for a branch around another. Memory bounds it: keys and values of 64 heads, 2048 of 8193
// entries of 256 bytes, 26.6 us, 5.1 TB/s.
template <class Unit>
__device__ __forceinline__ void keep_units(const KeepEntry& e, const int32_t* index, const char* src, char* dst, uint32_t begin)
{
    const uint32_t end = e.kept * e.units;
    uint32_t unit[kKeepEach], at[kKeepEach];
    Unit v[kKeepEach];
    const auto entry_of = [&](uint32_t k, auto&& divide) {
        const uint32_t p = min(begin + k * kBlock + threadIdx.x, end - 1), j = divide(p);
        unit[k]          = p - j * e.units;
        at[k]            = (uint32_t)index[j];
    };
    if (e.units_log < 32u)
    {
#pragma unroll
        for (uint32_t k = 0; k < kKeepEach; ++k) entry_of(k, [&](uint32_t p) { return p >> e.units_log; });
    }
    else
    {
#pragma unroll
        for (uint32_t k = 0; k < kKeepEach; ++k) entry_of(k, [&](uint32_t p) { return p / e.units; });
    }
#pragma unroll
    for (uint32_t k = 0; k < kKeepEach; ++k)
        v[k] = *reinterpret_cast<const Unit*>(src + (int64_t)min(at[k], e.n - 1) * e.src_row + (int64_t)unit[k] * (int64_t)sizeof(Unit));
#pragma unroll
    for (uint32_t k = 0; k < kKeepEach; ++k)
    {
        const uint32_t p = begin + k * kBlock + threadIdx.x;
        if (p < end) *reinterpret_cast<Unit*>(dst + (int64_t)p * (int64_t)sizeof(Unit)) = at[k] < e.n ? v[k] : nothing(v[k]);
    }
}

// Entries of one unit of 4 bytes, planes of floats mostly: a thread takes four neighbouring ones at a time, whose indices and results are 16 bytes (a scene of
// 2 M points, 353 MB, 72 us, 4.9 TB/s; unit by unit 92). The last four of an outer may be taken twice.
__device__ __forceinline__ void keep_words(const KeepEntry& e, const int32_t* index, const char* src, char* dst, uint32_t begin)
{
    const uint32_t end = e.kept;
    const auto word    = [&](uint32_t i) { return *reinterpret_cast<const uint32_t*>(src + (int64_t)min(i, e.n - 1) * e.src_row); };
    if (end < 4)
    {
        if (threadIdx.x >= end) return;
        const uint32_t i = (uint32_t)index[threadIdx.x];
        *reinterpret_cast<uint32_t*>(dst + threadIdx.x * 4) = i < e.n ? word(i) : 0u;
        return;
    }
    uint4 at[kKeepQuads], v[kKeepQuads];
    const auto place = [&](uint32_t k) { return min(begin + 4 * (k * kBlock + threadIdx.x), end - 4); };
#pragma unroll
    for (uint32_t k = 0; k < kKeepQuads; ++k) at[k] = load_four(reinterpret_cast<const char*>(index + place(k)));
#pragma unroll
    for (uint32_t k = 0; k < kKeepQuads; ++k) v[k] = make_uint4(word(at[k].x), word(at[k].y), word(at[k].z), word(at[k].w));
#pragma unroll
    for (uint32_t k = 0; k < kKeepQuads; ++k)
    {
        v[k].x = at[k].x < e.n ? v[k].x : 0u, v[k].y = at[k].y < e.n ? v[k].y : 0u;
        v[k].z = at[k].z < e.n ? v[k].z : 0u, v[k].w = at[k].w < e.n ? v[k].w : 0u;
        if (begin + 4 * (k * kBlock + threadIdx.x) < end) store_four(dst + (int64_t)place(k) * 4, v[k]);
    }
}

// Where there are no entries to take.
__device__ __forceinline__ void keep_nothing(const KeepEntry& e, char* dst, uint32_t begin)
{
    const uint64_t bytes = (uint64_t)e.kept * e.units << e.unit_log, each = (uint64_t)kKeepChunk << e.unit_log;
    for (uint64_t p = ((uint64_t)begin << e.unit_log) + threadIdx.x; p < min(bytes, ((uint64_t)begin << e.unit_log) + each); p += kBlock) dst[p] = 0;
}

__global__ void __launch_bounds__(kBlock) keep_rows_kernel(KeepLaunch a)
{
    const ChunkFinder<finder_groups(kKeepEntries)> find(a);
    const KeepEntry& e    = a.e[__builtin_amdgcn_readfirstlane(find(blockIdx.x))];
    const uint32_t chunk  = blockIdx.x - e.first_chunk, outer = chunk / e.chunks, begin = (chunk - outer * e.chunks) * kKeepChunk;
    const uint32_t of_row = (outer + e.outer_in_row) / e.per_index;
    const int32_t* index  = e.index + (int64_t)of_row * e.index_stride;
    const char* src       = e.src + (int64_t)outer * e.src_outer;
    char* dst             = e.dst + (int64_t)outer * e.dst_outer;
    if (e.n == 0) keep_nothing(e, dst, begin);
    else if (e.unit_log == 2 && e.units == 1) keep_words(e, index, src, dst, begin / kKeepChunk * kKeepWords);
    else if (e.unit_log == 4) keep_units<uint4>(e, index, src, dst, begin);
    else if (e.unit_log == 3) keep_units<uint2>(e, index, src, dst, begin);
    else if (e.unit_log == 2) keep_units<uint32_t>(e, index, src, dst, begin);
    else if (e.unit_log == 1) keep_units<uint16_t>(e, index, src, dst, begin);
    else keep_units<uint8_t>(e, index, src, dst, begin);
}
}  // namespace vetrast
