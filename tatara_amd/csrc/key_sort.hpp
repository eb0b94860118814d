// A stable counting sort by keys of up to 1024 values, the step that bucket rows and the
// embedding's gradient are built from.
//
// Items are cut into runs, one a workgroup, and a run into 16 of them, one a wave.  A
// key's items lie by workgroup, wave and place, so the place of an item is the number
// of items with smaller keys, plus those of its key in the workgroups, waves and lanes
// ahead.  With one workgroup all of that is one launch; with more, a first launch
// counts the keys of every run.  Counts are whole numbers: nothing depends on the order
// in which they are added.
//
// Bound by latency: 8192 items of 9 keys in one workgroup 7.8 us, 65536 in 64 of them 2.7 and
// 5.8, of 512 keys 2.7 and 9.3 (every workgroup adds up the counts of all; read one key at a
// time and not ahead 14.8).
#pragma once

#include "elem.hpp"

namespace tatara {
namespace {

constexpr uint32_t kMaxKeys = 1024;
constexpr uint32_t kSortWaves = 16;
constexpr uint32_t kSortThreads = kSortWaves * kWave;
constexpr int kHand = 8;  // items that a lane reads at once
constexpr uint32_t kMaxRuns = 256;
// Items that one workgroup sorts alone, and that a workgroup has at least.
constexpr uint32_t kAlone = 8192;
constexpr uint32_t kLeastRun = 1024;
// Counts of all runs at most (65536 items of 512 keys: 9.3 us, with twice as many 10.0).
constexpr uint32_t kMostCounts = 16384;

struct SortShape {
    uint32_t runs;  // workgroups
    uint32_t run;   // items of each, a multiple of kSortThreads
};

inline uint32_t most_runs(uint32_t keys) { return std::min(kMaxRuns, std::max(16u, kMostCounts / keys)); }

inline SortShape sort_shape(uint64_t items, uint32_t keys) {
    if (items <= kAlone) return {1, (uint32_t)(items + kSortThreads - 1) / kSortThreads * kSortThreads};
    const uint64_t runs = std::min<uint64_t>((items + kLeastRun - 1) / kLeastRun, most_runs(keys));
    const uint64_t run = ((items + runs - 1) / runs + kSortThreads - 1) / kSortThreads * kSortThreads;
    return {(uint32_t)((items + run - 1) / run), (uint32_t)run};
}

// A run's counts are read four at a time.
__host__ __device__ constexpr uint32_t in_fours(uint32_t keys) { return (keys + 3) / 4 * 4; }

// Bytes of the counts of all runs.
inline uint64_t sort_bytes(uint32_t keys) { return 4ull * most_runs(keys) * in_fours(keys); }

// The lanes with the same key (below 2^BITS) as this one, of those that are `in`.
template <int BITS>
__device__ __forceinline__ uint64_t same_key(bool in, uint32_t key) {
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
        const uint64_t set = __ballot(key >> b & 1);
        same &= key >> b & 1 ? set : ~set;
    }
    return same;
}

// Between the lanes' reads of their keys' counters, the additions of the first lane of each
// key, and the next reads: lanes read what others of the wave add to.  The wave's LDS accesses
// are done in their order, which the compiler has to keep; no instruction.
__device__ __forceinline__ void in_wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Exclusive sum over the workgroup's kSortThreads threads.
__device__ __forceinline__ uint32_t sum_ahead(uint32_t x, uint32_t* part) {
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    uint32_t s = x;
#pragma unroll
    for (int d = 1; d < (int)kWave; d *= 2) {
        const uint32_t o = __shfl_up(s, d);
        s += (int)lane >= d ? o : 0u;
    }
    if (lane == kWave - 1) part[wave] = s;
    __syncthreads();
    uint32_t ahead = 0;
#pragma unroll
    for (uint32_t w = 0; w < kSortWaves; ++w) ahead += w < wave ? part[w] : 0u;
    return ahead + s - x;
}

// What is sorted, Items, has
//   Item load(i)      item i,
//   key(item)         its key, below `keys`, or above for one that is left out,
//   put(i, item, key, first, rank)   for each that is not, with the first place of its key
//                     and its number in it,
//   drop(i)           for the others,
//   finish(firsts, keys)   at the end, with the first place of every key and, at [keys],
//                     the number of all.

// counts[run][in_fours(keys)].
template <typename Items>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(Items items, uint64_t n, uint32_t run, uint32_t keys,
                                                                  uint32_t* __restrict__ counts) {
    __shared__ uint32_t count[kMaxKeys];
    const uint32_t width = in_fours(keys);
    for (uint32_t e = threadIdx.x; e < width; e += kSortThreads) count[e] = 0;
    __syncthreads();
    const uint64_t first = (uint64_t)blockIdx.x * run;
    for (uint32_t at0 = 0; at0 < run; at0 += kSortThreads * kHand) {
        uint32_t key[kHand];
#pragma unroll
        for (int h = 0; h < kHand; ++h) {
            const uint32_t at = at0 + h * kSortThreads + threadIdx.x;
            key[h] = at < run && first + at < n ? items.key(items.load(first + at)) : kMaxKeys;
        }
#pragma unroll
        for (int h = 0; h < kHand; ++h)
            if (key[h] < keys) atomicAdd(&count[key[h]], 1u);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < width; e += kSortThreads) counts[(uint64_t)blockIdx.x * width + e] = count[e];
}

// What a workgroup of kSortThreads threads does, with sort_lds(keys) bytes of LDS.  ALONE:
// there is no other, and no counts.
template <int BITS, bool ALONE, typename Items>
__device__ __forceinline__ void sort_place(const Items& items, uint64_t n, uint32_t run, uint32_t keys,
                                           const uint32_t* __restrict__ counts, uint32_t* shared) {
    const uint32_t width = in_fours(keys);
    uint32_t* next = shared;                     // [wave][key]: the next item's place in its key
    uint32_t* total = next + kSortWaves * keys;  // [width]
    uint32_t* ahead = total + width;             // [width]: in the runs ahead of this one
    uint32_t* first = ahead + width;             // [keys + 1]
    uint32_t* part = first + keys + 1;           // [wave]
    const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const uint32_t mine = run / kSortWaves;  // items of a wave, a multiple of kWave
    const uint64_t from = (ALONE ? 0 : (uint64_t)blockIdx.x * run) + (uint64_t)wave * mine;
    typename Items::Item item[kHand];
    uint32_t key[kHand];
    auto read = [&](uint32_t at0) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < kHand; ++h) {
            const uint32_t at = at0 + h * kWave + lane;
            const bool here = at < mine && from + at < n;
            if (here) item[h] = items.load(from + at);
            key[h] = here ? items.key(item[h]) : kMaxKeys;
        }
    };
    // what is read of memory is on its way before the first barrier
    read(0);
    uint32_t all[4] = {}, before[4] = {};
    const uint32_t share = threadIdx.x / (width / 4), four = (threadIdx.x - share * (width / 4)) * 4;
    const uint32_t shares = kSortThreads / (width / 4);
    if (!ALONE && share < shares) {
#pragma unroll 8
        for (uint32_t b = share; b < gridDim.x; b += shares) {
            const uint4 c = *reinterpret_cast<const uint4*>(counts + b * width + four);
            const bool earlier = b < blockIdx.x;
            all[0] += c.x, all[1] += c.y, all[2] += c.z, all[3] += c.w;
            before[0] += earlier ? c.x : 0, before[1] += earlier ? c.y : 0;
            before[2] += earlier ? c.z : 0, before[3] += earlier ? c.w : 0;
        }
    }
    for (uint32_t i = threadIdx.x; i < kSortWaves * keys + 2 * width; i += kSortThreads) shared[i] = 0;
    __syncthreads();
    uint32_t* my_next = next + wave * keys;
    for (uint32_t at0 = 0; at0 < mine; at0 += kWave * kHand) {
        if (at0) read(at0);
#pragma unroll
        for (int h = 0; h < kHand; ++h)
            if (key[h] < keys) atomicAdd(&my_next[key[h]], 1u);
    }
    if (!ALONE && share < shares) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (all[j]) atomicAdd(&total[four + j], all[j]);
            if (before[j]) atomicAdd(&ahead[four + j], before[j]);
        }
    }
    __syncthreads();
    // kMaxKeys threads are enough for all keys
    const uint32_t e = threadIdx.x;
    if (e < keys) {
        uint32_t s = ahead[e], c[kSortWaves];
#pragma unroll
        for (uint32_t w = 0; w < kSortWaves; ++w) c[w] = next[w * keys + e];
#pragma unroll
        for (uint32_t w = 0; w < kSortWaves; ++w) {
            next[w * keys + e] = s;
            s += c[w];
        }
        if (ALONE) total[e] = s;
    }
    const uint32_t count = e < keys ? total[e] : 0u;
    const uint32_t start = sum_ahead(count, part);
    if (e < keys) first[e] = start;
    if (e + 1 == keys) first[keys] = start + count;
    __syncthreads();
    for (uint32_t at0 = 0; at0 < mine; at0 += kWave * kHand) {
        if (at0 || mine > kWave * kHand) read(at0);
#pragma unroll
        for (int h = 0; h < kHand; ++h) {
            if (at0 + h * kWave < mine) {
                const uint64_t i = from + at0 + h * kWave + lane;
                const bool in = key[h] < keys;
                const uint64_t same = same_key<BITS>(in, key[h]);
                const uint64_t below = same & ((1ull << lane) - 1);
                uint32_t rank = 0;
                if (in) rank = __hip_atomic_load(&my_next[key[h]], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                in_wave_order();
                if (in && below == 0) atomicAdd(&my_next[key[h]], (uint32_t)__popcll(same));
                in_wave_order();
                rank += (uint32_t)__popcll(below);
                if (in)
                    items.put(i, item[h], key[h], first[key[h]], rank);
                else if (i < n)
                    items.drop(i);
            }
        }
    }
    items.finish(first, keys);
}

template <typename Items, int BITS, bool ALONE>
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(Items items, uint64_t n, uint32_t run, uint32_t keys,
                                                                  const uint32_t* __restrict__ counts) {
    extern __shared__ uint32_t shared[];
    sort_place<BITS, ALONE>(items, n, run, keys, counts, shared);
}

inline uint32_t sort_lds(uint32_t keys) { return 4 * (kSortWaves * keys + 2 * in_fours(keys) + keys + 1 + kSortWaves); }

// Calls f with bits that tell the keys apart.
template <typename F>
void with_bits(uint32_t keys, F&& f) {
    if (keys <= 16)
        f(std::integral_constant<int, 4>{});
    else if (keys <= 128)
        f(std::integral_constant<int, 7>{});
    else
        f(std::integral_constant<int, 10>{});
}

template <typename Items>
int32_t launch_sort(const Items& items, uint64_t n, uint32_t keys, uint32_t* counts, hipStream_t stream) {
    const SortShape shape = sort_shape(std::max<uint64_t>(n, 1), keys);
    if (shape.runs > 1) {
        sort_count_kernel<<<shape.runs, kSortThreads, 0, stream>>>(items, n, shape.run, keys, counts);
        TATARA_LAUNCHED("sort_count");
    }
    with_bits(keys, [&](auto bits) {
        constexpr int BITS = decltype(bits)::value;
        if (shape.runs > 1)
            sort_place_kernel<Items, BITS, false>
                <<<shape.runs, kSortThreads, sort_lds(keys), stream>>>(items, n, shape.run, keys, counts);
        else
            sort_place_kernel<Items, BITS, true>
                <<<1, kSortThreads, sort_lds(keys), stream>>>(items, n, shape.run, keys, nullptr);
    });
    TATARA_LAUNCHED("sort_place");
    return kOk;
}

}  // namespace
}  // namespace tatara
