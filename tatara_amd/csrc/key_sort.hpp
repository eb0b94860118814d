// A stable counting sort by keys of up to 1024 values, the step that bucket rows and the
// embedding's gradient are built from.
//
// Items are cut into runs, one a workgroup, and a run into 16 of them, one a wave.  A
// key's items lie by workgroup, wave and place, so the place of an item is the number
// of items with smaller keys, plus those of its key in the workgroups, waves and lanes
// ahead.  With one workgroup all of that is one launch; with more, a first launch
// counts the keys of every run.  Counts are whole numbers: nothing depends on the order
// in which they are added.
#pragma once

#include "elem.hpp"

namespace tatara {
namespace {

constexpr uint32_t kMaxKeys = 1024;
constexpr uint32_t kSortWaves = 16;
constexpr uint32_t kSortThreads = kSortWaves * kWave;
constexpr uint32_t kMaxRuns = 256;
// Items that one workgroup sorts alone, and that a workgroup has at least.
constexpr uint32_t kAlone = 8192;
constexpr uint32_t kLeastRun = 1024;

struct SortShape {
    uint32_t runs;  // workgroups
    uint32_t run;   // items of each, a multiple of kSortThreads
};

// With more runs of many keys a workgroup would add up more counts than it has items.
inline uint32_t most_runs(uint32_t keys) { return std::min(kMaxRuns, std::max(16u, 32768u / keys)); }

inline SortShape sort_shape(uint64_t items, uint32_t keys) {
    if (items <= kAlone) return {1, (uint32_t)(items + kSortThreads - 1) / kSortThreads * kSortThreads};
    const uint64_t runs = std::min<uint64_t>((items + kLeastRun - 1) / kLeastRun, most_runs(keys));
    const uint64_t run = ((items + runs - 1) / runs + kSortThreads - 1) / kSortThreads * kSortThreads;
    return {(uint32_t)((items + run - 1) / run), (uint32_t)run};
}

// Bytes of the counts of all runs.
inline uint64_t sort_bytes(uint32_t keys) { return 4ull * most_runs(keys) * keys; }

// The lanes with the same key (below 2^bits) as this one, of those that are `in`.
__device__ __forceinline__ uint64_t same_key(bool in, uint32_t key, int bits) {
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot(key >> b & 1);
        same &= key >> b & 1 ? set : ~set;
    }
    return same;
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

// counts[run][key].  Keys: key(i) of item i, below `keys`, or kMaxKeys for an item that is
// left out.
template <typename Keys>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(Keys items, uint64_t n, uint32_t run, uint32_t keys,
                                                                  uint32_t* __restrict__ counts) {
    __shared__ uint32_t count[kMaxKeys];
    for (uint32_t e = threadIdx.x; e < keys; e += kSortThreads) count[e] = 0;
    __syncthreads();
    const uint64_t first = (uint64_t)blockIdx.x * run;
    for (uint32_t at = threadIdx.x; at < run; at += kSortThreads) {
        const uint32_t key = first + at < n ? items.key(first + at) : kMaxKeys;
        if (key < keys) atomicAdd(&count[key], 1u);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < keys; e += kSortThreads) counts[(uint64_t)blockIdx.x * keys + e] = count[e];
}

// Calls items.put(i, key, first place of its key, its number among them) for every item
// that is not left out and items.drop(i) for the others, then items.finish(firsts, keys)
// with the first place of every key and, at [keys], their number.
template <typename Keys>
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(Keys items, uint64_t n, uint32_t run, uint32_t keys,
                                                                  int bits, const uint32_t* __restrict__ counts) {
    extern __shared__ uint32_t shared[];
    uint32_t* next = shared;                                // [wave][key]: the next item's place in its key
    uint32_t* total = next + kSortWaves * keys;             // [key]
    uint32_t* ahead = total + keys;                         // [key]: in the runs ahead of this one
    uint32_t* first = ahead + keys;                         // [key + 1]
    uint32_t* part = first + keys + 1;                      // [wave]
    const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    for (uint32_t i = threadIdx.x; i < (kSortWaves + 2) * keys; i += kSortThreads) shared[i] = 0;
    __syncthreads();
    const uint32_t mine = run / kSortWaves;  // items of a wave, a multiple of kWave
    const uint64_t from = (uint64_t)blockIdx.x * run + (uint64_t)wave * mine;
    uint32_t* my_next = next + wave * keys;
    for (uint32_t at = lane; at < mine; at += kWave) {
        const uint32_t key = from + at < n ? items.key(from + at) : kMaxKeys;
        if (key < keys) atomicAdd(&my_next[key], 1u);
    }
    if (gridDim.x > 1) {
        for (uint32_t i = threadIdx.x; i < gridDim.x * keys; i += kSortThreads) {
            const uint32_t b = i / keys, e = i - b * keys, c = counts[i];
            if (c) {
                atomicAdd(&total[e], c);
                if (b < blockIdx.x) atomicAdd(&ahead[e], c);
            }
        }
    }
    __syncthreads();
    // kMaxKeys threads are enough for all keys
    const uint32_t e = threadIdx.x;
    if (e < keys) {
        uint32_t s = ahead[e];
        for (uint32_t w = 0; w < kSortWaves; ++w) {
            const uint32_t c = next[w * keys + e];
            next[w * keys + e] = s;
            s += c;
        }
        if (gridDim.x == 1) total[e] = s;
    }
    const uint32_t count = e < keys ? total[e] : 0u;
    const uint32_t start = sum_ahead(count, part);
    if (e < keys) first[e] = start;
    if (e + 1 == keys) first[keys] = start + count;
    __syncthreads();
    for (uint32_t at0 = 0; at0 < mine; at0 += kWave) {
        const uint64_t i = from + at0 + lane;
        const uint32_t key = i < n ? items.key(i) : kMaxKeys;
        const bool in = key < keys;
        const uint64_t same = same_key(in, key, bits);
        const uint64_t below = same & ((1ull << lane) - 1);
        uint32_t rank = 0;
        if (in) rank = __hip_atomic_load(&my_next[key], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        if (in && below == 0) atomicAdd(&my_next[key], (uint32_t)__popcll(same));  // behind the wave's loads
        rank += (uint32_t)__popcll(below);
        if (in)
            items.put(i, key, first[key], rank);
        else if (i < n)
            items.drop(i);
    }
    items.finish(first, keys);
}

inline uint32_t sort_lds(uint32_t keys) { return 4 * ((kSortWaves + 3) * keys + 1 + kSortWaves); }

template <typename Keys>
int32_t launch_sort(const Keys& items, uint64_t n, uint32_t keys, uint32_t* counts, hipStream_t stream) {
    const SortShape shape = sort_shape(std::max<uint64_t>(n, 1), keys);
    if (shape.runs > 1) {
        sort_count_kernel<<<shape.runs, kSortThreads, 0, stream>>>(items, n, shape.run, keys, counts);
        TATARA_LAUNCHED("sort_count");
    }
    int bits = 0;
    while ((1u << bits) < keys) ++bits;
    sort_place_kernel<<<shape.runs, kSortThreads, sort_lds(keys), stream>>>(items, n, shape.run, keys, bits, counts);
    TATARA_LAUNCHED("sort_place");
    return kOk;
}

}  // namespace
}  // namespace tatara
