// Element types of the operators that take f32, f16 or bf16 tensors: 16-byte
// pieces of a row and what the entry points check.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/tatara_hip.h"
#include "common.hpp"
#include "streams.hpp"

namespace tatara {

using f16_t = _Float16;
using bf16_t = __bf16;

constexpr uint32_t kWave = 64;

// V elements of a row, as they lie in memory.  A row may start at any element
// (a column range of a wider row), so the copies promise element alignment
// only; gfx950 takes unaligned 16-byte global accesses as one instruction.
template <typename T>
struct Piece {
    static constexpr int V = 16 / sizeof(T);
    T v[V];

    // `left` elements of the row remain at p; what lies past them becomes zero
    __device__ __forceinline__ void load(const T* p, int left) {
        if (left >= V) {
            __builtin_memcpy(v, p, 16);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = j < left ? p[j] : (T)0.0f;
        }
    }
    __device__ __forceinline__ void store(T* p, int left) const {
        if (left >= V) {
            __builtin_memcpy(p, v, 16);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < left) p[j] = v[j];
        }
    }
};

// n floats at any float address; past `left` they become `fill`
template <int N>
__device__ __forceinline__ void load_f32(float (&d)[N], const float* p, int left, float fill) {
    if (left >= N) {
        __builtin_memcpy(d, p, 4 * N);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) d[j] = j < left ? p[j] : fill;
    }
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

inline uint32_t elem_bytes(int32_t dtype) { return dtype == TATARA_F32 ? 4 : 2; }

// Whether the stream can take work of the current device.
int32_t check_stream(TataraStream* stream);

#define TATARA_REQUIRE_DTYPE(dtype) \
    TATARA_REQUIRE((dtype) == TATARA_F32 || (dtype) == TATARA_F16 || (dtype) == TATARA_BF16, "unknown element type")

#define TATARA_REQUIRE_ALIGNED(ptr, bytes) \
    TATARA_REQUIRE((uintptr_t)(ptr) % (bytes) == 0, #ptr " is not aligned to its element")

// The body is compiled once for each element type, as T.
#define TATARA_FOR_DTYPE(dtype, ...)       \
    do {                                   \
        if ((dtype) == TATARA_F32) {       \
            using T = float;               \
            __VA_ARGS__;                   \
        } else if ((dtype) == TATARA_F16) { \
            using T = ::tatara::f16_t;     \
            __VA_ARGS__;                   \
        } else {                           \
            using T = ::tatara::bf16_t;    \
            __VA_ARGS__;                   \
        }                                  \
    } while (0)

}  // namespace tatara
