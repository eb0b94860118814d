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

// V elements of a row, as they lie in memory.  A row may start at any element (a
// column range of a wider row), so the copies promise element alignment only;
// gfx950 takes unaligned 16-byte global accesses as one instruction.
template <typename T>
struct Piece {
    static constexpr int V = 16 / sizeof(T);
    T v[V];

    // The V elements from column c of a row of cols >= V, or, where fewer are
    // left, the row's last V: a load in no branch, which would be waited for there.
    // What it read is put right by fix(), when it is needed.
    __device__ __forceinline__ void load(const T* row, int c, int cols) {
        __builtin_memcpy(v, row + (c < cols - V ? c : cols - V), 16);
    }
    // `left` = cols - c elements first, zeros after them.
    __device__ __forceinline__ void fix(int left) {
        if (left < V) {
            unsigned __int128 bits;
            __builtin_memcpy(&bits, v, 16);
            bits = left <= 0 ? 0 : bits >> ((V - left) * (int)sizeof(T) * 8);
            __builtin_memcpy(v, &bits, 16);
        }
    }
    // of a row of fewer than V
    __device__ __forceinline__ void load_few(const T* row, int left) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = j < left ? row[j] : (T)0.0f;
    }
    // The 16 bytes are one vector: as elements they become stores of 12 and 4 bytes
    // (65536 x 1536 bf16 normalised with a residual: 164 us, so 145).
    __device__ __forceinline__ void store(T* p, int left) const {
        if (left >= V)
            *reinterpret_cast<Unaligned*>(p) = words();
        else
            store_few(p, left);
    }
    // The same, not kept in the caches.
    __device__ __forceinline__ void store_past(T* p, int left) const {
        if (left >= V) {
            __builtin_nontemporal_store(words(), reinterpret_cast<Unaligned*>(p));
            asm volatile("");  // else this becomes one store with that of another branch
        } else {
            store_few(p, left);
        }
    }
    // Has the compiler compute again what follows from the values, where it would keep it in
    // registers that a wide row does not have.
    __device__ __forceinline__ void forget() {
        Words w = words();
        asm volatile("" : "+v"(w));
        __builtin_memcpy(v, &w, 16);
    }

   private:
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    typedef Words Unaligned __attribute__((aligned(2)));
    __device__ __forceinline__ Words words() const {
        Words w;
        __builtin_memcpy(&w, v, 16);
        return w;
    }
    __device__ __forceinline__ void store_few(T* p, int left) const {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < left) p[j] = v[j];
    }
};

// N floats (4 or 8) from column c of a row, as Piece::load and fix.
template <int N>
struct Floats {
    Piece<float> p[N / 4];
    __device__ __forceinline__ void load(const float* row, int c, int cols) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) p[i].load(row, c + 4 * i, cols);
    }
    __device__ __forceinline__ void load_few(const float* row, int left) {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i / 4].v[i % 4] = i < left ? row[i] : 0.0f;
    }
    __device__ __forceinline__ void fix(int left) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) p[i].fix(left - 4 * i);
    }
    __device__ __forceinline__ float operator[](int i) const { return p[i / 4].v[i % 4]; }
};

// The lane's partner at step S of a join over groups of 2, 4, .. 64 lanes: another
// part of the group of 2^(S+1), so that after each step all lanes of that group
// hold the same.  Within 16 lanes a data-parallel modifier of the adding
// instruction, beyond a swap of half waves: no trip through LDS, whose wait a join
// of six would pay six times.
template <int S>
__device__ __forceinline__ uint32_t partner(uint32_t x) {
    if constexpr (S == 0) return __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xf, 0xf, true);   // lane ^ 1
    if constexpr (S == 1) return __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xf, 0xf, true);   // lane ^ 2
    if constexpr (S == 2) return __builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, true);  // 7 - lane of eight
    if constexpr (S == 3) return __builtin_amdgcn_update_dpp(0, x, 0x140, 0xf, 0xf, true);  // 15 - lane of sixteen
    if constexpr (S == 4) {
        const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)) & 16 ? r[0] : r[1];
    }
    if constexpr (S == 5) {
        const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)) & 32 ? r[0] : r[1];
    }
    return x;
}

// Joins over groups of G lanes (a power of two), the same in all lanes of a group.
template <int G, typename F>
__device__ __forceinline__ uint32_t group_join_u(uint32_t x, F&& f) {
    if constexpr (G > 1) x = f(x, partner<0>(x));
    if constexpr (G > 2) x = f(x, partner<1>(x));
    if constexpr (G > 4) x = f(x, partner<2>(x));
    if constexpr (G > 8) x = f(x, partner<3>(x));
    if constexpr (G > 16) x = f(x, partner<4>(x));
    if constexpr (G > 32) x = f(x, partner<5>(x));
    return x;
}
template <int G, typename F>
__device__ __forceinline__ float group_join(float x, F&& f) {
    return __uint_as_float(group_join_u<G>(__float_as_uint(x), [&](uint32_t a, uint32_t b) {
        return __float_as_uint(f(__uint_as_float(a), __uint_as_float(b)));
    }));
}
template <int G>
__device__ __forceinline__ float group_sum(float x) {
    return group_join<G>(x, [](float a, float b) { return a + b; });
}
template <int G>
__device__ __forceinline__ float group_max(float x) {
    return group_join<G>(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float x) { return group_sum<(int)kWave>(x); }

// Sum over the wave's lanes of the same place in groups of G; of use in the first
// group (the lanes of sixteen are turned round, so others add in another order).
template <int G, typename V, typename F>
__device__ __forceinline__ V column_join(V x, F&& f) {
    auto add = [&](uint32_t other) {
        V o;
        __builtin_memcpy(&o, &other, 4);
        x = f(x, o);
    };
    auto bits = [&] {
        uint32_t b;
        __builtin_memcpy(&b, &x, 4);
        return b;
    };
    if constexpr (G <= 1) add(partner<0>(bits()));
    if constexpr (G <= 2) add(partner<1>(bits()));
    if constexpr (G <= 4) add(__builtin_amdgcn_update_dpp(0, bits(), 0x124, 0xf, 0xf, true));  // turned by 4
    if constexpr (G <= 8) add(__builtin_amdgcn_update_dpp(0, bits(), 0x128, 0xf, 0xf, true));  // by 8
    if constexpr (G <= 16) add(partner<4>(bits()));
    if constexpr (G <= 32) add(partner<5>(bits()));
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
