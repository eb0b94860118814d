// What the norms of rows share: how many waves and registers a row takes, and the
// sums over them.
#pragma once

#include "elem.hpp"

namespace tatara {
namespace {

// Values of a row that a lane holds at most; with 16 waves on a row that is
// 32768 columns.
constexpr int kLaneValues = 32;
constexpr uint32_t kMaxCols = 16 * kWave * kLaneValues;
// Workgroups of the backward pass, each of which leaves a partial sum of dw and db:
// two a CU (65536 x 1536 bf16: 122 us, with four 130), one where rows are few
// (1009 x 769 f32: 8.8 us, with two 9.5).
constexpr uint32_t kGradBlocks = 512;
uint32_t grad_blocks(uint64_t units) {
    return (uint32_t)std::min<uint64_t>(units, units >= 2048 ? kGradBlocks : kGradBlocks / 2);
}

// Workgroups of the forward pass at most: a launch has room for 2^32 threads.
constexpr uint32_t kMaxGrid = 1u << 20;

// Sum over the W waves of a row; `slot` alternates so that one barrier a sum is enough.
template <int W>
__device__ __forceinline__ float row_sum(float x, float (*part)[W], int slot) {
    x = wave_sum(x);
    if constexpr (W > 1) {
        if (threadIdx.x % kWave == 0) part[slot][threadIdx.x / kWave] = x;
        __syncthreads();
        x = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) x += part[slot][i];
    }
    return x;
}

// The gradients of one or two parameters of `cols` values (the second of the columns
// from `cols` on) from the workgroups' partial sums of `width` values: 64 columns a
// workgroup, 16 waves that take every 16th partial, joined in order.
__global__ __launch_bounds__(1024) void norm_param_grad_kernel(const float* __restrict__ partial, uint32_t blocks,
                                                               uint32_t cols, uint32_t width, float* __restrict__ dw,
                                                               float* __restrict__ db) {
    __shared__ float part[16][kWave];
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t c = blockIdx.x * kWave + lane;
    float s = 0.0f;
    if (c < width)
#pragma unroll 8
        for (uint32_t b = wave; b < blocks; b += 16) s += partial[(uint64_t)b * width + c];
    part[wave][lane] = s;
    __syncthreads();
    if (wave || c >= width) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) s += part[i][lane];
    float* to = c < cols ? dw : db;
    if (to) to[c < cols ? c : c - cols] = s;
}

struct NormForm {
    int waves, pieces;  // waves on a row and 16-byte pieces a lane (0: less than one)
};

// 16-byte pieces that a lane holds with `waves` waves on a row, at most.  A wave
// alone is fastest where a row's values leave it registers for the next row's: up
// to 24 values a lane (40000 rows forward: 640 columns f32 34 us, with four waves
// 42; 1536 bf16 47 and 56; but 2048 f32 134 and 125, bf16 79 and 77), 16 in the f32
// backward pass (640: 57 and 80; 1536: 143 and 131).  Four waves go up to 32
// (16384 x 8192 f32: 211, with sixteen 249), backward 24 (bf16: 180 and 163).
constexpr int most_pieces(bool backward, int waves, int v) {
    const int values = waves == 1 ? (backward && v == 4 ? 16 : 24) : waves == 4 && backward ? 24 : kLaneValues;
    return values / v;
}
// Sixteen waves take what is too wide for four.
constexpr int least_pieces(bool backward, int waves, int v) {
    return waves == 16 ? most_pieces(backward, 4, v) / 4 + 1 : 1;
}

// Rows wide enough for it, or too few to fill the GPU with a wave each (backward,
// 1009 x 1536 f32: 13.1 us with one, 10.5 with four; from 2048 rows on 13.0 and
// 13.5), take several waves.
NormForm norm_form(bool backward, uint64_t rows, uint32_t cols, int v) {
    if (cols < (uint32_t)v) return {1, 0};
    for (int w : {1, 4}) {
        const int n = (int)ceil_div(cols, kWave * w * v);
        if (n > most_pieces(backward, w, v) || (w == 1 && rows < 1024 && n > 1)) continue;
        return {w, n == 5 ? 6 : n == 7 ? 8 : n};
    }
    const int n = (int)ceil_div(cols, kWave * 16 * v);
    return {16, n == 5 ? 6 : n == 7 ? 8 : n};
}

// Calls f with the form's constants.
template <typename T, bool BACKWARD, typename F>
void with_form(NormForm form, F&& f) {
    using std::integral_constant;
    auto pieces = [&](auto w) {
        constexpr int W = decltype(w)::value, V = Piece<T>::V;
        auto is = [&](auto n) {
            constexpr int N = decltype(n)::value;
            if constexpr (N >= least_pieces(BACKWARD, W, V) && N <= most_pieces(BACKWARD, W, V))
                if (form.pieces == N) f(w, n, std::false_type{});
        };
        is(integral_constant<int, 1>{});
        is(integral_constant<int, 2>{});
        is(integral_constant<int, 3>{});
        is(integral_constant<int, 4>{});
        is(integral_constant<int, 6>{});
        is(integral_constant<int, 8>{});
    };
    if (form.pieces == 0)
        f(integral_constant<int, 1>{}, integral_constant<int, 1>{}, std::true_type{});
    else if (form.waves == 1)
        pieces(integral_constant<int, 1>{});
    else if (form.waves == 4)
        pieces(integral_constant<int, 4>{});
    else
        pieces(integral_constant<int, 16>{});
}

}  // namespace
}  // namespace tatara
