// Layer norm of rows, forward and backward.
//
//   forward:  mean_r = sum_c x / C,  rstd_r = 1 / sqrt(sum_c (x - mean_r)^2 / C + eps),
//             y = (x - mean) rstd w + b
//   backward: h = (x - mean) rstd,  g = dy w,
//             dx = rstd (g - sum_c g / C - h sum_c (g h) / C),
//             dw = sum_r dy h,  db = sum_r dy
//
// Every sum is f32 and in a fixed order (no atomics), so results do not change
// from run to run.  The variance is of differences from the mean, which a row held
// in registers gives without a second read.
//
// Both passes read and write each value once and are bound by memory: 65536 x 1536
// take 152 us forward in f32 (5.3 TB/s; a copy of 2 GiB runs at 4.9) and 122 us
// backward in bf16 (4.9 TB/s).  Small ones are bound by their launches: 3.7 us
// forward, 6.7 backward (two launches) at 64 x 1536.  From 8193 columns on the backward
// pass's sixteen waves hold more than their registers (40 to 700 bytes a lane in
// scratch): 16384 x 12288 f32 469 us (5.2 TB/s), x 16384 1035 (3.1), 8192 x 32768 3068.
// (Calls of the C entry points, back to back.)
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

// FEW: rows of fewer elements than a piece has.
template <typename T, int W, int N, bool FEW>
__global__ __launch_bounds__(W == 16 ? 1024 : 256) void norm_forward_kernel(
    const T* __restrict__ x, int64_t x_stride, const float* __restrict__ weight, const float* __restrict__ bias,
    T* __restrict__ y, int64_t y_stride, float* __restrict__ mean, float* __restrict__ rstd, uint64_t rows,
    uint32_t cols, float eps) {
    constexpr int V = Piece<T>::V;
    __shared__ float part[2][W];
    const uint32_t lane = threadIdx.x % (kWave * W);
    auto column = [&](int i) { return (int)(i * kWave * W + lane) * V; };
    auto read = [&](auto& piece, const auto* from, int i) {
        if (FEW)
            piece.load_few(from, (int)cols - column(i));
        else
            piece.load(from, column(i), (int)cols);
    };
    auto fix = [&](auto& piece, int i) {
        if (!FEW) piece.fix((int)cols - column(i));
    };
    // more rows than the grid has room for are taken in turn
    constexpr int G = W == 1 ? 4 : 1;
    const uint64_t step = (uint64_t)gridDim.x * G;
    for (uint64_t row = (uint64_t)blockIdx.x * G + threadIdx.x / (kWave * W); row < rows; row += step) {
        Piece<T> in[N];
#pragma unroll
        for (int i = 0; i < N; ++i) read(in[i], x + (int64_t)row * x_stride, i);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            fix(in[i], i);
#pragma unroll
            for (int j = 0; j < V; ++j) s += (float)in[i].v[j];
        }
        const float m = row_sum<W>(s, part, 0) / (float)cols;
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int left = (int)cols - column(i);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = j < left ? (float)in[i].v[j] - m : 0.0f;
                s = fmaf(d, d, s);
            }
        }
        const float r = 1.0f / sqrtf(row_sum<W>(s, part, 1) / (float)cols + eps);
        if (lane == 0) {
            if (mean) mean[row] = m;
            if (rstd) rstd[row] = r;
        }
        T* yr = y + (int64_t)row * y_stride;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int left = (int)cols - column(i);
            if (left <= 0) break;
            Floats<V> w, b;
            if (weight) read(w, weight, i);
            if (bias) read(b, bias, i);
            if (weight) fix(w, i);
            if (bias) fix(b, i);
            Piece<T> out;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float h = ((float)in[i].v[j] - m) * r;
                out.v[j] = (T)fmaf(h, weight ? w[j] : 1.0f, bias ? b[j] : 0.0f);
            }
            out.store(yr + column(i), left);
        }
    }
}

template <typename T, int W, int N, bool FEW>
__global__ __launch_bounds__(W == 16 ? 1024 : 256) void norm_backward_kernel(
    const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride,
    const float* __restrict__ weight, const float* __restrict__ mean, const float* __restrict__ rstd,
    T* __restrict__ dx, int64_t dx_stride, float* __restrict__ partial, uint64_t rows, uint32_t cols) {
    constexpr int V = Piece<T>::V;
    constexpr int G = W == 1 ? 4 : 1;  // rows that the workgroup has in hand
    __shared__ float part[4][W];
    __shared__ float join[G == 1 ? 1 : (G - 1) * kWave * N * V];
    const uint32_t lane = threadIdx.x % (kWave * W), group = threadIdx.x / (kWave * W);
    auto column = [&](int i) { return (int)(i * kWave * W + lane) * V; };
    auto read = [&](auto& piece, const auto* from, int i) {
        if (FEW)
            piece.load_few(from, (int)cols - column(i));
        else
            piece.load(from, column(i), (int)cols);
    };
    auto fix = [&](auto& piece, int i) {
        if (!FEW) piece.fix((int)cols - column(i));
    };
    // the weight stays in registers where they last
    constexpr bool KEEP = N * V <= 24 || sizeof(T) == 2;
    float dw[N * V], db[N * V];
    Floats<V> kept[KEEP ? N : 1];
#pragma unroll
    for (int i = 0; i < N * V; ++i) dw[i] = db[i] = 0.0f;
    auto weights = [&](int i) {
        Floats<V> w;
        if (weight) {
            read(w, weight, i);
            fix(w, i);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) w.p[j / 4].v[j % 4] = 1.0f;
        }
        return w;
    };
    if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < N; ++i) kept[i] = weights(i);
    }
    Piece<T> px[N], pd[N];
    float m = 0.0f, r = 0.0f;
    auto read_row = [&](uint64_t row) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            read(px[i], x + (int64_t)row * x_stride, i);
            read(pd[i], dy + (int64_t)row * dy_stride, i);
        }
        m = mean[row];
        r = rstd[row];
    };
    int slot = 0;
    const uint64_t step = (uint64_t)gridDim.x * G;
    uint64_t row = (uint64_t)blockIdx.x * G + group;
    if (row < rows) read_row(row);
    for (; row < rows; row += step) {
        float h[N * V], g[N * V];
        float sg = 0.0f, sgh = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            fix(px[i], i);
            fix(pd[i], i);
            const Floats<V> w = KEEP ? kept[KEEP ? i : 0] : weights(i);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int e = i * V + j;
                // past the row's end dy is zero, and with it every sum's term
                const float d = (float)pd[i].v[j];
                h[e] = column(i) + j < (int)cols ? ((float)px[i].v[j] - m) * r : 0.0f;
                g[e] = d * w[j];
                sg += g[e];
                sgh = fmaf(g[e], h[e], sgh);
                dw[e] = fmaf(d, h[e], dw[e]);
                db[e] += d;
            }
        }
        const float scale = r;
        // the next row's values are on their way while this one's sums are joined
        const uint64_t next = row + step;
        read_row(next < rows ? next : row);
        const float a = row_sum<W>(sg, part, slot) / (float)cols;
        const float b = row_sum<W>(sgh, part, slot + 1) / (float)cols;
        slot ^= 2;
        T* to = dx + (int64_t)row * dx_stride;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            Piece<T> out;
#pragma unroll
            for (int j = 0; j < V; ++j) out.v[j] = (T)((g[i * V + j] - a - h[i * V + j] * b) * scale);
            out.store(to + column(i), (int)cols - column(i));
        }
    }
    if (!partial) return;
    float* to = partial + (uint64_t)blockIdx.x * 2 * cols;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* acc = which ? db : dw;
        if constexpr (G > 1) {
            if (which) __syncthreads();
            if (group > 0) {
#pragma unroll
                for (int i = 0; i < N * V; ++i) join[((group - 1) * N * V + i) * kWave + lane] = acc[i];
            }
            __syncthreads();
            if (group == 0) {
#pragma unroll
                for (int i = 0; i < N * V; ++i)
#pragma unroll
                    for (int o = 0; o < G - 1; ++o) acc[i] += join[(o * N * V + i) * kWave + lane];
            }
        }
        if (group == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = (i * kWave * W + lane) * V;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (c + j < (int)cols) to[(uint64_t)which * cols + c + j] = acc[i * V + j];
            }
        }
    }
}

// dw and db from the workgroups' partial sums: 64 columns a workgroup, 16
// waves that take every 16th partial, joined in order.
__global__ __launch_bounds__(1024) void norm_param_grad_kernel(const float* __restrict__ partial, uint32_t blocks,
                                                               uint32_t cols, float* __restrict__ dw,
                                                               float* __restrict__ db) {
    __shared__ float part[16][kWave];
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t c = blockIdx.x * kWave + lane;  // of both gradients' columns
    float s = 0.0f;
    if (c < 2 * cols)
#pragma unroll 8
        for (uint32_t b = wave; b < blocks; b += 16) s += partial[(uint64_t)b * 2 * cols + c];
    part[wave][lane] = s;
    __syncthreads();
    if (wave || c >= 2 * cols) return;
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

uint64_t partial_bytes(uint32_t cols) { return 4ull * kGradBlocks * 2 * cols; }

}  // namespace
}  // namespace tatara

using namespace tatara;

extern "C" {

int32_t tatara_op_layer_norm_forward(const void* x, int64_t x_stride, const float* weight, const float* bias, void* y,
                                     int64_t y_stride, float* mean, float* rstd, uint64_t rows, uint32_t cols,
                                     float eps, int32_t dtype, TataraStream* stream) {
    TATARA_REQUIRE_DTYPE(dtype);
    TATARA_REQUIRE(cols >= 1 && cols <= kMaxCols, "layer norm takes 1 to 32768 columns");
    TATARA_REQUIRE(rows < (1ull << 31), "too many rows");
    TATARA_REQUIRE(eps >= 0.0f, "eps must not be negative");
    if (rows == 0) return kOk;
    TATARA_REQUIRE(x && y, "null tensor");
    TATARA_REQUIRE(x_stride >= (int64_t)cols && y_stride >= (int64_t)cols, "a row stride is smaller than the row");
    TATARA_REQUIRE_ALIGNED(x, elem_bytes(dtype));
    TATARA_REQUIRE_ALIGNED(y, elem_bytes(dtype));
    if (int32_t st = check_stream(stream)) return st;
    TATARA_FOR_DTYPE(dtype, {
        with_form<T, false>(norm_form(false, rows, cols, Piece<T>::V), [&](auto w, auto n, auto few) {
            constexpr int W = decltype(w)::value;
            constexpr int N = decltype(n)::value;
            const uint32_t blocks = (uint32_t)std::min<uint64_t>(W == 1 ? (rows + 3) / 4 : rows, kMaxGrid);
            norm_forward_kernel<T, W, N, decltype(few)::value><<<blocks, W == 16 ? 1024 : 256, 0, raw(stream)>>>(
                static_cast<const T*>(x), x_stride, weight, bias, static_cast<T*>(y), y_stride, mean, rstd, rows,
                cols, eps);
        });
    });
    TATARA_LAUNCHED("norm_forward");
    return kOk;
}

int32_t tatara_op_layer_norm_backward_workspace(uint32_t cols, uint64_t* bytes) {
    TATARA_REQUIRE(bytes, "null output");
    TATARA_REQUIRE(cols >= 1 && cols <= kMaxCols, "layer norm takes 1 to 32768 columns");
    *bytes = partial_bytes(cols);
    return kOk;
}

int32_t tatara_op_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                                      const float* weight, const float* mean, const float* rstd, void* dx,
                                      int64_t dx_stride, float* dweight, float* dbias, uint64_t rows, uint32_t cols,
                                      int32_t dtype, void* workspace, uint64_t workspace_bytes,
                                      TataraStream* stream) {
    TATARA_REQUIRE_DTYPE(dtype);
    TATARA_REQUIRE(cols >= 1 && cols <= kMaxCols, "layer norm takes 1 to 32768 columns");
    TATARA_REQUIRE(rows < (1ull << 31), "too many rows");
    const bool params = dweight || dbias;
    TATARA_REQUIRE(!params || (workspace && workspace_bytes >= partial_bytes(cols)), "workspace too small");
    TATARA_REQUIRE_ALIGNED(workspace, 16);
    if (rows) {
        TATARA_REQUIRE(dy && x && mean && rstd && dx, "null tensor");
        TATARA_REQUIRE(dy_stride >= (int64_t)cols && x_stride >= (int64_t)cols && dx_stride >= (int64_t)cols,
                       "a row stride is smaller than the row");
        TATARA_REQUIRE_ALIGNED(dy, elem_bytes(dtype));
        TATARA_REQUIRE_ALIGNED(x, elem_bytes(dtype));
        TATARA_REQUIRE_ALIGNED(dx, elem_bytes(dtype));
    }
    if (int32_t st = check_stream(stream)) return st;
    float* partial = params ? static_cast<float*>(workspace) : nullptr;
    uint32_t blocks = 0;
    if (rows) {
        TATARA_FOR_DTYPE(dtype, {
            with_form<T, true>(norm_form(true, rows, cols, Piece<T>::V), [&](auto w, auto n, auto few) {
                constexpr int W = decltype(w)::value;
                constexpr int N = decltype(n)::value;
                blocks = grad_blocks(W == 1 ? (rows + 3) / 4 : rows);
                norm_backward_kernel<T, W, N, decltype(few)::value><<<blocks, W == 16 ? 1024 : 256, 0, raw(stream)>>>(
                    static_cast<const T*>(dy), dy_stride, static_cast<const T*>(x), x_stride, weight, mean, rstd,
                    static_cast<T*>(dx), dx_stride, partial, rows, cols);
            });
        });
        TATARA_LAUNCHED("norm_backward");
    }
    if (params) {
        norm_param_grad_kernel<<<ceil_div(2ull * cols, kWave), 1024, 0, raw(stream)>>>(partial, blocks, cols, dweight,
                                                                                       dbias);
        TATARA_LAUNCHED("norm_param_grad");
    }
    return kOk;
}

}  // extern "C"
