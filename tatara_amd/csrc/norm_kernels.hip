// Layer norm of rows, forward and backward.
//
//   forward:  mean_r = sum_c x / C,  rstd_r = 1 / sqrt(sum_c (x - mean_r)^2 / C + eps),
//             y = (x - mean) rstd w + b
//   backward: h = (x - mean) rstd,  g = dy w,
//             dx = rstd (g - sum_c g / C - h sum_c (g h) / C),
//             dw = sum_r dy h,  db = sum_r dy
//
// Every sum is f32 and in a fixed order (no atomics), so results do not change
// from run to run.
#include "elem.hpp"

namespace tatara {
namespace {

// Values of a row that a lane holds at most; with 16 waves on a row that is
// 32768 columns.
constexpr int kLaneValues = 32;
constexpr uint32_t kMaxCols = 16 * kWave * kLaneValues;
// Workgroups of the backward pass, each of which leaves a partial sum of dw and db.
constexpr uint32_t kGradBlocks = 512;

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

template <typename T, int W, int N>
__global__ __launch_bounds__(W == 16 ? 1024 : 256) void norm_forward_kernel(
    const T* __restrict__ x, int64_t x_stride, const float* __restrict__ weight, const float* __restrict__ bias,
    T* __restrict__ y, int64_t y_stride, float* __restrict__ mean, float* __restrict__ rstd, uint64_t rows,
    uint32_t cols, float eps) {
    constexpr int V = Piece<T>::V;
    __shared__ float part[2][W];
    const uint32_t lane = threadIdx.x % (kWave * W);
    const uint64_t row = (uint64_t)blockIdx.x * (blockDim.x / (kWave * W)) + threadIdx.x / (kWave * W);
    if (row >= rows) return;  // W > 1: one row a workgroup, so all of it returns
    const T* xr = x + (int64_t)row * x_stride;
    Piece<T> in[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (i * kWave * W + lane) * V;
        in[i].load(xr + c, (int)cols - c);
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) s += (float)in[i].v[j];
    const float m = row_sum<W>(s, part, 0) / (float)cols;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int left = (int)cols - (int)(i * kWave * W + lane) * V;
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
        const int c = (i * kWave * W + lane) * V;
        const int left = (int)cols - c;
        if (left <= 0) break;
        float w[V], b[V];
        if (weight) load_f32(w, weight + c, left, 0.0f);
        if (bias) load_f32(b, bias + c, left, 0.0f);
        Piece<T> out;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float h = ((float)in[i].v[j] - m) * r;
            out.v[j] = (T)fmaf(h, weight ? w[j] : 1.0f, bias ? b[j] : 0.0f);
        }
        out.store(yr + c, left);
    }
}

template <typename T, int W, int N>
__global__ __launch_bounds__(W == 16 ? 1024 : 256) void norm_backward_kernel(
    const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride,
    const float* __restrict__ weight, const float* __restrict__ mean, const float* __restrict__ rstd,
    T* __restrict__ dx, int64_t dx_stride, float* __restrict__ partial, uint64_t rows, uint32_t cols) {
    constexpr int V = Piece<T>::V;
    constexpr int G = W == 1 ? 4 : 1;  // rows that the workgroup has in hand
    __shared__ float part[4][W];
    __shared__ float join[G == 1 ? 1 : (G - 1) * kWave * N * V];
    const uint32_t lane = threadIdx.x % (kWave * W), group = threadIdx.x / (kWave * W);
    float dw[N * V], db[N * V];
#pragma unroll
    for (int i = 0; i < N * V; ++i) dw[i] = db[i] = 0.0f;
    int slot = 0;
    for (uint64_t row = (uint64_t)blockIdx.x * G + group; row < rows; row += (uint64_t)gridDim.x * G) {
        Piece<T> px[N], pd[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = (i * kWave * W + lane) * V;
            px[i].load(x + (int64_t)row * x_stride + c, (int)cols - c);
            pd[i].load(dy + (int64_t)row * dy_stride + c, (int)cols - c);
        }
        const float m = mean[row], r = rstd[row];
        float sg = 0.0f, sgh = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = (i * kWave * W + lane) * V;
            float w[V];
            if (weight) load_f32(w, weight + c, (int)cols - c, 0.0f);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                // past the row's end dy is zero, and with it every sum's term
                const float d = (float)pd[i].v[j], h = ((float)px[i].v[j] - m) * r;
                const float g = weight ? d * w[j] : d;
                sg += g;
                sgh = fmaf(g, h, sgh);
                dw[i * V + j] = fmaf(d, c + j < (int)cols ? h : 0.0f, dw[i * V + j]);
                db[i * V + j] += d;
            }
        }
        const float a = row_sum<W>(sg, part, slot) / (float)cols;
        const float b = row_sum<W>(sgh, part, slot + 1) / (float)cols;
        slot ^= 2;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = (i * kWave * W + lane) * V;
            const int left = (int)cols - c;
            if (left <= 0) break;
            float w[V];
            if (weight) load_f32(w, weight + c, left, 0.0f);
            Piece<T> out;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = (float)pd[i].v[j], h = ((float)px[i].v[j] - m) * r;
                const float g = weight ? d * w[j] : d;
                out.v[j] = (T)((g - a - h * b) * r);
            }
            out.store(dx + (int64_t)row * dx_stride + c, left);
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
    int waves, pieces;  // waves on a row and 16-byte pieces a lane
};

// Rows wide enough for it, or too few to fill the GPU with a wave each, take
// several waves.
NormForm norm_form(uint64_t rows, uint32_t cols, int v) {
    const int most = kLaneValues / v;
    for (int w : {1, 4, 16}) {
        const int n = (int)ceil_div(cols, kWave * w * v);
        if (n > most || (w == 1 && rows < 2048 && n > 1)) continue;
        return {w, n == 5 ? 6 : n == 7 ? 8 : n};
    }
    return {16, most};
}

// Calls f with the form's constants.
template <typename T, typename F>
void with_form(NormForm form, F&& f) {
    auto pieces = [&](auto w) {
        constexpr int W = decltype(w)::value;
        switch (form.pieces) {
            case 1: f(w, std::integral_constant<int, 1>{}); break;
            case 2: f(w, std::integral_constant<int, 2>{}); break;
            case 3: f(w, std::integral_constant<int, 3>{}); break;
            case 4: f(w, std::integral_constant<int, 4>{}); break;
            default:
                if constexpr (Piece<T>::V == 4) {
                    if (form.pieces == 6)
                        f(w, std::integral_constant<int, 6>{});
                    else
                        f(w, std::integral_constant<int, 8>{});
                }
        }
        (void)W;
    };
    if (form.waves == 1)
        pieces(std::integral_constant<int, 1>{});
    else if (form.waves == 4)
        pieces(std::integral_constant<int, 4>{});
    else
        pieces(std::integral_constant<int, 16>{});
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
        with_form<T>(norm_form(rows, cols, Piece<T>::V), [&](auto w, auto n) {
            constexpr int W = decltype(w)::value;
            constexpr int N = decltype(n)::value;
            norm_forward_kernel<T, W, N><<<W == 1 ? ceil_div(rows, 4) : (uint32_t)rows, W == 16 ? 1024 : 256, 0,
                                           raw(stream)>>>(static_cast<const T*>(x), x_stride, weight, bias,
                                                          static_cast<T*>(y), y_stride, mean, rstd, rows, cols, eps);
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
            with_form<T>(norm_form(rows, cols, Piece<T>::V), [&](auto w, auto n) {
                constexpr int W = decltype(w)::value;
                constexpr int N = decltype(n)::value;
                blocks = (uint32_t)std::min<uint64_t>(W == 1 ? (rows + 3) / 4 : rows, kGradBlocks);
                norm_backward_kernel<T, W, N><<<blocks, W == 16 ? 1024 : 256, 0, raw(stream)>>>(
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
