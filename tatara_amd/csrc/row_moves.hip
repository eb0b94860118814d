// Rows from the positions' order into another one and back: what a bucket's layers
// read and write, and what an embedding looks up.
//
// Both kernels go by positions, G lanes each (the power of two that holds a row, up to
// a wave), so that a position's own row is read or written once, however many choices it
// has, and the rows it meets elsewhere are whole ones.  A lane keeps the slots and
// weights of its position's K choices in registers.
#include "row_moves.hpp"

namespace tatara {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxGrid = 1u << 20;

// Sum over groups of `lanes` lanes.
__device__ __forceinline__ float lanes_sum(float x, uint32_t lanes) {
    auto add = [&](uint32_t other) { x += __uint_as_float(other); };
    if (lanes > 1) add(partner<0>(__float_as_uint(x)));
    if (lanes > 2) add(partner<1>(__float_as_uint(x)));
    if (lanes > 4) add(partner<2>(__float_as_uint(x)));
    if (lanes > 8) add(partner<3>(__float_as_uint(x)));
    if (lanes > 16) add(partner<4>(__float_as_uint(x)));
    if (lanes > 32) add(partner<5>(__float_as_uint(x)));
    return x;
}

template <typename T, bool FEW>
__device__ __forceinline__ void read(Piece<T>& p, const T* row, int c, int cols) {
    if (FEW)
        p.load_few(row, cols - c);
    else
        p.load(row, c, cols);
}
template <typename T, bool FEW>
__device__ __forceinline__ void fix(Piece<T>& p, int c, int cols) {
    if (!FEW) p.fix(cols - c);
}

// K: at least top_k; U: pieces of each row in hand.  FEW: rows of fewer elements than
// a piece has.
template <typename T, int K, int U, bool FEW>
__global__ __launch_bounds__(kThreads) void rows_back_kernel(RowsBack a, uint32_t lanes) {
    constexpr int V = Piece<T>::V;
    const uint32_t lane = threadIdx.x & (lanes - 1), per_block = kThreads / lanes;
    const int cols = (int)a.cols;
    const T* rows = static_cast<const T*>(a.rows);
    const uint64_t step = (uint64_t)gridDim.x * per_block;
    for (uint64_t t = (uint64_t)blockIdx.x * per_block + threadIdx.x / lanes; t < a.positions; t += step) {
        const T* from[K];
        float w[K];
        bool in[K];
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const uint64_t at = t * a.top_k + (j < (int)a.top_k ? j : 0);
            const uint32_t s = (uint32_t)a.slot[at];
            in[j] = j < (int)a.top_k && s < a.n_rows;
            w[j] = a.gate ? a.scale * a.gate[at] : a.scale;
            from[j] = rows + (int64_t)(in[j] ? s : 0) * a.rows_stride;
        }
        T* to = static_cast<T*>(a.y) + (int64_t)t * a.y_stride;
        for (int c0 = (int)lane * V; c0 < cols; c0 += (int)lanes * V * U) {
            Piece<T> p[K][U];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < K; ++j) read<T, FEW>(p[j][u], from[j], c0 + u * (int)lanes * V, cols);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u * (int)lanes * V;
                float y[V];
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] = 0.0f;
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    fix<T, FEW>(p[j][u], c, cols);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float v = w[j] * (float)p[j][u].v[e];
                        y[e] = !in[j] ? y[e] : j == 0 ? v : y[e] + v;
                    }
                }
                Piece<T> out;
#pragma unroll
                for (int e = 0; e < V; ++e) out.v[e] = (T)y[e];
                out.store(to + c, cols - c);
            }
        }
    }
}

// DOT: the gates' gradient too.  Behind the workgroups of positions, those from `blocks`
// on clear the rows without a source, kThreads of them each.
template <typename T, int K, int U, bool FEW, bool DOT>
__global__ __launch_bounds__(kThreads) void rows_out_kernel(RowsOut a, uint32_t lanes, uint32_t blocks) {
    constexpr int V = Piece<T>::V;
    const int cols = (int)a.cols;
    T* rows = static_cast<T*>(a.rows);
    if (blockIdx.x >= blocks) {
        __shared__ bool none[kThreads];
        const uint64_t items = a.positions * a.top_k;
        for (uint64_t first = (uint64_t)(blockIdx.x - blocks) * kThreads; first < a.n_rows;
             first += (uint64_t)(gridDim.x - blocks) * kThreads) {
            __syncthreads();
            const uint64_t mine = first + threadIdx.x;
            none[threadIdx.x] = mine < a.n_rows && (uint32_t)a.source[mine] >= items;
            __syncthreads();
            for (int r = 0; r < kThreads; ++r) {
                if (!none[r]) continue;
                Piece<T> zero;
#pragma unroll
                for (int e = 0; e < V; ++e) zero.v[e] = (T)0.0f;
                T* to = rows + (int64_t)(first + r) * a.rows_stride;
                for (int c = (int)threadIdx.x * V; c < cols; c += kThreads * V) zero.store(to + c, cols - c);
            }
        }
        return;
    }
    const uint32_t lane = threadIdx.x & (lanes - 1), per_block = kThreads / lanes;
    const uint64_t step = (uint64_t)blocks * per_block;
    const uint64_t rounds = (a.positions + step - 1) / step;
    for (uint64_t i = 0; i < rounds; ++i) {  // the same for every lane: the sums need them all
        const uint64_t mine = i * step + (uint64_t)blockIdx.x * per_block + threadIdx.x / lanes;
        const bool here = mine < a.positions;
        const uint64_t t = here ? mine : 0;
        int64_t at[K];
        float w[K], dot[K];
        bool in[K];
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const uint64_t item = t * a.top_k + (j < (int)a.top_k ? j : 0);
            const uint32_t s = (uint32_t)a.slot[item];
            in[j] = here && j < (int)a.top_k && s < a.n_rows;
            w[j] = a.gate ? a.gate[item] : 1.0f;
            at[j] = in[j] ? s : 0;
            dot[j] = 0.0f;
        }
        const T* x = static_cast<const T*>(a.x) + (int64_t)t * a.x_stride;
        const T* from = static_cast<const T*>(a.from);
        for (int c0 = (int)lane * V; c0 < cols; c0 += (int)lanes * V * U) {
            Piece<T> p[U], q[DOT ? K : 1][U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u * (int)lanes * V;
                read<T, FEW>(p[u], x, c, cols);
                if constexpr (DOT) {
#pragma unroll
                    for (int j = 0; j < K; ++j) read<T, FEW>(q[j][u], from + at[j] * a.from_stride, c, cols);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u * (int)lanes * V;
                fix<T, FEW>(p[u], c, cols);
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    if constexpr (DOT) {
                        fix<T, FEW>(q[j][u], c, cols);
#pragma unroll
                        for (int e = 0; e < V; ++e) dot[j] = fmaf((float)p[u].v[e], (float)q[j][u].v[e], dot[j]);
                    }
                    if (!in[j]) continue;
                    Piece<T> out = p[u];
                    if (a.gate) {
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            float v = w[j] * (float)p[u].v[e];
                            // f16: kept from becoming one instruction that rounds once where others
                            // round twice, so that drows is the same with and without dgate
                            asm("" : "+v"(v));
                            out.v[e] = (T)v;
                        }
                    }
                    out.store(rows + at[j] * a.rows_stride + c, cols - c);
                }
            }
        }
        if constexpr (DOT) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const float s = lanes_sum(dot[j], lanes);
                if (here && lane == 0 && j < (int)a.top_k) a.dgate[t * a.top_k + j] = in[j] ? s : 0.0f;
            }
        }
    }
}

// Calls f with K.
template <typename F>
void with_top(uint32_t top_k, F&& f) {
    using std::integral_constant;
    if (top_k == 1)
        f(integral_constant<int, 1>{});
    else if (top_k == 2)
        f(integral_constant<int, 2>{});
    else if (top_k <= 4)
        f(integral_constant<int, 4>{});
    else
        f(integral_constant<int, 16>{});
}

// Lanes that hold a row, a power of two up to a wave.
uint32_t row_lanes(uint32_t cols, int v) {
    uint32_t lanes = 1;
    while (lanes < kWave && lanes * v < cols) lanes *= 2;
    return lanes;
}

uint32_t position_blocks(uint64_t positions, uint32_t lanes) {
    const uint64_t per_block = kThreads / lanes;
    return (uint32_t)std::min<uint64_t>((positions + per_block - 1) / per_block, kMaxGrid);
}

}  // namespace

int32_t launch_rows_back(const RowsBack& a, int32_t dtype, hipStream_t stream) {
    if (a.positions == 0) return kOk;
    TATARA_FOR_DTYPE(dtype, {
        constexpr int V = Piece<T>::V;
        const uint32_t lanes = row_lanes(a.cols, V), blocks = position_blocks(a.positions, lanes);
        with_top(a.top_k, [&](auto k) {
            constexpr int K = decltype(k)::value, U = K == 1 ? 4 : K == 2 ? 2 : 1;
            if (a.cols < (uint32_t)V)
                rows_back_kernel<T, K, 1, true><<<blocks, kThreads, 0, stream>>>(a, lanes);
            else
                rows_back_kernel<T, K, U, false><<<blocks, kThreads, 0, stream>>>(a, lanes);
        });
    });
    TATARA_LAUNCHED("rows_back");
    return kOk;
}

int32_t launch_rows_out(const RowsOut& a, int32_t dtype, hipStream_t stream) {
    if (a.positions == 0 && a.n_rows == 0) return kOk;
    TATARA_FOR_DTYPE(dtype, {
        constexpr int V = Piece<T>::V;
        const uint32_t lanes = row_lanes(a.cols, V), blocks = position_blocks(a.positions, lanes);
        const uint32_t clear = (uint32_t)std::min<uint64_t>((a.n_rows + kThreads - 1) / kThreads, kMaxGrid);
        with_top(a.top_k, [&](auto k) {
            constexpr int K = decltype(k)::value, U = K == 1 ? 4 : K == 2 ? 2 : 1;
            auto launch = [&](auto few, auto dot) {
                constexpr bool FEW = decltype(few)::value, DOT = decltype(dot)::value;
                rows_out_kernel<T, K, FEW ? 1 : DOT ? U : 4, FEW, DOT>
                    <<<blocks + clear, kThreads, 0, stream>>>(a, lanes, blocks);
            };
            auto with_dot = [&](auto few) { a.dgate ? launch(few, std::true_type{}) : launch(few, std::false_type{}); };
            a.cols < (uint32_t)V ? with_dot(std::true_type{}) : with_dot(std::false_type{});
        });
    });
    TATARA_LAUNCHED("rows_out");
    return kOk;
}

}  // namespace tatara
