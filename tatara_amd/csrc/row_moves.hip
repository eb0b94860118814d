// Rows from the positions' order into another one and back: what a bucket's layers
// read and write, and what an embedding looks up.
//
// Both kernels go by positions, G lanes each (the power of two that holds a row, up to
// a wave), so that a position's own row is read or written once, however many choices it
// has, and the rows it meets elsewhere are whole ones.  A lane keeps the slots and
// weights of its position's K choices in registers.
//
// Bound by memory: 65536 x 1536 f32 gathered 146 us (805 MB, 5.5 TB/s), 32768 x 768 f16 with
// two choices back with the gates' gradient 49 (252 MB, 5.1), 65536 x 768 bf16 of a table of
// 1629 rows 22.4 (writes at 4.5; the table comes from the last-level cache as often as the
// rows written push it out of the L2).  More positions in hand a lane are no faster.  Five to
// sixteen choices share one form (16381 x 512 bf16 back: four 16.3 us, five 42.0, eight 47.0,
// sixteen 64.9, of which bytes take 17, 20, 30 and 57; 8192 x 1536 f32, eight 94 and 91).
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

// K: at least top_k; U: pieces of each row in hand.  FEW: rows of fewer elements than a
// piece has.
template <typename T, int K, int U, bool FEW>
__global__ __launch_bounds__(kThreads) void rows_back_kernel(RowsBack a, uint32_t lanes, bool past) {
    constexpr int V = Piece<T>::V;
    const uint32_t lane = threadIdx.x & (lanes - 1), groups = kThreads / lanes;
    const int cols = (int)a.cols;
    const T* rows = static_cast<const T*>(a.rows);
    const uint64_t step = (uint64_t)gridDim.x * groups;
    for (uint64_t t = (uint64_t)blockIdx.x * groups + threadIdx.x / lanes; t < a.positions; t += step) {
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
                for (int e = 0; e < V; ++e) {
                    asm("" : "+v"(y[e]));  // f16: rounded to f32 first in every form
                    out.v[e] = (T)y[e];
                }
                if (past)
                    out.store_past(to + c, cols - c);
                else
                    out.store(to + c, cols - c);
            }
        }
    }
}

// DOT: the gates' gradient too.  The first `clear` workgroups clear the rows without a
// source, of which a wave looks at `clear_rows`.
template <typename T, int K, int U, bool FEW, bool DOT>
__global__ __launch_bounds__(kThreads) void rows_out_kernel(RowsOut a, uint32_t lanes, uint32_t clear,
                                                           uint32_t clear_rows) {
    constexpr int V = Piece<T>::V;
    const int cols = (int)a.cols;
    T* rows = static_cast<T*>(a.rows);
    if (blockIdx.x < clear) {
        const uint64_t items = a.positions * a.top_k;
        const uint32_t lane = threadIdx.x % kWave;
        Piece<T> zero;
#pragma unroll
        for (int e = 0; e < V; ++e) zero.v[e] = (T)0.0f;
        constexpr uint32_t WAVES = kThreads / kWave;
        for (uint64_t first = ((uint64_t)blockIdx.x * WAVES + threadIdx.x / kWave) * clear_rows; first < a.n_rows;
             first += (uint64_t)clear * WAVES * clear_rows) {
            const uint64_t mine = first + lane;
            const bool look = lane < clear_rows && mine < a.n_rows;
            uint64_t none = __ballot(look && (uint32_t)a.source[look ? mine : first] >= items);
            for (; none; none &= none - 1) {
                T* to = rows + (int64_t)(first + __builtin_ctzll(none)) * a.rows_stride;
                for (int c = (int)lane * V; c < cols; c += kWave * V) zero.store(to + c, cols - c);
            }
        }
        return;
    }
    const uint32_t lane = threadIdx.x & (lanes - 1), groups = kThreads / lanes;
    const uint64_t step = (uint64_t)(gridDim.x - clear) * groups;
    const uint64_t rounds = (a.positions + step - 1) / step;
    for (uint64_t i = 0; i < rounds; ++i) {  // the same for every lane: the sums need them all
        const uint64_t mine = i * step + (uint64_t)(blockIdx.x - clear) * groups + threadIdx.x / lanes;
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
            Piece<T> p[U], r[DOT ? K : 1][U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u * (int)lanes * V;
                read<T, FEW>(p[u], x, c, cols);
                if constexpr (DOT) {
#pragma unroll
                    for (int j = 0; j < K; ++j) read<T, FEW>(r[j][u], from + at[j] * a.from_stride, c, cols);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u * (int)lanes * V;
                fix<T, FEW>(p[u], c, cols);
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    if constexpr (DOT) {
                        fix<T, FEW>(r[j][u], c, cols);
#pragma unroll
                        for (int e = 0; e < V; ++e) dot[j] = fmaf((float)p[u].v[e], (float)r[j][u].v[e], dot[j]);
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

// How a row of `cols` lies over lanes: a power of two of them that holds it, up to a wave,
// of which half or a quarter if that leaves fewer idle (768 columns of 16 bits: 3 pieces
// of 32 lanes, not 2 of 64 with half of one empty), and pieces a lane has in hand.
struct RowForm {
    uint32_t lanes;
    int pieces;
};
RowForm row_form(uint32_t cols, int v, int most_pieces) {
    const uint32_t n = ceil_div(cols, v);
    uint32_t lanes = 1;
    while (lanes < kWave && lanes < n) lanes *= 2;
    if (lanes == kWave) {
        uint32_t best = ceil_div(n, kWave) * kWave;
        for (uint32_t l = kWave / 2; l >= 16; l /= 2)
            if (ceil_div(n, l) * l < best && ceil_div(n, l) <= 4) lanes = l, best = ceil_div(n, l) * l;
    }
    const uint32_t rounds = ceil_div(n, lanes);
    return {lanes, (int)ceil_div(rounds, ceil_div(rounds, most_pieces))};
}

// Calls f with the pieces in hand.
template <int MOST, typename F>
void with_pieces(int pieces, F&& f) {
    auto is = [&](auto u) {
        if constexpr (decltype(u)::value <= MOST)
            if (pieces == decltype(u)::value) f(u);
    };
    is(std::integral_constant<int, 1>{});
    is(std::integral_constant<int, 2>{});
    is(std::integral_constant<int, 3>{});
    is(std::integral_constant<int, 4>{});
}

// Whether rows are written past the caches: from half the last-level cache (256 MB) on they
// would push out what a reader finds there.  Rows of a table looked up and then normalised
// (bf16): 65536 x 1536, 201 MB, 48 us and with the norm 136, past the caches 40 and 124;
// 65536 x 768 22.5 and 61.7, past them 18.6 and 68.
bool past_caches(uint64_t bytes) { return bytes >= 128ull << 20; }

uint32_t position_blocks(uint64_t positions, uint32_t lanes) {
    const uint64_t groups = kThreads / lanes;
    return (uint32_t)std::min<uint64_t>((positions + groups - 1) / groups, kMaxGrid);
}

}  // namespace

int32_t launch_rows_back(const RowsBack& a, int32_t dtype, hipStream_t stream) {
    if (a.positions == 0) return kOk;
    TATARA_FOR_DTYPE(dtype, {
        constexpr int V = Piece<T>::V;
        const bool past = past_caches(a.positions * a.cols * sizeof(T));
        with_top(a.top_k, [&](auto k) {
            constexpr int K = decltype(k)::value, MOST = K <= 4 ? 4 : 1;
            if (a.cols < (uint32_t)V) {
                rows_back_kernel<T, K, 1, true>
                    <<<position_blocks(a.positions, 1), kThreads, 0, stream>>>(a, 1, past);
                return;
            }
            const RowForm form = row_form(a.cols, V, MOST);
            with_pieces<MOST>(form.pieces, [&](auto u) {
                rows_back_kernel<T, K, decltype(u)::value, false>
                    <<<position_blocks(a.positions, form.lanes), kThreads, 0, stream>>>(a, form.lanes, past);
            });
        });
    });
    TATARA_LAUNCHED("rows_back");
    return kOk;
}

int32_t launch_rows_out(const RowsOut& a, int32_t dtype, hipStream_t stream) {
    if (a.positions == 0 && a.n_rows == 0) return kOk;
    TATARA_FOR_DTYPE(dtype, {
        constexpr int V = Piece<T>::V;
        // few rows a wave where there are few: it clears them one after the other
        uint32_t clear_rows = 1;
        while (clear_rows < kWave && a.n_rows > 4096ull * clear_rows) clear_rows *= 2;
        const uint32_t clear = (uint32_t)std::min<uint64_t>(
            (a.n_rows + kThreads / kWave * clear_rows - 1) / (kThreads / kWave * clear_rows), kMaxGrid);
        with_top(a.top_k, [&](auto k) {
            auto launch = [&](auto dot) {
                constexpr bool DOT = decltype(dot)::value;
                constexpr int K = decltype(k)::value, MOST = !DOT || K <= 4 ? 4 : 1;
                if (a.cols < (uint32_t)V) {
                    rows_out_kernel<T, K, 1, true, DOT>
                        <<<clear + position_blocks(a.positions, 1), kThreads, 0, stream>>>(a, 1, clear,
                                                                                             clear_rows);
                    return;
                }
                const RowForm form = row_form(a.cols, V, MOST);
                with_pieces<MOST>(form.pieces, [&](auto u) {
                    rows_out_kernel<T, K, decltype(u)::value, false, DOT>
                        <<<clear + position_blocks(a.positions, form.lanes), kThreads, 0, stream>>>(a, form.lanes,
                                                                                                    clear, clear_rows);
                });
            };
            a.dgate ? launch(std::true_type{}) : launch(std::false_type{});
        });
    });
    TATARA_LAUNCHED("rows_out");
    return kOk;
}

}  // namespace tatara
