// Root-mean-square norm of rows with the residual's addition, with an output in 8
// bits, and its gradient.
//
//   s = x + residual, rounded to the element type (as it is stored),
//   rstd_r = 1 / sqrt(sum_c s^2 / C + eps),  y = s rstd w
//   8 bits: of each group of a row's columns, scale = max(max |y|, 2^-100) / M and
//           q = round(y / scale), M = 448 (e4m3) or 127 (whole numbers)
//   backward: h = s rstd,  g = dy w,
//             ds = rstd (g - h sum_c (g h) / C) + dtotal,  dw = sum_r dy h
//
// Every sum is f32 and in a fixed order (no atomics).
//
// A row stays in registers between its sum and its use, so each value is read and
// written once: bound by memory, 65536 x 1536 bf16 with a residual and its sum 144 us
// (5.6 TB/s; a copy of 400 MB runs at 5.4).  In 8 bits also by instructions, 140 a lane of
// eight values: 16381 x 2048 f16 with scales of 128 columns 21 to 23 us (100 MB; a plain cast
// 21.8).  A row alone takes 3 us, the backward pass of 1009 x 769 f32 7.8 (2049 x 769
// in two launches 8.6).
#include "norm_rows.hpp"

namespace tatara {
namespace {

// Workgroups of an output in 8 bits at most: four rows each of 16384, so that the weight is
// loaded once for them (16381 x 2048 f16: 23.0 us, with one row each 25.0, with 2048 23.4).
constexpr uint32_t kBits8Blocks = 4096;

// Whether the weight's gradient is made beside dx by workgroups of its own, which read dy and
// the sum again, instead of from the others' partial sums by a second launch: up to 1024 rows
// of 4 MB, an XCD's L2.  In a graph, with dtotal, f32 100 x 769 3.0 us and by two launches 6.5,
// 1000 x 32 4.0 and 4.8, 1024 x 1024 6.6 and 7.8, bf16 512 x 4096 5.5 and 11.2, 1024 x 2048 7.8 and
// 9.6; slower only in rows that start inside a line, f32 1009 x 769 8.3 and 7.6, where calls from
// the host take 8.2 and 11.0.  Of more rows f32 1500 x 256 5.5 and 6.1, but 2048 x 32 5.8 and 5.4,
// 2048 x 128 6.2 and 5.4, bf16 2048 x 256 7.7 and 5.8; of more bytes f32 1024 x 1536 11.4 and 9.5,
// 512 x 4096 12.8 and 11.1.
bool weight_beside(uint64_t rows, uint64_t row_bytes) { return rows <= 1024 && rows * row_bytes <= 4u << 20; }

// Lanes on a row for it.
constexpr uint32_t kWeightLanes = 4;

// The larger; NaN if either is.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Sum over the L lanes of a row, or its W waves.
template <int W, int L>
__device__ __forceinline__ float lanes_sum(float x, float (*part)[W], int slot) {
    if constexpr (L < (int)kWave)
        return group_sum<L>(x);
    else
        return row_sum<W>(x, part, slot);
}

// The largest of what they hold.
template <int W, int L>
__device__ __forceinline__ float lanes_max(float x, float (*part)[W], int slot) {
    x = group_join<L>(x, larger);
    if constexpr (W > 1) {
        if (threadIdx.x % kWave == 0) part[slot][threadIdx.x / kWave] = x;
        __syncthreads();
        x = part[slot][0];
#pragma unroll
        for (int i = 1; i < W; ++i) x = larger(x, part[slot][i]);
    }
    return x;
}

// V values as 8-bit ones, of which the first `left` are stored.
template <int V>
__device__ __forceinline__ void store_8bit(uint8_t* to, const float* v, bool e4m3, int left) {
    uint32_t word[V / 4];
    if (e4m3) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const int low = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
            word[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], low, true);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            word[i] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) word[i] |= ((uint32_t)(int32_t)rintf(v[4 * i + j]) & 0xffu) << (8 * j);
        }
    }
    if (left >= V) {
        __builtin_memcpy(to, word, V);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < left) to[j] = (uint8_t)(word[j / 4] >> (8 * (j % 4)));
    }
}

// Where y goes.
struct RmsOut {
    void* y;  // of the element type, or of 8 bits
    int64_t stride;
    float* scale;     // 8 bits: [rows][groups]
    uint32_t groups;  // of a row
    uint32_t lanes;   // that a group lies in; 0: the whole row
    bool e4m3;
};

// W waves on a row, or L lanes of one with one piece each; N pieces a lane.  FEW: rows of
// fewer elements than a piece has.  BITS8: an output in 8 bits.  total may be
// x or residual: a row's loads stand ahead of its sum, and its stores behind.
template <typename T, int W, int L, int N, bool FEW, bool ADD, bool BITS8>
__global__ __launch_bounds__(W == 16 ? 1024 : 256) void rms_forward_kernel(
    const T* x, int64_t x_stride, const T* residual, int64_t residual_stride, const float* __restrict__ weight,
    T* total, int64_t total_stride, RmsOut out, float* __restrict__ rstd, uint64_t rows, uint32_t cols, float eps) {
    constexpr int V = Piece<T>::V;
    __shared__ float part[2][W];
    __shared__ float part_max[2][W];
    const uint32_t lane = threadIdx.x % (L * W);
    uint32_t group = threadIdx.x / (L * W);
    if constexpr (L == kWave) group = __builtin_amdgcn_readfirstlane(group);
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
    constexpr int G = W == 1 ? 256 / L : 1;  // rows that the workgroup has in hand
    // the weight stays in registers over the workgroup's rows: as f32 it has up to twice
    // the bytes of a row
    constexpr bool KEEP = BITS8 && W < 16 && (N * V <= 24 || sizeof(T) == 2);
    Floats<V> kept[KEEP ? N : 1];
    auto weights = [&](int i) {
        const float* from = weight;
        if constexpr (W == 16) asm volatile("" : "+s"(from));  // else they are all kept
        Floats<V> w;
        if (from) {
            read(w, from, i);
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
    // An output in 8 bits has few workgroups, and reads a row while it works on the last.
    constexpr bool AHEAD = BITS8 && W < 16;
    Piece<T> px[N], pr[ADD ? N : 1];
    auto read_row = [&](uint64_t row) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            read(px[i], x + (int64_t)row * x_stride, i);
            if constexpr (ADD) read(pr[i], residual + (int64_t)row * residual_stride, i);
        }
    };
    const uint64_t step = (uint64_t)gridDim.x * G;
    uint64_t row = (uint64_t)blockIdx.x * G + group;
    if (AHEAD && row < rows) read_row(row);
    int slot = 0;
    for (; row < rows; row += step, slot ^= 1) {
        if (!AHEAD) read_row(row);
        Piece<T> in[N], more[ADD ? N : 1];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            in[i] = px[i];
            if constexpr (ADD) more[i] = pr[i];
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            fix(in[i], i);
            if constexpr (ADD) fix(more[i], i);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if constexpr (ADD) in[i].v[j] = (T)((float)in[i].v[j] + (float)more[i].v[j]);
                const float v = (float)in[i].v[j];
                s = fmaf(v, v, s);
            }
        }
        if constexpr (AHEAD) {  // behind the last row nothing uses what is read
            const uint64_t next = row + step;
            read_row(next < rows ? next : row);
        }
        const float r = rsqrtf(lanes_sum<W, L>(s, part, slot) / (float)cols + eps);
        if (lane == 0 && rstd) rstd[row] = r;
        if constexpr (ADD) {
            if (total) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    in[i].store(total + (int64_t)row * total_stride + column(i), (int)cols - column(i));
            }
        }
        auto normed = [&](int i, float* y) {
            const Floats<V> w = KEEP ? kept[KEEP ? i : 0] : weights(i);
#pragma unroll
            for (int j = 0; j < V; ++j) y[j] = (float)in[i].v[j] * r * w[j];
        };
        if constexpr (!BITS8) {
            T* to = static_cast<T*>(out.y) + (int64_t)row * out.stride;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int left = (int)cols - column(i);
                if (left <= 0) break;
                float y[V];
                normed(i, y);
                Piece<T> piece;
#pragma unroll
                for (int j = 0; j < V; ++j) piece.v[j] = (T)y[j];
                piece.store(to + column(i), left);
            }
        } else {
            // NaN and infinity reach the largest: past the row's end a value is NaN only if
            // rstd is not finite, and then so is none of the row
            constexpr bool TWICE = W == 16;  // y is made again for its second use
            float y[TWICE ? 1 : N][V], top[N], all = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float* yi = y[TWICE ? 0 : i];
                normed(i, yi);
                top[i] = 0.0f;
#pragma unroll
                for (int j = 0; j < V; ++j) top[i] = larger(top[i], fabsf(yi[j]));
                all = larger(all, top[i]);
            }
            if (out.lanes == 0) {
                all = lanes_max<W, L>(all, part_max, slot);
#pragma unroll
                for (int i = 0; i < N; ++i) top[i] = all;
            } else {
                auto join = [&](auto s) {
                    constexpr int S = decltype(s)::value;
                    if (L >> S > 1 && out.lanes >> S > 1) {
#pragma unroll
                        for (int i = 0; i < N; ++i)
                            top[i] = larger(top[i], __uint_as_float(partner<S>(__float_as_uint(top[i]))));
                    }
                };
                join(std::integral_constant<int, 0>{});
                join(std::integral_constant<int, 1>{});
                join(std::integral_constant<int, 2>{});
                join(std::integral_constant<int, 3>{});
                join(std::integral_constant<int, 4>{});
            }
            uint8_t* to = static_cast<uint8_t*>(out.y) + (int64_t)row * out.stride;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int left = (int)cols - column(i);
                if (left <= 0) break;
                // Products with reciprocals: three roundings of f32 and one unit of the
                // reciprocal off y / scale, which shows where that lies on the border of two
                // results; the largest, off M by as much, rounds to M.
                const bool finite = top[i] < INFINITY;
                float scale = fmaxf(top[i], 0x1p-100f) * (out.e4m3 ? 1.0f / 448.0f : 1.0f / 127.0f);
                const float inv = __builtin_amdgcn_rcpf(scale);
                if constexpr (TWICE) {
                    in[i].forget();
                    normed(i, y[0]);
                }
                float v[V];
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = y[TWICE ? 0 : i][j] * inv;
                if (__ballot(!finite)) {
                    // a group with a value that is not finite has the scale NaN, and zeros
                    scale = finite ? scale : __uint_as_float(0x7fc00000u);
#pragma unroll
                    for (int j = 0; j < V; ++j) v[j] = finite ? v[j] : 0.0f;
                }
                store_8bit<V>(to + column(i), v, out.e4m3, left);
                const uint32_t in_group = out.lanes ? lane % out.lanes : lane + i;
                if (in_group == 0)
                    out.scale[row * out.groups + (out.lanes ? (uint32_t)column(i) / (out.lanes * V) : 0)] = scale;
            }
        }
    }
}

// dw of a few columns over all rows, by a workgroup: four lanes with a piece each and a
// group of rows for each four of them, joined in order.  Of few rows this needs no second
// launch, since rstd is known.
template <typename T, int THREADS, bool FEW>
__device__ __forceinline__ void weight_columns(const T* __restrict__ dy, int64_t dy_stride,
                                               const T* __restrict__ total, int64_t total_stride,
                                               const float* __restrict__ rstd, float* __restrict__ dweight,
                                               uint32_t rows, uint32_t cols, uint32_t block) {
    constexpr int V = Piece<T>::V, WAVES = THREADS / kWave;
    __shared__ float join[WAVES][kWeightLanes * V];
    const uint32_t lane = threadIdx.x % kWeightLanes;
    const int c = (int)((block * kWeightLanes + lane) * V), left = (int)cols - c;
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.0f;
    constexpr uint32_t GROUPS = THREADS / kWeightLanes;
    constexpr int HAND = 8;  // rows that a lane reads at once
    for (uint32_t row0 = threadIdx.x / kWeightLanes; row0 < rows; row0 += GROUPS * HAND) {
        Piece<T> s[HAND], d[HAND];
        float r[HAND];
#pragma unroll
        for (int k = 0; k < HAND; ++k) {
            const uint32_t row = row0 + k * GROUPS < rows ? row0 + k * GROUPS : row0;
            const T *sr = total + (int64_t)row * total_stride, *dr = dy + (int64_t)row * dy_stride;
            if (FEW) {
                s[k].load_few(sr, left);
                d[k].load_few(dr, left);
            } else {
                s[k].load(sr, min(c, (int)cols), (int)cols);
                d[k].load(dr, min(c, (int)cols), (int)cols);
            }
            r[k] = rstd[row];
        }
#pragma unroll
        for (int k = 0; k < HAND; ++k) {
            if (row0 + k * GROUPS >= rows) break;
            if (!FEW) {
                s[k].fix(left);
                d[k].fix(left);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] = fmaf((float)d[k].v[j], (float)s[k].v[j] * r[k], acc[j]);
        }
    }
    const uint32_t wave = threadIdx.x / kWave;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float sum = column_join<(int)kWeightLanes>(acc[j], [](float x, float y) { return x + y; });
        if (threadIdx.x % kWave < kWeightLanes) join[wave][lane * V + j] = sum;
    }
    __syncthreads();
    const uint32_t mine = threadIdx.x, at = block * kWeightLanes * V + mine;
    if (mine >= kWeightLanes * V || at >= cols) return;
    float sum = join[0][mine];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += join[w][mine];
    dweight[at] = sum;
}

// dx may be dtotal, as total above.  With a partial, every workgroup leaves its sums of dw
// there; with a dweight, the workgroups from `dx_blocks` on make it.
template <typename T, int W, int L, int N, bool FEW, bool ADD>
__global__ __launch_bounds__(W == 16 ? 1024 : 256) void rms_backward_kernel(
    const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ total, int64_t total_stride,
    const float* __restrict__ weight, const float* __restrict__ rstd, const T* dtotal, int64_t dtotal_stride, T* dx,
    int64_t dx_stride, float* __restrict__ partial, float* __restrict__ dweight, uint32_t dx_blocks, uint64_t rows,
    uint32_t cols) {
    constexpr int V = Piece<T>::V;
    constexpr int G = W == 1 ? 256 / L : 1;  // rows that the workgroup has in hand
    if (blockIdx.x >= dx_blocks) {
        weight_columns<T, W == 16 ? 1024 : 256, FEW>(dy, dy_stride, total, total_stride, rstd, dweight, (uint32_t)rows,
                                                     cols, blockIdx.x - dx_blocks);
        return;
    }
    __shared__ float part[2][W];
    __shared__ float join[W > 1 ? 1 : 3 * kWave * N * V];
    const uint32_t lane = threadIdx.x % (L * W);
    uint32_t group = threadIdx.x / (L * W);
    if constexpr (L == kWave) group = __builtin_amdgcn_readfirstlane(group);
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
    // The weight stays in registers where they last.  Of the widest rows, values are made
    // again for their second use and none is read ahead (f32 4096 x 32768 1037 us, so 707, with
    // dtotal 8192 x 16384 724 and 402; but bf16 16384 x 8192 158 and 189).
    constexpr bool LEAN = W == 16 && (N * V > 16 || (N * V > 8 && (ADD || sizeof(T) == 4)));
    constexpr bool KEEP = !LEAN && N * V <= 24;
    float dw[N * V];
    Floats<V> kept[KEEP ? N : 1];
#pragma unroll
    for (int i = 0; i < N * V; ++i) dw[i] = 0.0f;
    auto weights = [&](int i) {
        const float* from = weight;
        if constexpr (LEAN) asm volatile("" : "+s"(from));  // else they are all kept
        Floats<V> w;
        if (from) {
            read(w, from, i);
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
    Piece<T> ps[N], pd[N], pt[ADD ? N : 1];
    float r = 0.0f;
    auto read_row = [&](uint64_t row) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            read(ps[i], total + (int64_t)row * total_stride, i);
            read(pd[i], dy + (int64_t)row * dy_stride, i);
            if constexpr (ADD) read(pt[i], dtotal + (int64_t)row * dtotal_stride, i);
        }
        r = rstd[row];
    };
    int slot = 0;
    const uint64_t step = (uint64_t)dx_blocks * G;
    uint64_t row = (uint64_t)blockIdx.x * G + group;
    if (!LEAN && row < rows) read_row(row);
    for (; row < rows; row += step, slot ^= 1) {
        if (LEAN) read_row(row);
        float h[LEAN ? V : N * V], g[LEAN ? V : N * V];
        Piece<T> add[ADD ? N : 1];
        float sgh = 0.0f;
        auto terms = [&](int i, float* hi, float* gi) {
            const Floats<V> w = KEEP ? kept[KEEP ? i : 0] : weights(i);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                // past the row's end both are zero (NaN if rstd is not finite, and then so is
                // what is in the row)
                hi[j] = (float)ps[i].v[j] * r;
                gi[j] = (float)pd[i].v[j] * w[j];
            }
        };
#pragma unroll
        for (int i = 0; i < N; ++i) {
            fix(ps[i], i);
            fix(pd[i], i);
            if constexpr (ADD) {
                fix(pt[i], i);
                add[i] = pt[i];
            }
            float *hi = h + (LEAN ? 0 : i * V), *gi = g + (LEAN ? 0 : i * V);
            terms(i, hi, gi);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                sgh = fmaf(gi[j], hi[j], sgh);
                dw[i * V + j] = fmaf((float)pd[i].v[j], hi[j], dw[i * V + j]);
            }
        }
        const float scale = r;
        // the next row's values are on their way while this one's sum is joined (behind the
        // last row nothing uses what is read)
        const uint64_t next = row + step;
        if (!LEAN) read_row(next < rows ? next : row);
        const float b = lanes_sum<W, L>(sgh, part, slot) / (float)cols;
        T* to = dx + (int64_t)row * dx_stride;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float *hi = h + (LEAN ? 0 : i * V), *gi = g + (LEAN ? 0 : i * V);
            if constexpr (LEAN) {
                ps[i].forget();
                pd[i].forget();
                terms(i, hi, gi);
            }
            Piece<T> out;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = (gi[j] - hi[j] * b) * scale;
                if constexpr (ADD)
                    out.v[j] = (T)(d + (float)add[i].v[j]);
                else
                    out.v[j] = (T)d;
            }
            out.store(to + column(i), (int)cols - column(i));
        }
    }
    if (!partial) return;
    float* to = partial + (uint64_t)blockIdx.x * cols;
    if constexpr (L < (int)kWave) {  // over the wave's rows; the first L lanes have the sums
#pragma unroll
        for (int i = 0; i < N * V; ++i) dw[i] = column_join<L>(dw[i], [](float x, float y) { return x + y; });
    }
    const uint32_t wave = W == 1 ? threadIdx.x / kWave : 0, place = W == 1 ? threadIdx.x % kWave : lane;
    if constexpr (W == 1) {
        if (wave > 0) {
#pragma unroll
            for (int i = 0; i < N * V; ++i) join[((wave - 1) * N * V + i) * kWave + place] = dw[i];
        }
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int i = 0; i < N * V; ++i)
#pragma unroll
                for (int o = 0; o < 3; ++o) dw[i] += join[(o * N * V + i) * kWave + place];
        }
    }
    if (wave == 0 && (L == (int)kWave || place < L)) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = column(i);
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c + j < (int)cols) to[c + j] = dw[i * V + j];
        }
    }
}

// Calls f with the waves, lanes and pieces of a row.  Rows that half a wave holds share a
// wave (65536 x 32 f32: forward 13.3 us, backward 22.8 with a wave each).
template <typename T, bool BACKWARD, typename F>
void with_rms_form(uint64_t rows, uint32_t cols, F&& f) {
    using std::integral_constant;
    constexpr int V = Piece<T>::V;
    const integral_constant<int, 1> one;
    auto lanes = [&](auto l) { f(one, l, one, std::false_type{}); };
    if (cols < (uint32_t)V)
        f(one, one, one, std::true_type{});
    else if (cols <= 2 * V)
        lanes(integral_constant<int, 2>{});
    else if (cols <= 4 * V)
        lanes(integral_constant<int, 4>{});
    else if (cols <= 8 * V)
        lanes(integral_constant<int, 8>{});
    else if (cols <= 16 * V)
        lanes(integral_constant<int, 16>{});
    else if (cols <= 32 * V)
        lanes(integral_constant<int, 32>{});
    else
        with_form<T, BACKWARD>(norm_form(BACKWARD, rows, cols, V), [&](auto w, auto n, auto few) {
            f(w, integral_constant<int, (int)kWave>{}, n, few);
        });
}

uint64_t partial_bytes(uint32_t cols) { return 4ull * kGradBlocks * cols; }

int32_t check_forward(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                      const void* total, int64_t total_stride, const void* y, int64_t y_stride, uint64_t rows,
                      uint32_t cols, float eps, int32_t dtype) {
    TATARA_REQUIRE_DTYPE(dtype);
    TATARA_REQUIRE(cols >= 1 && cols <= kMaxCols, "RMS norm takes 1 to 32768 columns");
    TATARA_REQUIRE(rows < (1ull << 31), "too many rows");
    TATARA_REQUIRE(eps >= 0.0f, "eps must not be negative");
    TATARA_REQUIRE(residual || !total, "a sum is asked for, and no residual given");
    if (rows == 0) return kOk;
    TATARA_REQUIRE(x && y, "null tensor");
    TATARA_REQUIRE(x_stride >= (int64_t)cols && y_stride >= (int64_t)cols &&
                       (!residual || residual_stride >= (int64_t)cols) && (!total || total_stride >= (int64_t)cols),
                   "a row stride is smaller than the row");
    TATARA_REQUIRE(!total || ((total != x || total_stride == x_stride) &&
                              (total != residual || total_stride == residual_stride)),
                   "in place the strides are the same");
    TATARA_REQUIRE_ALIGNED(x, elem_bytes(dtype));
    TATARA_REQUIRE_ALIGNED(residual, elem_bytes(dtype));
    TATARA_REQUIRE_ALIGNED(total, elem_bytes(dtype));
    return kOk;
}

template <bool BITS8>
void launch_forward(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                    const float* weight, void* total, int64_t total_stride, const RmsOut& out, float* rstd,
                    uint64_t rows, uint32_t cols, float eps, int32_t dtype, hipStream_t stream) {
    TATARA_FOR_DTYPE(dtype, {
        with_rms_form<T, false>(rows, cols, [&](auto w, auto l, auto n, auto few) {
            constexpr int W = decltype(w)::value, L = decltype(l)::value, G = W == 1 ? 256 / L : 1;
            constexpr int N = decltype(n)::value;
            constexpr bool FEW = decltype(few)::value;
            const uint32_t blocks =
                (uint32_t)std::min<uint64_t>((rows + G - 1) / G, BITS8 ? kBits8Blocks : kMaxGrid);
            const uint32_t threads = W == 16 ? 1024 : 256;
            if (residual)
                rms_forward_kernel<T, W, L, N, FEW, true, BITS8><<<blocks, threads, 0, stream>>>(
                    static_cast<const T*>(x), x_stride, static_cast<const T*>(residual), residual_stride, weight,
                    static_cast<T*>(total), total_stride, out, rstd, rows, cols, eps);
            else
                rms_forward_kernel<T, W, L, N, FEW, false, BITS8><<<blocks, threads, 0, stream>>>(
                    static_cast<const T*>(x), x_stride, nullptr, 0, weight, nullptr, 0, out, rstd, rows, cols, eps);
        });
    });
}

}  // namespace
}  // namespace tatara

using namespace tatara;

extern "C" {

int32_t tatara_op_rms_norm_forward(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                                   const float* weight, void* total, int64_t total_stride, void* y, int64_t y_stride,
                                   float* rstd, uint64_t rows, uint32_t cols, float eps, int32_t dtype,
                                   TataraStream* stream) {
    if (int32_t st = check_forward(x, x_stride, residual, residual_stride, total, total_stride, y, y_stride, rows,
                                   cols, eps, dtype))
        return st;
    TATARA_REQUIRE_ALIGNED(y, elem_bytes(dtype));
    if (rows == 0) return kOk;
    if (int32_t st = check_stream(stream)) return st;
    launch_forward<false>(x, x_stride, residual, residual_stride, weight, total, total_stride,
                          RmsOut{y, y_stride, nullptr, 0, 0, false}, rstd, rows, cols, eps, dtype, raw(stream));
    TATARA_LAUNCHED("rms_forward");
    return kOk;
}

int32_t tatara_op_rms_norm_forward_8bit(const void* x, int64_t x_stride, const void* residual,
                                        int64_t residual_stride, const float* weight, void* total,
                                        int64_t total_stride, void* q, int64_t q_stride, float* scale, float* rstd,
                                        uint64_t rows, uint32_t cols, uint32_t group, float eps, int32_t dtype,
                                        int32_t format, TataraStream* stream) {
    TATARA_REQUIRE(format == TATARA_E4M3 || format == TATARA_I8, "unknown 8-bit format");
    TATARA_REQUIRE(group == 0 || group == 32 || group == 64 || group == 128,
                   "a scale stands for 32, 64 or 128 columns, or for a row (0)");
    if (int32_t st = check_forward(x, x_stride, residual, residual_stride, total, total_stride, q, q_stride, rows,
                                   cols, eps, dtype))
        return st;
    if (rows == 0) return kOk;
    TATARA_REQUIRE(scale, "null tensor");
    if (int32_t st = check_stream(stream)) return st;
    const uint32_t v = 16 / elem_bytes(dtype);
    launch_forward<true>(x, x_stride, residual, residual_stride, weight, total, total_stride,
                         RmsOut{q, q_stride, scale, group ? ceil_div(cols, group) : 1, group / v,
                                format == TATARA_E4M3},
                         rstd, rows, cols, eps, dtype, raw(stream));
    TATARA_LAUNCHED("rms_forward_8bit");
    return kOk;
}

int32_t tatara_op_rms_norm_backward_workspace(uint32_t cols, uint64_t* bytes) {
    TATARA_REQUIRE(bytes, "null output");
    TATARA_REQUIRE(cols >= 1 && cols <= kMaxCols, "RMS norm takes 1 to 32768 columns");
    *bytes = partial_bytes(cols);
    return kOk;
}

int32_t tatara_op_rms_norm_backward(const void* dy, int64_t dy_stride, const void* total, int64_t total_stride,
                                    const float* weight, const float* rstd, const void* dtotal,
                                    int64_t dtotal_stride, void* dx, int64_t dx_stride, float* dweight, uint64_t rows,
                                    uint32_t cols, int32_t dtype, void* workspace, uint64_t workspace_bytes,
                                    TataraStream* stream) {
    TATARA_REQUIRE_DTYPE(dtype);
    TATARA_REQUIRE(cols >= 1 && cols <= kMaxCols, "RMS norm takes 1 to 32768 columns");
    TATARA_REQUIRE(rows < (1ull << 31), "too many rows");
    TATARA_REQUIRE(!dweight || (workspace && workspace_bytes >= partial_bytes(cols)), "workspace too small");
    TATARA_REQUIRE_ALIGNED(workspace, 16);
    if (rows) {
        TATARA_REQUIRE(dy && total && rstd && dx, "null tensor");
        TATARA_REQUIRE(dy_stride >= (int64_t)cols && total_stride >= (int64_t)cols && dx_stride >= (int64_t)cols &&
                           (!dtotal || dtotal_stride >= (int64_t)cols),
                       "a row stride is smaller than the row");
        TATARA_REQUIRE(dx != dtotal || dx_stride == dtotal_stride, "in place the strides are the same");
        TATARA_REQUIRE_ALIGNED(dy, elem_bytes(dtype));
        TATARA_REQUIRE_ALIGNED(total, elem_bytes(dtype));
        TATARA_REQUIRE_ALIGNED(dtotal, elem_bytes(dtype));
        TATARA_REQUIRE_ALIGNED(dx, elem_bytes(dtype));
        // the weight's workgroups may read what others have written by then
        TATARA_REQUIRE(dx != dy && dx != total, "dx must not be dy or the sum");
    }
    if (int32_t st = check_stream(stream)) return st;
    const bool beside = dweight && rows && weight_beside(rows, (uint64_t)cols * elem_bytes(dtype));
    float* partial = dweight && !beside ? static_cast<float*>(workspace) : nullptr;
    uint32_t blocks = 0;
    if (rows) {
        TATARA_FOR_DTYPE(dtype, {
            with_rms_form<T, true>(rows, cols, [&](auto w, auto l, auto n, auto few) {
                constexpr int W = decltype(w)::value, L = decltype(l)::value, G = W == 1 ? 256 / L : 1;
                constexpr int N = decltype(n)::value;
                constexpr bool FEW = decltype(few)::value;
                const uint64_t units = (rows + G - 1) / G;
                blocks = beside ? (uint32_t)units : grad_blocks(units);
                const uint32_t more = beside ? ceil_div(cols, kWeightLanes * Piece<T>::V) : 0;
                auto launch = [&](auto add) {
                    rms_backward_kernel<T, W, L, N, FEW, decltype(add)::value>
                        <<<blocks + more, W == 16 ? 1024 : 256, 0, raw(stream)>>>(
                            static_cast<const T*>(dy), dy_stride, static_cast<const T*>(total), total_stride, weight,
                            rstd, static_cast<const T*>(dtotal), dtotal_stride, static_cast<T*>(dx), dx_stride,
                            partial, dweight, blocks, rows, cols);
                };
                dtotal ? launch(std::true_type{}) : launch(std::false_type{});
            });
        });
        TATARA_LAUNCHED("rms_backward");
    }
    if (dweight && !beside) {
        norm_param_grad_kernel<<<ceil_div(cols, kWave), 1024, 0, raw(stream)>>>(partial, blocks, cols, cols, dweight,
                                                                                nullptr);
        TATARA_LAUNCHED("rms_weight_grad");
    }
    return kOk;
}

}  // extern "C"
