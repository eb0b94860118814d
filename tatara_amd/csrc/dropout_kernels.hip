// Dropout from a counter-based generator, whose mask is never stored.
//
//   u_rc = word c % 4 of Philox4x32-10 (Salmon et al., Parallel random numbers: as
//          easy as 1, 2, 3, SC 2011) at counter (c / 4, row, step's low and high
//          half) with the seed as the key,
//   y_rc = u_rc >= round(p 2^32) ? x_rc / (1 - p) : 0, plus the residual
//
// The gradient is the same call on dy without a residual.  A value's number depends on
// its row, column, step and seed alone, so neither strides nor the launch's shape nor
// how a batch is cut (first_row) change the mask.
//
// Bound by memory, with the generator's products (twenty of 32 x 32 bits for four values, a
// quarter of the usual rate) behind the loads: 65536 x 1536 bf16 with a residual 109 us
// (604 MB, 5.5 TB/s), of which instructions take about 75.  A lane has four pieces of 16
// bytes in hand (16384 x 1536 bf16 22.9 us in a graph, with one 24.8), in a small call too, which
// is bound by them: 1021 x 130 f32 are 33 workgroups on 256 CUs, 4.0 us, with one piece a lane 2.7.
#include "elem.hpp"

namespace tatara {
namespace {

constexpr int kThreads = 256;
constexpr int kPieces = 4;  // 16-byte pieces a lane has in hand
constexpr uint32_t kMaxGrid = 1u << 20;
constexpr uint32_t kMaxCols = 1u << 24;

struct Words {
    uint32_t v[4];
};

// a * b in 64 bits is one instruction; the keys are the same in all lanes.
__device__ __forceinline__ Words philox(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p = (uint64_t)a * 0xD2511F53u, q = (uint64_t)c * 0xCD9E8D57u;
        a = (uint32_t)(q >> 32) ^ b ^ k0;
        b = (uint32_t)q;
        c = (uint32_t)(p >> 32) ^ d ^ k1;
        d = (uint32_t)p;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{a, b, c, d}};
}

// A workgroup takes kThreads * kPieces consecutive pieces of the rows, `per_row` of
// them a row.  FEW: rows of fewer elements than a piece has.  In place, a row's last piece
// is read again by elements where it is not a whole one: what stands for it otherwise, the
// row's last 16 bytes, another wave may have written by then.
template <typename T, bool FEW, bool ADD, bool IN_PLACE>
__global__ __launch_bounds__(kThreads) void dropout_kernel(
    const T* x, int64_t x_stride, const T* residual, int64_t residual_stride, T* y, int64_t y_stride, uint64_t pieces,
    uint32_t per_row, uint32_t cols, uint32_t first_row, uint32_t threshold, float scale, uint32_t key0, uint32_t key1,
    uint64_t step, const uint64_t* __restrict__ more_steps) {
    constexpr int V = Piece<T>::V;
    if (more_steps) step += *more_steps;
    constexpr uint32_t kAtOnce = kThreads * kPieces;
    for (uint64_t first = (uint64_t)blockIdx.x * kAtOnce; first < pieces; first += (uint64_t)gridDim.x * kAtOnce) {
        const uint32_t first_in = (uint32_t)(first % per_row);
        const uint64_t row0 = first / per_row;
        Piece<T> in[kPieces], add[ADD ? kPieces : 1];
        uint64_t row[kPieces];
        int col[kPieces];
        bool here[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            uint32_t at = i * kThreads + threadIdx.x;
            here[i] = first + at < pieces;
            at = here[i] ? at : 0;
            const uint32_t down = (first_in + at) / per_row;
            row[i] = row0 + down;
            col[i] = (int)(first_in + at - down * per_row) * V;
            const T* xr = x + (int64_t)row[i] * x_stride;
            const T* rr = ADD ? residual + (int64_t)row[i] * residual_stride : nullptr;
            if (FEW) {
                in[i].load_few(xr, (int)cols);
                if constexpr (ADD) add[i].load_few(rr, (int)cols);
            } else {
                in[i].load(xr, col[i], (int)cols);
                if constexpr (ADD) add[i].load(rr, col[i], (int)cols);
            }
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int left = (int)cols - col[i];
            uint32_t u[V];
#pragma unroll
            for (int b = 0; b < V / 4; ++b) {
                const Words w = philox((uint32_t)col[i] / 4 + b, (uint32_t)row[i] + first_row, (uint32_t)step,
                                       (uint32_t)(step >> 32), key0, key1);
#pragma unroll
                for (int j = 0; j < 4; ++j) u[4 * b + j] = w.v[j];
            }
            if (!FEW) {
                if (IN_PLACE && left < V) {
                    in[i].load_few(x + (int64_t)row[i] * x_stride + col[i], left);
                    if constexpr (ADD) add[i].load_few(residual + (int64_t)row[i] * residual_stride + col[i], left);
                } else {
                    in[i].fix(left);
                    if constexpr (ADD) add[i].fix(left);
                }
            }
            Piece<T> out;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                // what is dropped is zero whatever it was
                float v = u[j] >= threshold ? (float)in[i].v[j] * scale : 0.0f;
                if constexpr (ADD) v += (float)add[i].v[j];
                asm("" : "+v"(v));  // f16: rounded to f32 first in every form of this kernel
                out.v[j] = (T)v;
            }
            if (here[i]) out.store(y + (int64_t)row[i] * y_stride + col[i], left);
        }
    }
}

}  // namespace
}  // namespace tatara

using namespace tatara;

extern "C" int32_t tatara_op_dropout(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                                     void* y, int64_t y_stride, uint64_t rows, uint32_t cols, double p, uint64_t seed,
                                     uint64_t step, const uint64_t* more_steps, uint32_t first_row, int32_t dtype,
                                     TataraStream* stream) {
    TATARA_REQUIRE_DTYPE(dtype);
    TATARA_REQUIRE(cols >= 1 && cols <= kMaxCols, "dropout takes 1 to 2^24 columns");
    TATARA_REQUIRE(rows < (1ull << 31) && rows + first_row <= (1ull << 32), "too many rows");
    TATARA_REQUIRE(p >= 0.0 && p < 1.0, "p must be in [0, 1)");
    if (rows == 0) return kOk;
    TATARA_REQUIRE(x && y, "null tensor");
    TATARA_REQUIRE(x_stride >= (int64_t)cols && y_stride >= (int64_t)cols &&
                       (!residual || residual_stride >= (int64_t)cols),
                   "a row stride is smaller than the row");
    TATARA_REQUIRE_ALIGNED(x, elem_bytes(dtype));
    TATARA_REQUIRE_ALIGNED(residual, elem_bytes(dtype));
    TATARA_REQUIRE_ALIGNED(y, elem_bytes(dtype));
    TATARA_REQUIRE_ALIGNED(more_steps, 8);
    TATARA_REQUIRE((y != x || y_stride == x_stride) && (y != residual || y_stride == residual_stride),
                   "in place the strides are the same");
    if (int32_t st = check_stream(stream)) return st;
    // p next to 1 rounds to 2^32, which no number reaches
    const uint32_t threshold = (uint32_t)std::min(nearbyint(p * 0x1p32), 0x1p32 - 1.0);
    const float scale = (float)(1.0 / (1.0 - p));
    TATARA_FOR_DTYPE(dtype, {
        constexpr int V = Piece<T>::V;
        const uint32_t per_row = ceil_div(cols, V);
        const uint64_t pieces = rows * per_row;
        constexpr uint64_t AT_ONCE = kThreads * kPieces;
        const uint32_t blocks = (uint32_t)std::min<uint64_t>((pieces + AT_ONCE - 1) / AT_ONCE, kMaxGrid);
        auto launch = [&](auto few, auto add, auto in_place) {
            dropout_kernel<T, decltype(few)::value, decltype(add)::value, decltype(in_place)::value>
                <<<blocks, kThreads, 0, raw(stream)>>>(
                    static_cast<const T*>(x), x_stride, static_cast<const T*>(residual), residual_stride,
                    static_cast<T*>(y), y_stride, pieces, per_row, cols, first_row, threshold, scale, (uint32_t)seed,
                    (uint32_t)(seed >> 32), step, more_steps);
        };
        auto with_place = [&](auto few, auto add) {
            (y == x || y == residual) && cols % V ? launch(few, add, std::true_type{})
                                                  : launch(few, add, std::false_type{});
        };
        auto with_add = [&](auto few) {
            residual ? with_place(few, std::true_type{}) : with_place(few, std::false_type{});
        };
        cols < (uint32_t)V ? with_add(std::true_type{}) : with_add(std::false_type{});
    });
    TATARA_LAUNCHED("dropout");
    return kOk;
}
