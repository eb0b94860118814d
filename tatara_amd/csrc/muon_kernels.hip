// Orthogonalised updates (Muon): a batch of matrices U of one shape becomes
//
//   X_0 = U / (|U|_F + 1e-7),  A = X X^T,  B = a I + b A + c A^2,  X <- B X,
//
// X standing with its shorter side first, for a number of steps.  With (a, b,
// c) = (3.4445, -4.7750, 2.0315) every singular value of X_0 in (0, 1] is taken
// near 1 (the scalar map a s + b s^3 + c s^5 keeps [0, 1.2024] and raises small
// values by a), so X ends as an approximation of U's orthogonal factor.  Muon
// takes U from the gradient's momentum and subtracts lr scale X from the
// weights.
//
// The products run on the f16 matrix cores with f32 sums.  A value v of X, A or
// B is held as two f16 numbers of 2^14 v, hi = f16(2^14 v) and lo = f16(2^14 v
// - hi): 22 bits, and |v| < 4 cannot overflow (|X| <= 1.21, |A| <= 1.46, |B| <=
// 3.45 by the map above).  A product takes hi hi + hi lo + lo hi, three f16
// products at 16 times the f32 matrix rate each, and leaves out lo lo, 2^-22 of
// the result.  Errors against 64-bit steps are those of f32 products (1e-6 to
// 1e-5 of |X|, from the sums' rounding).
#include "elem.hpp"
#include "muon_tiles.hpp"

namespace tatara {
namespace {

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr double kNormEps = 1e-7;
constexpr float kHeld = 16384.0f;             // a held value's factor
constexpr float kUnheld = 1.0f / 16384.0f;
constexpr float kProduct = 1.0f / (16384.0f * 16384.0f);
constexpr uint32_t kPad = 64;                 // sides of the held matrices are multiples of it
constexpr uint32_t kNormParts = 512;          // partial sums of a matrix's norm, at most
constexpr uint32_t kMaxSide = 32768;

using half8 = f16_t __attribute__((ext_vector_type(8)));
using half4 = f16_t __attribute__((ext_vector_type(4)));
using floatx16 = float __attribute__((ext_vector_type(16)));

// Where a held matrix has the hi of (row, col); lo lies kLow further.  Four rows'
// 16 columns of hi fill a 128-byte line, the next line has their lo: a stage's
// loads take whole lines, also where a stage is of 16 columns.  Loads of
// half lines ran at 22 to 27 bytes a clock and CU, of whole ones at 35.
using Held = f16_t*;
constexpr uint32_t kLow = 64;
__device__ __forceinline__ uint64_t held_at(uint64_t row, uint32_t col, uint32_t cols) {
    return ((row / 4) * (cols / 16) + col / 16) * 128 + row % 4 * 16 + col % 16;
}

// v less an f16 number, in one instruction of both widths: the factor is hidden from
// the compiler, which would widen the number and subtract.
__device__ __forceinline__ float less(float v, f16_t h) {
    float minus = -1.0f;
    asm("" : "+s"(minus));
    return fmaf((float)h, minus, v);
}

__device__ __forceinline__ void split(float v, f16_t& hi, f16_t& lo) {
    const float s = v * kHeld;
    hi = (f16_t)s;
    lo = (f16_t)less(s, hi);
}

// Where a step's U comes from: a gradient alone, or a gradient and the
// momentum that it has been added to.
struct Source {
    const void* grad;
    float* momentum;  // null: U = grad
    int64_t row_stride, batch_stride;
    uint32_t rows, cols;
    float beta, mix;  // f32 of beta and of 1 - beta, each rounded once
    int32_t nesterov;
};

// 1 / (sqrt(sum of squares) + 1e-7) as a power of two and a factor near 1, so that
// f32 products with a matrix's values neither overflow nor lose bits at any size.
struct Inverse {
    float power, factor;
    __device__ __forceinline__ explicit Inverse(double squares) {
        const double norm = sqrt(squares) + kNormEps;
        const int e = norm > 1.0 && norm < 1e300 ? ilogb(norm) : 0;
        power = (float)ldexp(1.0, -e);
        factor = (float)(ldexp(1.0, e) / norm);
    }
    __device__ __forceinline__ float times(float x) const { return x * power * factor; }
};

constexpr int kPiece = 8;  // elements of a row that a thread takes at once

// Eight elements of U from (row, col) on, zeros past the row's end.
template <typename T, bool FIRST>
__device__ __forceinline__ void source_values(const Source& s, uint32_t b, uint32_t row, uint32_t col,
                                              float (&u)[kPiece]) {
    const T* g = static_cast<const T*>(s.grad) + (int64_t)b * s.batch_stride + (int64_t)row * s.row_stride + col;
    const int left = (int)s.cols - (int)col;
    Piece<T> p[kPiece / Piece<T>::V];
    float m[kPiece];
    float* at = s.momentum + ((uint64_t)b * s.rows + row) * s.cols + col;
    if (left >= kPiece) {
        __builtin_memcpy(p, g, sizeof(p));
        if (s.momentum) __builtin_memcpy(m, at, sizeof(m));
    } else {
#pragma unroll
        for (int j = 0; j < kPiece; ++j) {
            p[j / Piece<T>::V].v[j % Piece<T>::V] = j < left ? g[j] : (T)0.0f;
            m[j] = s.momentum && j < left ? at[j] : 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < kPiece; ++j) {
        const float gv = (float)p[j / Piece<T>::V].v[j % Piece<T>::V];
        if (!s.momentum) {
            u[j] = gv;
            continue;
        }
        if (FIRST) m[j] = s.beta * m[j] + s.mix * gv;
        u[j] = s.nesterov ? s.mix * gv + s.beta * m[j] : m[j];
    }
    if (FIRST && s.momentum) {
        if (left >= kPiece) {
            __builtin_memcpy(at, m, sizeof(m));
        } else {
#pragma unroll
            for (int j = 0; j < kPiece; ++j)
                if (j < left) at[j] = m[j];
        }
    }
}

// Sum over the workgroup's 256 threads, the same in all of them.
__device__ __forceinline__ double block_sum(double x, double (&join)[256 / kWave]) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    if (threadIdx.x % kWave == 0) join[threadIdx.x / kWave] = x;
    __syncthreads();
    return join[0] + join[1] + join[2] + join[3];
}

// Adds the gradient to the momentum and leaves partial sums of |U|^2.  Squares
// are summed in 64 bits: no gradient's size overflows or vanishes.  Bound by memory:
// 45 of 1629 x 1536 f32 (1.35 GB read and written) 0.23 ms.
template <typename T>
__global__ __launch_bounds__(256) void muon_moment_kernel(Source s, double* __restrict__ parts) {
    __shared__ double join[256 / kWave];
    const uint32_t b = blockIdx.y, row_pieces = (s.cols + kPiece - 1) / kPiece, n = s.rows * row_pieces;
    double sum = 0.0;
#pragma unroll 2
    for (uint32_t e = blockIdx.x * 256 + threadIdx.x; e < n; e += gridDim.x * 256) {
        const uint32_t row = e / row_pieces;
        float u[kPiece];
        source_values<T, true>(s, b, row, (e - row * row_pieces) * kPiece, u);
#pragma unroll
        for (int j = 0; j < kPiece; ++j) sum = fma((double)u[j], (double)u[j], sum);
    }
    sum = block_sum(sum, join);
    if (threadIdx.x == 0) parts[(uint64_t)b * kNormParts + blockIdx.x] = sum;
}

// Writes X_0 as U lies (straight, [rows up][cols up]) and transposed, 64 x 64 a
// workgroup.  U is formed again from gradient and momentum, which costs no more than
// to have kept it.  Bound by memory: 45 of 1629 x 1536 f32 (1.82 GB) 0.35 ms.
template <typename T>
__global__ __launch_bounds__(256) void muon_split_kernel(Source s, const double* __restrict__ parts, uint32_t n_parts,
                                                         Held straight, Held turned, uint32_t rows_up,
                                                         uint32_t cols_up) {
    __shared__ float tile[64][65];
    __shared__ double join[256 / kWave];
    const uint32_t b = blockIdx.z, r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
    const uint64_t first = 2ull * b * rows_up * cols_up;
    // two pieces a thread; of the straight matrix, then of the turned one
    float u[2][kPiece];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t r = r0 + threadIdx.x / 8 + i * 32, c = c0 + threadIdx.x % 8 * 8;
        if (r < s.rows && c < s.cols) {
            source_values<T, false>(s, b, r, c, u[i]);
        } else {
#pragma unroll
            for (int j = 0; j < kPiece; ++j) u[i][j] = 0.0f;
        }
    }
    double sum = 0.0;
    for (uint32_t i = threadIdx.x; i < n_parts; i += 256) sum += parts[(uint64_t)b * kNormParts + i];
    const Inverse inv(block_sum(sum, join));
    auto put = [&](Held to, const float (&v)[kPiece]) {
        half8 hi, lo;
#pragma unroll
        for (int j = 0; j < kPiece; ++j) {
            f16_t h, l;
            split(v[j], h, l);
            hi[j] = h;
            lo[j] = l;
        }
        *reinterpret_cast<half8*>(to) = hi;
        *reinterpret_cast<half8*>(to + kLow) = lo;
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t r = threadIdx.x / 8 + i * 32, c = threadIdx.x % 8 * 8;
#pragma unroll
        for (int j = 0; j < kPiece; ++j) tile[r][c + j] = u[i][j] = inv.times(u[i][j]);
        put(straight + first + held_at(r0 + r, c0 + c, cols_up), u[i]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t c = threadIdx.x / 8 + i * 32, r = threadIdx.x % 8 * 8;
#pragma unroll
        for (int j = 0; j < kPiece; ++j) u[i][j] = tile[r + j][c];
        put(turned + first + held_at(c0 + c, r0 + r, rows_up), u[i]);
    }
}

// Where X goes after the last step: to `out`, or into the weights.
struct Target {
    void* out;
    int64_t row_stride, batch_stride;
    float* weights;
    float keep, rate, min_w, max_w;  // w = clamp(keep w - rate X)
};

__device__ __forceinline__ float updated(const Target& t, float w, float x) {
    const float u = fmaf(-t.rate, x, t.keep * w);
    return u < t.min_w ? t.min_w : (u > t.max_w ? t.max_w : u);
}

using floatx4 = float __attribute__((ext_vector_type(4)));

struct Halves {
    half4 hi, lo;
};

using half2 = f16_t __attribute__((ext_vector_type(2)));
using floatx2 = float __attribute__((ext_vector_type(2)));

__device__ __forceinline__ half4 to_halves(const floatx4& v) {
    const half2 a = __builtin_convertvector(__builtin_shufflevector(v, v, 0, 1), half2);
    const half2 b = __builtin_convertvector(__builtin_shufflevector(v, v, 2, 3), half2);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3);
}
// Of values that have their factor already.
__device__ __forceinline__ Halves split_held(const floatx4& v) {
    Halves h;
    h.hi = to_halves(v);
    floatx4 rest;
#pragma unroll
    for (int r = 0; r < 4; ++r) rest[r] = less(v[r], h.hi[r]);
    h.lo = to_halves(rest);
    return h;
}

__device__ __forceinline__ half8 join8(const half4& a, const half4& b) {
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
// Products of 16 x 16 blocks, which fill the 32 values of k of an instruction by
// twos; which k a lane's values stand for does not matter as long as both operands
// agree.  (16x16x16 takes as long for half the work, and one right behind a
// 16x16x32 whose sum it adds to has been seen to read that sum too early.)
__device__ __forceinline__ floatx4 mfma32(const half8& a, const half8& b, const floatx4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// Two blocks: lo hi, hi lo, hi hi of both.
__device__ __forceinline__ void products(const Halves& a0, const Halves& a1, const Halves& b0, const Halves& b1,
                                         floatx4& low, floatx4& mid, floatx4& c) {
    const half8 ah = join8(a0.hi, a1.hi), bh = join8(b0.hi, b1.hi);
    low = mfma32(join8(a0.lo, a1.lo), bh, low);
    mid = mfma32(ah, join8(b0.lo, b1.lo), mid);
    c = mfma32(ah, bh, c);
}
// One block: a's hi, then its lo, with both halves of b (lo lo comes for nothing).
__device__ __forceinline__ floatx4 product(const half8& a_hi, const half8& a_lo, const Halves& b, floatx4 c) {
    const half8 both = join8(b.hi, b.lo);
    c = mfma32(a_lo, both, c);
    return mfma32(a_hi, both, c);
}
__device__ __forceinline__ floatx4 product(const Halves& a, const Halves& b, const floatx4& c) {
    return product(join8(a.hi, a.hi), join8(a.lo, a.lo), b, c);
}

// Four elements of a row: at a byte offset from the matrix that is the same for all
// lanes, plus the lane's.  WHOLE: every lane's four exist, and nothing is worked out
// a load.  Otherwise `left` exist, with zeros in the place of the others; their
// loads are in no branch, which would wait for each: they read the matrix's start.
template <bool WHOLE, typename V>
__device__ __forceinline__ floatx4 load4(const V* base, uint32_t uniform, uint32_t lane, int left) {
    const char* p = reinterpret_cast<const char*>(base);
    floatx4 f;
    if (WHOLE) {
        V v[4];
        __builtin_memcpy(v, p + uniform + lane, sizeof(v));
#pragma unroll
        for (int r = 0; r < 4; ++r) f[r] = (float)v[r];
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const V v = *reinterpret_cast<const V*>(p + (r < left ? uniform + lane + r * (uint32_t)sizeof(V) : 0u));
            f[r] = r < left ? (float)v : 0.0f;
        }
    }
    return f;
}
template <bool WHOLE, typename V>
__device__ __forceinline__ void store4(V* base, uint32_t uniform, uint32_t lane, int left, const floatx4& f) {
    V* p = reinterpret_cast<V*>(reinterpret_cast<char*>(base) + uniform + lane);
    const V v[4] = {(V)f[0], (V)f[1], (V)f[2], (V)f[3]};
    if (WHOLE) {
        __builtin_memcpy(p, v, sizeof(v));
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r < left) p[r] = v[r];
    }
}

// All steps of a matrix of a few rows in one workgroup: X stays in registers, in
// blocks of 16 x 16, MB rows of blocks and NT columns of them a wave.  An MFMA
// result's lane holds four rows of a column, which is also how 16x16x16 takes its
// right operand, so B X needs no rearrangement; X X^T takes the blocks
// transposed, which a product with the identity gives (exactly: one term a sum).
// Each wave sums X X^T over its columns, the workgroup adds the waves' sums in
// order.  One launch and one CU a matrix: 9 of 16 x 1536 take 19.2 us, five steps of
// 2.4 us, each bound by the issue of its conversions and products (270 instructions
// a wave, four waves a SIMD).
// All 16 waves also where columns do not fill them: they share the sums and B (16 x 16:
// 8 us, with one wave 22; 64 x 64: 38, with four 75).
constexpr uint32_t kSmallWaves = 16;
template <int MB, int NT, typename T>
__global__ __launch_bounds__(kSmallWaves* kWave) void muon_small_kernel(Source s, Target t, uint32_t steps) {
    constexpr uint32_t waves = kSmallWaves;
    constexpr int NB = MB * (MB + 1) / 2, CHUNK = NB < 4 ? NB : 4, PITCH = MB * 16 + 4;
    __shared__ __align__(16) float gram[MB * 16][PITCH];
    __shared__ __align__(16) f16_t poly_hi[MB * 16][PITCH], poly_lo[MB * 16][PITCH];
    // one more, so that four waves' sums that are read together lie in different banks
    __shared__ floatx4 parts[waves][CHUNK * kWave + 1];
    __shared__ double join[waves];
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t col = lane % 16, row4 = lane / 16 * 4;
    const bool flipped = s.rows > s.cols;
    const uint32_t m = flipped ? s.cols : s.rows, n = flipped ? s.rows : s.cols, b = blockIdx.x;
    half4 identity;
#pragma unroll
    for (int r = 0; r < 4; ++r) identity[r] = row4 + r == col ? (f16_t)1.0f : (f16_t)0.0f;
    const half8 of_hi = join8(identity, half4{}), of_lo = join8(half4{}, identity);
    const floatx4 zero = {};
    // a block transposed, exactly: a sum of one term
    auto turn16 = [&](const Halves& h) {
        Halves o;
        o.hi = to_halves(mfma32(join8(h.hi, h.lo), of_hi, zero));
        o.lo = to_halves(mfma32(join8(h.hi, h.lo), of_lo, zero));
        return o;
    };
    // A lane reads and writes four neighbours of a row of U, neighbouring lanes the
    // next ones (lane by lane from row to row, loads took ten times as long), which
    // LDS puts where the products take them.  A lane's part of the offset is the
    // same for all its blocks, the rest the same for all lanes.
    const uint32_t my_row = lane / 4, my_col = lane % 4 * 4;
    auto moved = [&](int slot, const Halves& h, uint32_t from, uint32_t to) {
        half8* at = reinterpret_cast<half8*>(parts[wave] + slot % CHUNK * kWave);
        // 16 columns' pieces lie 64 bytes apart; turned, they cover all banks
        from ^= from / 16;
        to ^= to / 16;
        at[from] = join8(h.hi, h.lo);
        __builtin_amdgcn_wave_barrier();
        const half8 v = at[to];
        __builtin_amdgcn_wave_barrier();
        Halves o;
        o.hi = __builtin_shufflevector(v, v, 0, 1, 2, 3);
        o.lo = __builtin_shufflevector(v, v, 4, 5, 6, 7);
        return o;
    };
    const uint64_t first = (uint64_t)b * s.rows * s.cols;
    const uint32_t y0 = __builtin_amdgcn_readfirstlane(wave) * 16;
    auto left = [&](int ib, int tt) {
        const uint32_t y = tt * waves * 16 + y0;
        const uint32_t r = flipped ? y + my_row : ib * 16 + my_row, c = flipped ? ib * 16 + my_col : y + my_col;
        return r < s.rows ? (int)s.cols - (int)c : 0;
    };
    auto uniform = [&](int64_t row_stride, uint32_t size, int ib, int tt) {
        const uint32_t pitch = (uint32_t)row_stride * size, y = tt * waves * 16 + y0;
        return flipped ? y * pitch + ib * 16 * size : ib * 16 * pitch + y * size;
    };
    auto mine = [&](int64_t row_stride, uint32_t size) {
        return my_row * (uint32_t)row_stride * size + my_col * size;
    };
    // all of the wave's blocks lie inside
    const bool whole = m == MB * 16 && (NT - 1) * waves * 16 + y0 + 16 <= n;
    // The weights are read with the rest where registers last (6 blocks a lane).
    constexpr bool EARLY = MB * NT <= 6;
    floatx4 u[MB][NT], w[EARLY ? MB : 1][EARLY ? NT : 1];
    auto read = [&](auto is_whole) {
        constexpr bool WHOLE = decltype(is_whole)::value;
        const T* g = static_cast<const T*>(s.grad) + (int64_t)b * s.batch_stride;
        const uint32_t g_lane = mine(s.row_stride, sizeof(T)), w_lane = mine(s.cols, 4);
#pragma unroll
        for (int tt = 0; tt < NT; ++tt)
#pragma unroll
            for (int ib = 0; ib < MB; ++ib)
                u[ib][tt] = load4<WHOLE>(g, uniform(s.row_stride, sizeof(T), ib, tt), g_lane, left(ib, tt));
        if (!s.momentum) return;
        float* mom = s.momentum + first;
        // columns of blocks whose loads go out together, ahead of their stores
        constexpr int BATCH = EARLY ? NT : (6 + MB - 1) / MB;
#pragma unroll
        for (int t0 = 0; t0 < NT; t0 += BATCH) {
            floatx4 mo[BATCH][MB];
#pragma unroll
            for (int q = 0; q < BATCH && t0 + q < NT; ++q)
#pragma unroll
                for (int ib = 0; ib < MB; ++ib)
                    mo[q][ib] = load4<WHOLE>((const float*)mom, uniform(s.cols, 4, ib, t0 + q), w_lane, left(ib, t0 + q));
            if constexpr (EARLY) {  // momentum comes with weights
#pragma unroll
                for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                    for (int ib = 0; ib < MB; ++ib)
                        w[ib][tt] = load4<WHOLE>((const float*)t.weights + first, uniform(s.cols, 4, ib, tt), w_lane,
                                                 left(ib, tt));
            }
#pragma unroll
            for (int q = 0; q < BATCH && t0 + q < NT; ++q)
#pragma unroll
                for (int ib = 0; ib < MB; ++ib) {
                    const floatx4 gv = u[ib][t0 + q], m1 = s.beta * mo[q][ib] + s.mix * gv;
                    store4<WHOLE>(mom, uniform(s.cols, 4, ib, t0 + q), w_lane, left(ib, t0 + q), m1);
                    u[ib][t0 + q] = s.nesterov ? s.mix * gv + s.beta * m1 : m1;  // zeros stay zeros
                }
        }
    };
    if (whole)
        read(std::true_type{});
    else
        read(std::false_type{});
    double sum = 0.0;
#pragma unroll
    for (int ib = 0; ib < MB; ++ib)
#pragma unroll
        for (int tt = 0; tt < NT; ++tt)
#pragma unroll
            for (int r = 0; r < 4; ++r) sum = fma((double)u[ib][tt][r], (double)u[ib][tt][r], sum);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) join[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < (int)waves; ++i) sum += join[i];
    const Inverse inv(sum);
    // X as it is held; its f32 values only pass through
    Halves x[MB][NT];
#pragma unroll
    for (int ib = 0; ib < MB; ++ib)
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
            floatx4 v;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = inv.times(u[ib][tt][r]) * kHeld;
            x[ib][tt] = moved(ib * NT + tt, split_held(v), lane, col * 4 + row4 / 4);
        }
    if (!flipped) {
#pragma unroll
        for (int ib = 0; ib < MB; ++ib)
#pragma unroll
            for (int tt = 0; tt < NT; ++tt) x[ib][tt] = turn16(x[ib][tt]);
    }

#pragma unroll 1
    for (uint32_t step = 0; step < steps; ++step) {
        floatx4 low[NB], mid[NB], acc[NB];
#pragma unroll
        for (int k = 0; k < NB; ++k) low[k] = mid[k] = acc[k] = zero;
#pragma unroll
        for (int tt = 0; tt < NT; tt += 2) {
            Halves rows[2][MB];
#pragma unroll
            for (int o = 0; o < 2 && tt + o < NT; ++o)
#pragma unroll
                for (int ib = 0; ib < MB; ++ib) rows[o][ib] = turn16(x[ib][tt + o]);
            int k = 0;
#pragma unroll
            for (int ib = 0; ib < MB; ++ib)
#pragma unroll
                for (int jb = ib; jb < MB; ++jb, ++k) {
                    // separate sums where there are too few blocks to fill the wait for one
                    floatx4 &l = MB == 1 ? low[k] : acc[k], &m_ = MB == 1 ? mid[k] : acc[k];
                    if (tt + 1 < NT)
                        products(rows[0][ib], rows[1][ib], rows[0][jb], rows[1][jb], l, m_, acc[k]);
                    else
                        acc[k] = product(rows[0][ib], rows[0][jb], acc[k]);
                }
            if (MB > 1) __builtin_amdgcn_sched_barrier(0);  // more columns' blocks at once would not fit
        }
        if (MB == 1) acc[0] += low[0] + mid[0];
#pragma unroll
        for (int k0 = 0; k0 < NB; k0 += CHUNK) {
#pragma unroll
            for (int k = 0; k < CHUNK; ++k)
                if (k0 + k < NB) parts[wave][k * kWave + lane] = acc[k0 + k];
            __syncthreads();
            const uint32_t have = (NB - k0 < CHUNK ? NB - k0 : CHUNK) * 256;
            // four lanes an element, four waves' sums a lane
            for (uint32_t q = threadIdx.x; q < have * 4; q += waves * kWave) {
                const uint32_t e = q / 4, w0 = q % 4 * 4;
                float v = 0.0f;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
                    v += reinterpret_cast<const float*>(parts[w0 + i])[e];
                v += __shfl_xor(v, 1);
                v += __shfl_xor(v, 2);
                v *= kUnheld;  // with its factor
                if (w0) continue;
                uint32_t k = k0 + e / 256, ib = 0;
                while (k >= MB - ib) k -= MB - ib, ++ib;
                const uint32_t jb = ib + k, l = e % 256 / 4;
                const uint32_t i = ib * 16 + l / 16 * 4 + e % 4, j = jb * 16 + l % 16;
                gram[i][j] = v;
                if (ib != jb) gram[j][i] = v;
            }
            __syncthreads();
        }
        // block (ib, jb) of B, four rows of a column a lane
        auto poly = [&](uint32_t ib, uint32_t jb) {
            floatx4 v = zero;
#pragma unroll
            for (int kb = 0; kb < MB; ++kb)
                v = product(split_held(*reinterpret_cast<const floatx4*>(&gram[ib * 16 + col][kb * 16 + row4])),
                            split_held(*reinterpret_cast<const floatx4*>(&gram[jb * 16 + col][kb * 16 + row4])), v);
            const floatx4 old = *reinterpret_cast<const floatx4*>(&gram[jb * 16 + col][ib * 16 + row4]);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                v[r] = fmaf(kC * kProduct, v[r], fmaf(kB * kUnheld, old[r], ib == jb && row4 + r == col ? kA : 0.0f));
            // without the factor, so that B X has X's: of B's entries, up to 3.45, no
            // more than 2^-25 is lost to f16's smallest numbers
            return split_held(v);
        };
        // B is symmetric: four rows of a column are four columns of a row, as the
        // left operand takes them.  One block every wave computes for itself.
        Halves only;
        if constexpr (MB == 1) {
            only = poly(0, 0);
        } else {
            if (wave < MB * MB) {
                const uint32_t ib = wave / MB, jb = wave % MB;
                const Halves h = poly(ib, jb);
                *reinterpret_cast<half4*>(&poly_hi[jb * 16 + col][ib * 16 + row4]) = h.hi;
                *reinterpret_cast<half4*>(&poly_lo[jb * 16 + col][ib * 16 + row4]) = h.lo;
            }
            __syncthreads();
        }
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
            Halves cols[MB];
#pragma unroll
            for (int kb = 0; kb < MB; ++kb) cols[kb] = x[kb][tt];
#pragma unroll
            for (int ib = 0; ib < MB; ++ib) {
                floatx4 v = zero;
                auto block = [&](int kb) {
                    if (MB == 1) return only;
                    Halves h;
                    h.hi = *reinterpret_cast<const half4*>(&poly_hi[ib * 16 + col][kb * 16 + row4]);
                    h.lo = *reinterpret_cast<const half4*>(&poly_lo[ib * 16 + col][kb * 16 + row4]);
                    return h;
                };
#pragma unroll
                for (int kb = 0; kb + 1 < MB; kb += 2)
                    products(block(kb), block(kb + 1), cols[kb], cols[kb + 1], v, v, v);
                if (MB % 2) v = product(block(MB - 1), cols[MB - 1], v);
                x[ib][tt] = split_held(v);
            }
            if (MB > 1) __builtin_amdgcn_sched_barrier(0);
        }
    }
    auto write = [&](auto is_whole) {
        constexpr bool WHOLE = decltype(is_whole)::value;
        const uint32_t w_lane = mine(s.cols, 4), o_lane = mine(t.row_stride, sizeof(T));
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
            if constexpr (!EARLY) {
                if (t.weights) {
#pragma unroll
                    for (int ib = 0; ib < MB; ++ib)
                        u[ib][tt] = load4<WHOLE>((const float*)t.weights + first, uniform(s.cols, 4, ib, tt), w_lane,
                                                 left(ib, tt));
                }
            }
#pragma unroll
            for (int ib = 0; ib < MB; ++ib) {
                const Halves h =
                    moved(ib * NT + tt, flipped ? x[ib][tt] : turn16(x[ib][tt]), col * 4 + row4 / 4, lane);
                floatx4 v;
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = ((float)h.hi[r] + (float)h.lo[r]) * kUnheld;
                if (t.weights) {
                    const floatx4 old = EARLY ? w[EARLY ? ib : 0][EARLY ? tt : 0] : u[ib][tt];
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = updated(t, old[r], v[r]);
                    store4<WHOLE>(t.weights + first, uniform(s.cols, 4, ib, tt), w_lane, left(ib, tt), v);
                } else {
                    store4<WHOLE>(static_cast<T*>(t.out) + (int64_t)b * t.batch_stride,
                                  uniform(t.row_stride, sizeof(T), ib, tt), o_lane, left(ib, tt), v);
                }
            }
        }
    };
    if (whole)
        write(std::true_type{});
    else
        write(std::false_type{});
}

// What becomes of a product's tile.
enum Epilogue { kGram, kPoly, kApply, kOut, kUpdate };

struct ProductArgs {
    Held p, q;           // [m][k] and [n][k]: the product is p q^T
    uint32_t m, n, k;    // multiples of kPad
    uint32_t tiles_m, tiles_n, tiles;  // of one matrix's product
    Held old;            // kPoly: A
    Held to, turned;     // results as they lie and (kApply) transposed
    // kOut, kUpdate: the caller's matrices, [rows][cols]; flipped: X is their transpose
    Target target;
    uint32_t rows, cols;
    int32_t flipped;
};

// A stage lies in LDS by blocks of 16 columns, in each the rows of p, then of q, four
// rows' 16 pieces together as they lie in memory (hi of the four rows, then lo).
// Within those the place turns with the row, so that 16 rows of one piece cover all
// of LDS's banks.
__device__ __forceinline__ uint32_t turn(uint32_t row) {
    return (row / 4 & 1) | (row / 4 & 2) << 2;
}
__device__ __forceinline__ uint32_t place(uint32_t row, uint32_t low, uint32_t half) {
    return row / 4 * 16 + ((low * 8 + row % 4 * 2 + half) ^ turn(row));
}

// 16 bytes a lane from global memory to LDS, the wave's 64 in a row from `to`.
__device__ __forceinline__ void load_to_lds(const f16_t* from, half8* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// Waits until at most N of the wave's loads are on their way and its LDS reads
// are done, then for the workgroup.
template <int N>
__device__ __forceinline__ void arrive() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A wave's strip of 32 rows in LDS, f32: filled from MFMA results, read in rows.
template <typename L>
struct Strip {
    static constexpr int PITCH = StripShape<L>::PITCH;
    float* base;
    uint32_t lane;

    // block t of the strip, its rows along the strip's
    __device__ __forceinline__ void put_along(const floatx16& v, int t) const {
#pragma unroll
        for (int r = 0; r < 16; ++r) base[(r / 4 * 8 + lane / 32 * 4 + r % 4) * PITCH + t * 32 + lane % 32] = v[r];
    }
    // block t, transposed
    __device__ __forceinline__ void put_across(const floatx16& v, int t) const {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float4 q = {v[g * 4], v[g * 4 + 1], v[g * 4 + 2], v[g * 4 + 3]};
            *reinterpret_cast<float4*>(base + lane % 32 * PITCH + t * 32 + g * 8 + lane / 32 * 4) = q;
        }
    }
    // Between filling a strip and reading it, and before the next filling: lanes read what
    // others wrote.  The wave's LDS accesses are done in their order, which the compiler
    // has to keep; no instruction.
    __device__ __forceinline__ static void exchange() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    // the strip as rows of a held matrix from (row, col) on, of which `left`
    // columns exist (a multiple of 32: the side is one of 64, a strip starts at one of 32)
    template <int WIDTH>
    __device__ __forceinline__ void store(Held to, uint32_t row, uint32_t col, uint32_t cols, int32_t left) const {
        constexpr int LANES = WIDTH / 8;  // of a row
        const uint32_t c = lane % LANES * 8;
        exchange();
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += (int)kWave / LANES) {
            const uint32_t r = r0 + lane / LANES;
            half8 hi, lo;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                f16_t h, l;
                split(base[r * PITCH + c + j], h, l);
                hi[j] = h;
                lo[j] = l;
            }
            if ((int32_t)c < left) {
                f16_t* at = to + held_at(row + r, col + c, cols);
                *reinterpret_cast<half8*>(at) = hi;
                *reinterpret_cast<half8*>(at + kLow) = lo;
            }
        }
        exchange();
    }
    // its values one by one, a batch's loads ahead of its stores:
    // store(row, column, value, load(row, column))
    template <int WIDTH, typename F, typename G>
    __device__ __forceinline__ void each(F&& load, G&& store) const {
        constexpr int ROWS = (int)kWave / WIDTH, BATCH = 8;
        const uint32_t c = lane % WIDTH;
        exchange();
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += BATCH * ROWS) {
            float old[BATCH];
#pragma unroll
            for (int q = 0; q < BATCH; ++q) old[q] = load(r0 + q * ROWS + lane / WIDTH, c);
#pragma unroll
            for (int q = 0; q < BATCH; ++q) {
                const uint32_t r = r0 + q * ROWS + lane / WIDTH;
                store(r, c, base[r * PITCH + c], old[q]);
            }
        }
        exchange();
    }
};

// hi hi + hi lo + lo hi of every product, whatever the result's type (T, of kOut alone).
// Early steps that multiply hi alone (11 bits) would take a fifth off a bf16 result
// (2048 x 1024: three of five 209 us, none 267) and are not taken: what they leave of it
// has no bound near its own rounding of 1.7e-3.  One of five leaves 3e-6 of a full-rank
// matrix of 256, but 2e-3 of one whose rows are all alike: its one singular value is at
// 1 from the start, and what rounding puts beside it grows in the steps that follow.
//
// 45 of 1629 x 1536 f32, a step: X X^T 0.60 ms, B 0.58, B X 1.15 (1.31 into the
// weights), 930 TFLOP/s of f16 products in tiles of 128.  There the card's power is
// the bound: matrix cores are busy in 57% of cycles at a clock of about 1.6 GHz,
// tiles of 256 x 256 and 256 x 128 reach the same rate.  Small ones are bound by
// latency: 6 to 8 us a launch (5 of 257 x 391).
template <int EPI, typename T, typename L>
__global__ __launch_bounds__(L::THREADS) void muon_product_kernel(ProductArgs a) {
    constexpr int BM = L::BM, BN = L::BN, TM = L::TM, TN = L::TN;
    constexpr int S = L::S, LOADS = L::LOADS;
    constexpr int DOWN = StripShape<L>::DOWN, OVER = StripShape<L>::OVER;
    constexpr int STAGE = L::PIECES, BLOCK = (BM + BN) * 4;  // pieces, of a stage and of 16 columns
    using Lds = ProductLds<L>;
    __shared__ half8 lds[Lds::BYTES / 16];
    // neighbouring tiles on one XCD, so that its L2 holds the panels they share
    const uint32_t bid = xcd_swizzle(blockIdx.x, gridDim.x);
    const uint32_t b = bid / a.tiles, at = bid % a.tiles;
    uint32_t ti, tj;
    if (EPI == kGram || EPI == kPoly) {
        // the result is symmetric: tiles that reach the diagonal or lie right of it
        ti = 0;
        uint32_t left = at;
        for (;;) {
            const uint32_t skip = ti * BM / BN, row = a.tiles_n - skip;
            if (left < row) {
                tj = skip + left;
                break;
            }
            left -= row;
            ++ti;
        }
    } else {
        ti = at % a.tiles_m;
        tj = at / a.tiles_m;
    }
    const uint32_t i0 = ti * BM, j0 = tj * BN;
    const uint64_t p_at = 2ull * b * a.m * a.k, q_at = 2ull * b * a.n * a.k;
    const uint32_t tid = threadIdx.x, lane = tid % kWave, group = tid / kWave / (L::WR * L::WC);
    const uint32_t wave = tid / kWave % (L::WR * L::WC);
    const uint32_t wi = wave / L::WC * (TM * 32), wj = wave % L::WC * (TN * 32);
    floatx16 acc[TM][TN] = {};
    const f16_t* from[LOADS];
#pragma unroll
    for (int s = 0; s < LOADS; ++s) {
        const uint32_t e = s * L::THREADS + tid, at = e % BLOCK, four = at / 16;
        const uint32_t piece = at % 16 ^ turn(four * 4), row = four * 4 + piece % 8 / 2;
        // rows past the matrix (its side is a multiple of 64, not of the tile) are not stored
        const uint32_t r = row < BM ? min(i0 + row, a.m - 1) : min(j0 + row - BM, a.n - 1);
        from[s] = (row < BM ? a.p + p_at : a.q + q_at) + held_at(r, e / BLOCK * 16 + piece % 2 * 8, a.k) +
                  piece / 8 * kLow;
    }
    const uint32_t wave0 = __builtin_amdgcn_readfirstlane(tid / kWave) * kWave;
    auto fetch = [&](uint32_t stage, uint32_t k0) {
#pragma unroll
        for (int s = 0; s < LOADS; ++s) load_to_lds(from[s] + k0 * 8, &lds[stage * STAGE + s * L::THREADS + wave0]);
    };
    const uint32_t stages = a.k / L::KS;
    for (uint32_t s = 0; s + 1 < S && s < stages; ++s) fetch(s, s * L::KS);
    uint32_t buf = 0;
    for (uint32_t it = 0; it < stages; ++it) {
        // this stage has arrived, and nobody reads the one before it any more
        if (it + S - 1 <= stages)
            arrive<(S - 2) * LOADS>();
        else
            arrive<0>();
        if (it + S - 1 < stages) fetch(buf == 0 ? S - 1 : buf - 1, (it + S - 1) * L::KS);
        // the next 16 values of k are read while these are multiplied
        constexpr int STEPS = L::KS / 16 / L::KG;
        half8 fp[2][2][TM], fq[2][2][TN];  // [this, next][hi, lo][block]
        auto read = [&](int kk) {
            const half8* from_lds = lds + buf * STAGE + (kk * L::KG + group) * BLOCK;
#pragma unroll
            for (int lo = 0; lo < 2; ++lo) {
                // in the order of the products below
#pragma unroll
                for (int x = 0; x < TM; ++x) {
                    const uint32_t row = wi + x * 32 + lane % 32;
                    fp[kk % 2][1 - lo][x] = from_lds[place(row, 1 - lo, lane / 32)];
                }
#pragma unroll
                for (int y = 0; y < TN; ++y) {
                    const uint32_t row = BM + wj + y * 32 + lane % 32;
                    fq[kk % 2][lo][y] = from_lds[place(row, lo, lane / 32)];
                }
            }
        };
        read(0);
#pragma unroll
        for (int kk = 0; kk < STEPS; ++kk) {
            if (kk + 1 < STEPS) read(kk + 1);
            const int c = kk % 2;
#pragma unroll
            for (int pass = 2; pass >= 0; --pass)  // lo hi, hi lo, hi hi
#pragma unroll
                for (int x = 0; x < TM; ++x)
#pragma unroll
                    for (int y = 0; y < TN; ++y)
                        acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[c][pass == 2][x], fq[c][pass == 1][y],
                                                                           acc[x][y], 0, 0, 0);
        }
        buf = buf + 1 == S ? 0 : buf + 1;
    }
    // A lane holds, of each 32 x 32 block, four groups of four consecutive rows of
    // one column.  Strips of 32 rows (or columns) go through LDS, a region a wave,
    // so that they are stored in whole rows.
    arrive<0>();
    if constexpr (L::KG > 1) {
        floatx4* sums = reinterpret_cast<floatx4*>(lds);
        if (group > 0) {
#pragma unroll
            for (int x = 0; x < TM; ++x)
#pragma unroll
                for (int y = 0; y < TN; ++y)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        sums[Lds::sum(group, wave, (x * TN + y) * 4 + q, lane)] =
                            floatx4{acc[x][y][q * 4], acc[x][y][q * 4 + 1], acc[x][y][q * 4 + 2], acc[x][y][q * 4 + 3]};
        }
        __syncthreads();
        if (group > 0) return;  // no barrier follows: a wave's strip holds none of the sums
#pragma unroll
        for (int x = 0; x < TM; ++x)
#pragma unroll
            for (int y = 0; y < TN; ++y)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int o = 1; o < L::KG; ++o) {
                        const floatx4 v = sums[Lds::sum(o, wave, (x * TN + y) * 4 + q, lane)];
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[x][y][q * 4 + r] += v[r];
                    }
    }
    const Strip<L> strip{reinterpret_cast<float*>(lds) + Lds::strip(wave) / 4, lane};
    const uint64_t first = 2ull * b * a.m * a.n;
#pragma unroll
    for (int x = 0; x < TM; ++x) {
        const uint32_t i = i0 + wi + x * 32;
        if (EPI == kPoly && i < a.m) {
            // A is symmetric: four rows of a column are four columns of a row
            half4 hi[TN][4], lo[TN][4];
#pragma unroll
            for (int y = 0; y < TN; ++y)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const uint32_t j = min(j0 + wj + y * 32 + lane % 32, a.n - 1);
                    const f16_t* o = a.old + first + held_at(j, i + g * 8 + lane / 32 * 4, a.m);
                    hi[y][g] = *reinterpret_cast<const half4*>(o);
                    lo[y][g] = *reinterpret_cast<const half4*>(o + kLow);
                }
#pragma unroll
            for (int y = 0; y < TN; ++y)
#pragma unroll
                for (int g = 0; g < 4; ++g)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float o = ((float)hi[y][g][r] + (float)lo[y][g][r]) * kUnheld;
                        const float v = acc[x][y][g * 4 + r] * kProduct;
                        const bool diagonal = i + g * 8 + lane / 32 * 4 + r == j0 + wj + y * 32 + lane % 32;
                        acc[x][y][g * 4 + r] = fmaf(kC, v, fmaf(kB, o, diagonal ? kA : 0.0f));
                    }
        } else {
#pragma unroll
            for (int y = 0; y < TN; ++y)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[x][y][r] *= kProduct;
        }
    }
    if (EPI == kOut || EPI == kUpdate) {
        auto read = [&](uint32_t row, uint32_t col) {
            if (EPI == kOut || row >= a.rows || col >= a.cols) return 0.0f;
            return a.target.weights[((uint64_t)b * a.rows + row) * a.cols + col];
        };
        auto write = [&](uint32_t row, uint32_t col, float v, float w) {
            if (row >= a.rows || col >= a.cols) return;
            if (EPI == kOut) {
                static_cast<T*>(a.target.out)[(int64_t)b * a.target.batch_stride +
                                              (int64_t)row * a.target.row_stride + col] = (T)v;
            } else {
                a.target.weights[((uint64_t)b * a.rows + row) * a.cols + col] = updated(a.target, w, v);
            }
        };
        if (a.flipped) {
#pragma unroll
            for (int y = 0; y < TN; ++y)
#pragma unroll
                for (int x = 0; x < TM; x += DOWN) {
                    const uint32_t j = j0 + wj + y * 32, i = i0 + wi + x * 32;
#pragma unroll
                    for (int t = 0; t < DOWN; ++t) strip.put_across(acc[x + t][y], t);
                    strip.template each<DOWN * 32>(
                        [&](uint32_t r, uint32_t c) { return read(j + r, i + c); },
                        [&](uint32_t r, uint32_t c, float v, float w) { write(j + r, i + c, v, w); });
                }
        } else {
#pragma unroll
            for (int x = 0; x < TM; ++x)
#pragma unroll
                for (int y = 0; y < TN; y += OVER) {
                    const uint32_t j = j0 + wj + y * 32, i = i0 + wi + x * 32;
#pragma unroll
                    for (int t = 0; t < OVER; ++t) strip.put_along(acc[x][y + t], t);
                    strip.template each<OVER * 32>(
                        [&](uint32_t r, uint32_t c) { return read(i + r, j + c); },
                        [&](uint32_t r, uint32_t c, float v, float w) { write(i + r, j + c, v, w); });
                }
        }
        return;
    }
#pragma unroll
    for (int x = 0; x < TM; ++x)
#pragma unroll
        for (int y = 0; y < TN; y += OVER) {
            const uint32_t i = i0 + wi + x * 32, j = j0 + wj + y * 32;
#pragma unroll
            for (int t = 0; t < OVER; ++t) strip.put_along(acc[x][y + t], t);
            strip.template store<OVER * 32>(a.to + first, i, j, a.n, i < a.m ? a.n - j : 0);
        }
    // a symmetric result's other half; a tile on the diagonal has both
    if (EPI == kApply || j0 >= i0 + BM) {
#pragma unroll
        for (int y = 0; y < TN; ++y)
#pragma unroll
            for (int x = 0; x < TM; x += DOWN) {
                const uint32_t i = i0 + wi + x * 32, j = j0 + wj + y * 32;
#pragma unroll
                for (int t = 0; t < DOWN; ++t) strip.put_across(acc[x + t][y], t);
                strip.template store<DOWN * 32>((EPI == kApply ? a.turned : a.to) + first, j, i, a.m,
                                                j < a.n ? a.m - i : 0);
            }
    }
}

template <int EPI, typename L>
uint32_t count_tiles(ProductArgs& p) {
    p.tiles_m = ceil_div(p.m, L::BM);
    p.tiles_n = ceil_div(p.n, L::BN);
    p.tiles = p.tiles_m * p.tiles_n;
    if (EPI == kGram || EPI == kPoly) {
        p.tiles = 0;
        for (uint32_t i = 0; i < p.tiles_m; ++i) p.tiles += p.tiles_n - i * L::BM / L::BN;
    }
    return p.tiles;
}

template <int EPI, typename T, typename L>
void launch_tiles(ProductArgs p, uint32_t batch, hipStream_t stream) {
    const uint32_t tiles = count_tiles<EPI, L>(p);
    muon_product_kernel<EPI, T, L><<<tiles * batch, L::THREADS, 0, stream>>>(p);
}

// Tiles of 128, two workgroups a CU that fill each other's waits, from two rounds
// of the GPU's CUs on.  Below, tiles of 64, with two groups of waves for one
// workgroup on a CU; two stages of them let a second workgroup onto a CU (30 of 200
// x 200: 130 us, three stages 163), three go further where it would have nothing to
// do (3 of 512 x 512: 142, two 150).  What bounds such a product is what a CU's loads
// bring to LDS, so where CUs are left over the tiles are of 64 x 32 (3 of 512 x 512:
// 137) and 32 x 32, four groups of waves and four stages (512 x 512: 102, tiles of 64
// 127; 257 x 391: 82 and 103; 3 of 512 x 512 139).
template <int EPI, typename T>
void launch_product(ProductArgs p, uint32_t batch, hipStream_t stream) {
    constexpr uint64_t kCus = 256;
    const uint64_t narrow = (uint64_t)batch * count_tiles<EPI, Narrow>(p);
    if ((uint64_t)batch * count_tiles<EPI, Wide>(p) >= 2 * kCus)
        launch_tiles<EPI, T, Wide>(p, batch, stream);
    else if (narrow > kCus)
        launch_tiles<EPI, T, Narrow>(p, batch, stream);
    else if (narrow > kCus / 2)
        launch_tiles<EPI, T, Deep>(p, batch, stream);
    else if (narrow > kCus * 3 / 8)
        launch_tiles<EPI, T, Half>(p, batch, stream);
    else
        launch_tiles<EPI, T, Tiny>(p, batch, stream);
}

struct Step {
    Held x, xt, next_xt, gram, poly;
    uint32_t m, n;
    bool last;
};

template <typename T>
void launch_step(const Step& s, const Source& from, const Target& t, uint32_t batch, hipStream_t stream) {
    ProductArgs p{};
    p.p = p.q = s.x;
    p.m = p.n = s.m;
    p.k = s.n;
    p.to = s.gram;
    launch_product<kGram, float>(p, batch, stream);
    p.p = p.q = p.old = s.gram;
    p.k = s.m;
    p.to = s.poly;
    launch_product<kPoly, float>(p, batch, stream);
    p.p = s.poly;
    p.q = s.xt;
    p.n = s.n;
    p.to = s.x;
    p.turned = s.next_xt;
    p.target = t;
    p.rows = from.rows;
    p.cols = from.cols;
    p.flipped = from.rows > from.cols;
    if (!s.last)
        launch_product<kApply, float>(p, batch, stream);
    else if (t.weights)
        launch_product<kUpdate, float>(p, batch, stream);
    else
        launch_product<kOut, T>(p, batch, stream);
}

uint32_t up(uint32_t n) { return (n + kPad - 1) / kPad * kPad; }

// The workspace's parts, by their byte offsets.
struct Layout {
    uint64_t parts, x, xt[2], a, b, bytes;
    uint32_t m, n;
    Layout(uint32_t batch, uint32_t rows, uint32_t cols) {
        m = up(std::min(rows, cols));
        n = up(std::max(rows, cols));
        const uint64_t full = (uint64_t)batch * m * n, side = (uint64_t)batch * m * m;
        uint64_t at = 0;
        auto take = [&](uint64_t n_bytes) {
            const uint64_t o = at;
            at += (n_bytes + 255) / 256 * 256;
            return o;
        };
        parts = take(sizeof(double) * kNormParts * (uint64_t)batch);
        x = take(4 * full);
        xt[0] = take(4 * full);
        xt[1] = take(4 * full);
        a = take(4 * side);
        b = take(4 * side);
        bytes = at;
    }
};

Held held(void* ws, uint64_t offset) { return reinterpret_cast<Held>(static_cast<uint8_t*>(ws) + offset); }

// Columns of blocks that a wave of muon_small_kernel holds, 0 where a workgroup
// cannot hold the matrix: twelve blocks a wave are 48 of its 128 registers.  From eight
// blocks on they do not last beside a step's sums, and 40 to 330 bytes a lane go to
// scratch.  What it can hold is faster there all the same (one of
// 16 x 1536: 16 us, by products 82; 32 x 1536, 12 blocks, 38 and 82; 64 x 512, 8 blocks,
// 53 and 66) or as fast on one CU (64 x 768, 12 blocks: 73 and 70).
uint32_t small_blocks(uint32_t rows, uint32_t cols) {
    const uint32_t mb = ceil_div(std::min(rows, cols), 16), nt = ceil_div(std::max(rows, cols), 256);
    if (mb > 4 || nt * mb > 12) return 0;
    for (uint32_t have : {1u, 2u, 3u, 4u, 6u, 12u})
        if (nt <= have && have * mb <= 12) return have;
    return 0;
}

template <typename T>
int32_t launch_small(const Source& s, const Target& t, uint32_t batch, uint32_t steps, hipStream_t stream) {
    const uint32_t mb = ceil_div(std::min(s.rows, s.cols), 16), nt = small_blocks(s.rows, s.cols);
    auto go = [&](auto m, auto n) {
        muon_small_kernel<decltype(m)::value, decltype(n)::value, T><<<batch, kSmallWaves * kWave, 0, stream>>>(s, t, steps);
    };
    auto with_columns = [&](auto m) {
        constexpr int MB = decltype(m)::value;
        using std::integral_constant;
        if (nt == 1) return go(m, integral_constant<int, 1>{});
        if (nt == 2) return go(m, integral_constant<int, 2>{});
        if (nt == 3) return go(m, integral_constant<int, 3>{});
        if constexpr (MB <= 3)
            if (nt == 4) return go(m, integral_constant<int, 4>{});
        if constexpr (MB <= 2)
            if (nt == 6) return go(m, integral_constant<int, 6>{});
        if constexpr (MB == 1)
            if (nt == 12) return go(m, integral_constant<int, 12>{});
    };
    if (mb == 1)
        with_columns(std::integral_constant<int, 1>{});
    else if (mb == 2)
        with_columns(std::integral_constant<int, 2>{});
    else if (mb == 3)
        with_columns(std::integral_constant<int, 3>{});
    else
        with_columns(std::integral_constant<int, 4>{});
    TATARA_LAUNCHED("muon_small");
    return kOk;
}

template <typename T>
int32_t launch_products(const Source& s, const Target& t, uint32_t batch, uint32_t steps, void* ws,
                        hipStream_t stream) {
    const Layout l(batch, s.rows, s.cols);
    const bool flipped = s.rows > s.cols;
    double* parts = reinterpret_cast<double*>(static_cast<uint8_t*>(ws) + l.parts);
    const Held x = held(ws, l.x), ga = held(ws, l.a), gb = held(ws, l.b), xt[2] = {held(ws, l.xt[0]), held(ws, l.xt[1])};
    const uint32_t n_parts = std::min<uint32_t>(kNormParts, ceil_div((uint64_t)s.rows * ceil_div(s.cols, kPiece), 256));
    muon_moment_kernel<T><<<dim3(n_parts, batch), 256, 0, stream>>>(s, parts);
    TATARA_LAUNCHED("muon_moment");
    muon_split_kernel<T><<<dim3(up(s.cols) / 64, up(s.rows) / 64, batch), 256, 0, stream>>>(
        s, parts, n_parts, flipped ? xt[0] : x, flipped ? x : xt[0], up(s.rows), up(s.cols));
    TATARA_LAUNCHED("muon_split");
    for (uint32_t i = 0; i < steps; ++i) {
        Step step{};
        step.x = x;
        step.xt = xt[i % 2];
        step.next_xt = xt[(i + 1) % 2];
        step.gram = ga;
        step.poly = gb;
        step.m = l.m;
        step.n = l.n;
        step.last = i + 1 == steps;
        launch_step<T>(step, s, t, batch, stream);
        TATARA_LAUNCHED("muon_product");
    }
    return kOk;
}

template <typename T>
int32_t launch_steps(const Source& s, const Target& t, uint32_t batch, uint32_t steps, void* ws, hipStream_t stream) {
    // its offsets within a matrix are of 32 bits
    const bool near = (uint64_t)s.rows * std::max(s.row_stride, t.row_stride) < (1u << 29);
    if (near && small_blocks(s.rows, s.cols)) return launch_small<T>(s, t, batch, steps, stream);
    return launch_products<T>(s, t, batch, steps, ws, stream);
}

int32_t check_matrices(uint32_t batch, uint32_t rows, uint32_t cols, int32_t dtype) {
    TATARA_REQUIRE_DTYPE(dtype);
    TATARA_REQUIRE(rows >= 1 && rows <= kMaxSide && cols >= 1 && cols <= kMaxSide, "a matrix has sides of 1 to 32768");
    TATARA_REQUIRE(batch <= 65535, "at most 65535 matrices");
    return kOk;
}

}  // namespace
}  // namespace tatara

using namespace tatara;

extern "C" {

int32_t tatara_op_orthogonalise_workspace(uint32_t batch, uint32_t rows, uint32_t cols, int32_t dtype,
                                          uint64_t* bytes) {
    TATARA_REQUIRE(bytes, "null output");
    if (int32_t st = check_matrices(batch, rows, cols, dtype)) return st;
    *bytes = Layout(batch, rows, cols).bytes;
    return kOk;
}

int32_t tatara_op_orthogonalise(const void* in, int64_t in_row_stride, int64_t in_batch_stride, void* out,
                                int64_t out_row_stride, int64_t out_batch_stride, uint32_t batch, uint32_t rows,
                                uint32_t cols, int32_t dtype, uint32_t steps, void* workspace,
                                uint64_t workspace_bytes, TataraStream* stream) {
    if (int32_t st = check_matrices(batch, rows, cols, dtype)) return st;
    TATARA_REQUIRE(steps >= 1 && steps <= 32, "steps must be 1 to 32");
    if (batch == 0) return kOk;
    TATARA_REQUIRE(in && out, "null tensor");
    TATARA_REQUIRE(in_row_stride >= (int64_t)cols && out_row_stride >= (int64_t)cols,
                   "a row stride is smaller than the row");
    TATARA_REQUIRE(batch == 1 || (in_batch_stride >= 0 &&
                                  out_batch_stride >= (int64_t)(rows - 1) * out_row_stride + (int64_t)cols),
                   "a matrix stride is smaller than the matrix");
    TATARA_REQUIRE_ALIGNED(in, elem_bytes(dtype));
    TATARA_REQUIRE_ALIGNED(out, elem_bytes(dtype));
    TATARA_REQUIRE(workspace && workspace_bytes >= Layout(batch, rows, cols).bytes, "workspace too small");
    TATARA_REQUIRE_ALIGNED(workspace, 16);
    if (int32_t st = check_stream(stream)) return st;
    const Source s{in, nullptr, in_row_stride, in_batch_stride, rows, cols, 0.0f, 0.0f, 0};
    const Target t{out, out_row_stride, out_batch_stride, nullptr, 0.0f, 0.0f, 0.0f, 0.0f};
    TATARA_FOR_DTYPE(dtype, return launch_steps<T>(s, t, batch, steps, workspace, raw(stream)));
}

int32_t tatara_op_muon_step(float* weights, float* momentum, const void* grad, uint32_t batch, uint32_t rows,
                            uint32_t cols, int32_t grad_dtype, double beta, int32_t nesterov, float lr, float decay,
                            float scale, float min_w, float max_w, uint32_t steps, void* workspace,
                            uint64_t workspace_bytes, TataraStream* stream) {
    if (int32_t st = check_matrices(batch, rows, cols, grad_dtype)) return st;
    TATARA_REQUIRE(steps >= 1 && steps <= 32, "steps must be 1 to 32");
    TATARA_REQUIRE(beta >= 0.0 && beta < 1.0, "beta must be in [0, 1)");
    TATARA_REQUIRE(min_w <= max_w, "min_w must not exceed max_w");
    if (batch == 0) return kOk;
    TATARA_REQUIRE(weights && momentum && grad, "null tensor");
    TATARA_REQUIRE_ALIGNED(weights, 4);
    TATARA_REQUIRE_ALIGNED(momentum, 4);
    TATARA_REQUIRE_ALIGNED(grad, elem_bytes(grad_dtype));
    TATARA_REQUIRE(workspace && workspace_bytes >= Layout(batch, rows, cols).bytes, "workspace too small");
    TATARA_REQUIRE_ALIGNED(workspace, 16);
    if (int32_t st = check_stream(stream)) return st;
    const Source s{grad, momentum, (int64_t)cols, (int64_t)rows * cols, rows, cols, (float)beta,
                   (float)(1.0 - beta), nesterov};
    const Target t{nullptr, 0, 0, weights, (float)(1.0 - (double)lr * decay), lr * scale, min_w, max_w};
    TATARA_FOR_DTYPE(grad_dtype, return launch_steps<T>(s, t, batch, steps, workspace, raw(stream)));
}

}  // extern "C"
