// Orthogonalised updates (Muon): a batch of matrices U of one shape becomes
//
//   X_0 = U / (|U|_F + 1e-7),  A = X X^T,  B = b A + c A^2,  X <- a X + B X,
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
// 2.9 by the map above).  A product takes hi hi + hi lo + lo hi, three f16
// products at 16 times the f32 matrix rate each, and leaves out lo lo, 2^-22 of
// the result.  Errors against 64-bit steps are those of f32 products (1e-6 to
// 1e-5 of |X|, from the sums' rounding).
#include "elem.hpp"

namespace tatara {
namespace {

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr double kNormEps = 1e-7;
constexpr float kHeld = 16384.0f;             // a held value's factor
constexpr float kUnheld = 1.0f / 16384.0f;
constexpr float kProduct = 1.0f / (16384.0f * 16384.0f);
constexpr uint32_t kPad = 64;                 // sides of the held matrices are multiples of it
constexpr uint32_t kNormParts = 128;          // partial sums of a matrix's norm
constexpr uint32_t kMaxSide = 32768;

using half8 = f16_t __attribute__((ext_vector_type(8)));
using half4 = f16_t __attribute__((ext_vector_type(4)));
using floatx16 = float __attribute__((ext_vector_type(16)));

// A matrix held as two f16 planes.
struct Held {
    f16_t* hi;
    f16_t* lo;
};

__device__ __forceinline__ void split(float v, f16_t& hi, f16_t& lo) {
    const float s = v * kHeld;
    hi = (f16_t)s;
    lo = (f16_t)(s - (float)hi);
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

template <typename T>
__device__ __forceinline__ float source_value(const Source& s, uint64_t at, float g) {
    if (!s.momentum) return g;
    const float m = s.momentum[at];
    return s.nesterov ? s.mix * g + s.beta * m : m;
}

// Adds the gradient to the momentum and leaves partial sums of |U|^2.  Squares
// are summed in 64 bits: no gradient's size overflows or vanishes.
template <typename T>
__global__ __launch_bounds__(256) void muon_moment_kernel(Source s, double* __restrict__ parts) {
    __shared__ double join[256 / kWave];
    const uint32_t b = blockIdx.y;
    const T* g = static_cast<const T*>(s.grad) + (int64_t)b * s.batch_stride;
    const uint64_t n = (uint64_t)s.rows * s.cols;
    double sum = 0.0;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) {
        const uint64_t r = i / s.cols;
        const float gv = (float)g[(int64_t)r * s.row_stride + (int64_t)(i - r * s.cols)];
        if (s.momentum) {
            const uint64_t at = b * n + i;
            s.momentum[at] = s.beta * s.momentum[at] + s.mix * gv;
        }
        const double u = (double)source_value<T>(s, b * n + i, gv);
        sum += u * u;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (threadIdx.x % kWave == 0) join[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) parts[(uint64_t)b * kNormParts + blockIdx.x] = join[0] + join[1] + join[2] + join[3];
}

// Writes X_0 as U lies (straight, [rows up][cols up]) and transposed.
template <typename T>
__global__ __launch_bounds__(256) void muon_split_kernel(Source s, const double* __restrict__ parts, uint32_t n_parts,
                                                         Held straight, Held turned, uint32_t rows_up,
                                                         uint32_t cols_up) {
    __shared__ float tile[64][65];
    const uint32_t b = blockIdx.z, r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
    double sum = 0.0;
    for (uint32_t i = 0; i < n_parts; ++i) sum += parts[(uint64_t)b * kNormParts + i];
    const double inv = 1.0 / (sqrt(sum) + kNormEps);
    const T* g = static_cast<const T*>(s.grad) + (int64_t)b * s.batch_stride;
    const uint64_t n = (uint64_t)s.rows * s.cols, plane = (uint64_t)b * rows_up * cols_up;
    const uint32_t c = threadIdx.x % 64, q = threadIdx.x / 64;
    for (uint32_t r = q; r < 64; r += 4) {
        float v = 0.0f;
        if (r0 + r < s.rows && c0 + c < s.cols) {
            const float gv = (float)g[(int64_t)(r0 + r) * s.row_stride + c0 + c];
            v = (float)((double)source_value<T>(s, b * n + (uint64_t)(r0 + r) * s.cols + c0 + c, gv) * inv);
        }
        tile[r][c] = v;
        const uint64_t at = plane + (uint64_t)(r0 + r) * cols_up + c0 + c;
        split(v, straight.hi[at], straight.lo[at]);
    }
    __syncthreads();
    for (uint32_t r = q; r < 64; r += 4) {
        const uint64_t at = plane + (uint64_t)(c0 + r) * rows_up + r0 + c;
        split(tile[c][r], turned.hi[at], turned.lo[at]);
    }
}

// What becomes of a product's tile.
enum Epilogue { kGram, kPoly, kApply, kOut, kUpdate };

struct ProductArgs {
    Held p, q;           // [m][k] and [n][k]: the product is p q^T
    uint32_t m, n, k;    // multiples of kPad
    Held old;            // kPoly: A; kApply and later: X transposed, before the step
    Held to, turned;     // results as they lie and (kApply) transposed
    // kOut, kUpdate: the caller's matrices, [rows][cols]; flipped: X is their transpose
    void* out;
    int64_t out_row_stride, out_batch_stride;
    uint32_t rows, cols;
    int32_t flipped;
    float* weights;
    float keep, rate, min_w, max_w;  // w = clamp(keep w - rate X)
};

// 128 x 128 of p q^T: four waves of 64 x 64, 32 values of k a stage.
template <int EPI, typename T>
__global__ __launch_bounds__(256) void muon_product_kernel(ProductArgs a) {
    constexpr uint32_t TILE = 128, KS = 32, CH = KS / 8;  // 16-byte pieces of a row's stage
    __shared__ half8 lds[2][4][TILE * CH];                // [buffer][p hi, p lo, q hi, q lo][row, piece]
    const uint32_t b = blockIdx.z;
    uint32_t ti, tj;
    if (EPI == kGram || EPI == kPoly) {  // the result is symmetric: tiles on and right of the diagonal
        const uint32_t nt = (a.n + TILE - 1) / TILE;
        uint32_t left = blockIdx.x;
        ti = 0;
        while (left >= nt - ti) left -= nt - ti, ++ti;
        tj = ti + left;
    } else {
        const uint32_t nt = (a.n + TILE - 1) / TILE;
        ti = blockIdx.x / nt;
        tj = blockIdx.x % nt;
    }
    const uint32_t i0 = ti * TILE, j0 = tj * TILE;
    const uint64_t p_at = (uint64_t)b * a.m * a.k, q_at = (uint64_t)b * a.n * a.k;
    const uint32_t tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const uint32_t wi = wave / 2 * 64, wj = wave % 2 * 64;
    floatx16 acc[2][2] = {};
    half8 next[8];
    auto fetch = [&](uint32_t k0) {
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const uint32_t e = (s % 2) * 256 + tid, row = e / CH, piece = e % CH;
            const bool isq = s >= 4, islo = (s / 2) % 2;
            // rows past the matrix (its side is a multiple of 64, not of the tile) are not stored
            const uint32_t r = isq ? min(j0 + row, a.n - 1) : min(i0 + row, a.m - 1);
            const f16_t* base = isq ? (islo ? a.q.lo : a.q.hi) + q_at : (islo ? a.p.lo : a.p.hi) + p_at;
            next[s] = *reinterpret_cast<const half8*>(base + (uint64_t)r * a.k + k0 + piece * 8);
        }
    };
    // pieces of rows four apart share banks: the piece's place turns with the row
    auto place = [](uint32_t row, uint32_t piece) { return row * CH + (piece ^ ((row >> 2) & 3)); };
    auto put = [&](int buf) {
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const uint32_t e = (s % 2) * 256 + tid;
            lds[buf][s / 2][place(e / CH, e % CH)] = next[s];
        }
    };
    fetch(0);
    put(0);
    __syncthreads();
    int buf = 0;
    for (uint32_t k0 = 0; k0 < a.k; k0 += KS) {
        const bool more = k0 + KS < a.k;
        if (more) fetch(k0 + KS);
#pragma unroll
        for (uint32_t kk = 0; kk < KS / 16; ++kk) {
            half8 fp[2][2], fq[2][2];  // [hi, lo][block of 32]
#pragma unroll
            for (int pl = 0; pl < 2; ++pl)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const uint32_t piece = kk * 2 + lane / 32;
                    fp[pl][t] = lds[buf][pl][place(wi + t * 32 + lane % 32, piece)];
                    fq[pl][t] = lds[buf][2 + pl][place(wj + t * 32 + lane % 32, piece)];
                }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[1][x], fq[0][y], acc[x][y], 0, 0, 0);
                    acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[0][x], fq[1][y], acc[x][y], 0, 0, 0);
                    acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[0][x], fq[0][y], acc[x][y], 0, 0, 0);
                }
        }
        if (more) put(buf ^ 1);
        __syncthreads();
        buf ^= 1;
    }
    // a lane holds, for four groups of rows, four consecutive rows of one column
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const uint32_t i = i0 + wi + x * 32 + g * 8 + (lane / 32) * 4, j = j0 + wj + y * 32 + lane % 32;
                if (i >= a.m || j >= a.n) continue;
                float v[4];
                half4 hi, lo;
                // the same elements of the transposed matrix, four in a row
                const uint64_t across = (uint64_t)b * a.m * a.n + (uint64_t)j * a.m + i;
                if (EPI != kGram) {
                    hi = *reinterpret_cast<const half4*>(a.old.hi + across);
                    lo = *reinterpret_cast<const half4*>(a.old.lo + across);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float s = acc[x][y][g * 4 + r] * kProduct;
                    const float o = EPI == kGram ? 0.0f : ((float)hi[r] + (float)lo[r]) * kUnheld;
                    v[r] = EPI == kGram ? s : EPI == kPoly ? fmaf(kC, s, kB * o) : fmaf(kA, o, s);
                }
                if (EPI == kOut || EPI == kUpdate) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const uint32_t row = a.flipped ? j : i + r, col = a.flipped ? i + r : j;
                        if (row >= a.rows || col >= a.cols) continue;
                        if (EPI == kOut) {
                            static_cast<T*>(a.out)[(int64_t)b * a.out_batch_stride + (int64_t)row * a.out_row_stride +
                                                   col] = (T)v[r];
                        } else {
                            float* w = a.weights + ((uint64_t)b * a.rows + row) * a.cols + col;
                            const float u = fmaf(-a.rate, v[r], a.keep * *w);
                            *w = u < a.min_w ? a.min_w : (u > a.max_w ? a.max_w : u);
                        }
                    }
                    continue;
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    f16_t h, l;
                    split(v[r], h, l);
                    hi[r] = h;
                    lo[r] = l;
                    const uint64_t at = (uint64_t)b * a.m * a.n + (uint64_t)(i + r) * a.n + j;
                    a.to.hi[at] = h;
                    a.to.lo[at] = l;
                }
                if (EPI == kApply || ti != tj) {
                    const Held& t = EPI == kApply ? a.turned : a.to;
                    *reinterpret_cast<half4*>(t.hi + across) = hi;
                    *reinterpret_cast<half4*>(t.lo + across) = lo;
                }
            }
}

uint32_t up(uint32_t n) { return (n + kPad - 1) / kPad * kPad; }

// The workspace's parts, by their byte offsets.
struct Layout {
    uint64_t parts, x, xt[2], a, b, bytes;
    uint64_t side, full;  // elements of one plane of all A and of all X
    uint32_t m, n;
    Layout(uint32_t batch, uint32_t rows, uint32_t cols) {
        m = up(std::min(rows, cols));
        n = up(std::max(rows, cols));
        full = (uint64_t)batch * m * n;
        side = (uint64_t)batch * m * m;
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

Held held(void* ws, uint64_t offset, uint64_t plane) {
    f16_t* p = reinterpret_cast<f16_t*>(static_cast<uint8_t*>(ws) + offset);
    return {p, p + plane};
}

struct Target {
    void* out;
    int64_t row_stride, batch_stride;
    float* weights;
    float keep, rate, min_w, max_w;
};

template <typename T>
int32_t launch_steps(const Source& s, const Target& t, uint32_t batch, uint32_t steps, void* ws, hipStream_t stream) {
    const Layout l(batch, s.rows, s.cols);
    const bool flipped = s.rows > s.cols;
    double* parts = reinterpret_cast<double*>(static_cast<uint8_t*>(ws) + l.parts);
    const Held x = held(ws, l.x, l.full), ga = held(ws, l.a, l.side), gb = held(ws, l.b, l.side);
    const Held xt[2] = {held(ws, l.xt[0], l.full), held(ws, l.xt[1], l.full)};
    const uint32_t n_parts = std::min<uint32_t>(kNormParts, ceil_div((uint64_t)s.rows * s.cols, 2048));
    muon_moment_kernel<T><<<dim3(n_parts, batch), 256, 0, stream>>>(s, parts);
    TATARA_LAUNCHED("muon_moment");
    muon_split_kernel<T><<<dim3(up(s.cols) / 64, up(s.rows) / 64, batch), 256, 0, stream>>>(
        s, parts, n_parts, flipped ? xt[0] : x, flipped ? x : xt[0], up(s.rows), up(s.cols));
    TATARA_LAUNCHED("muon_split");
    const uint32_t tm = ceil_div(l.m, 128), tn = ceil_div(l.n, 128);
    for (uint32_t i = 0; i < steps; ++i) {
        ProductArgs p{};
        p.p = p.q = x;
        p.m = p.n = l.m;
        p.k = l.n;
        p.to = ga;
        muon_product_kernel<kGram, T><<<dim3(tm * (tm + 1) / 2, 1, batch), 256, 0, stream>>>(p);
        TATARA_LAUNCHED("muon_gram");
        p.p = p.q = p.old = ga;
        p.k = l.m;
        p.to = gb;
        muon_product_kernel<kPoly, T><<<dim3(tm * (tm + 1) / 2, 1, batch), 256, 0, stream>>>(p);
        TATARA_LAUNCHED("muon_poly");
        p.p = gb;
        p.q = p.old = xt[i % 2];
        p.n = l.n;
        p.to = x;
        p.turned = xt[(i + 1) % 2];
        p.out = t.out;
        p.out_row_stride = t.row_stride;
        p.out_batch_stride = t.batch_stride;
        p.rows = s.rows;
        p.cols = s.cols;
        p.flipped = flipped;
        p.weights = t.weights;
        p.keep = t.keep;
        p.rate = t.rate;
        p.min_w = t.min_w;
        p.max_w = t.max_w;
        const dim3 grid(tm * tn, 1, batch);
        if (i + 1 < steps)
            muon_product_kernel<kApply, T><<<grid, 256, 0, stream>>>(p);
        else if (t.weights)
            muon_product_kernel<kUpdate, T><<<grid, 256, 0, stream>>>(p);
        else
            muon_product_kernel<kOut, T><<<grid, 256, 0, stream>>>(p);
        TATARA_LAUNCHED("muon_apply");
    }
    return kOk;
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
