// The learned choice among a LayerStack's buckets: softmax over a position's
// logits, its k best buckets, how often each bucket is taken, and the loss that
// keeps the buckets balanced, with the gradient of both.
//
//   p_t = softmax(l_t),  S_t = the k largest logits (equal ones: lowest bucket first),
//   gate_tj = p_tS_tj  or, renormalised,  p_tS_tj / sum_j p_tS_tj,
//   count_e = #{(t, j): S_tj = e},  P_e = sum_t p_te,  N = positions that count,
//   loss = balance E / (k N^2) sum_e count_e P_e
//
// count is a step function of the logits, so the loss's gradient goes through P
// alone: with h_te = dL/dp_te,  dl_te = p_te (h_te - sum_j p_tj h_tj).
//
// A logit of -infinity masks the bucket for the position: p = 0, never chosen
// (bucket -1 and gate 0 where fewer than k are left).  A position with valid = 0
// or without an unmasked bucket does not count: p = 0, no choice, no gradient.
// NaN orders above every number.
//
// Sums over positions are f32 (counts: integers) in a fixed order, so results
// do not change from run to run.
#include "elem.hpp"

namespace tatara {
namespace {

constexpr uint32_t kMaxBuckets = 1024;
constexpr uint32_t kMaxTop = 16;
constexpr uint32_t kGateBlocks = 512;  // workgroups, each of which leaves a partial sum
constexpr int kThreads = 256;

// A partial sum's place: probability and count of every bucket, then the
// positions that count.
struct Partial {
    float prob;
    int32_t count;
};

// Orders floats as unsigned integers: NaN above +infinity, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kMaskedKey = 0x007fffffu;  // of -infinity; every smaller key stands for "none"

template <int G>
__device__ __forceinline__ float group_max(float x) {
#pragma unroll
    for (int o = 1; o < G; o <<= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
template <int G>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
    for (int o = 1; o < G; o <<= 1) x += __shfl_xor(x, o);
    return x;
}

// A position's logits, V consecutive buckets a lane and G lanes a position.
template <typename T, int V, int G>
struct Row {
    float p[V];       // logits, then probabilities
    uint32_t key[V];  // 0 past the last bucket
    float top, total;
    bool counts;

    __device__ __forceinline__ void load(const T* row, uint32_t buckets, uint32_t first, bool use) {
        T raw[V];
        const int left = use ? (int)buckets - (int)first : 0;
        if (left >= V) {
            __builtin_memcpy(raw, row + first, sizeof(T) * V);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) raw[j] = j < left ? row[first + j] : (T)0.0f;
        }
        bool any = false;
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float x = j < left ? (float)raw[j] : -INFINITY;
            p[j] = x;
            key[j] = j < left ? order_key(x) : 0u;
            m = fmaxf(m, x);
            any |= key[j] > kMaskedKey;
        }
        top = group_max<G>(m);
        // fmaxf passes over a NaN, which reaches the sum through its own exponential
        counts = group_max<G>(any ? 1.0f : 0.0f) > 0.0f;
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            p[j] = counts ? expf(p[j] - top) : 0.0f;
            s += p[j];
        }
        total = group_sum<G>(s);
#pragma unroll
        for (int j = 0; j < V; ++j) p[j] = counts ? p[j] / total : 0.0f;
    }
};

__device__ __forceinline__ void write_totals(const float* prob, const int32_t* count, int32_t counted,
                                             uint32_t buckets, float scale, float* prob_out, int32_t* count_out,
                                             int32_t* counted_out, float* loss, double* join) {
    double s = 0.0;
    for (uint32_t e = threadIdx.x; e < buckets; e += blockDim.x) {
        prob_out[e] = prob[e];
        count_out[e] = count[e];
        s += (double)count[e] * (double)prob[e];
    }
    join[threadIdx.x] = s;
    for (uint32_t o = blockDim.x / 2; o > 0; o >>= 1) {
        __syncthreads();
        if (threadIdx.x < o) join[threadIdx.x] += join[threadIdx.x + o];
    }
    if (threadIdx.x == 0) {
        *counted_out = counted;
        const double n = counted > 0 ? (double)counted : 1.0;
        *loss = (float)((double)scale * join[0] / (n * n));
    }
}

// scale = balance E / k
template <typename T, int V, int G>
__global__ __launch_bounds__(kThreads) void gate_forward_kernel(
    const T* __restrict__ logits, int64_t stride, const uint8_t* __restrict__ valid, uint64_t positions,
    uint32_t buckets, uint32_t top_k, int32_t renormalise, int32_t* __restrict__ bucket, float* __restrict__ gate,
    Partial* __restrict__ partial, float scale, float* __restrict__ prob_out, int32_t* __restrict__ count_out,
    int32_t* __restrict__ counted_out, float* __restrict__ loss) {
    constexpr int E = V * G, WAVES = kThreads / kWave;
    __shared__ float sum_p[WAVES][E];
    __shared__ int32_t sum_c[WAVES][E];
    __shared__ int32_t sum_n[WAVES];
    __shared__ double join[kThreads];
    const uint32_t lane = threadIdx.x % G, first = lane * V;
    float acc_p[V];
    int32_t acc_c[V], acc_n = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) acc_p[j] = 0.0f, acc_c[j] = 0;
    const uint64_t step = (uint64_t)gridDim.x * (kThreads / G);
    const uint64_t rounds = (positions + step - 1) / step;
    for (uint64_t i = 0; i < rounds; ++i) {  // the same for every lane: the sums below need them all
        const uint64_t t = i * step + (uint64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
        const bool use = t < positions && (!valid || valid[t < positions ? t : 0] != 0);
        Row<T, V, G> row;
        row.load(logits + (int64_t)(t < positions ? t : 0) * stride, buckets, first, use);
#pragma unroll
        for (int j = 0; j < V; ++j) acc_p[j] += row.p[j];
        acc_n += row.counts && lane == 0;
        float mine[kMaxTop], chosen = 0.0f;  // static indices: the rounds are unrolled
        int32_t at[kMaxTop];
#pragma unroll
        for (int r = 0; r < (int)kMaxTop; ++r) {
            mine[r] = 0.0f;
            at[r] = -1;
            if (r >= (int)top_k) continue;
            // the largest key, and of equal ones the lowest bucket
            uint64_t best = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const uint64_t k = ((uint64_t)row.key[j] << 32) | (0xffffffffu - (first + j));
                best = k > best ? k : best;
            }
#pragma unroll
            for (int o = 1; o < G; o <<= 1) {
                const uint64_t other = __shfl_xor((unsigned long long)best, o);
                best = other > best ? other : best;
            }
            const bool taken = row.counts && (uint32_t)(best >> 32) > kMaskedKey;
            const uint32_t e = 0xffffffffu - (uint32_t)best;
            float p = 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const bool here = taken && e == first + j;
                p += here ? row.p[j] : 0.0f;
                acc_c[j] += here;
                if (here) row.key[j] = 0u;
            }
            mine[r] = group_sum<G>(p);
            chosen += mine[r];
            if (taken) at[r] = (int32_t)e;
        }
        if (t < positions && lane == 0) {
#pragma unroll
            for (int r = 0; r < (int)kMaxTop; ++r) {
                if (r >= (int)top_k) break;
                bucket[t * top_k + r] = at[r];
                gate[t * top_k + r] = at[r] < 0 ? 0.0f : renormalise ? mine[r] / chosen : mine[r];
            }
        }
    }
    // over the positions of the wave, then of the workgroup
#pragma unroll
    for (int o = G; o < (int)kWave; o <<= 1) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            acc_p[j] += __shfl_xor(acc_p[j], o);
            acc_c[j] += __shfl_xor(acc_c[j], o);
        }
        acc_n += __shfl_xor(acc_n, o);
    }
    const uint32_t wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave < G) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            sum_p[wave][first + j] = acc_p[j];
            sum_c[wave][first + j] = acc_c[j];
        }
        if (lane == 0) sum_n[wave] = acc_n;
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < buckets; e += kThreads) {
#pragma unroll
        for (int w = 1; w < WAVES; ++w) {
            sum_p[0][e] += sum_p[w][e];
            sum_c[0][e] += sum_c[w][e];
        }
    }
    int32_t n = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) n += sum_n[w];
    if (gridDim.x > 1) {
        Partial* to = partial + (uint64_t)blockIdx.x * (buckets + 1);
        for (uint32_t e = threadIdx.x; e < buckets; e += kThreads) to[e] = {sum_p[0][e], sum_c[0][e]};
        if (threadIdx.x == 0) to[buckets] = {0.0f, n};
        return;
    }
    write_totals(sum_p[0], sum_c[0], n, buckets, scale, prob_out, count_out, counted_out, loss, join);
}

// Joins the workgroups' partial sums, in their order.
__global__ __launch_bounds__(1024) void gate_totals_kernel(const Partial* __restrict__ partial, uint32_t blocks,
                                                           uint32_t buckets, float scale,
                                                           float* __restrict__ prob_out,
                                                           int32_t* __restrict__ count_out,
                                                           int32_t* __restrict__ counted_out,
                                                           float* __restrict__ loss) {
    __shared__ float prob[kMaxBuckets + 1];
    __shared__ int32_t count[kMaxBuckets + 1];
    __shared__ double join[1024];
    const uint32_t lane = threadIdx.x % kWave;
    // a wave a bucket: lane by lane over the workgroups
    for (uint32_t e = threadIdx.x / kWave; e <= buckets; e += 1024 / kWave) {
        float p = 0.0f;
        int32_t c = 0;
        for (uint32_t b = lane; b < blocks; b += kWave) {
            const Partial v = partial[(uint64_t)b * (buckets + 1) + e];
            p += v.prob;
            c += v.count;
        }
        p = wave_sum(p);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o);
        if (lane == 0) prob[e] = p, count[e] = c;
    }
    __syncthreads();
    write_totals(prob, count, count[buckets], buckets, scale, prob_out, count_out, counted_out, loss, join);
}

// scale = dloss balance E / k
template <typename T, int V, int G>
__global__ __launch_bounds__(kThreads) void gate_backward_kernel(
    const T* __restrict__ logits, int64_t stride, const uint8_t* __restrict__ valid, uint64_t positions,
    uint32_t buckets, uint32_t top_k, int32_t renormalise, const int32_t* __restrict__ bucket,
    const float* __restrict__ dgate, const int32_t* __restrict__ count, const int32_t* __restrict__ counted,
    float scale, T* __restrict__ dlogits, int64_t dstride) {
    const uint32_t lane = threadIdx.x % G, first = lane * V;
    float base[V];
    {
        const float n = (float)(counted[0] > 0 ? counted[0] : 1);
#pragma unroll
        for (int j = 0; j < V; ++j) base[j] = first + j < buckets ? scale * (float)count[first + j] / n / n : 0.0f;
    }
    const uint64_t step = (uint64_t)gridDim.x * (kThreads / G);
    const uint64_t rounds = (positions + step - 1) / step;
    for (uint64_t i = 0; i < rounds; ++i) {
        const uint64_t t = i * step + (uint64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
        const bool in = t < positions;
        const bool use = in && (!valid || valid[t] != 0);
        Row<T, V, G> row;
        row.load(logits + (int64_t)(in ? t : 0) * stride, buckets, first, use);
        float h[V];
#pragma unroll
        for (int j = 0; j < V; ++j) h[j] = base[j];
        if (dgate) {
            float total = 1.0f, along = 0.0f;
            if (renormalise) {
                float s = 0.0f, sd = 0.0f;
                for (uint32_t r = 0; r < top_k; ++r) {
                    const int32_t e = use ? bucket[t * top_k + r] : -1;
                    const float d = e >= 0 ? dgate[t * top_k + r] : 0.0f;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float p = e == (int32_t)(first + j) ? row.p[j] : 0.0f;
                        s += p;
                        sd = fmaf(p, d, sd);
                    }
                }
                s = group_sum<G>(s);
                sd = group_sum<G>(sd);
                total = s == 0.0f ? 1.0f : s;
                along = sd / total;
            }
            for (uint32_t r = 0; r < top_k; ++r) {
                const int32_t e = use ? bucket[t * top_k + r] : -1;
                const float d = e >= 0 ? dgate[t * top_k + r] : 0.0f;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (e == (int32_t)(first + j)) h[j] += (d - along) / total;
            }
        }
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) s = fmaf(row.p[j], h[j], s);
        s = group_sum<G>(s);
        T out[V];
#pragma unroll
        for (int j = 0; j < V; ++j) out[j] = (T)(row.p[j] * (h[j] - s));
        const int left = in ? (int)buckets - (int)first : 0;
        T* to = dlogits + (int64_t)(in ? t : 0) * dstride + first;
        if (left >= V) {
            __builtin_memcpy(to, out, sizeof(T) * V);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < left) to[j] = out[j];
        }
    }
}

// Calls f with V and G: eight buckets a lane, sixteen from 513 on.
template <typename F>
void with_lanes(uint32_t buckets, F&& f) {
    using std::integral_constant;
    const integral_constant<int, 8> v8;
    if (buckets <= 8)
        f(v8, integral_constant<int, 1>{});
    else if (buckets <= 16)
        f(v8, integral_constant<int, 2>{});
    else if (buckets <= 32)
        f(v8, integral_constant<int, 4>{});
    else if (buckets <= 64)
        f(v8, integral_constant<int, 8>{});
    else if (buckets <= 128)
        f(v8, integral_constant<int, 16>{});
    else if (buckets <= 256)
        f(v8, integral_constant<int, 32>{});
    else if (buckets <= 512)
        f(v8, integral_constant<int, 64>{});
    else
        f(integral_constant<int, 16>{}, integral_constant<int, 64>{});
}

uint64_t gate_bytes(uint32_t buckets) { return sizeof(Partial) * (uint64_t)kGateBlocks * (buckets + 1); }

int32_t check_gate(uint64_t positions, uint32_t buckets, uint32_t top_k, int32_t dtype) {
    TATARA_REQUIRE_DTYPE(dtype);
    TATARA_REQUIRE(buckets >= 1 && buckets <= kMaxBuckets, "the gate takes 1 to 1024 buckets");
    TATARA_REQUIRE(top_k >= 1 && top_k <= kMaxTop && top_k <= buckets,
                   "top_k must be 1 to 16 and no more than the buckets");
    TATARA_REQUIRE(positions * top_k < (1ull << 31) && positions < (1ull << 31), "too many positions");
    return kOk;
}

}  // namespace
}  // namespace tatara

using namespace tatara;

extern "C" {

int32_t tatara_op_bucket_gate_workspace(uint32_t buckets, uint64_t* bytes) {
    TATARA_REQUIRE(bytes, "null output");
    TATARA_REQUIRE(buckets >= 1 && buckets <= kMaxBuckets, "the gate takes 1 to 1024 buckets");
    *bytes = gate_bytes(buckets);
    return kOk;
}

int32_t tatara_op_bucket_gate_forward(const void* logits, int64_t stride, const uint8_t* valid, uint64_t positions,
                                      uint32_t buckets, uint32_t top_k, int32_t renormalise, float balance,
                                      int32_t dtype, int32_t* bucket, float* gate, int32_t* count, float* prob_sum,
                                      int32_t* counted, float* loss, void* workspace, uint64_t workspace_bytes,
                                      TataraStream* stream) {
    if (int32_t st = check_gate(positions, buckets, top_k, dtype)) return st;
    TATARA_REQUIRE(count && prob_sum && counted && loss, "null output");
    TATARA_REQUIRE(!positions || (logits && bucket && gate), "null tensor");
    TATARA_REQUIRE(!positions || stride >= (int64_t)buckets, "the row stride is smaller than the row");
    TATARA_REQUIRE(workspace && workspace_bytes >= gate_bytes(buckets), "workspace too small");
    TATARA_REQUIRE_ALIGNED(logits, elem_bytes(dtype));
    TATARA_REQUIRE_ALIGNED(workspace, 16);
    if (int32_t st = check_stream(stream)) return st;
    const float scale = balance * (float)buckets / (float)top_k;
    Partial* partial = static_cast<Partial*>(workspace);
    uint32_t blocks = 1;
    TATARA_FOR_DTYPE(dtype, {
        with_lanes(buckets, [&](auto v, auto g) {
            constexpr int V = decltype(v)::value;
            constexpr int G = decltype(g)::value;
            blocks = std::max(1u, (uint32_t)std::min<uint64_t>(ceil_div(positions, kThreads / G), kGateBlocks));
            gate_forward_kernel<T, V, G><<<blocks, kThreads, 0, raw(stream)>>>(
                static_cast<const T*>(logits), stride, valid, positions, buckets, top_k, renormalise, bucket, gate,
                partial, scale, prob_sum, count, counted, loss);
        });
    });
    TATARA_LAUNCHED("gate_forward");
    if (blocks > 1) {
        gate_totals_kernel<<<1, 1024, 0, raw(stream)>>>(partial, blocks, buckets, scale, prob_sum, count, counted,
                                                        loss);
        TATARA_LAUNCHED("gate_totals");
    }
    return kOk;
}

int32_t tatara_op_bucket_gate_backward(const void* logits, int64_t stride, const uint8_t* valid, uint64_t positions,
                                       uint32_t buckets, uint32_t top_k, int32_t renormalise, float balance,
                                       int32_t dtype, const int32_t* bucket, const int32_t* count,
                                       const int32_t* counted, const float* dgate, float dloss, void* dlogits,
                                       int64_t dlogits_stride, TataraStream* stream) {
    if (int32_t st = check_gate(positions, buckets, top_k, dtype)) return st;
    if (positions == 0) return kOk;
    TATARA_REQUIRE(logits && bucket && count && counted && dlogits, "null tensor");
    TATARA_REQUIRE(stride >= (int64_t)buckets && dlogits_stride >= (int64_t)buckets,
                   "a row stride is smaller than the row");
    TATARA_REQUIRE_ALIGNED(logits, elem_bytes(dtype));
    TATARA_REQUIRE_ALIGNED(dlogits, elem_bytes(dtype));
    if (int32_t st = check_stream(stream)) return st;
    const float scale = dloss * balance * (float)buckets / (float)top_k;
    TATARA_FOR_DTYPE(dtype, {
        with_lanes(buckets, [&](auto v, auto g) {
            constexpr int V = decltype(v)::value;
            constexpr int G = decltype(g)::value;
            const uint32_t blocks = (uint32_t)std::min<uint64_t>(ceil_div(positions, kThreads / G), 2048);
            gate_backward_kernel<T, V, G><<<blocks, kThreads, 0, raw(stream)>>>(
                static_cast<const T*>(logits), stride, valid, positions, buckets, top_k, renormalise, bucket, dgate,
                count, counted, scale, static_cast<T*>(dlogits), dlogits_stride);
        });
    });
    TATARA_LAUNCHED("gate_backward");
    return kOk;
}

}  // extern "C"
