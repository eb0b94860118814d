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
constexpr uint32_t kGateBlocks = 256;  // workgroups, each of which leaves a partial sum (512 are no faster)
constexpr int kThreads = 256;
constexpr uint32_t kArrivals = 16;
constexpr uint32_t kZeroed = 4096;  // bytes of the workspace that begin as zero

// Partial sums of a workgroup: of every bucket the probability (low half) and the
// count, then the positions that count.
struct Workspace {
    // Counts of workgroups that have left their sums, zero between calls, a cache
    // line each: of every kArrivals-th workgroup, then of those groups that are
    // full.  (65536 x 9 with all of 512 workgroups on one count: 15 us, so 10.)
    uint32_t arrived[kArrivals + 1][32];
    uint32_t unused[kZeroed / 4 - (kArrivals + 1) * 32];
    uint64_t partial[];
};
static_assert(sizeof(Workspace) == kZeroed, "what the caller clears");

// Whether this is the last of the launch's workgroups to ask; the counts are zero
// again when it is.
__device__ __forceinline__ bool arrives_last(Workspace* ws) {
    auto count = [&](uint32_t i, uint32_t members) {
        const uint32_t n = __hip_atomic_fetch_add(&ws->arrived[i][0], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (n + 1 != members) return false;
        __hip_atomic_store(&ws->arrived[i][0], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return true;
    };
    const uint32_t i = blockIdx.x % kArrivals;
    return count(i, (gridDim.x - i + kArrivals - 1) / kArrivals) && count(kArrivals, min(gridDim.x, kArrivals));
}

__device__ __forceinline__ void put_partial(Workspace* ws, uint32_t block, uint32_t e, uint32_t buckets, float prob,
                                            int32_t count) {
    __hip_atomic_store(&ws->partial[(uint64_t)block * (buckets + 1) + e],
                       (uint64_t)(uint32_t)count << 32 | __float_as_uint(prob), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t get_partial(Workspace* ws, uint32_t block, uint32_t e, uint32_t buckets) {
    return __hip_atomic_load(&ws->partial[(uint64_t)block * (buckets + 1) + e], __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
}

// Orders floats as unsigned integers: NaN above +infinity, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kMaskedKey = 0x007fffffu;  // of -infinity; every smaller key stands for "none"

// The largest of the group's lanes.
template <int G>
__device__ __forceinline__ uint64_t group_best(uint64_t x) {
    auto step = [&](auto s) {
        constexpr int S = decltype(s)::value;
        if constexpr (G >> S > 1) {
            const uint64_t other = (uint64_t)partner<S>((uint32_t)(x >> 32)) << 32 | partner<S>((uint32_t)x);
            x = other > x ? other : x;
        }
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    step(std::integral_constant<int, 2>{});
    step(std::integral_constant<int, 3>{});
    step(std::integral_constant<int, 4>{});
    step(std::integral_constant<int, 5>{});
    return x;
}

// A position's logits, V consecutive buckets a lane and G lanes a position.
template <typename T, int V, int G>
struct Row {
    static constexpr int PV = Piece<T>::V;
    Piece<T> raw[V / PV];
    float p[V];       // probabilities
    uint32_t key[V];  // of the logits; 0 past the last bucket
    bool counts;

    // Loads in no branch, which would be waited for there.
    __device__ __forceinline__ void load(const T* row, uint32_t buckets, uint32_t first) {
        if (buckets >= PV) {
#pragma unroll
            for (int i = 0; i < V / PV; ++i) raw[i].load(row, first + i * PV, buckets);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const T v = row[first + j < buckets ? first + j : 0];
                raw[j / PV].v[j % PV] = v;
            }
        }
    }
    __device__ __forceinline__ void softmax(uint32_t buckets, uint32_t first, bool use) {
        const int left = (int)buckets - (int)first;
        if (buckets >= PV) {
#pragma unroll
            for (int i = 0; i < V / PV; ++i) raw[i].fix(left - i * PV);
        }
        float m = -INFINITY, any = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float x = j < left ? (float)raw[j / PV].v[j % PV] : -INFINITY;
            p[j] = x;
            key[j] = j < left ? order_key(x) : 0u;
            m = fmaxf(m, x);
            any = key[j] > kMaskedKey ? 1.0f : any;
        }
        // fmaxf passes over a NaN, which reaches the sum through its own exponential
        const float top = group_max<G>(m);
        counts = use && group_max<G>(any) > 0.0f;
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            p[j] = counts ? expf(p[j] - top) : 0.0f;
            s += p[j];
        }
        const float inv = counts ? 1.0f / group_sum<G>(s) : 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) p[j] *= inv;
    }
};

// By the workgroup's first wave.
__device__ __forceinline__ void write_totals(const float* prob, const int32_t* count, int32_t counted,
                                             uint32_t buckets, float scale, float* prob_out, int32_t* count_out,
                                             int32_t* counted_out, float* loss) {
    float s = 0.0f;
    for (uint32_t e = threadIdx.x; e < buckets; e += kWave) {
        prob_out[e] = prob[e];
        count_out[e] = count[e];
        s = fmaf((float)count[e], prob[e], s);
    }
    s = wave_sum(s);
    if (threadIdx.x == 0) {
        *counted_out = counted;
        const float n = (float)max(counted, 1);
        *loss = scale * s / n / n;
    }
}

// One launch: a lane holds eight buckets of a position, so that most positions need
// one to eight lanes and few joins.  Bound by latency, not bytes (65536 x 9 f32, 2.9
// MB: 8.7 us a call, 9.3 the kernel under a profiler): a load, the softmax and the
// choice, then the partial sums' way past the L2 and back.  As two launches it took
// 11.4 us.  With many buckets the choice and the join, four buckets a round, are most
// of it: 65536 x 64 32 us, 65536 x 256 117, 16384 x 1024 with two choices 321, where the
// backward pass, which has neither, takes 14, 40 and 70 for twice the bytes.
// scale = balance E / k.  K: at least top_k, for registers without an index.
template <typename T, int V, int G, int K>
__global__ __launch_bounds__(kThreads) void gate_forward_kernel(
    const T* __restrict__ logits, int64_t stride, const uint8_t* __restrict__ valid, uint64_t positions,
    uint32_t buckets, uint32_t top_k, int32_t renormalise, int32_t* __restrict__ bucket, float* __restrict__ gate,
    Workspace* __restrict__ ws, float scale, float* __restrict__ prob_out, int32_t* __restrict__ count_out,
    int32_t* __restrict__ counted_out, float* __restrict__ loss) {
    constexpr int E = V * G, WAVES = kThreads / kWave;
    __shared__ float sum_p[WAVES][E];
    __shared__ int32_t sum_c[WAVES][E];
    __shared__ int32_t sum_n[WAVES];
    __shared__ bool last;
    const uint32_t lane = threadIdx.x % G, first = lane * V;
    float acc_p[V];
    int32_t acc_c[V], acc_n = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) acc_p[j] = 0.0f, acc_c[j] = 0;
    const uint64_t step = (uint64_t)gridDim.x * (kThreads / G);
    const uint64_t rounds = (positions + step - 1) / step;
    for (uint64_t i = 0; i < rounds; ++i) {  // the same for every lane: the sums below need them all
        const uint64_t t = i * step + (uint64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
        const bool in = t < positions;
        Row<T, V, G> row;
        row.load(logits + (int64_t)(in ? t : 0) * stride, buckets, first);
        const uint8_t ok = valid ? valid[in ? t : 0] : 1;
        row.softmax(buckets, first, in && ok != 0);
#pragma unroll
        for (int j = 0; j < V; ++j) acc_p[j] += row.p[j];
        acc_n += row.counts && lane == 0;
        float mine[K], chosen = 0.0f;
        int32_t at[K];
#pragma unroll
        for (int r = 0; r < K; ++r) {
            mine[r] = 0.0f;
            at[r] = -1;
            if (K > 1 && r >= (int)top_k) continue;
            // the largest key, and of equal ones the lowest bucket
            uint64_t best = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const uint64_t k = ((uint64_t)row.key[j] << 32) | (0xffffffffu - (first + j));
                best = k > best ? k : best;
            }
            best = group_best<G>(best);
            const bool taken = row.counts && (uint32_t)(best >> 32) > kMaskedKey;
            const uint32_t e = 0xffffffffu - (uint32_t)best;
            float p = 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const bool here = taken && e == first + j;
                p += here ? row.p[j] : 0.0f;
                acc_c[j] += here;
                row.key[j] = here ? 0u : row.key[j];
            }
            mine[r] = group_sum<G>(p);
            chosen += mine[r];
            at[r] = taken ? (int32_t)e : -1;
        }
        if (in && lane == 0) {
#pragma unroll
            for (int r = 0; r < K; ++r) {
                if (K > 1 && r >= (int)top_k) break;
                bucket[t * top_k + r] = at[r];
                gate[t * top_k + r] = at[r] < 0 ? 0.0f : renormalise ? mine[r] / chosen : mine[r];
            }
        }
    }
    // over the positions of the wave, then of the workgroup
    auto add = [](auto x, auto y) { return x + y; };
#pragma unroll
    for (int j = 0; j < V; ++j) {
        acc_p[j] = column_join<G>(acc_p[j], add);
        acc_c[j] = column_join<G>(acc_c[j], add);
    }
    acc_n = column_join<G>(acc_n, add);
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
    if (buckets > kWave) __syncthreads();  // else one wave has them all
    int32_t n = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) n += sum_n[w];
    if (gridDim.x > 1) {
        // The last workgroup to get here joins all partial sums, in their order.
        // They are atomic stores of agent scope, which gfx950 writes through the XCD's
        // L2 (sc1) and whose vmcnt falls when they have arrived; each wave waits for
        // its own ahead of the barrier, and a thread behind it counts the workgroup.
        // The last one reads them by atomic loads of that scope, past its L2.  That is
        // the sequence that a release and an acquire of agent scope become on this chip
        // less the write-back and invalidation of the whole L2, which they need for
        // plain stores alone (65536 x 9 with them: 12.2 us instead of 8.7).
        for (uint32_t e = threadIdx.x; e <= buckets; e += kThreads)
            put_partial(ws, blockIdx.x, e, buckets, e < buckets ? sum_p[0][e] : 0.0f, e < buckets ? sum_c[0][e] : n);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) last = arrives_last(ws);
        __syncthreads();
        if (!last) return;
        // a wave a bucket, lane by lane over the workgroups
        const uint32_t l = threadIdx.x % kWave;
        for (uint32_t e = wave; e <= buckets; e += WAVES) {
            float p[kGateBlocks / kWave];
            int32_t c[kGateBlocks / kWave];
#pragma unroll
            for (int k = 0; k < (int)(kGateBlocks / kWave); ++k) {
                const uint32_t b = k * kWave + l;
                const uint64_t v = get_partial(ws, b < gridDim.x ? b : 0, e, buckets);
                p[k] = b < gridDim.x ? __uint_as_float((uint32_t)v) : 0.0f;
                c[k] = b < gridDim.x ? (int32_t)(v >> 32) : 0;
            }
#pragma unroll
            for (int k = 1; k < (int)(kGateBlocks / kWave); ++k) p[0] += p[k], c[0] += c[k];
            p[0] = column_join<1>(p[0], add);
            c[0] = column_join<1>(c[0], add);
            if (l == 0) {
                if (e < buckets)
                    sum_p[0][e] = p[0], sum_c[0][e] = c[0];
                else
                    sum_n[0] = c[0];
            }
        }
        __syncthreads();
        n = sum_n[0];
    }
    if (wave == 0)
        write_totals(sum_p[0], sum_c[0], n, buckets, scale, prob_out, count_out, counted_out, loss);
}

// The softmax again from the logits, which costs less than to have kept it.  Bound by
// latency: 65536 x 9 f32 (5.2 MB) 5.5 us, 16381 x 64 bf16 with four choices 7.5; with
// many buckets by its loads and joins: 65536 x 64 f32 13.6 us (7 of bytes), 65536 x 256
// 40 (27), 16384 x 1024 with two choices 70 (27).
// scale = dloss balance E / k
template <typename T, int V, int G, int K>
__global__ __launch_bounds__(kThreads) void gate_backward_kernel(
    const T* __restrict__ logits, int64_t stride, const uint8_t* __restrict__ valid, uint64_t positions,
    uint32_t buckets, uint32_t top_k, int32_t renormalise, const int32_t* __restrict__ bucket,
    const float* __restrict__ dgate, const int32_t* __restrict__ count, const int32_t* __restrict__ counted,
    float scale, T* __restrict__ dlogits, int64_t dstride) {
    const uint32_t lane = threadIdx.x % G, first = lane * V;
    const uint64_t step = (uint64_t)gridDim.x * (kThreads / G);
    const uint64_t rounds = (positions + step - 1) / step;
    int32_t counts[V], n_counted = counted[0];
#pragma unroll
    for (int j = 0; j < V; ++j) counts[j] = count[first + j < buckets ? first + j : 0];
    for (uint64_t i = 0; i < rounds; ++i) {
        const uint64_t t = i * step + (uint64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
        const bool in = t < positions;
        const uint64_t at = in ? t : 0;
        Row<T, V, G> row;
        row.load(logits + (int64_t)at * stride, buckets, first);
        const uint8_t ok = valid ? valid[at] : 1;
        int32_t e[K];
        float d[K];
#pragma unroll
        for (int r = 0; r < K; ++r) {
            const uint64_t c = at * top_k + (r < (int)top_k ? r : 0);
            e[r] = dgate ? bucket[c] : -1;
            d[r] = dgate ? dgate[c] : 0.0f;
        }
        row.softmax(buckets, first, in && ok != 0);
#pragma unroll
        for (int r = 0; r < K; ++r) {
            if (r >= (int)top_k || !row.counts) e[r] = -1;
            d[r] = e[r] >= 0 ? d[r] : 0.0f;
        }
        float total = 1.0f, along = 0.0f;
        if (renormalise) {
            float s = 0.0f, sd = 0.0f;
#pragma unroll
            for (int r = 0; r < K; ++r)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float p = e[r] == (int32_t)(first + j) ? row.p[j] : 0.0f;
                    s += p;
                    sd = fmaf(p, d[r], sd);
                }
            s = group_sum<G>(s);
            sd = group_sum<G>(sd);
            total = s == 0.0f ? 1.0f : s;
            along = sd / total;
        }
        const float n = (float)(n_counted > 0 ? n_counted : 1);
        float h[V], s = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            h[j] = first + j < buckets ? scale * (float)counts[j] / n / n : 0.0f;
#pragma unroll
            for (int r = 0; r < K; ++r) h[j] += e[r] == (int32_t)(first + j) ? (d[r] - along) / total : 0.0f;
            s = fmaf(row.p[j], h[j], s);
        }
        s = group_sum<G>(s);
        T* to = dlogits + (int64_t)at * dstride + first;
        const int left = in ? (int)buckets - (int)first : 0;
#pragma unroll
        for (int j0 = 0; j0 < V; j0 += Piece<T>::V) {
            Piece<T> out;
#pragma unroll
            for (int j = 0; j < Piece<T>::V; ++j)
                out.v[j] = (T)(row.counts ? row.p[j0 + j] * (h[j0 + j] - s) : 0.0f);  // 0 also where h is infinite
            out.store(to + j0, left - j0);
        }
    }
}

// Calls f with V, G and K: eight buckets a lane, sixteen from 513 on.
template <typename F>
void with_lanes(uint32_t buckets, uint32_t top_k, F&& f) {
    using std::integral_constant;
    auto with_top = [&](auto v, auto g) {
        if (top_k == 1)
            f(v, g, integral_constant<int, 1>{});
        else if (top_k <= 4)
            f(v, g, integral_constant<int, 4>{});
        else
            f(v, g, integral_constant<int, 16>{});
    };
    const integral_constant<int, 8> v8;
    if (buckets <= 8)
        with_top(v8, integral_constant<int, 1>{});
    else if (buckets <= 16)
        with_top(v8, integral_constant<int, 2>{});
    else if (buckets <= 32)
        with_top(v8, integral_constant<int, 4>{});
    else if (buckets <= 64)
        with_top(v8, integral_constant<int, 8>{});
    else if (buckets <= 128)
        with_top(v8, integral_constant<int, 16>{});
    else if (buckets <= 256)
        with_top(v8, integral_constant<int, 32>{});
    else if (buckets <= 512)
        with_top(v8, integral_constant<int, 64>{});
    else
        with_top(integral_constant<int, 16>{}, integral_constant<int, 64>{});
}

uint64_t gate_bytes(uint32_t buckets) {
    return sizeof(Workspace) + sizeof(uint64_t) * (uint64_t)kGateBlocks * (buckets + 1);
}

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
    TATARA_FOR_DTYPE(dtype, {
        with_lanes(buckets, top_k, [&](auto v, auto g, auto k) {
            constexpr int V = decltype(v)::value;
            constexpr int G = decltype(g)::value;
            const uint32_t blocks =
                std::max(1u, (uint32_t)std::min<uint64_t>(ceil_div(positions, kThreads / G), kGateBlocks));
            gate_forward_kernel<T, V, G, decltype(k)::value><<<blocks, kThreads, 0, raw(stream)>>>(
                static_cast<const T*>(logits), stride, valid, positions, buckets, top_k, renormalise, bucket, gate,
                static_cast<Workspace*>(workspace), scale, prob_sum, count, counted, loss);
        });
    });
    TATARA_LAUNCHED("gate_forward");
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
        with_lanes(buckets, top_k, [&](auto v, auto g, auto k) {
            constexpr int V = decltype(v)::value;
            constexpr int G = decltype(g)::value;
            const uint32_t blocks = (uint32_t)std::min<uint64_t>(ceil_div(positions, kThreads / G), 2048);
            gate_backward_kernel<T, V, G, decltype(k)::value><<<blocks, kThreads, 0, raw(stream)>>>(
                static_cast<const T*>(logits), stride, valid, positions, buckets, top_k, renormalise, bucket, dgate,
                count, counted, scale, static_cast<T*>(dlogits), dlogits_stride);
        });
    });
    TATARA_LAUNCHED("gate_backward");
    return kOk;
}

}  // extern "C"
