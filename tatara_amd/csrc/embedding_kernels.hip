// Rows of a table by a position's token, scaled, and the table's gradient.
//
//   y_i = scale table_{token_i},   dtable_v = scale sum over i with token_i = v of dy_i
//
// A token outside 0..V - 1 stands for none: its row is zeros, and it has no gradient.
//
// The gradient sorts the positions by token (a stable radix sort of up to three digits)
// and adds each token's rows in the positions' order, in f32: no atomics, and every row
// of dtable is written once.  The sorted positions are cut into chunks of equal length, so
// that a token that nearly all positions have is summed as fast as others.  A chunk's
// first and last token may reach into its neighbours: their sums go to `partial` and are
// joined in order by a last launch, a workgroup for 256 columns of a token, which is what one
// token that is in all chunks costs more.
//
// 65536 x 1536 f32 of 73305 rows, 453 MB of them zeros or sums: 217 us, of which the sums and
// zeros take 182 (853 MB, 4.7 TB/s, as a copy of that size), four launches of the sort 29 and the
// join 9.  With one token in all positions 251 us, the join 42 of them; of 1000 rows 141 instead of
// 112, of 2 rows 107 instead of 99 (floor 81).  1000 x 768 of 2000 rows: 16.5 us in three launches;
// up to 256 positions take one.
#include "key_sort.hpp"
#include "row_moves.hpp"

namespace tatara {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxVocab = 1u << 28;
// Rows of the table that a workgroup looks up at most, and clears where no position has one.
constexpr uint32_t kClearRows = 128;
constexpr int kBatch = 8;  // rows that a lane has in hand
// Waves that have a chunk each, at most (200000 x 256 f32 of 9 rows: with 1024 62 us, 2048 49, 4096
// 55), and chunks, of which wide rows take several waves each.
constexpr uint32_t kMostWaves = 2048, kMostChunks = 1024;
// Positions of a chunk at least; twice as many of narrow rows, whose waves have several chunks
// (65536 x 16 f32 of 81 rows: 25 us, so 19.4).
constexpr uint32_t kLeastChunk = 8;

// Positions that need no sort: a thread each where rows are cleared.
constexpr uint32_t kFewPositions = 256;
static_assert(kFewPositions <= kThreads && kClearRows <= kThreads, "one turn of a workgroup");

// A position and its token.
struct alignas(8) Place {
    uint32_t key, at;
};

// A pass of the radix sort.  The first one reads the tokens, of which those that stand
// for none become `vocab`, behind the others.
struct Digit {
    const int32_t* token;
    const Place* in;
    Place* out;
    uint32_t vocab, shift, mask;

    using Item = Place;
    __device__ __forceinline__ Item load(uint64_t i) const {
        if (token) return {min((uint32_t)token[i], vocab), (uint32_t)i};
        return in[i];
    }
    __device__ __forceinline__ uint32_t key(Item item) const { return item.key >> shift & mask; }
    __device__ __forceinline__ void put(uint64_t, Item item, uint32_t, uint32_t first, uint32_t rank) const {
        out[first + rank] = item;
    }
    __device__ __forceinline__ void drop(uint64_t) const {}
    __device__ __forceinline__ void finish(const uint32_t*, uint32_t) const {}
};

// The passes go from one list to the other.
__host__ __device__ __forceinline__ Digit digit_of(int pass, int bits, const int32_t* token, uint32_t vocab,
                                                   uint32_t mask, Place* even, Place* odd) {
    return {pass ? nullptr : token, pass % 2 ? even : odd, pass % 2 ? odd : even, vocab, (uint32_t)(pass * bits), mask};
}

// All passes, of positions that one workgroup sorts.
template <int BITS>
__global__ __launch_bounds__(kSortThreads) void embedding_sort_kernel(const int32_t* token, uint32_t n, uint32_t run,
                                                                      uint32_t vocab, int passes, int bits,
                                                                      uint32_t keys, uint32_t mask, Place* even,
                                                                      Place* odd) {
    extern __shared__ uint32_t shared[];
    for (int pass = 0; pass < passes; ++pass) {
        asm volatile("" : "+s"(n), "+s"(keys));  // else what no pass changes is kept in registers that there are not
        sort_place<BITS, true>(digit_of(pass, bits, token, vocab, mask, even, odd), n, run, keys, nullptr, shared);
        __syncthreads();  // this pass's places are written before the next one reads them
    }
}

struct Sorted {
    const Place* place;  // [n], by token
    uint32_t n, chunk, chunks;
    __device__ __forceinline__ uint32_t key(uint64_t i) const { return place[i].key; }
};

// Zeros in the rows that no position has.
__device__ __forceinline__ void clear_rows_of(const bool* none, uint32_t rows, float* table, uint32_t cols) {
    const uint32_t per_row = (cols + 3) / 4;
    Piece<float> zero;
#pragma unroll
    for (int e = 0; e < 4; ++e) zero.v[e] = 0.0f;
    if (per_row >= kWave) {  // a row a wave
        for (uint32_t r = threadIdx.x / kWave; r < rows; r += kThreads / kWave) {
            if (!none[r]) continue;
            float* to = table + (uint64_t)r * cols;
            for (uint32_t c = threadIdx.x % kWave * 4; c < cols; c += kWave * 4) zero.store(to + c, (int)(cols - c));
        }
    } else {
        for (uint32_t i = threadIdx.x; i < rows * per_row; i += kThreads) {
            const uint32_t r = i / per_row, c = (i - r * per_row) * 4;
            if (none[r]) zero.store(table + (uint64_t)r * cols + c, (int)(cols - c));
        }
    }
}

// A group of G lanes adds the rows of a chunk, V columns a lane; rows wider than a wave
// are cut into `slabs`.  `clear` workgroups write the rows of the table that no position
// has.
template <typename T, int G, bool FEW>
__global__ __launch_bounds__(kThreads) void embedding_sum_kernel(const T* __restrict__ dy, int64_t dy_stride, Sorted s,
                                                                 uint32_t vocab, uint32_t cols, float scale,
                                                                 float* __restrict__ dtable,
                                                                 float* __restrict__ partial, uint32_t clear,
                                                                 uint32_t clear_rows, uint32_t slabs) {
    constexpr int V = Piece<T>::V;
    // the workgroups that clear lie evenly among the others, which read where they write
    const uint32_t cleared = (uint32_t)((uint64_t)blockIdx.x * clear / gridDim.x);
    const bool clears = cleared != (uint32_t)((uint64_t)(blockIdx.x + 1) * clear / gridDim.x);
    if (clears) {
        __shared__ bool none[kClearRows];
        // eight lanes look for a row, for TURNS of them at once
        constexpr uint32_t LANES = 8, ROWS = kThreads / LANES, TURNS = kClearRows / ROWS;
        const uint32_t lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
        for (uint64_t first = (uint64_t)cleared * clear_rows; first < vocab; first += (uint64_t)clear * clear_rows) {
            __syncthreads();
            uint32_t lo[TURNS], hi[TURNS];  // the first place with a key of the row or above lies in lo..hi
#pragma unroll
            for (uint32_t q = 0; q < TURNS; ++q) lo[q] = 0, hi[q] = q * ROWS + group < clear_rows ? s.n : 0;
            for (bool more = true; more;) {
                uint32_t wide = 0;
#pragma unroll
                for (uint32_t q = 0; q < TURNS; ++q) {
                    // a lane looks at the last place of each of LANES parts
                    const uint32_t part = max((hi[q] - lo[q] + LANES - 1) / LANES, 1u);
                    const uint32_t mine = lo[q] + (lane + 1) * part - 1;
                    const uint64_t v = first + q * ROWS + group;
                    const uint64_t below = __ballot(mine < hi[q] && s.key(mine < hi[q] ? mine : 0) < v);
                    const uint32_t mask = (uint32_t)(below >> (threadIdx.x % kWave - lane)) & ((1u << LANES) - 1);
                    lo[q] += __popc(mask) * part;
                    hi[q] = min(hi[q], lo[q] + part - 1);
                    wide |= hi[q] - lo[q];
                }
                more = __ballot(wide) != 0;
            }
#pragma unroll
            for (uint32_t q = 0; q < TURNS; ++q) {
                const uint64_t v = first + q * ROWS + group;
                if (lane == 0) none[q * ROWS + group] = v < vocab && !(lo[q] < s.n && s.key(lo[q]) == v);
            }
            __syncthreads();
            clear_rows_of(none, clear_rows, dtable + first * cols, cols);
        }
        return;
    }
    uint32_t unit = (blockIdx.x - cleared) * (kThreads / G) + threadIdx.x / G;
    if (G == kWave) unit = __builtin_amdgcn_readfirstlane(unit);
    const uint32_t chunk = unit / slabs;
    if (chunk >= s.chunks) return;
    const int c = (int)((unit - chunk * slabs) * kWave + threadIdx.x % G) * V, left = (int)cols - c;
    if (left <= 0) return;
    const uint32_t begin = chunk * s.chunk, end = min(begin + s.chunk, s.n);
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.0f;
    // whether the token's first row lies in the chunk
    bool began = begin == 0 || s.key(begin - 1) != s.key(begin);
    bool open = false;
    auto flush = [&](float* to, float by) {
#pragma unroll
        for (int h = 0; h < V / 4; ++h) {
            Piece<float> out;
#pragma unroll
            for (int e = 0; e < 4; ++e) out.v[e] = acc[4 * h + e] * by;
            out.store(to + c + 4 * h, left - 4 * h);
        }
    };
    for (uint32_t i0 = begin; i0 < end; i0 += kBatch) {
        uint32_t key[kBatch + 1], at[kBatch];
#pragma unroll
        for (int j = 0; j <= kBatch; ++j) {
            const Place place = s.place[min(i0 + j, s.n - 1)];
            key[j] = place.key;
            if (j < kBatch) at[j] = place.at;
        }
        Piece<T> p[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (FEW)
                p[j].load_few(dy + (int64_t)at[j] * dy_stride, (int)cols);
            else
                p[j].load(dy + (int64_t)at[j] * dy_stride, c, (int)cols);
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (i0 + j >= end || key[j] >= vocab) break;
            if (!FEW) p[j].fix(left);
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] += (float)p[j].v[e];
            open = i0 + j + 1 < s.n && key[j + 1] == key[j];
            if (!open) {
                if (began)
                    flush(dtable + (uint64_t)key[j] * cols, scale);
                else
                    flush(partial + (uint64_t)chunk * 2 * cols, 1.0f);
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] = 0.0f;
                began = true;
            }
        }
    }
    if (open) flush(partial + ((uint64_t)chunk * 2 + began) * cols, 1.0f);
}

// The rows of tokens that reach over several chunks, of 256 columns.  A wave looks at a
// chunk: where a token begins in it and goes on, it adds the sums of the chunks that the
// token is in, and if they are many the workgroup's waves take a part of them each.
template <int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void embedding_join_kernel(Sorted s, uint32_t vocab, uint32_t cols,
                                                                       float scale, const float* __restrict__ partial,
                                                                       float* __restrict__ dtable, uint32_t slabs) {
    constexpr uint32_t FEW = 16;
    __shared__ float join[WAVES - 1][kWave * 4];
    __shared__ uint32_t many[WAVES];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const uint32_t chunk0 = blockIdx.x / slabs * WAVES;
    const int c = (int)((blockIdx.x % slabs) * kWave + lane) * 4, left = (int)cols - c;
    // the chunks that the token is in which begins in this one, 0 if it ends there
    auto chain = [&](uint32_t chunk) {
        const uint64_t begin = (uint64_t)chunk * s.chunk, next = begin + s.chunk;
        if (next >= s.n) return 0u;
        const uint32_t key = s.key(next);
        if (key >= vocab || s.key(next - 1) != key || (begin > 0 && s.key(begin - 1) == key)) return 0u;
        uint32_t more = 0, got;
        do {
            const uint64_t place = next + (uint64_t)(more + lane) * s.chunk;
            got = (uint32_t)__popcll(__ballot(place < s.n && s.key(place < s.n ? place : 0) == key));
            more += got;
        } while (got == kWave);
        return more + 1;
    };
    float acc[4];
    auto add = [&](uint32_t chunk, uint32_t from, uint32_t to) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = 0.0f;
#pragma unroll 8
        for (uint32_t t = from; t < to; ++t) {
            const float* row = partial + ((uint64_t)(chunk + t) * 2 + (t == 0)) * cols;
            Piece<float> p;
            if (cols < 4) {
                p.load_few(row, left);
            } else {
                p.load(row, min(c, (int)cols), (int)cols);
                p.fix(left);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += p.v[e];
        }
    };
    auto write = [&](uint32_t chunk) {
        if (left <= 0) return;
        Piece<float> out;
#pragma unroll
        for (int e = 0; e < 4; ++e) out.v[e] = acc[e] * scale;
        out.store(dtable + (uint64_t)s.key((uint64_t)(chunk + 1) * s.chunk) * cols + c, left);
    };
    const uint32_t mine = chain(chunk0 + wave);
    if (mine && mine <= FEW) {
        add(chunk0 + wave, 0, mine);
        write(chunk0 + wave);
    }
    if (lane == 0) many[wave] = mine > FEW ? mine : 0;
    __syncthreads();
    for (uint32_t w = 0; w < WAVES; ++w) {
        const uint32_t terms = many[w];
        if (!terms) continue;
        add(chunk0 + w, (uint32_t)((uint64_t)terms * wave / WAVES), (uint32_t)((uint64_t)terms * (wave + 1) / WAVES));
        if (wave) {
#pragma unroll
            for (int e = 0; e < 4; ++e) join[wave - 1][lane * 4 + e] = acc[e];
        }
        __syncthreads();
        if (!wave) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int o = 0; o < WAVES - 1; ++o) acc[e] += join[o][lane * 4 + e];
            write(chunk0 + w);
        }
        __syncthreads();
    }
}

// The whole gradient of few positions in one launch, without a sort: a wave a position and
// 64 V columns adds the rows of all positions with its token if none ahead of it has that token.
// (64 x 256 f32 of 1000 rows 2.5 us, by sort, sum and join 11.6; 256 x 1536 of 2 rows, 128
// positions each, 11.0 and 12.)
template <typename T, bool FEW>
__global__ __launch_bounds__(kThreads) void embedding_few_kernel(const T* __restrict__ dy, int64_t dy_stride,
                                                                 const int32_t* __restrict__ token, uint32_t n,
                                                                 uint32_t vocab, uint32_t cols, float scale,
                                                                 float* __restrict__ dtable, uint32_t clear,
                                                                 uint32_t clear_rows, uint32_t slabs) {
    constexpr int V = Piece<T>::V;
    if (blockIdx.x < clear) {
        __shared__ bool none[kClearRows];
        for (uint64_t first = (uint64_t)blockIdx.x * clear_rows; first < vocab; first += (uint64_t)clear * clear_rows) {
            __syncthreads();
            if (threadIdx.x < clear_rows) none[threadIdx.x] = first + threadIdx.x < vocab;
            __syncthreads();
            if (threadIdx.x < n) {
                const uint64_t row = (uint64_t)(uint32_t)token[threadIdx.x] - first;  // wraps below it
                if (row < clear_rows) none[row] = false;
            }
            __syncthreads();
            clear_rows_of(none, clear_rows, dtable + first * cols, cols);
        }
        return;
    }
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t unit = (blockIdx.x - clear) * (kThreads / kWave) + wave;
    const uint32_t i = unit / slabs, lane = threadIdx.x % kWave;
    if (i >= n) return;
    const uint32_t key = (uint32_t)token[i];
    uint64_t same[kFewPositions / kWave];
#pragma unroll
    for (uint32_t k = 0; k < kFewPositions / kWave; ++k) {
        const uint32_t j = k * kWave + lane;
        same[k] = __ballot(j < n && (uint32_t)token[j < n ? j : 0] == key);
    }
    if (key >= vocab) return;
#pragma unroll
    for (uint32_t k = 0; k < kFewPositions / kWave; ++k) {
        const uint64_t ahead = i >= (k + 1) * kWave ? ~0ull : i > k * kWave ? (1ull << (i - k * kWave)) - 1 : 0;
        if (same[k] & ahead) return;
    }
    const int c = (int)((unit - i * slabs) * kWave + lane) * V, left = (int)cols - c;
    if (left <= 0) return;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.0f;
    auto add = [&](auto hand, uint64_t& from, uint32_t base) __attribute__((always_inline)) {
        constexpr int HAND = decltype(hand)::value;
        Piece<T> p[HAND];
        const uint64_t all = from;
        uint32_t at = 0;
#pragma unroll
        for (int k = 0; k < HAND; ++k) {  // behind the last the last again
            at = from ? base + (uint32_t)__builtin_ctzll(from) : at;
            from &= from - 1;
            const T* row = dy + (int64_t)at * dy_stride;
            if (FEW)
                p[k].load_few(row, (int)cols);
            else
                p[k].load(row, c, (int)cols);
        }
        const int count = __popcll(all);
#pragma unroll
        for (int k = 0; k < HAND; ++k) {
            if (!FEW) p[k].fix(left);
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] = k < count ? acc[e] + (float)p[k].v[e] : acc[e];
        }
    };
#pragma unroll
    for (uint32_t k = 0; k < kFewPositions / kWave; ++k)
        while (same[k]) {
            if (__popcll(same[k]) <= 2)
                add(std::integral_constant<int, 2>{}, same[k], k * kWave);
            else
                add(std::integral_constant<int, 16>{}, same[k], k * kWave);
        }
#pragma unroll
    for (int h = 0; h < V / 4; ++h) {
        Piece<float> out;
#pragma unroll
        for (int e = 0; e < 4; ++e) out.v[e] = acc[4 * h + e] * scale;
        out.store(dtable + (uint64_t)key * cols + c + 4 * h, left - 4 * h);
    }
}

// Lanes of a row.
uint32_t sum_lanes(uint32_t cols, int v) {
    const uint32_t pieces = ceil_div(cols, v);
    return pieces <= 4 ? 4 : pieces <= 16 ? 16 : pieces <= 32 ? 32 : kWave;
}

struct Plan {
    int passes, bits;  // of the sort
    uint32_t keys;
    uint32_t chunk, chunks;
    uint64_t counts, list, partial, bytes;  // where the workspace's parts begin; two lists
};

uint64_t whole_lines(uint64_t bytes) { return (bytes + 127) / 128 * 128; }

Plan plan(uint64_t n, uint32_t vocab, uint32_t cols, int32_t dtype) {
    Plan p;
    int bits = 0;
    while (bits < 32 && (uint64_t)vocab >> bits) ++bits;  // the largest key is vocab itself
    p.passes = (bits + 9) / 10;
    p.bits = (bits + p.passes - 1) / p.passes;
    p.keys = p.passes == 1 ? vocab + 1 : 1u << p.bits;
    // chunks enough to fill the GPU, of rows enough that few of them are joined
    const uint32_t v = 16 / elem_bytes(dtype), lanes = sum_lanes(cols, v), slabs = ceil_div(cols, lanes * v);
    const uint64_t most = (uint64_t)std::max(kMostChunks, kMostWaves / slabs) * (kWave / lanes);
    p.chunk = lanes == kWave ? kLeastChunk : 2 * kLeastChunk;
    while ((n + p.chunk - 1) / p.chunk > most) p.chunk *= 2;
    p.chunks = (uint32_t)((n + p.chunk - 1) / p.chunk);
    p.counts = 0;
    p.list = whole_lines(sort_bytes(p.keys));
    p.partial = p.list + 2 * whole_lines(sizeof(Place) * n);
    // of any smaller number of positions too
    const uint64_t some = std::min<uint64_t>((n + kLeastChunk - 1) / kLeastChunk, most);
    p.bytes = std::max<uint64_t>(p.partial + 8 * some * cols, 128);
    return p;
}

int32_t check_embedding(uint64_t positions, uint32_t vocab, uint32_t cols, int32_t dtype) {
    TATARA_REQUIRE_DTYPE(dtype);
    TATARA_REQUIRE(vocab >= 1 && vocab <= kMaxVocab, "a table has 1 to 2^28 rows");
    TATARA_REQUIRE(cols >= 1 && cols <= kMaxRowCols, "rows have 1 to 32768 columns");
    TATARA_REQUIRE(positions < (1ull << 31), "too many positions");
    return kOk;
}

}  // namespace
}  // namespace tatara

using namespace tatara;

extern "C" {

int32_t tatara_op_embedding_forward(const int32_t* token, uint64_t positions, const void* table, int64_t table_stride,
                                    uint32_t vocab, uint32_t cols, float scale, void* y, int64_t y_stride,
                                    int32_t dtype, TataraStream* stream) {
    if (int32_t st = check_embedding(positions, vocab, cols, dtype)) return st;
    if (positions == 0) return kOk;
    TATARA_REQUIRE(token && table && y, "null tensor");
    TATARA_REQUIRE(table_stride >= (int64_t)cols && y_stride >= (int64_t)cols, "a row stride is smaller than the row");
    TATARA_REQUIRE_ALIGNED(table, elem_bytes(dtype));
    TATARA_REQUIRE_ALIGNED(y, elem_bytes(dtype));
    if (int32_t st = check_stream(stream)) return st;
    return launch_rows_back(
        RowsBack{table, table_stride, vocab, token, nullptr, scale, y, y_stride, positions, 1, cols}, dtype,
        raw(stream));
}

int32_t tatara_op_embedding_backward_workspace(uint64_t positions, uint32_t vocab, uint32_t cols, int32_t dtype,
                                               uint64_t* bytes) {
    TATARA_REQUIRE(bytes, "null output");
    if (int32_t st = check_embedding(positions, vocab, cols, dtype)) return st;
    *bytes = plan(positions, vocab, cols, dtype).bytes;
    return kOk;
}

int32_t tatara_op_embedding_backward(const void* dy, int64_t dy_stride, const int32_t* token, uint64_t positions,
                                     uint32_t vocab, uint32_t cols, float scale, float* dtable, int32_t dtype,
                                     void* workspace, uint64_t workspace_bytes, TataraStream* stream) {
    if (int32_t st = check_embedding(positions, vocab, cols, dtype)) return st;
    TATARA_REQUIRE(dtable && (!positions || (dy && token)), "null tensor");
    TATARA_REQUIRE(!positions || dy_stride >= (int64_t)cols, "the row stride is smaller than the row");
    TATARA_REQUIRE_ALIGNED(dy, elem_bytes(dtype));
    const Plan p = plan(positions, vocab, cols, dtype);
    TATARA_REQUIRE(workspace && workspace_bytes >= p.bytes, "workspace too small");
    TATARA_REQUIRE_ALIGNED(workspace, 16);
    if (int32_t st = check_stream(stream)) return st;
    // of a small table few rows a workgroup, which clears them at one CU's rate
    const uint32_t clear_rows = std::max(4u, std::min(kClearRows, vocab / 1024));
    const uint32_t clear = std::min(ceil_div(vocab, clear_rows), 1u << 20);
    if (positions <= kFewPositions) {
        TATARA_FOR_DTYPE(dtype, {
            const uint32_t slabs = ceil_div(cols, kWave * Piece<T>::V);
            const uint32_t blocks = clear + ceil_div(positions * slabs, kThreads / kWave);
            auto launch = [&](auto few) {
                embedding_few_kernel<T, decltype(few)::value><<<blocks, kThreads, 0, raw(stream)>>>(
                    static_cast<const T*>(dy), dy_stride, token, (uint32_t)positions, vocab, cols, scale, dtable,
                    clear, clear_rows, slabs);
            };
            cols < (uint32_t)Piece<T>::V ? launch(std::true_type{}) : launch(std::false_type{});
        });
        TATARA_LAUNCHED("embedding_few");
        return kOk;
    }
    char* base = static_cast<char*>(workspace);
    Place* list[2];
    for (int i = 0; i < 2; ++i)
        list[i] = reinterpret_cast<Place*>(base + p.list + i * whole_lines(sizeof(Place) * positions));
    float* partial = reinterpret_cast<float*>(base + p.partial);
    const uint32_t mask = p.passes == 1 ? ~0u : p.keys - 1;
    const SortShape shape = sort_shape(positions, p.keys);
    if (shape.runs == 1) {
        with_bits(p.keys, [&](auto bits) {
            embedding_sort_kernel<decltype(bits)::value><<<1, kSortThreads, sort_lds(p.keys), raw(stream)>>>(
                token, (uint32_t)positions, shape.run, vocab, p.passes, p.bits, p.keys, mask, list[0], list[1]);
        });
        TATARA_LAUNCHED("embedding_sort");
    }
    for (int i = 0; shape.runs > 1 && i < p.passes; ++i)
        if (int32_t st = launch_sort(digit_of(i, p.bits, token, vocab, mask, list[0], list[1]), positions, p.keys,
                                     reinterpret_cast<uint32_t*>(base + p.counts), raw(stream)))
            return st;
    const Sorted s{list[(p.passes - 1) % 2], (uint32_t)positions, p.chunk, p.chunks};
    TATARA_FOR_DTYPE(dtype, {
        constexpr int V = Piece<T>::V;
        const uint32_t lanes = sum_lanes(cols, V), slabs = ceil_div(cols, lanes * V);
        auto launch = [&](auto g, auto few) {
            constexpr int G = decltype(g)::value;
            const uint32_t blocks = clear + ceil_div((uint64_t)p.chunks * slabs, kThreads / G);
            embedding_sum_kernel<T, G, decltype(few)::value><<<blocks, kThreads, 0, raw(stream)>>>(
                static_cast<const T*>(dy), dy_stride, s, vocab, cols, scale, dtable, partial, clear, clear_rows,
                slabs);
        };
        using std::integral_constant;
        if (cols < (uint32_t)V)
            launch(integral_constant<int, 4>{}, std::true_type{});
        else if (lanes == 4)
            launch(integral_constant<int, 4>{}, std::false_type{});
        else if (lanes == 16)
            launch(integral_constant<int, 16>{}, std::false_type{});
        else if (lanes == 32)
            launch(integral_constant<int, 32>{}, std::false_type{});
        else
            launch(integral_constant<int, 64>{}, std::false_type{});
    });
    TATARA_LAUNCHED("embedding_sum");
    if (p.chunks > 1) {
        const uint32_t slabs = ceil_div(cols, kWave * 4);
        auto launch = [&](auto waves) {
            constexpr int WAVES = decltype(waves)::value;
            embedding_join_kernel<WAVES><<<ceil_div(p.chunks - 1, WAVES) * slabs, WAVES * kWave, 0, raw(stream)>>>(
                s, vocab, cols, scale, partial, dtable, slabs);
        };
        // sixteen waves where a token is in many chunks (65536 x 1536 f32 of 2 tokens: the call 104
        // us, so 97; of 73305 217 and 222)
        if (positions / vocab > 16ull * p.chunk)
            launch(std::integral_constant<int, 16>{});
        else
            launch(std::integral_constant<int, 4>{});
        TATARA_LAUNCHED("embedding_join");
    }
    return kOk;
}

}  // extern "C"
