// The rows of each bucket side by side, for its layers, and back in the positions' order.
//
//   sort:    the choices (t, j) by bucket, and in a bucket by t and j; row r is that of
//            choice source_r, choice (t, j) has row slot_tj
//   gather:  rows_r = x_{source_r / k}
//   combine: y_t = sum_j gate_tj rows_{slot_tj}
//   and back: dx_t = sum_j drows_{slot_tj};  drows_r = gate dy,  dgate_tj = dy_t . rows_{slot_tj}
//
// Packed, a bucket's rows follow the one's before it; with a capacity, bucket e has
// rows e capacity to (e + 1) capacity - 1, and what does not fit has no row.  Sums are
// f32 in the choices' order: no atomics.
#include "key_sort.hpp"
#include "row_moves.hpp"

namespace tatara {
namespace {

struct Choices {
    const int32_t* bucket;
    int32_t* slot;
    int32_t* source;
    int32_t* offset;
    uint64_t n_rows;
    uint32_t capacity;  // 0: packed

    using Item = uint32_t;
    __device__ __forceinline__ Item load(uint64_t i) const { return (uint32_t)bucket[i]; }
    __device__ __forceinline__ uint32_t key(Item e) const { return e; }
    __device__ __forceinline__ void put(uint64_t i, Item, uint32_t e, uint32_t first, uint32_t rank) const {
        const bool fits = !capacity || rank < capacity;
        const uint32_t row = capacity ? e * capacity + rank : first + rank;
        slot[i] = fits ? (int32_t)row : -1;
        if (fits) source[row] = (int32_t)i;
    }
    __device__ __forceinline__ void drop(uint64_t i) const { slot[i] = -1; }
    // The rows that no choice has.
    __device__ __forceinline__ void finish(const uint32_t* first, uint32_t keys) const {
        const uint64_t threads = (uint64_t)gridDim.x * kSortThreads;
        const uint64_t me = (uint64_t)blockIdx.x * kSortThreads + threadIdx.x;
        if (capacity) {
            for (uint64_t r = me; r < n_rows; r += threads) {
                const uint32_t e = (uint32_t)r / capacity;
                if ((uint32_t)r - e * capacity >= first[e + 1] - first[e]) source[r] = -1;
            }
        } else {
            for (uint64_t r = first[keys] + me; r < n_rows; r += threads) source[r] = -1;
        }
        if (blockIdx.x == 0)
            for (uint32_t e = threadIdx.x; e <= keys; e += kSortThreads) offset[e] = (int32_t)first[e];
    }
};

int32_t check_choices(uint64_t positions, uint32_t top_k) {
    TATARA_REQUIRE(top_k >= 1 && top_k <= kMaxTop, "top_k must be 1 to 16");
    TATARA_REQUIRE(positions < (1ull << 31) && positions * top_k < (1ull << 31), "too many positions");
    return kOk;
}

int32_t check_rows(uint64_t positions, uint32_t top_k, uint64_t n_rows, uint32_t cols, int32_t dtype) {
    TATARA_REQUIRE_DTYPE(dtype);
    if (int32_t st = check_choices(positions, top_k)) return st;
    TATARA_REQUIRE(n_rows < (1ull << 31), "too many rows");
    TATARA_REQUIRE(cols >= 1 && cols <= kMaxRowCols, "rows have 1 to 32768 columns");
    return kOk;
}

}  // namespace
}  // namespace tatara

using namespace tatara;

extern "C" {

int32_t tatara_op_bucket_rows_workspace(uint32_t buckets, uint64_t* bytes) {
    TATARA_REQUIRE(bytes, "null output");
    TATARA_REQUIRE(buckets >= 1 && buckets <= kMaxKeys, "rows are sorted by 1 to 1024 buckets");
    *bytes = sort_bytes(buckets);
    return kOk;
}

int32_t tatara_op_bucket_rows_sort(const int32_t* bucket, uint64_t positions, uint32_t buckets, uint32_t top_k,
                                   uint32_t capacity, int32_t* slot, int32_t* source, int32_t* offset,
                                   void* workspace, uint64_t workspace_bytes, TataraStream* stream) {
    TATARA_REQUIRE(buckets >= 1 && buckets <= kMaxKeys, "rows are sorted by 1 to 1024 buckets");
    if (int32_t st = check_choices(positions, top_k)) return st;
    const uint64_t items = positions * top_k;
    const uint64_t n_rows = capacity ? (uint64_t)buckets * capacity : items;
    TATARA_REQUIRE(n_rows < (1ull << 31), "too many rows");
    TATARA_REQUIRE(offset && (!items || (bucket && slot)) && (!n_rows || source), "null tensor");
    TATARA_REQUIRE(workspace && workspace_bytes >= sort_bytes(buckets), "workspace too small");
    TATARA_REQUIRE_ALIGNED(workspace, 16);
    if (int32_t st = check_stream(stream)) return st;
    return launch_sort(Choices{bucket, slot, source, offset, n_rows, capacity}, items, buckets,
                       static_cast<uint32_t*>(workspace), raw(stream));
}

int32_t tatara_op_bucket_rows_gather(const void* x, int64_t x_stride, const int32_t* slot, const int32_t* source,
                                     uint64_t positions, uint32_t top_k, void* rows, int64_t rows_stride,
                                     uint64_t n_rows, uint32_t cols, int32_t dtype, TataraStream* stream) {
    if (int32_t st = check_rows(positions, top_k, n_rows, cols, dtype)) return st;
    if (n_rows == 0) return kOk;
    TATARA_REQUIRE((!positions || (x && slot)) && source && rows, "null tensor");
    TATARA_REQUIRE((!positions || x_stride >= (int64_t)cols) && rows_stride >= (int64_t)cols,
                   "a row stride is smaller than the row");
    TATARA_REQUIRE_ALIGNED(x, elem_bytes(dtype));
    TATARA_REQUIRE_ALIGNED(rows, elem_bytes(dtype));
    if (int32_t st = check_stream(stream)) return st;
    return launch_rows_out(RowsOut{x, x_stride, slot, source, nullptr, nullptr, 0, nullptr, rows, rows_stride, n_rows,
                                   positions, top_k, cols},
                           dtype, raw(stream));
}

int32_t tatara_op_bucket_rows_combine(const void* rows, int64_t rows_stride, uint64_t n_rows, const int32_t* slot,
                                      const float* gate, uint64_t positions, uint32_t top_k, void* y,
                                      int64_t y_stride, uint32_t cols, int32_t dtype, TataraStream* stream) {
    if (int32_t st = check_rows(positions, top_k, n_rows, cols, dtype)) return st;
    if (positions == 0) return kOk;
    TATARA_REQUIRE(n_rows >= 1, "positions without rows");
    TATARA_REQUIRE(rows && slot && y, "null tensor");
    TATARA_REQUIRE(rows_stride >= (int64_t)cols && y_stride >= (int64_t)cols, "a row stride is smaller than the row");
    TATARA_REQUIRE_ALIGNED(rows, elem_bytes(dtype));
    TATARA_REQUIRE_ALIGNED(y, elem_bytes(dtype));
    if (int32_t st = check_stream(stream)) return st;
    return launch_rows_back(RowsBack{rows, rows_stride, n_rows, slot, gate, 1.0f, y, y_stride, positions, top_k, cols},
                            dtype, raw(stream));
}

int32_t tatara_op_bucket_rows_combine_backward(const void* dy, int64_t dy_stride, const void* rows,
                                               int64_t rows_stride, uint64_t n_rows, const int32_t* slot,
                                               const int32_t* source, const float* gate, uint64_t positions,
                                               uint32_t top_k, void* drows, int64_t drows_stride, float* dgate,
                                               uint32_t cols, int32_t dtype, TataraStream* stream) {
    if (int32_t st = check_rows(positions, top_k, n_rows, cols, dtype)) return st;
    TATARA_REQUIRE(n_rows >= 1 || positions == 0, "positions without rows");
    if (n_rows == 0) return kOk;
    TATARA_REQUIRE((!positions || (dy && slot && gate)) && source && drows && (!dgate || !positions || rows),
                   "null tensor");
    TATARA_REQUIRE((!positions || dy_stride >= (int64_t)cols) && drows_stride >= (int64_t)cols &&
                       (!dgate || !positions || rows_stride >= (int64_t)cols),
                   "a row stride is smaller than the row");
    TATARA_REQUIRE_ALIGNED(dy, elem_bytes(dtype));
    TATARA_REQUIRE_ALIGNED(rows, elem_bytes(dtype));
    TATARA_REQUIRE_ALIGNED(drows, elem_bytes(dtype));
    if (int32_t st = check_stream(stream)) return st;
    return launch_rows_out(RowsOut{dy, dy_stride, slot, source, gate, rows, rows_stride, dgate, drows, drows_stride,
                                   n_rows, positions, top_k, cols},
                           dtype, raw(stream));
}

}  // extern "C"
