// Rows that move between the positions' order and another one (row_moves.hip).
#pragma once

#include "elem.hpp"

namespace tatara {

constexpr uint32_t kMaxTop = 16;
constexpr uint32_t kMaxRowCols = 32768;

// y[t] = sum over j of w * rows[slot[t][j]], w = scale, times gate[t][j] if there is
// a gate; a slot outside 0..n_rows - 1 adds nothing.
struct RowsBack {
    const void* rows;
    int64_t rows_stride;
    uint64_t n_rows;
    const int32_t* slot;  // [positions][top_k]
    const float* gate;
    float scale;
    void* y;
    int64_t y_stride;
    uint64_t positions;
    uint32_t top_k, cols;
};
int32_t launch_rows_back(const RowsBack& a, int32_t dtype, hipStream_t stream);

// rows[slot[t][j]] = gate[t][j] * x[t] (1 without a gate), dgate[t][j] = x[t] . from[slot[t][j]]
// if asked for (0 without a row), and zeros in every row whose source is outside
// 0..positions * top_k - 1.
struct RowsOut {
    const void* x;
    int64_t x_stride;
    const int32_t* slot;
    const int32_t* source;  // [n_rows]
    const float* gate;
    const void* from;
    int64_t from_stride;
    float* dgate;
    void* rows;
    int64_t rows_stride;
    uint64_t n_rows, positions;
    uint32_t top_k, cols;
};
int32_t launch_rows_out(const RowsOut& a, int32_t dtype, hipStream_t stream);

}  // namespace tatara
