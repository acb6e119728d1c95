// Index arithmetic of the packed prompt attention (include/qwen2_decode.h), for the
// kernel and, compiled by the host's compiler alone, for its tests.
#pragma once

#include "qwen2_paged.h"

namespace w4g64 {

// A sequence's rows from its two bounds, within [0, rows_end()] whatever they are.
struct PackedRows {
    int begin, end;
};
__host__ __device__ inline PackedRows packed_rows(int begin, int end, int rows) {
    PackedRows s;
    s.begin = begin < 0 ? 0 : (begin > rows ? rows : begin);
    s.end = end < s.begin ? s.begin : (end > rows ? rows : end);
    return s;
}

// Rows of no sequence, those before the first one's and those behind the last one's, none
// twice whatever the bounds are: how many there are, and the i-th.
struct FreeRows {
    int before, end;
};
__host__ __device__ inline FreeRows free_rows(const int32_t* cu_rows, int batch, int rows) {
    const int end = rows_end(cu_rows, batch, rows), first = cu_rows[0];
    return FreeRows{first < 0 ? 0 : first < end ? first : end, end};
}
__host__ __device__ inline int free_count(const FreeRows& f, int rows) { return f.before + (rows - f.end); }
__host__ __device__ inline int free_row(const FreeRows& f, int i) { return i < f.before ? i : f.end + (i - f.before); }

}  // namespace w4g64
