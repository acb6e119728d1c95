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

}  // namespace w4g64
