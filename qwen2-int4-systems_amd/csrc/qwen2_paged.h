// Addressing of the paged key/value cache (include/qwen2_decode.h), for the
// kernels and, compiled by the host's compiler alone, for their tests: every
// index that a kernel takes from device memory passes through one of these.
#pragma once

#include <stdint.h>

namespace w4g64 {

// A paged cache as a kernel sees it.  Strides in elements.
struct PagedView {
    uint16_t* k;
    uint16_t* v;
    int64_t k_page, k_head, k_position;
    int64_t v_page, v_head, v_position;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* cu_rows;
    const int32_t* lengths;
    int batch;
    int kv_heads;
    int num_pages;
    int page_shift;   // log2 of the page size
    int table_width;
};

// The rows of one sequence, bounded by [0, rows] whatever cu_rows holds, and
// the position of its first one (negative where lengths says less than n).
// The kernels give rows_end() for `rows`: no sequence reaches past the last one.
struct SequenceRows {
    int begin, end;
    int64_t first;
};
__host__ __device__ inline SequenceRows sequence_rows(const int32_t* cu_rows, const int32_t* lengths, int sequence,
                                                      int rows) {
    SequenceRows s;
    const int begin = cu_rows[sequence], end = cu_rows[sequence + 1];
    s.begin = begin < 0 ? 0 : (begin > rows ? rows : begin);
    s.end = end < s.begin ? s.begin : (end > rows ? rows : end);
    s.first = (int64_t)lengths[sequence] - (s.end - s.begin);
    return s;
}

// The end of the last sequence's rows, bounded by [0, rows] whatever cu_rows
// holds, and the row behind it that is a workgroup's first one (in 64 bits: the
// sum of two bounds of 31).
__host__ __device__ inline int rows_end(const int32_t* cu_rows, int batch, int rows) {
    const int end = cu_rows[batch];
    return end < 0 ? 0 : (end > rows ? rows : end);
}
__host__ __device__ inline int64_t rest_row(const int32_t* cu_rows, int batch, int rows, unsigned workgroup) {
    return (int64_t)rows_end(cu_rows, batch, rows) + workgroup;
}

// The page of a position, or -1: outside the table, or not a page of the pool.
__host__ __device__ inline int checked_page(int page, int num_pages) { return page >= 0 && page < num_pages ? page : -1; }
__host__ __device__ inline int page_of(const int32_t* table_row, int table_width, int page_shift, int num_pages,
                                       int64_t position) {
    if (position < 0 || (position >> page_shift) >= table_width) return -1;
    return checked_page(table_row[position >> page_shift], num_pages);
}

}  // namespace w4g64
