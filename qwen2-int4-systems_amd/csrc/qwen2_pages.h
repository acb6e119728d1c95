// Index arithmetic of the page operators (include/qwen2_decode.h), for the kernels
// and, compiled by the host's compiler alone, for their tests: every index that a
// kernel takes from device memory passes through one of these.
#pragma once

#include <stdint.h>

namespace w4g64 {

// Whether a table's entry is a page of the pool.
__host__ __device__ inline bool names_page(int entry, int pages) { return entry >= 0 && entry < pages; }

// Pages of a length (none where it is negative), and how many of them a table's row
// can name.
__host__ __device__ inline int pages_needed(int length, int page_shift) {
    return length <= 0 ? 0 : (int)(((int64_t)length + (int64_t(1) << page_shift) - 1) >> page_shift);
}
__host__ __device__ inline int pages_wanted(int length, int page_shift, int width) {
    const int need = pages_needed(length, page_shift);
    return need < width ? need : width;
}

// The columns of a row that part `part` of `parts` sees to: as many 64s as each needs at
// most, from the first on (worked out without a sign: a part's end may pass 2^31 - 1).
struct ColumnPart {
    int from, end;
};
__host__ __device__ inline ColumnPart column_part(int width, int part, int parts) {
    const uint32_t columns = (uint32_t)width, least = 64 * (uint32_t)parts, each = (columns + least - 1) / least * 64;
    const uint32_t from = (uint32_t)part * each, end = from + each;
    return ColumnPart{(int)(from < columns ? from : columns), (int)(end < columns ? end : columns)};
}

}  // namespace w4g64
