// What the entry points of packed prompts and of pages refuse by sizes and strides alone
// (the status of set_error), for the host calls to ask before they copy an argument.
#pragma once

#include <stdint.h>

#include "../../include/qwen2_decode.h"

namespace w4g64 {

// (k_row, v_row: elements from a row of keys, of values, to the next)
int packed_attention_sizes(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t k_row,
                           int64_t v_row, int dtype, float scale);
int paged_resize_sizes(int64_t batch, int64_t table_width, int64_t num_pages, int64_t page_size);
int paged_fork_sizes(const qwen2_page_pool* pool, int64_t batch, int64_t children, int64_t table_width);
int paged_compact_sizes(const qwen2_page_pool* pool, int64_t batch, int64_t table_width);

}  // namespace w4g64
