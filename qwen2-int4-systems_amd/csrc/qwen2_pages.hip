// Giving out, forking and compacting the pages of a paged cache
// (qwen2_paged_resize, qwen2_paged_fork, qwen2_paged_compact, include/qwen2_decode.h).
//
// All three come down to ranks: the i-th page wanted is the i-th free one, the i-th
// page that moves goes to the i-th hole.  Pages are counted in groups of kGroup (four
// ballots of a wave, whose bits are ranks within the group), the groups' counts are
// summed up, and a second look at the pages writes the lists.
//   few     one workgroup does all of that, with barriers between: up to kFewPages
//           pages and kFewEntries table entries;
//   many    one launch counts, one lists, one applies.
// Answers go to new arrays: what a kernel reads nobody changes, and the only atomics
// are whole numbers' sums, so that the same inputs give the same answer.  Keys and
// values are copied from pages in use to pages that are free, which no other copy
// reads: in any order.
//
// Indices from device memory (entries, lengths, parents) are bounded before they are
// used; what names no page is left out.
#include <hip/hip_runtime.h>

#include "qwen2_decode.h"
#include "qwen2_pages.h"
#include "w4g64_device.h"
#include "w4g64_internal.h"

namespace w4g64 {
namespace {

constexpr int kThreads = 1024;           // of the workgroups that count, list and plan
constexpr int kWaves = kThreads / 64;
constexpr int kGroup = 256;              // pages counted together, by one wave
constexpr int kFewPages = 1 << 16;
constexpr int kFewEntries = 1 << 15;
constexpr int64_t kMostPages = 1 << 24;  // (a workgroup sums up the counts before its own)
constexpr int kCopyThreads = 256;

__device__ __forceinline__ int lane_id() { return threadIdx.x & 63; }
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
__device__ __forceinline__ int bits_before(uint64_t mask, int lane) {
    return __popcll(mask & ((uint64_t(1) << lane) - 1));
}

// Sum over the workgroup's threads, the same in all of them; `meet` holds kWaves words.
__device__ __forceinline__ int block_sum(int v, int* meet) {
    const int lane = lane_id(), wave = wave_id();
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if (lane == 0) meet[wave] = v;
    __syncthreads();
    int sum = 0;
    for (int w = 0; w < kWaves; ++w) sum += meet[w];
    return sum;
}

// Sum over the threads before this one, and over all.
__device__ __forceinline__ int block_before(int v, int* meet, int& all) {
    const int lane = lane_id(), wave = wave_id();
    int upto = v;
    for (int d = 1; d < 64; d <<= 1) {
        const int other = __shfl_up(upto, d);
        if (lane >= d) upto += other;
    }
    __syncthreads();
    if (lane == 63) meet[wave] = upto;
    __syncthreads();
    int before = 0;
    all = 0;
    for (int w = 0; w < kWaves; ++w) {
        before += w < wave ? meet[w] : 0;
        all += meet[w];
    }
    return before + upto - v;
}

// One group of pages as a wave sees it: bit l of free[i] is page 256 g + 64 i + l.
struct Group {
    uint64_t free[4];
    int there[4];  // the lane's pages' users
    __device__ __forceinline__ void load(const int32_t* users, int pages, int group) {
        const int lane = lane_id();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t p = (int64_t)group * kGroup + 64 * i + lane;
            there[i] = p < pages ? users[p] : -1;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) free[i] = __ballot(there[i] == 0);
    }
    __device__ __forceinline__ int count() const {
        return __popcll(free[0]) + __popcll(free[1]) + __popcll(free[2]) + __popcll(free[3]);
    }
};

// Writes the free pages of rank below `limit` to list[rank]; `before`: the rank of the
// group's first one.
__device__ __forceinline__ void list_group(const Group& g, int group, int before, int limit, int32_t* list) {
    const int lane = lane_id();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int rank = before + bits_before(g.free[i], lane);
        if (g.there[i] == 0 && rank < limit) list[rank] = group * kGroup + 64 * i + lane;
        before += __popcll(g.free[i]);
    }
}

// The free pages' counts of all groups (one workgroup): counts[g]; with `copy`, the
// users besides.
__device__ __forceinline__ void count_groups(const int32_t* users, int pages, int32_t* counts, int32_t* copy) {
    const int groups = (pages + kGroup - 1) / kGroup;
    for (int g = wave_id(); g < groups; g += kWaves) {
        Group x;
        x.load(users, pages, g);
        if (lane_id() == 0) counts[g] = x.count();
        if (copy)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int p = g * kGroup + 64 * i + lane_id();
                if (p < pages) copy[p] = x.there[i];
            }
    }
}

// Counts to sums before (in place, one workgroup); returns the sum of all.
__device__ __forceinline__ int sum_groups(int32_t* counts, int groups, int* meet) {
    int sum = 0;
    for (int base = 0; base < groups; base += kThreads) {
        const int g = base + (int)threadIdx.x;
        int all;
        const int before = block_before(g < groups ? counts[g] : 0, meet, all);
        if (g < groups) counts[g] = sum + before;
        sum += all;
    }
    __syncthreads();
    return sum;
}

// The first `limit` free pages in order, by one workgroup, from the sums of
// sum_groups().
__device__ __forceinline__ void list_free(const int32_t* users, int pages, const int32_t* sums, int limit, int32_t* list) {
    const int groups = (pages + kGroup - 1) / kGroup;
    for (int g = wave_id(); g < groups; g += kWaves) {
        const int before = sums[g];
        if (before >= limit) break;
        Group x;
        x.load(users, pages, g);
        list_group(x, g, before, limit, list);
    }
}

// ---- resize ----

struct ResizeArgs {
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* users;
    int32_t* new_table;
    int32_t* new_users;
    int32_t* missing;
    int32_t* want;    // [batch]: pages that a row gets
    int32_t* counts;  // [groups]
    int32_t* list;    // free pages in order
    int64_t table_stride;
    int batch, width, pages, page_shift, most;  // most: entries of the list
    int row_blocks;
};

// A row's entries in [0, upto) that name no page (one wave).
__device__ __forceinline__ int lacking(const ResizeArgs& a, int b) {
    const int upto = pages_wanted(a.lengths[b], a.page_shift, a.width);
    const int32_t* row = a.table + b * a.table_stride;
    int lacks = 0;
    for (int c0 = 0; c0 < upto; c0 += 256) {
        int entry[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = c0 + 64 * i + lane_id();
            entry[i] = c < upto ? row[c] : 0;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            lacks += __popcll(__ballot(c0 + 64 * i + lane_id() < upto && !names_page(entry[i], a.pages)));
    }
    return lacks;
}

// A row's new entries (one wave): free pages from rank `start` on where one is wanted
// (there are `free` in the list), pages given up where none is.
__device__ __forceinline__ void resize_row(const ResizeArgs& a, int b, int64_t start, int free) {
    const int need = pages_needed(a.lengths[b], a.page_shift);
    const int upto = min(need, a.width);
    const int32_t* row = a.table + b * a.table_stride;
    int32_t* to = a.new_table + (int64_t)b * a.width;
    int held = 0;
    for (int c0 = 0; c0 < a.width; c0 += 256) {
        int entry[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = c0 + 64 * i + lane_id();
            entry[i] = c < a.width ? row[c] : -1;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = c0 + 64 * i + lane_id();
            const bool named = names_page(entry[i], a.pages);
            const uint64_t wants = __ballot(c < upto && !named);
            int e = named ? entry[i] : -1;
            if (c >= upto) {
                if (named) atomicAdd(a.new_users + e, -1);
                e = -1;
            } else if (!named) {
                const int64_t rank = start + bits_before(wants, lane_id());
                if (rank < free) {
                    e = a.list[rank];
                    atomicAdd(a.new_users + e, 1);
                }
            }
            if (c < a.width) to[c] = e;
            held += __popcll(__ballot(e >= 0));
            start += __popcll(wants);
        }
    }
    if (lane_id() == 0) a.missing[b] = need - held;
}

__global__ __launch_bounds__(kThreads) void resize_few_kernel(ResizeArgs a) {
    __shared__ int meet[kWaves];
    count_groups(a.users, a.pages, a.counts, a.new_users);
    for (int b = wave_id(); b < a.batch; b += kWaves) {
        const int lacks = lacking(a, b);
        if (lane_id() == 0) a.want[b] = lacks;
    }
    __syncthreads();
    const int wanted = sum_groups(a.want, a.batch, meet);
    const int free = min(sum_groups(a.counts, (a.pages + kGroup - 1) / kGroup, meet), wanted);
    list_free(a.users, a.pages, a.counts, free, a.list);
    __syncthreads();
    for (int b = wave_id(); b < a.batch; b += kWaves) resize_row(a, b, a.want[b], free);
}

// Many: rows' wants by the first workgroups, pages' counts by the others.
__global__ __launch_bounds__(kThreads) void resize_count_kernel(ResizeArgs a) {
    if ((int)blockIdx.x < a.row_blocks) {
        const int b = (int)blockIdx.x * kWaves + wave_id();
        if (b >= a.batch) return;
        const int lacks = lacking(a, b);
        if (lane_id() == 0) a.want[b] = lacks;
        return;
    }
    const int g = ((int)blockIdx.x - a.row_blocks) * kWaves + wave_id();
    if ((int64_t)g * kGroup >= a.pages) return;
    Group x;
    x.load(a.users, a.pages, g);
    if (lane_id() == 0) a.counts[g] = x.count();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t p = (int64_t)g * kGroup + 64 * i + lane_id();
        if (p < a.pages) a.new_users[p] = x.there[i];
    }
}

// The sum of counts[0 .. n) by one workgroup.
__device__ __forceinline__ int sum_of(const int32_t* counts, int n, int* meet) {
    int sum = 0;
    for (int i = (int)threadIdx.x; i < n; i += kThreads) sum += counts[i];
    return block_sum(sum, meet);
}

__global__ __launch_bounds__(kThreads) void resize_list_kernel(ResizeArgs a) {
    __shared__ int meet[kWaves];
    const int groups = (a.pages + kGroup - 1) / kGroup;
    const int first = (int)blockIdx.x * kWaves;
    int before = sum_of(a.counts, first, meet);
    if (before >= a.most) return;
    const int g = first + wave_id();
    if (g >= groups) return;
    for (int i = first; i < g; ++i) before += a.counts[i];
    Group x;
    x.load(a.users, a.pages, g);
    list_group(x, g, before, a.most, a.list);
}

__global__ __launch_bounds__(kThreads) void resize_apply_kernel(ResizeArgs a) {
    __shared__ int meet[kWaves];
    const int free = min(sum_of(a.counts, (a.pages + kGroup - 1) / kGroup, meet), a.most);
    const int first = (int)blockIdx.x * kWaves;
    int64_t start = sum_of(a.want, first, meet);
    const int b = first + wave_id();
    if (b >= a.batch) return;
    for (int i = first; i < b; ++i) start += a.want[i];
    resize_row(a, b, start, free);
}

// ---- copies between pages ----

struct Pool {
    uint16_t* data[2];  // keys, values
    int64_t layer[2], page[2], head[2], position[2];
    int layers, pieces;  // 16-byte pieces of a position
    int kv_heads, page_size;
};

// `count` positions of a page of one layer (keys or values) to another page, by the
// workgroup: pieces in the order of the larger stride.
__device__ __forceinline__ void copy_page(const Pool& p, int which, int layer, int from, int to, int count) {
    const uint16_t* base = p.data[which] + layer * p.layer[which];
    const uint16_t* source = base + from * p.page[which];
    uint16_t* target = const_cast<uint16_t*>(base) + to * p.page[which];
    const bool by_head = p.head[which] >= p.position[which];
    const int inner = by_head ? count : p.kv_heads;
    const int64_t inner_step = by_head ? p.position[which] : p.head[which];
    const int64_t outer_step = by_head ? p.head[which] : p.position[which];
    const int total = p.kv_heads * count * p.pieces;
    constexpr int kAtOnce = 4;
    for (int base_piece = 0; base_piece < total; base_piece += kAtOnce * kCopyThreads) {
        u32x4 x[kAtOnce];
        int64_t at[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int piece = base_piece + i * kCopyThreads + (int)threadIdx.x;
            const int row = piece / p.pieces, d = piece - row * p.pieces;
            const int outer = row / inner;
            at[i] = outer * outer_step + (row - outer * inner) * inner_step + 8 * d;
            if (piece < total) x[i] = *(const u32x4*)(source + at[i]);
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
            if (base_piece + i * kCopyThreads + (int)threadIdx.x < total) *(u32x4*)(target + at[i]) = x[i];
    }
}

// ---- fork ----

struct ForkArgs {
    Pool pool;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* users;
    const int32_t* parents;
    int32_t* new_table;
    int32_t* new_lengths;
    int32_t* new_users;
    int32_t* missing;
    int32_t* first;   // [batch]: a row's first child (children if it has none)
    int32_t* born;    // [batch]: how many it has
    int32_t* target;  // [children]: the page of a child's copy, -1 if it has none, or -2 where one was wanted
    int32_t* counts;  // [groups]
    int32_t* list;    // [children]: free pages
    int64_t table_stride;
    int batch, children, width, pages, page_shift;
    int counted;      // counts and new_users were made by a launch before
    int row_blocks, old_blocks;
};

// A row's last page if it is there and not full: its column, or -1.
__device__ __forceinline__ int partial_column(const ForkArgs& a, int b) {
    const int length = max(a.lengths[b], 0);
    const int column = length >> a.page_shift;
    if (!(length & ((1 << a.page_shift) - 1)) || column >= a.width) return -1;
    return names_page(a.table[b * a.table_stride + column], a.pages) ? column : -1;
}
// Whether only this row names that page.
__device__ __forceinline__ bool sole(const ForkArgs& a, int b, int column) {
    return a.users[a.table[b * a.table_stride + column]] == 1;
}

__global__ __launch_bounds__(kThreads) void fork_count_kernel(ForkArgs a) {
    const int g = (int)blockIdx.x * kWaves + wave_id();
    if ((int64_t)g * kGroup >= a.pages) return;
    Group x;
    x.load(a.users, a.pages, g);
    if (lane_id() == 0) a.counts[g] = x.count();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t p = (int64_t)g * kGroup + 64 * i + lane_id();
        if (p < a.pages) a.new_users[p] = x.there[i];
    }
}

// One workgroup: who copies, and to which page.
__global__ __launch_bounds__(kThreads) void fork_plan_kernel(ForkArgs a) {
    __shared__ int meet[kWaves];
    const int tid = (int)threadIdx.x;
    for (int b = tid; b < a.batch; b += kThreads) a.first[b] = a.children, a.born[b] = 0;
    if (!a.counted) count_groups(a.users, a.pages, a.counts, a.new_users);
    __syncthreads();
    for (int i = tid; i < a.children; i += kThreads) {
        const int parent = a.parents[i];
        if (parent < 0 || parent >= a.batch) continue;
        atomicMin(a.first + parent, i);
        atomicAdd(a.born + parent, 1);
    }
    __syncthreads();
    int copies = 0;
    for (int base = 0; base < a.children; base += kThreads) {
        const int i = base + tid;
        bool copy = false;
        if (i < a.children) {
            const int parent = a.parents[i];
            if (parent >= 0 && parent < a.batch) {
                const int column = partial_column(a, parent);
                copy = column >= 0 && (__hip_atomic_load(a.first + parent, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != i ||
                                       !sole(a, parent, column));
            }
        }
        int all;
        const int rank = copies + block_before(copy, meet, all);
        if (i < a.children) a.target[i] = copy ? rank : -1;
        copies += all;
    }
    const int free = min(sum_groups(a.counts, (a.pages + kGroup - 1) / kGroup, meet), copies);
    list_free(a.users, a.pages, a.counts, free, a.list);
    __syncthreads();
    for (int i = tid; i < a.children; i += kThreads) {
        const int rank = a.target[i];
        if (rank >= 0) a.target[i] = rank < free ? a.list[rank] : -2;
    }
}

// Workgroups of three kinds: new rows, one wave each; old rows' users, one wave each;
// copies, one child, layer and side (keys, values) each.
__global__ __launch_bounds__(kCopyThreads) void fork_apply_kernel(ForkArgs a) {
    const int block = (int)blockIdx.x;
    constexpr int kRows = kCopyThreads / 64;
    if (block < a.row_blocks) {
        const int i = block * kRows + wave_id();
        if (i >= a.children) return;
        const int parent = a.parents[i];
        const bool there = parent >= 0 && parent < a.batch;
        const int length = there ? max(a.lengths[parent], 0) : 0;
        const int upto = pages_wanted(length, a.page_shift, a.width);
        const int target = a.target[i];
        const int column = there ? partial_column(a, parent) : -1;
        const int32_t* row = a.table + (there ? parent : 0) * a.table_stride;
        for (int c = lane_id(); c < a.width; c += 64) {
            int e = c < upto ? row[c] : -1;
            if (!names_page(e, a.pages)) e = -1;
            if (c == column && target != -1) {
                e = target;
                if (e >= 0) atomicAdd(a.new_users + e, 1);
                else e = -1;
            }
            a.new_table[(int64_t)i * a.width + c] = e;
        }
        if (lane_id() == 0) {
            a.new_lengths[i] = length;
            a.missing[i] = target == -2;
        }
        return;
    }
    if (block < a.row_blocks + a.old_blocks) {
        const int b = (block - a.row_blocks) * kRows + wave_id();
        if (b >= a.batch) return;
        const int born = a.born[b];
        const int upto = pages_wanted(a.lengths[b], a.page_shift, a.width);
        const int column = partial_column(a, b);
        // children that hold the row's last page itself
        const int kept = column >= 0 && born > 0 && sole(a, b, column);
        for (int c = lane_id(); c < a.width; c += 64) {
            const int e = a.table[b * a.table_stride + c];
            const int change = (c == column ? kept : c < upto ? born : 0) - 1;
            if (change && names_page(e, a.pages)) atomicAdd(a.new_users + e, change);
        }
        return;
    }
    const int64_t item = block - a.row_blocks - a.old_blocks;
    const int i = (int)(item / (2 * a.pool.layers)), rest = (int)(item - (int64_t)i * 2 * a.pool.layers);
    const int target = a.target[i];
    if (target < 0) return;
    const int parent = a.parents[i];
    const int length = a.lengths[parent];
    copy_page(a.pool, rest & 1, rest >> 1, a.table[parent * a.table_stride + (length >> a.page_shift)], target,
              length & ((1 << a.page_shift) - 1));
}

// ---- compact ----

// What becomes of a page: kStays; kGone (free, behind the live ones); kMoves + i, to
// the i-th hole; kHole + i, taken by the i-th page that moves.
constexpr int32_t kStays = -1, kGone = -2, kMoves = 0, kHole = 1 << 30;

struct CompactArgs {
    Pool pool;
    const int32_t* table;
    const int32_t* users;
    int32_t* new_table;
    int32_t* new_users;
    int32_t* moved_to;
    int32_t* fate;    // [pages]
    int32_t* counts;  // [groups]
    int32_t* holes;   // [pages / 2]
    int32_t* movers;  // [pages / 2]
    int32_t* moves;   // [1]
    int64_t table_stride;
    int batch, width, pages;
    int page_blocks, copy_blocks;
};

// A group's pages; `before`: the free pages before it, `live`: all in use, `low`: free
// pages below `live`.
__device__ __forceinline__ void settle_group(const CompactArgs& a, const Group& g, int group, int before, int live, int low) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t p64 = (int64_t)group * kGroup + 64 * i + lane_id();
        const int free_before = before + bits_before(g.free[i], lane_id());
        before += __popcll(g.free[i]);
        if (p64 >= a.pages) continue;
        const int p = (int)p64;
        if (g.there[i] == 0) {
            a.fate[p] = p < live ? kHole + free_before : kGone;
            if (p < live) a.holes[free_before] = p;
        } else if (p < live) {
            a.fate[p] = kStays;
        } else {
            const int rank = p - free_before - (live - low);
            a.fate[p] = kMoves + rank;
            a.movers[rank] = p;
        }
    }
}

// Free pages below `live`, from the sums of free pages before each group.
__device__ __forceinline__ int free_below(const CompactArgs& a, int live, int before) {
    const int group = live / kGroup;  // (live <= pages: its group's pages below `live` exist)
    Group x;
    x.load(a.users, a.pages, group);
    int low = before;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int edge = live - group * kGroup - 64 * i;  // bits below it count
        const uint64_t mask = edge <= 0 ? 0 : edge >= 64 ? ~uint64_t(0) : (uint64_t(1) << edge) - 1;
        low += __popcll(x.free[i] & mask);
    }
    return low;
}

__global__ __launch_bounds__(kThreads) void compact_few_kernel(CompactArgs a) {
    __shared__ int meet[kWaves];
    const int groups = (a.pages + kGroup - 1) / kGroup;
    count_groups(a.users, a.pages, a.counts, nullptr);
    __syncthreads();
    const int free = sum_groups(a.counts, groups, meet);
    const int live = a.pages - free;
    const int low = free_below(a, live, live / kGroup < groups ? a.counts[live / kGroup] : free);
    for (int g = wave_id(); g < groups; g += kWaves) {
        Group x;
        x.load(a.users, a.pages, g);
        settle_group(a, x, g, a.counts[g], live, low);
    }
    if (threadIdx.x == 0) *a.moves = low;
}

__global__ __launch_bounds__(kThreads) void compact_count_kernel(CompactArgs a) {
    const int g = (int)blockIdx.x * kWaves + wave_id();
    if ((int64_t)g * kGroup >= a.pages) return;
    Group x;
    x.load(a.users, a.pages, g);
    if (lane_id() == 0) a.counts[g] = x.count();
}

__global__ __launch_bounds__(kThreads) void compact_list_kernel(CompactArgs a) {
    __shared__ int meet[kWaves];
    const int groups = (a.pages + kGroup - 1) / kGroup;
    const int live = a.pages - sum_of(a.counts, groups, meet);
    const int low = free_below(a, live, sum_of(a.counts, min(live / kGroup, groups), meet));
    const int first = (int)blockIdx.x * kWaves;
    int before = sum_of(a.counts, first, meet);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.moves = low;
    const int g = first + wave_id();
    if (g >= groups) return;
    for (int i = first; i < g; ++i) before += a.counts[i];
    Group x;
    x.load(a.users, a.pages, g);
    settle_group(a, x, g, before, live, low);
}

// Copies by the first workgroups, which go through all there are; then pages, then
// table entries.
__global__ __launch_bounds__(kCopyThreads) void compact_apply_kernel(CompactArgs a) {
    int block = (int)blockIdx.x;
    if (block < a.copy_blocks) {
        const int64_t items = (int64_t)*a.moves * 2 * a.pool.layers;
        for (int64_t item = block; item < items; item += a.copy_blocks) {
            const int i = (int)(item / (2 * a.pool.layers)), rest = (int)(item - (int64_t)i * 2 * a.pool.layers);
            copy_page(a.pool, rest & 1, rest >> 1, a.movers[i], a.holes[i], a.pool.page_size);
        }
        return;
    }
    block -= a.copy_blocks;
    auto place = [&](int p) {
        const int32_t f = a.fate[p];
        return f == kStays ? p : f >= kMoves && f < kHole ? a.holes[f - kMoves] : -1;
    };
    if (block < a.page_blocks) {
        const int64_t p = (int64_t)block * kCopyThreads + threadIdx.x;
        if (p >= a.pages) return;
        const int32_t f = a.fate[p];
        a.moved_to[p] = place((int)p);
        a.new_users[p] = f == kStays ? a.users[p] : f >= kHole ? a.users[a.movers[f - kHole]] : 0;
        return;
    }
    block -= a.page_blocks;
    const int64_t at = (int64_t)block * kCopyThreads + threadIdx.x;
    if (at >= (int64_t)a.batch * a.width) return;
    const int b = (int)(at / a.width), c = (int)(at - (int64_t)b * a.width);
    const int e = a.table[b * a.table_stride + c];
    a.new_table[at] = names_page(e, a.pages) ? place(e) : -1;
}

// ---- host ----

int64_t blocks_of(int64_t n, int64_t per) { return (n + per - 1) / per; }
int64_t groups_of(int64_t pages) { return blocks_of(pages, kGroup); }

bool aligned4(std::initializer_list<const void*> all) {
    for (const void* p : all)
        if (!p || ((uintptr_t)p & 3)) return false;
    return true;
}

// The sizes that all three have.
int check_sizes(const char* op, int64_t batch, int64_t width, int64_t pages) {
    if (batch < 0 || batch > (1 << 20) || width <= 0 || width > 0x7FFFFFFF || pages <= 0)
        return set_error(W4G64_STATUS_INVALID_VALUE,
                         "%s needs a batch in [0, 2^20], table_width in [1, 2^31) and num_pages above 0, got %lld, %lld and %lld", op,
                         (long long)batch, (long long)width, (long long)pages);
    if (pages > kMostPages || batch * width > 0x7FFFFFFF)
        return set_error(W4G64_STATUS_UNSUPPORTED, "%s takes up to 2^24 pages and 2^31 - 1 table entries, got %lld and %lld", op,
                         (long long)pages, (long long)(batch * width));
    return W4G64_STATUS_OK;
}

int shift_of(int64_t page_size) {
    for (int shift = 4; shift <= 20; ++shift)
        if (int64_t(1) << shift == page_size) return shift;
    return -1;
}

int pool_view(const char* op, const qwen2_page_pool* p, Pool* view) {
    if (!p || !p->k || !p->v || (((uintptr_t)p->k | (uintptr_t)p->v) & 15))
        return set_error(W4G64_STATUS_INVALID_VALUE, "%s: pools must be non-null and 16-byte aligned", op);
    if (p->layers <= 0 || p->layers > 0xFFFF || p->kv_heads <= 0 || p->kv_heads > 0xFFFF || shift_of(p->page_size) < 0)
        return set_error(W4G64_STATUS_INVALID_VALUE,
                         "%s: layers and kv_heads must be in [1, 2^16) and page_size a power of two in [16, 2^20], got %lld, "
                         "%lld and %lld", op, (long long)p->layers, (long long)p->kv_heads, (long long)p->page_size);
    if (p->head_dim <= 0 || p->head_dim % 8 || p->head_dim > 1024 || p->kv_heads * p->page_size * p->head_dim > (1 << 30))
        return set_error(W4G64_STATUS_UNSUPPORTED,
                         "%s: head_dim must be a multiple of 8 up to 1024 and a page at most 2^30 elements, got %lld", op,
                         (long long)p->head_dim);
    const int64_t strides[] = {p->k_layer, p->k_page, p->k_head, p->k_position, p->v_layer, p->v_page, p->v_head, p->v_position};
    for (int64_t s : strides)
        if (s < 0 || s % 8)
            return set_error(W4G64_STATUS_INVALID_VALUE, "%s: pool strides must be multiples of 8 elements, not negative", op);
    *view = Pool{{(uint16_t*)p->k, (uint16_t*)p->v}, {p->k_layer, p->v_layer}, {p->k_page, p->v_page}, {p->k_head, p->v_head},
                 {p->k_position, p->v_position}, (int)p->layers, (int)(p->head_dim / 8), (int)p->kv_heads, (int)p->page_size};
    return W4G64_STATUS_OK;
}

int check_workspace(const char* op, int64_t need, const void* workspace, int64_t bytes) {
    if (need && (!workspace || bytes < need || ((uintptr_t)workspace & 3)))
        return set_error(W4G64_STATUS_WORKSPACE, "%s needs %lld workspace bytes, 4-byte aligned, got %lld", op, (long long)need,
                         (long long)(workspace ? bytes : 0));
    return W4G64_STATUS_OK;
}

int launched(const char* op) {
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return set_error(W4G64_STATUS_HIP_ERROR, "%s launch failed: %s", op, hipGetErrorString(err));
    return clear_error();
}

int64_t most_given(int64_t batch, int64_t width, int64_t pages) { return batch * width < pages ? batch * width : pages; }

}  // namespace
}  // namespace w4g64

using namespace w4g64;

extern "C" {

int64_t qwen2_paged_resize_workspace_bytes(int64_t batch, int64_t table_width, int64_t num_pages) {
    if (check_sizes("paged_resize", batch, table_width, num_pages)) return 0;
    return 4 * (batch + groups_of(num_pages) + most_given(batch, table_width, num_pages));
}

int qwen2_paged_resize(const int32_t* page_table, int64_t table_stride, const int32_t* lengths, const int32_t* page_users,
                       int32_t* new_table, int32_t* new_users, int32_t* missing, int64_t batch, int64_t table_width,
                       int64_t num_pages, int64_t page_size, void* workspace, int64_t workspace_bytes, void* stream) {
    int status = check_sizes("paged_resize", batch, table_width, num_pages);
    if (status) return status;
    if (shift_of(page_size) < 0)
        return set_error(W4G64_STATUS_INVALID_VALUE, "page_size must be a power of two in [16, 2^20], got %lld", (long long)page_size);
    if (!aligned4({page_users, new_users}) || (batch && !aligned4({page_table, lengths, new_table, missing})))
        return set_error(W4G64_STATUS_INVALID_VALUE, "paged_resize pointers must be non-null, 4-byte aligned device pointers");
    status = check_workspace("paged_resize", qwen2_paged_resize_workspace_bytes(batch, table_width, num_pages), workspace,
                             workspace_bytes);
    if (status) return status;
    ResizeArgs a{};
    a.table = page_table, a.table_stride = table_stride, a.lengths = lengths, a.users = page_users;
    a.new_table = new_table, a.new_users = new_users, a.missing = missing;
    a.want = (int32_t*)workspace, a.counts = a.want + batch, a.list = a.counts + groups_of(num_pages);
    a.batch = (int)batch, a.width = (int)table_width, a.pages = (int)num_pages, a.page_shift = shift_of(page_size);
    a.most = (int)most_given(batch, table_width, num_pages);
    const hipStream_t s = (hipStream_t)stream;
    if (num_pages <= kFewPages && batch * table_width <= kFewEntries) {
        hipLaunchKernelGGL(resize_few_kernel, dim3(1), dim3(kThreads), 0, s, a);
        return launched("paged_resize");
    }
    a.row_blocks = (int)blocks_of(batch, kWaves);
    const int64_t lists = blocks_of(groups_of(num_pages), kWaves);
    hipLaunchKernelGGL(resize_count_kernel, dim3((unsigned)(a.row_blocks + lists)), dim3(kThreads), 0, s, a);
    if (batch) {
        hipLaunchKernelGGL(resize_list_kernel, dim3((unsigned)lists), dim3(kThreads), 0, s, a);
        hipLaunchKernelGGL(resize_apply_kernel, dim3((unsigned)a.row_blocks), dim3(kThreads), 0, s, a);
    }
    return launched("paged_resize");
}

int64_t qwen2_paged_fork_workspace_bytes(int64_t batch, int64_t children, int64_t num_pages) {
    if (batch < 0 || children < 0 || num_pages <= 0) return 0;
    return 4 * (2 * batch + 2 * children + groups_of(num_pages));
}

int qwen2_paged_fork(const qwen2_page_pool* pool, const int32_t* page_table, int64_t table_stride, const int32_t* lengths,
                     const int32_t* page_users, const int32_t* parents, int32_t* new_table, int32_t* new_lengths,
                     int32_t* new_users, int32_t* missing, int64_t batch, int64_t children, int64_t table_width,
                     void* workspace, int64_t workspace_bytes, void* stream) {
    ForkArgs a{};
    int status = pool_view("paged_fork", pool, &a.pool);
    if (!status) status = check_sizes("paged_fork", batch, table_width, pool->num_pages);
    if (!status) status = check_sizes("paged_fork", children, table_width, pool->num_pages);
    if (status) return status;
    if (!aligned4({page_users, new_users}) || (batch && !aligned4({page_table, lengths})) ||
        (children && !aligned4({parents, new_table, new_lengths, missing})))
        return set_error(W4G64_STATUS_INVALID_VALUE, "paged_fork pointers must be non-null, 4-byte aligned device pointers");
    const int64_t copies = children * 2 * pool->layers;
    if (copies > 0x7FFFFF)  // (of 2^32 threads a launch)
        return set_error(W4G64_STATUS_UNSUPPORTED, "paged_fork call is too large: %lld copies", (long long)copies);
    status = check_workspace("paged_fork", qwen2_paged_fork_workspace_bytes(batch, children, pool->num_pages), workspace,
                             workspace_bytes);
    if (status) return status;
    a.table = page_table, a.table_stride = table_stride, a.lengths = lengths, a.users = page_users, a.parents = parents;
    a.new_table = new_table, a.new_lengths = new_lengths, a.new_users = new_users, a.missing = missing;
    a.first = (int32_t*)workspace, a.born = a.first + batch, a.target = a.born + batch, a.list = a.target + children;
    a.counts = a.list + children;
    a.batch = (int)batch, a.children = (int)children, a.width = (int)table_width, a.pages = (int)pool->num_pages;
    a.page_shift = shift_of(pool->page_size);
    const hipStream_t s = (hipStream_t)stream;
    a.counted = pool->num_pages > kFewPages;
    if (a.counted)
        hipLaunchKernelGGL(fork_count_kernel, dim3((unsigned)blocks_of(groups_of(pool->num_pages), kWaves)), dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kThreads), 0, s, a);
    a.row_blocks = (int)blocks_of(children, kCopyThreads / 64), a.old_blocks = (int)blocks_of(batch, kCopyThreads / 64);
    const int64_t blocks = a.row_blocks + a.old_blocks + copies;
    if (blocks) hipLaunchKernelGGL(fork_apply_kernel, dim3((unsigned)blocks), dim3(kCopyThreads), 0, s, a);
    return launched("paged_fork");
}

int64_t qwen2_paged_compact_workspace_bytes(int64_t num_pages) {
    return num_pages <= 0 ? 0 : 4 * (num_pages + groups_of(num_pages) + 2 * (num_pages / 2) + 1);
}

int qwen2_paged_compact(const qwen2_page_pool* pool, const int32_t* page_table, int64_t table_stride,
                        const int32_t* page_users, int32_t* new_table, int32_t* new_users, int32_t* moved_to, int64_t batch,
                        int64_t table_width, void* workspace, int64_t workspace_bytes, void* stream) {
    CompactArgs a{};
    int status = pool_view("paged_compact", pool, &a.pool);
    if (!status) status = check_sizes("paged_compact", batch, table_width, pool->num_pages);
    if (status) return status;
    if (!aligned4({page_users, new_users, moved_to}) || (batch && !aligned4({page_table, new_table})))
        return set_error(W4G64_STATUS_INVALID_VALUE, "paged_compact pointers must be non-null, 4-byte aligned device pointers");
    const int64_t pages = pool->num_pages;
    status = check_workspace("paged_compact", qwen2_paged_compact_workspace_bytes(pages), workspace, workspace_bytes);
    if (status) return status;
    a.table = page_table, a.table_stride = table_stride, a.users = page_users;
    a.new_table = new_table, a.new_users = new_users, a.moved_to = moved_to;
    a.fate = (int32_t*)workspace, a.counts = a.fate + pages, a.holes = a.counts + groups_of(pages);
    a.movers = a.holes + pages / 2, a.moves = a.movers + pages / 2;
    a.batch = (int)batch, a.width = (int)table_width, a.pages = (int)pages;
    const hipStream_t s = (hipStream_t)stream;
    if (pages <= kFewPages) {
        hipLaunchKernelGGL(compact_few_kernel, dim3(1), dim3(kThreads), 0, s, a);
    } else {
        const unsigned lists = (unsigned)blocks_of(groups_of(pages), kWaves);
        hipLaunchKernelGGL(compact_count_kernel, dim3(lists), dim3(kThreads), 0, s, a);
        hipLaunchKernelGGL(compact_list_kernel, dim3(lists), dim3(kThreads), 0, s, a);
    }
    // (eight workgroups a CU go through the copies; no more than there can be)
    const int64_t most = pages / 2 * 2 * pool->layers;
    a.copy_blocks = (int)(most < 2048 ? most : 2048);
    a.page_blocks = (int)blocks_of(pages, kCopyThreads);
    const int64_t blocks = a.copy_blocks + a.page_blocks + blocks_of(batch * table_width, kCopyThreads);
    hipLaunchKernelGGL(compact_apply_kernel, dim3((unsigned)blocks), dim3(kCopyThreads), 0, s, a);
    return launched("paged_compact");
}

}  // extern "C"
