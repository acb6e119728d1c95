// Giving out, forking and compacting the pages of a paged cache
// (qwen2_paged_resize, qwen2_paged_fork, qwen2_paged_compact, include/qwen2_decode.h).
//
// All three come down to ranks: the i-th page wanted is the i-th free one, the i-th
// page that moves goes to the i-th hole.  Pages are counted in groups of kGroup (four
// ballots of a wave, whose bits are ranks within the group), the groups' counts are
// summed up, and a second look at the pages writes the lists.
//   few     one launch, every workgroup of which works all of that out for itself, in
//           LDS, and then does its part of what follows: a launch costs a caller 3.6 us.
//           Each goes through up to 64 KB of users and, but for a compaction, the old
//           table (of a fork, the first one does).  us of a resize of empty rows, few /
//           many, a call by itself (as part of a graph): 64 x 80 entries 7.4 / 12.7 (7.9 /
//           8.6), 128 x 64 9.0 / 12.3 (9.5 / 8.7), 256 x 64 14.3 / 12.8 (15.0 / 8.9); of a
//           fork to as many rows 128 x 64 8.7 / 14.1 (9.1 / 10.0), 192 x 64 12.4 / 14.1 (13.0
//           / 9.9);
//   many    one launch counts, one lists, one applies.
// Answers go to new arrays: what a kernel reads nobody changes, and the only atomics
// are whole numbers' sums, so that the same inputs give the same answer.  Keys and
// values are copied from pages in use to pages that are free, which no other copy
// reads: in any order.
//
// What bounds them.  Few: the launch and loads that depend on each other (6 to 8 us of a
// kernel).  Copies of pages: memory; 977 pages of 8 layers moved, 256 MB read and
// written, take 51.7 of a compaction's 53 us (4.95 TB/s; a large copy 5.18).  A resize of
// 511 rows of up to 2048 pages, a ninth of them given up and a ninth cut back: 3.2 + 4.6 +
// 10.5 us, 5.5 of it atomics on the users of some 90000 pages.
//
// Indices from device memory (entries, lengths, parents) are bounded before they are
// used; what names no page is left out.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "qwen2_decode.h"
#include "qwen2_paged_device.h"
#include "qwen2_pages.h"
#include "serving_sizes.h"
#include "w4g64_internal.h"

namespace w4g64 {
namespace {

constexpr int kThreads = 1024;           // of the workgroups that count, list and plan
constexpr int kWaves = kThreads / 64;
constexpr int kGroup = 256;              // pages counted together, by one wave
constexpr int kFewPages = 1 << 14;
constexpr int kFewRows = kThreads;       // (one of a thread)
constexpr int kFewResize = 1 << 13, kFewFork = 3 << 12;  // entries of the old table
constexpr int64_t kMostPages = 1 << 24;  // (a workgroup sums up the counts before its own)
constexpr int kMostCopyThreads = 256;

__device__ __forceinline__ int lane_id() { return threadIdx.x & 63; }
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
// Bits of the lanes before this one.
__device__ __forceinline__ int bits_before(uint64_t mask) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

__device__ __forceinline__ int last_lane(int v) { return __builtin_amdgcn_readlane(v, 63); }

// Sum over the waves before this one of what each brings (the same in its lanes), and
// over all; `meet` holds kWaves words.
__device__ __forceinline__ int waves_before(int v, int* meet, int& all) {
    const int lane = lane_id(), wave = wave_id();
    __syncthreads();
    if (lane == 0) meet[wave] = v;
    __syncthreads();
    const int upto = running_sum(lane < kWaves ? meet[lane] : 0);
    all = last_lane(upto);
    return __builtin_amdgcn_readlane(upto, wave) - v;
}
// Over the threads before this one, and over all.
__device__ __forceinline__ int block_before(int v, int* meet, int& all) {
    const int upto = running_sum(v);
    return waves_before(last_lane(upto), meet, all) + upto - v;
}
// How many threads before this one say yes, and how many do.
__device__ __forceinline__ int block_rank(bool yes, int* meet, int& all) {
    const uint64_t mask = __ballot(yes);
    const int before = waves_before(__popcll(mask), meet, all);
    return before + bits_before(mask);
}
// Sum over the workgroup's threads, the same in all of them.
__device__ __forceinline__ int block_sum(int v, int* meet) {
    int all;
    waves_before(last_lane(running_sum(v)), meet, all);
    return all;
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
    // Free ones among the first n.
    __device__ __forceinline__ int count_below(int n) const {
        int sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int edge = n - 64 * i;  // bits below it count
            sum += __popcll(free[i] & (edge <= 0 ? 0 : edge >= 64 ? ~uint64_t(0) : (uint64_t(1) << edge) - 1));
        }
        return sum;
    }
};

// Writes the free pages of rank below `limit` to list[rank]; `before`: the rank of the
// group's first one.
__device__ __forceinline__ void list_group(const Group& g, int group, int before, int limit, int32_t* list) {
    const int lane = lane_id();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int rank = before + bits_before(g.free[i]);
        if (g.there[i] == 0 && rank < limit) list[rank] = group * kGroup + 64 * i + lane;
        before += __popcll(g.free[i]);
    }
}

// Few: all groups of the pool, wave w's being w, w + kWaves, ...
struct Groups {
    static constexpr int kMost = kFewPages / kGroup, kEach = kMost / kWaves;
    static_assert(kMost == 64, "one of a lane");
    Group x[kEach];
    int upto;  // lane g: free pages up to and with group g
    __device__ __forceinline__ void load(const int32_t* users, int pages) {
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            x[k] = Group{{}, {-1, -1, -1, -1}};
            if (group(k) * kGroup < pages) x[k].load(users, pages, group(k));
        }
    }
    // (before a barrier; sum() after it)
    __device__ __forceinline__ void tell(int* counts) const {
        const int wave = wave_id();
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            if (lane_id() == 0) counts[wave + kWaves * k] = x[k].count();
    }
    __device__ __forceinline__ int sum(const int* counts) {
        upto = running_sum(counts[lane_id()]);
        return last_lane(upto);
    }
    __device__ __forceinline__ int group(int k) const { return wave_id() + kWaves * k; }
    __device__ __forceinline__ int before(int k) const { return __builtin_amdgcn_readlane(upto, group(k)) - x[k].count(); }
    // The free pages of ranks below `limit`, in order.
    __device__ __forceinline__ void list(int limit, int32_t* to) const {
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int first = before(k);
            if (x[k].count() && first < limit) list_group(x[k], group(k), first, limit, to);
        }
    }
};

// The sum of counts[first .. at), fewer than 64 (one wave).
__device__ __forceinline__ int sum_between(const int32_t* counts, int first, int at) {
    return last_lane(running_sum(first + lane_id() < at ? counts[first + lane_id()] : 0));
}

// The sum of counts[0 .. n) by one workgroup.
__device__ __forceinline__ int sum_of(const int32_t* counts, int n, int* meet) {
    int sum = 0;
    for (int i = (int)threadIdx.x; i < n; i += kThreads) sum += counts[i];
    return block_sum(sum, meet);
}

// ---- resize ----

struct ResizeArgs {
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* cached;  // may be null
    const int32_t* users;
    int32_t* new_table;
    int32_t* new_users;
    int32_t* missing;
    // many:
    int32_t* want;    // [batch]: pages that a row lacks
    int32_t* start;   // [batch]: those of the rows before it
    int32_t* free;    // [1]: free pages, no more than the list holds
    int32_t* counts;  // [groups]
    int32_t* list;    // free pages in order
    int64_t table_stride;
    int batch, width, pages, page_shift, most;  // most: entries of the list
    int list_blocks;
    Divisor by_width;
};

// The first column of row b that may be given a page: those before it hold cached
// positions, and a page given there would hold what another sequence left in it.
__device__ __forceinline__ int first_given(const ResizeArgs& a, int b) {
    return a.cached ? pages_needed(a.cached[b], a.page_shift) : 0;
}

// 256 columns of a row from c0, below `end`, by one wave.  (Columns go up to 2^31 - 1, and
// the ones looked at past the last go by: they are counted in 32 bits without a sign.)
struct Columns {
    int entry[4];
    __device__ __forceinline__ void load(const int32_t* row, uint32_t c0, uint32_t end) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t c = c0 + 64 * i + lane_id();
            entry[i] = c < end ? row[c] : -1;
        }
    }
};

// Entries in [from, upto), of column `given` or a later one, that name no page (one
// wave); `x`: the first 256 columns.
__device__ __forceinline__ int lacking(const ResizeArgs& a, const int32_t* row, uint32_t from, uint32_t upto, uint32_t given,
                                       Columns x) {
    int lacks = 0;
    for (uint32_t c0 = from; c0 < upto; c0 += 256) {
        if (c0 > from) x.load(row, c0, upto);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t c = c0 + 64 * i + lane_id();
            lacks += __popcll(__ballot(c >= given && c < upto && !names_page(x.entry[i], a.pages)));
        }
    }
    return lacks;
}

// The new entries of columns [from, end) of row b (one wave): free pages from rank
// `start` on where one is wanted (list[rank], below `free`; from column `given` on), none
// behind the length.
// With kCount the users of pages given and given up change besides.  `x`: the first of
// the columns.  Returns how many entries name a page.
template <bool kCount>
__device__ __forceinline__ int resize_columns(const ResizeArgs& a, int b, uint32_t from, uint32_t end, int64_t start, int free,
                                              const int32_t* list, int length, uint32_t given, Columns x) {
    const uint32_t upto = pages_wanted(length, a.page_shift, a.width), reach = upto < end ? upto : end;
    const int32_t* row = a.table + b * a.table_stride;
    int32_t* to = a.new_table + (int64_t)b * a.width;
    int held = 0;
    for (uint32_t c0 = from; c0 < end; c0 += 256) {
        if (c0 > from) x.load(row, c0, end);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t c = c0 + 64 * i + lane_id();
            const bool named = names_page(x.entry[i], a.pages);
            const uint64_t wants = __ballot(c >= given && c < reach && !named);
            int e = named ? x.entry[i] : -1;
            if (c >= upto) {
                if (kCount && named) atomicAdd(a.new_users + e, -1);
                e = -1;
            } else if (!named && c >= given && c < end) {
                const int64_t rank = start + bits_before(wants);
                if (rank < free) {
                    e = list[rank];
                    if (kCount) atomicAdd(a.new_users + e, 1);
                }
            }
            if (c < end) to[c] = e;
            held += __popcll(__ballot(e >= 0));
            start += __popcll(wants);
        }
    }
    return held;
}

// Few: use(b, c, length of b, entry) for all entries of the table, by one workgroup;
// eight loads of a thread on their way at once.
template <class Args, class F>
__device__ __forceinline__ void each_entry(const Args& a, int entries, F use) {
    constexpr int kAtOnce = 8;
    for (int base = 0; base < entries; base += kAtOnce * kThreads) {
        int row[kAtOnce], column[kAtOnce], length[kAtOnce], entry[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int at = base + i * kThreads + (int)threadIdx.x;
            row[i] = a.by_width(min(at, entries - 1)), column[i] = at - row[i] * a.width;
            length[i] = a.lengths[row[i]];
            entry[i] = column[i] < a.width ? a.table[row[i] * a.table_stride + column[i]] : -1;
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
            if (column[i] < a.width) use(row[i], column[i], length[i], entry[i]);
    }
}

// Few.  The first workgroup writes the users, every other one kWaves rows.  (kCached: with
// cached positions; a form without them, which costs a call 0.2 us less.)
template <bool kCached>
__global__ __launch_bounds__(kThreads) void resize_few_kernel(ResizeArgs a) {
    __shared__ int counts[Groups::kMost], want[kFewRows], given[kFewPages];
    const int tid = (int)threadIdx.x;
    // what this wave's row needs at the end is on its way from the start
    const int b = ((int)blockIdx.x - 1) * kWaves + wave_id();
    const bool mine = blockIdx.x > 0 && b < a.batch;
    Columns row{};
    if (mine) row.load(a.table + b * a.table_stride, 0, a.width);
    const int row_length = mine ? a.lengths[b] : 0, row_given = kCached && mine ? first_given(a, b) : 0;
    Groups free_pages;
    free_pages.load(a.users, a.pages);
    want[tid] = 0;
    if (blockIdx.x == 0)  // there: less those given up
        for (int p = tid; p < a.pages; p += kThreads) given[p] = 0;
    free_pages.tell(counts);
    __syncthreads();
    const int entries = a.batch * a.width;
    const bool first = blockIdx.x == 0;
    each_entry(a, entries, [&](int b, int c, int length, int entry) {
        const bool named = names_page(entry, a.pages);
        if (c < pages_needed(length, a.page_shift)) {
            if (!named && (!kCached || c >= first_given(a, b))) atomicAdd(want + b, 1);
        } else if (first && named) {
            atomicAdd(given + entry, -1);
        }
    });
    __syncthreads();
    // rows' wants before this wave's row, and all
    int start = 0, wanted = 0;
    for (int i = lane_id(); i < a.batch; i += 64) {
        const int w = want[i];
        wanted += w;
        start += i < b ? w : 0;
    }
    start = last_lane(running_sum(start)), wanted = last_lane(running_sum(wanted));
    const int free = min(free_pages.sum(counts), wanted);
    if (first) {
#pragma unroll
        for (int k = 0; k < Groups::kEach; ++k) {
            const Group& x = free_pages.x[k];
            if (free_pages.group(k) * kGroup >= a.pages) break;
            int before = free_pages.before(k);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int p = free_pages.group(k) * kGroup + 64 * i + lane_id();
                const bool taken = x.there[i] == 0 && before + bits_before(x.free[i]) < free;
                if (p < a.pages) a.new_users[p] = x.there[i] + given[p] + taken;
                before += __popcll(x.free[i]);
            }
        }
        return;
    }
    free_pages.list(free, given);
    __syncthreads();
    if (!mine) return;
    const int held = resize_columns<false>(a, b, 0, a.width, start, free, given, row_length, row_given, row);
    if (lane_id() == 0) a.missing[b] = pages_needed(row_length, a.page_shift) - held;
}

// Many.  A row by a workgroup of kRowWaves, each a part of its columns.
constexpr int kRowWaves = 8;
// Rows' wants by the first workgroups, pages' counts by the others.
__global__ __launch_bounds__(64 * kRowWaves) void resize_count_kernel(ResizeArgs a) {
    __shared__ int meet[kRowWaves];
    if ((int)blockIdx.x < a.batch) {
        const int b = (int)blockIdx.x, wave = wave_id(), lane = lane_id();
        const ColumnPart part = column_part(a.width, wave, kRowWaves);
        const int32_t* row = a.table + b * a.table_stride;
        Columns first;
        first.load(row, part.from, part.end);
        const int upto = min(part.end, pages_wanted(a.lengths[b], a.page_shift, a.width));
        const int lacks = lacking(a, row, part.from, upto, first_given(a, b), first);
        if (lane == 0) meet[wave] = lacks;
        __syncthreads();
        int all = 0;
        for (int w = 0; w < kRowWaves; ++w) all += meet[w];
        if (threadIdx.x == 0) a.want[b] = all;
        return;
    }
    const int g = ((int)blockIdx.x - a.batch) * kRowWaves + wave_id();
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

// The free pages in order (as many as there are entries), and the rows' starts.
__global__ __launch_bounds__(kThreads) void resize_list_kernel(ResizeArgs a) {
    __shared__ int meet[kWaves];
    const int groups = (a.pages + kGroup - 1) / kGroup;
    if ((int)blockIdx.x < a.list_blocks) {
        const int first = (int)blockIdx.x * kWaves, g = first + wave_id();
        int before = sum_of(a.counts, first, meet);
        if (before >= a.most || g >= groups) return;
        before += sum_between(a.counts, first, g);
        Group x;
        x.load(a.users, a.pages, g);
        list_group(x, g, before, a.most, a.list);
        return;
    }
    const int first = ((int)blockIdx.x - a.list_blocks) * kThreads;
    const int before = sum_of(a.want, first, meet), b = first + (int)threadIdx.x;
    int all;
    const int start = before + block_before(b < a.batch ? a.want[b] : 0, meet, all);
    if (b < a.batch) a.start[b] = start;
    if (first == 0) {
        const int free = sum_of(a.counts, groups, meet);
        if (threadIdx.x == 0) *a.free = min(free, a.most);
    }
}

__global__ __launch_bounds__(64 * kRowWaves) void resize_apply_kernel(ResizeArgs a) {
    __shared__ int meet[kRowWaves];
    const int b = (int)blockIdx.x, wave = wave_id(), lane = lane_id();
    const ColumnPart part = column_part(a.width, wave, kRowWaves);
    const int32_t* row = a.table + b * a.table_stride;
    Columns first;
    first.load(row, part.from, part.end);
    const int free = *a.free, length = a.lengths[b], given = first_given(a, b);
    int64_t start = a.start[b];
    const int lacks = lacking(a, row, part.from, min(part.end, pages_wanted(length, a.page_shift, a.width)), given, first);
    if (lane == 0) meet[wave] = lacks;
    __syncthreads();
    for (int w = 0; w < wave; ++w) start += meet[w];
    __syncthreads();
    const int held = resize_columns<true>(a, b, part.from, part.end, start, free, a.list, length, given, first);
    if (lane == 0) meet[wave] = held;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < kRowWaves; ++w) all += meet[w];
    if (threadIdx.x == 0) a.missing[b] = pages_needed(length, a.page_shift) - all;
}

// ---- copies between pages ----

struct Pool {
    uint16_t* data[2];  // keys, values
    int64_t layer[2], page[2], head[2], position[2];
    int layers, pieces;  // 16-byte pieces of a position
    int kv_heads, page_size;
    int threads;         // that copy a page together: so many that each has kAtOnce pieces, a wave at least
};
constexpr int kAtOnce = 4;  // loads of a thread on their way

// `count` positions of a page of one layer (keys or values) to another page, by
// p.threads threads: pieces in the order of the larger stride.  Past the caches, as
// nothing reads them again soon: 256 MB (977 pages of 8 layers) take 53.8 us so, 60.0
// through them.
__device__ __forceinline__ void copy_page(const Pool& p, int which, int layer, int from, int to, int count) {
    const int tid = (int)threadIdx.x & (p.threads - 1);
    const uint16_t* base = p.data[which] + layer * p.layer[which];
    const uint16_t* source = base + from * p.page[which];
    uint16_t* target = const_cast<uint16_t*>(base) + to * p.page[which];
    const bool by_head = p.head[which] >= p.position[which];
    const int inner = by_head ? count : p.kv_heads;
    const int64_t inner_step = by_head ? p.position[which] : p.head[which];
    const int64_t outer_step = by_head ? p.head[which] : p.position[which];
    const int total = p.kv_heads * count * p.pieces;
    for (int first = tid; first < total; first += kAtOnce * p.threads) {
        u32x4 x[kAtOnce];
        int64_t at[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int piece = first + i * p.threads;
            const int row = piece / p.pieces, d = piece - row * p.pieces;
            const int outer = row / inner;
            at[i] = outer * outer_step + (row - outer * inner) * inner_step + 8 * d;
            if (piece < total) x[i] = __builtin_nontemporal_load((const u32x4*)(source + at[i]));
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
            if (first + i * p.threads < total) __builtin_nontemporal_store(x[i], (u32x4*)(target + at[i]));
    }
}

// The copies of a workgroup of kThreads: `blocks` such workgroups go through `items`.
template <class F>
__device__ __forceinline__ void each_copy(const Pool& p, int64_t items, int block, int blocks, F copy) {
    const int together = kThreads / p.threads;
    for (int64_t item = (int64_t)block * together + __builtin_amdgcn_readfirstlane((int)threadIdx.x / p.threads); item < items;
         item += (int64_t)blocks * together) {
        const int r = (int)(item / (2 * p.layers)), rest = (int)(item - (int64_t)r * 2 * p.layers);
        copy(r, rest & 1, rest >> 1);
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
    // many:
    int32_t* first;   // [batch]: a row's first child (children if it has none)
    int32_t* born;    // [batch]: how many it has
    int32_t* rank;    // [children]: of a child's copy among those of its kThreads children, -1 if it has none
    int32_t* copies;  // [children / kThreads]
    int32_t* free;    // [1]: free pages, no more than the list holds
    int32_t* counts;  // [groups]
    int32_t* list;    // [children]: free pages
    int64_t table_stride;
    int batch, children, width, pages, page_shift;
    int chunks;       // of 256 columns in a row
    int list_blocks, row_blocks, old_blocks, copy_blocks;
    Divisor by_width;
};

// What a fork asks of an old row: its length, and its last page if that is there and not
// full (column -1 if not).
struct Old {
    int length, column, page;
    bool sole;  // only this row names that page
};
__device__ __forceinline__ Old old_row(const ForkArgs& a, int b) {
    Old r;
    r.length = max(a.lengths[b], 0);
    r.column = r.length >> a.page_shift;
    r.page = -1;
    if ((r.length & ((1 << a.page_shift) - 1)) && r.column < a.width) r.page = a.table[b * a.table_stride + r.column];
    if (!names_page(r.page, a.pages)) r.column = -1;
    r.sole = r.column >= 0 && a.users[r.page] == 1;
    return r;
}

// A chunk of row i of the answer, columns from c0 (one wave), a copy of row `parent` (-1:
// none); `target`: the page of its copy, -1 if it has none, -2 where none was free.
template <bool kCount>
__device__ __forceinline__ void fork_chunk(const ForkArgs& a, int i, int c0, int parent, int length, int target) {
    const int upto = pages_wanted(length, a.page_shift, a.width);
    const int column = length >> a.page_shift;  // (where there is a copy)
    const int32_t* row = a.table + max(parent, 0) * a.table_stride;
    Columns x;
    x.load(row, c0, upto);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int c = c0 + 64 * k + lane_id();
        int e = names_page(x.entry[k], a.pages) ? x.entry[k] : -1;
        if (target != -1 && c == column) {
            e = target < 0 ? -1 : target;
            if (kCount && e >= 0) atomicAdd(a.new_users + e, 1);
        }
        if (c < a.width) a.new_table[(int64_t)i * a.width + c] = e;
    }
    if (c0 == 0 && lane_id() == 0) {
        a.new_lengths[i] = length;
        a.missing[i] = target == -2;
    }
}

// By what the users of column c's page of an old row change: children that hold it less
// the row itself.
__device__ __forceinline__ int fork_change(int c, int upto, int column, int born, bool kept) {
    return (c == column ? kept : c < upto ? born : 0) - 1;
}

// Few.  The first workgroup writes the users, the next row_blocks new rows, the others
// copy.
__global__ __launch_bounds__(kThreads) void fork_few_kernel(ForkArgs a) {
    // of children: parent[], length[], target[]; of copies: source[], filled[], list[]
    __shared__ int meet[kWaves], counts[Groups::kMost], first[kFewRows], born[kFewRows], parent[kFewRows], length[kFewRows],
        target[kFewRows], source[kFewRows], filled[kFewRows], list[kFewRows], change[kFewPages];
    const int tid = (int)threadIdx.x;
    int block = (int)blockIdx.x;
    // thread t: child t and, in the first workgroup, row t of the old batch
    int mine = tid < a.children ? a.parents[tid] : -1;
    if (mine >= a.batch) mine = -1;
    Groups free_pages;
    free_pages.load(a.users, a.pages);
    Old from{0, -1, -1, false}, old{0, -1, -1, false};
    if (mine >= 0) from = old_row(a, mine);
    if (block == 0) {
        if (tid < a.batch) old = old_row(a, tid);
        for (int p = tid; p < a.pages; p += kThreads) change[p] = 0;
    }
    first[tid] = a.children, born[tid] = 0;
    parent[tid] = max(mine, -1), length[tid] = from.length;
    free_pages.tell(counts);
    __syncthreads();
    if (mine >= 0) {
        atomicMin(first + mine, tid);
        atomicAdd(born + mine, 1);
    }
    __syncthreads();
    const bool copy = from.column >= 0 && (first[mine] != tid || !from.sole);
    int copies;
    const int rank = block_rank(copy, meet, copies);
    const int free = min(free_pages.sum(counts), copies);
    free_pages.list(free, list);
    if (copy) source[rank] = from.page, filled[rank] = from.length;
    __syncthreads();
    target[tid] = !copy ? -1 : rank < free ? list[rank] : -2;
    if (block == 0) {
        // (now of the old batch's rows: entries in use, the last page's column, and whether a
        // child keeps it)
        first[tid] = pages_wanted(old.length, a.page_shift, a.width), source[tid] = old.column;
        filled[tid] = old.sole && born[tid] > 0;
        if (tid < free) change[list[tid]] = 1;
        __syncthreads();
        const int entries = a.batch * a.width;
        each_entry(a, entries, [&](int b, int c, int, int entry) {
            const int by = fork_change(c, first[b], source[b], born[b], filled[b]);
            if (by && names_page(entry, a.pages)) atomicAdd(change + entry, by);
        });
        __syncthreads();
        for (int p = tid; p < a.pages; p += kThreads) a.new_users[p] = a.users[p] + change[p];
        return;
    }
    __syncthreads();
    if (--block < a.row_blocks) {
        const int item = block * kWaves + wave_id(), i = item / a.chunks;
        if (i < a.children) fork_chunk<false>(a, i, 256 * (item - i * a.chunks), parent[i], length[i], target[i]);
        return;
    }
    each_copy(a.pool, (int64_t)free * 2 * a.pool.layers, block - a.row_blocks, a.copy_blocks, [&](int r, int which, int layer) {
        copy_page(a.pool, which, layer, source[r], list[r], filled[r] & ((1 << a.page_shift) - 1));
    });
}

// Many.  Rows' children by the first workgroup, pages' counts by the others.
__global__ __launch_bounds__(kThreads) void fork_count_kernel(ForkArgs a) {
    const int tid = (int)threadIdx.x, lane = lane_id();
    if (blockIdx.x > 0) {
        const int g = ((int)blockIdx.x - 1) * kWaves + wave_id();
        if ((int64_t)g * kGroup >= a.pages) return;
        Group x;
        x.load(a.users, a.pages, g);
        if (lane == 0) a.counts[g] = x.count();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t p = (int64_t)g * kGroup + 64 * i + lane;
            if (p < a.pages) a.new_users[p] = x.there[i];
        }
        return;
    }
    for (int b = tid; b < a.batch; b += kThreads) a.first[b] = a.children, a.born[b] = 0;
    __syncthreads();
    for (int base = 0; base < a.children; base += 8 * kThreads) {
        int parent[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = base + k * kThreads + tid;
            parent[k] = i < a.children ? a.parents[i] : -1;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool there = parent[k] >= 0 && parent[k] < a.batch;
            const uint64_t all = __ballot(there);
            if (!all) continue;
            // (children of one row side by side go as one: 100000 of one row take 2800 us otherwise)
            const int head = __ffsll((unsigned long long)all) - 1;
            const bool alike = __ballot(there && parent[k] != __builtin_amdgcn_readlane(parent[k], head)) == 0;
            if (alike ? lane == head : there) {
                atomicMin(a.first + parent[k], base + k * kThreads + tid);
                atomicAdd(a.born + parent[k], alike ? __popcll(all) : 1);
            }
        }
    }
}

// Which children copy, and the free pages in order (as many as there are children).
__global__ __launch_bounds__(kThreads) void fork_list_kernel(ForkArgs a) {
    __shared__ int meet[kWaves];
    const int groups = (a.pages + kGroup - 1) / kGroup;
    if ((int)blockIdx.x < a.list_blocks) {
        const int first = (int)blockIdx.x * kWaves, g = first + wave_id();
        int before = sum_of(a.counts, first, meet);
        if (before >= a.children || g >= groups) return;
        before += sum_between(a.counts, first, g);
        Group x;
        x.load(a.users, a.pages, g);
        list_group(x, g, before, a.children, a.list);
        return;
    }
    const int block = (int)blockIdx.x - a.list_blocks, i = block * kThreads + (int)threadIdx.x;
    bool copy = false;
    if (i < a.children) {
        const int parent = a.parents[i];
        if (parent >= 0 && parent < a.batch) {
            const Old from = old_row(a, parent);
            copy = from.column >= 0 && (a.first[parent] != i || !from.sole);
        }
    }
    int copies;
    const int rank = block_rank(copy, meet, copies);
    if (i < a.children) a.rank[i] = copy ? rank : -1;
    if (threadIdx.x == 0) a.copies[block] = copies;
    if (block == 0) {
        const int free = sum_of(a.counts, groups, meet);
        if (threadIdx.x == 0) *a.free = min(free, a.children);
    }
}

// The page of child i's copy, as fork_chunk() takes it (one wave).
__device__ __forceinline__ int target_of(const ForkArgs& a, int i) {
    const int mine = a.rank[i], free = *a.free;
    if (mine < 0) return -1;
    int before = 0;
    for (int b = lane_id(); b < i / kThreads; b += 64) before += a.copies[b];
    const int rank = last_lane(running_sum(before)) + mine;
    return rank < free ? a.list[rank] : -2;
}

// Workgroups of three kinds: new rows, a chunk a wave; old rows' users, so too; copies.
__global__ __launch_bounds__(kThreads) void fork_apply_kernel(ForkArgs a) {
    const int block = (int)blockIdx.x;
    if (block < a.row_blocks + a.old_blocks) {
        const int item = (block < a.row_blocks ? block : block - a.row_blocks) * kWaves + wave_id();
        const int i = item / a.chunks, c0 = 256 * (item - i * a.chunks);
        if (block < a.row_blocks) {
            if (i >= a.children) return;
            const int parent = a.parents[i];
            const bool there = parent >= 0 && parent < a.batch;
            fork_chunk<true>(a, i, c0, there ? parent : -1, there ? max(a.lengths[parent], 0) : 0, target_of(a, i));
            return;
        }
        if (i >= a.batch) return;
        Columns x;
        x.load(a.table + i * a.table_stride, c0, a.width);
        const int born = a.born[i];
        const Old old = old_row(a, i);
        const int upto = pages_wanted(old.length, a.page_shift, a.width);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int by = fork_change(c0 + 64 * k + lane_id(), upto, old.column, born, old.sole && born > 0);
            if (by && names_page(x.entry[k], a.pages)) atomicAdd(a.new_users + x.entry[k], by);
        }
        return;
    }
    each_copy(a.pool, (int64_t)a.children * 2 * a.pool.layers, block - a.row_blocks - a.old_blocks, a.copy_blocks,
              [&](int i, int which, int layer) {
                  const int target = target_of(a, i);
                  if (target < 0) return;
                  const int parent = a.parents[i], length = a.lengths[parent];
                  copy_page(a.pool, which, layer, a.table[parent * a.table_stride + (length >> a.page_shift)], target,
                            length & ((1 << a.page_shift) - 1));
              });
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
    // many:
    int32_t* fate;    // [pages]
    int32_t* counts;  // [groups]
    int32_t* holes;   // [pages / 2]
    int32_t* movers;  // [pages / 2]
    int32_t* moves;   // [1]
    int64_t table_stride;
    int batch, width, pages;
    int page_blocks, table_blocks, copy_blocks;
    Divisor by_width;
};

// A group's pages; `before`: the free pages before it, `live`: all in use, `low`: free
// pages below `live`.
__device__ __forceinline__ void settle_group(const CompactArgs& a, const Group& g, int group, int before, int live, int low) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t p64 = (int64_t)group * kGroup + 64 * i + lane_id();
        const int free_before = before + bits_before(g.free[i]);
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
    return before + x.count_below(live % kGroup);
}

// Few: `to` says where a page lies now: kFree, or the page, or kRank and its rank among
// those that move.  The first workgroup writes what is said of pages, the next
// table_blocks table entries, the others copy.
// (two workgroups a CU copy faster than one: eight waves a SIMD, no more scalar registers
// than that leaves)
__global__ __launch_bounds__(kThreads, 8) void compact_few_kernel(CompactArgs a) {
    constexpr uint16_t kFree = 0xFFFF, kRank = 0x8000;
    static_assert(kFewPages / 2 + kRank < kFree && kFewPages <= kRank, "all told apart");
    __shared__ int counts[Groups::kMost], below[kWaves];
    __shared__ uint16_t to[kFewPages], holes[kFewPages / 2], movers[kFewPages / 2];
    const int tid = (int)threadIdx.x;
    Groups all;
    all.load(a.users, a.pages);
    all.tell(counts);
    __syncthreads();
    const int live = a.pages - all.sum(counts);
    // free pages below `live`: those of the groups before its own, and of that one's first pages
    int low = 0;
#pragma unroll
    for (int k = 0; k < Groups::kEach; ++k)
        if (all.group(k) == live / kGroup) low = all.before(k) + all.x[k].count_below(live % kGroup);
    const int wave = wave_id();
    if (lane_id() == 0) below[wave] = low;
    __syncthreads();
    low = live < kFewPages ? below[live / kGroup % kWaves] : 0;  // (no group is left: none is free)
#pragma unroll
    for (int k = 0; k < Groups::kEach; ++k) {
        const Group& x = all.x[k];
        if (all.group(k) * kGroup >= a.pages) break;
        int before = all.before(k);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = all.group(k) * kGroup + 64 * i + lane_id();
            const int free_before = before + bits_before(x.free[i]);
            before += __popcll(x.free[i]);
            if (p >= a.pages) continue;
            if (x.there[i] == 0) {
                to[p] = kFree;
                if (p < live) holes[free_before] = (uint16_t)p;
            } else if (p < live) {
                to[p] = (uint16_t)p;
            } else {
                const int rank = p - free_before - (live - low);
                to[p] = (uint16_t)(kRank + rank);
                movers[rank] = (uint16_t)p;
            }
        }
    }
    __syncthreads();
    auto place = [&](int p) {
        const uint16_t t = to[p];
        return t == kFree ? -1 : t >= kRank ? (int)holes[t - kRank] : (int)t;
    };
    int block = (int)blockIdx.x;
    if (block == 0) {
        for (int p = tid; p < a.pages; p += kThreads) {
            const int now = place(p);
            a.moved_to[p] = now;
            if (now >= 0) a.new_users[now] = a.users[p];
            if (p >= live) a.new_users[p] = 0;
        }
        return;
    }
    if (--block < a.table_blocks) {
        for (int64_t at = (int64_t)block * kThreads + tid; at < (int64_t)a.batch * a.width; at += (int64_t)a.table_blocks * kThreads) {
            const int b = a.by_width((int)at), e = a.table[b * a.table_stride + ((int)at - b * a.width)];
            a.new_table[at] = names_page(e, a.pages) ? place(e) : -1;
        }
        return;
    }
    each_copy(a.pool, (int64_t)low * 2 * a.pool.layers, block - a.table_blocks, a.copy_blocks, [&](int r, int which, int layer) {
        copy_page(a.pool, which, layer, movers[r], holes[r], a.pool.page_size);
    });
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
    before += sum_between(a.counts, first, g);
    Group x;
    x.load(a.users, a.pages, g);
    settle_group(a, x, g, before, live, low);
}

// Pages by the first workgroups, then table entries, then copies.
__global__ __launch_bounds__(kThreads) void compact_apply_kernel(CompactArgs a) {
    int block = (int)blockIdx.x;
    auto place = [&](int p) {
        const int32_t f = a.fate[p];
        return f == kStays ? p : f >= kMoves && f < kHole ? a.holes[f - kMoves] : -1;
    };
    if (block < a.page_blocks) {
        const int64_t p = (int64_t)block * kThreads + threadIdx.x;
        if (p >= a.pages) return;
        const int32_t f = a.fate[p];
        a.moved_to[p] = place((int)p);
        a.new_users[p] = f == kStays ? a.users[p] : f >= kHole ? a.users[a.movers[f - kHole]] : 0;
        return;
    }
    block -= a.page_blocks;
    if (block < a.table_blocks) {
        const int64_t at = (int64_t)block * kThreads + threadIdx.x;
        if (at >= (int64_t)a.batch * a.width) return;
        const int b = a.by_width((int)at), e = a.table[b * a.table_stride + ((int)at - b * a.width)];
        a.new_table[at] = names_page(e, a.pages) ? place(e) : -1;
        return;
    }
    each_copy(a.pool, (int64_t)*a.moves * 2 * a.pool.layers, block - a.table_blocks, a.copy_blocks, [&](int r, int which, int layer) {
        copy_page(a.pool, which, layer, a.movers[r], a.holes[r], a.pool.page_size);
    });
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
                 {p->k_position, p->v_position}, (int)p->layers, (int)(p->head_dim / 8), (int)p->kv_heads, (int)p->page_size, 64};
    while (view->threads < kMostCopyThreads && view->threads * kAtOnce < p->kv_heads * p->page_size * p->head_dim / 8) view->threads *= 2;
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

// Whether a resize's or fork's sizes are few; a compaction's are where the pages are.
bool few(int64_t rows, int64_t width, int64_t pages, int64_t entries) {
    return rows <= kFewRows && rows * width <= entries && pages <= kFewPages;
}
// (and a fork's new rows keep no more workgroups busy than run at once: each plans)
bool few_fork(int64_t batch, int64_t children, int64_t width, int64_t pages) {
    return few(batch, width, pages, kFewFork) && children <= kFewRows && children * blocks_of(width, 256) <= 256 * kWaves;
}
// Workgroups for `items` copies at most: two a CU, or as many as have something to do.
int copy_blocks(const Pool& pool, int64_t items) {
    const int64_t blocks = blocks_of(items, kThreads / pool.threads);
    return (int)(blocks < 512 ? blocks : 512);
}

}  // namespace

int paged_resize_sizes(int64_t batch, int64_t table_width, int64_t num_pages, int64_t page_size) {
    const int status = check_sizes("paged_resize", batch, table_width, num_pages);
    if (status) return status;
    if (shift_of(page_size) < 0)
        return set_error(W4G64_STATUS_INVALID_VALUE, "page_size must be a power of two in [16, 2^20], got %lld", (long long)page_size);
    return clear_error();
}

int paged_fork_sizes(const qwen2_page_pool* pool, int64_t batch, int64_t children, int64_t table_width) {
    Pool view;
    int status = pool_view("paged_fork", pool, &view);
    if (!status) status = check_sizes("paged_fork", batch, table_width, pool->num_pages);
    return status ? status : check_sizes("paged_fork", children, table_width, pool->num_pages);
}

int paged_compact_sizes(const qwen2_page_pool* pool, int64_t batch, int64_t table_width) {
    Pool view;
    const int status = pool_view("paged_compact", pool, &view);
    return status ? status : check_sizes("paged_compact", batch, table_width, pool->num_pages);
}

}  // namespace w4g64

using namespace w4g64;

extern "C" {

int64_t qwen2_paged_resize_workspace_bytes(int64_t batch, int64_t table_width, int64_t num_pages) {
    if (check_sizes("paged_resize", batch, table_width, num_pages)) return 0;
    return few(batch, table_width, num_pages, kFewResize) ? 0
                                              : 4 * (2 * batch + 1 + groups_of(num_pages) + most_given(batch, table_width, num_pages));
}

int qwen2_paged_resize(const int32_t* page_table, int64_t table_stride, const int32_t* lengths, const int32_t* page_users,
                       int32_t* new_table, int32_t* new_users, int32_t* missing, int64_t batch, int64_t table_width,
                       int64_t num_pages, int64_t page_size, void* workspace, int64_t workspace_bytes, void* stream) {
    return qwen2_paged_resize_cached(page_table, table_stride, lengths, nullptr, page_users, new_table, new_users, missing, batch,
                                     table_width, num_pages, page_size, workspace, workspace_bytes, stream);
}

int qwen2_paged_resize_cached(const int32_t* page_table, int64_t table_stride, const int32_t* lengths, const int32_t* cached,
                              const int32_t* page_users, int32_t* new_table, int32_t* new_users, int32_t* missing,
                              int64_t batch, int64_t table_width, int64_t num_pages, int64_t page_size, void* workspace,
                              int64_t workspace_bytes, void* stream) {
    int status = paged_resize_sizes(batch, table_width, num_pages, page_size);
    if (status) return status;
    if (!aligned4({page_users, new_users}) || (batch && !aligned4({page_table, lengths, new_table, missing})) ||
        ((uintptr_t)cached & 3))
        return set_error(W4G64_STATUS_INVALID_VALUE, "paged_resize pointers (`cached` alone may be null) must be non-null, 4-byte aligned device pointers");
    status = check_workspace("paged_resize", qwen2_paged_resize_workspace_bytes(batch, table_width, num_pages), workspace,
                             workspace_bytes);
    if (status) return status;
    ResizeArgs a{};
    a.table = page_table, a.table_stride = table_stride, a.lengths = lengths, a.cached = cached, a.users = page_users;
    a.new_table = new_table, a.new_users = new_users, a.missing = missing;
    a.batch = (int)batch, a.width = (int)table_width, a.pages = (int)num_pages, a.page_shift = shift_of(page_size);
    a.by_width = divisor(table_width);
    const hipStream_t s = (hipStream_t)stream;
    if (few(batch, table_width, num_pages, kFewResize)) {
        const dim3 grid((unsigned)(1 + blocks_of(batch, kWaves)));
        if (cached) hipLaunchKernelGGL(resize_few_kernel<true>, grid, dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL(resize_few_kernel<false>, grid, dim3(kThreads), 0, s, a);
        return launched("paged_resize");
    }
    a.want = (int32_t*)workspace, a.start = a.want + batch, a.free = a.start + batch, a.counts = a.free + 1;
    a.list = a.counts + groups_of(num_pages);
    a.most = (int)most_given(batch, table_width, num_pages);
    a.list_blocks = (int)blocks_of(groups_of(num_pages), kWaves);
    hipLaunchKernelGGL(resize_count_kernel, dim3((unsigned)(batch + blocks_of(groups_of(num_pages), kRowWaves))),
                       dim3(64 * kRowWaves), 0, s, a);
    if (batch) {
        hipLaunchKernelGGL(resize_list_kernel, dim3((unsigned)(a.list_blocks + blocks_of(batch, kThreads))), dim3(kThreads), 0, s, a);
        hipLaunchKernelGGL(resize_apply_kernel, dim3((unsigned)batch), dim3(64 * kRowWaves), 0, s, a);
    }
    return launched("paged_resize");
}

int64_t qwen2_paged_fork_workspace_bytes(int64_t batch, int64_t children, int64_t table_width, int64_t num_pages) {
    if (batch < 0 || children < 0 || table_width <= 0 || num_pages <= 0) return 0;
    if (few_fork(batch, children, table_width, num_pages)) return 0;
    return 4 * (2 * batch + 2 * children + blocks_of(children, kThreads) + 1 + groups_of(num_pages));
}

int qwen2_paged_fork(const qwen2_page_pool* pool, const int32_t* page_table, int64_t table_stride, const int32_t* lengths,
                     const int32_t* page_users, const int32_t* parents, int32_t* new_table, int32_t* new_lengths,
                     int32_t* new_users, int32_t* missing, int64_t batch, int64_t children, int64_t table_width,
                     void* workspace, int64_t workspace_bytes, void* stream) {
    ForkArgs a{};
    int status = paged_fork_sizes(pool, batch, children, table_width);
    if (status) return status;
    pool_view("paged_fork", pool, &a.pool);
    if (!aligned4({page_users, new_users}) || (batch && !aligned4({page_table, lengths})) ||
        (children && !aligned4({parents, new_table, new_lengths, missing})))
        return set_error(W4G64_STATUS_INVALID_VALUE, "paged_fork pointers must be non-null, 4-byte aligned device pointers");
    const int64_t copies = children * 2 * pool->layers;
    status = check_workspace("paged_fork", qwen2_paged_fork_workspace_bytes(batch, children, table_width, pool->num_pages), workspace,
                             workspace_bytes);
    if (status) return status;
    a.table = page_table, a.table_stride = table_stride, a.lengths = lengths, a.users = page_users, a.parents = parents;
    a.new_table = new_table, a.new_lengths = new_lengths, a.new_users = new_users, a.missing = missing;
    a.batch = (int)batch, a.children = (int)children, a.width = (int)table_width, a.pages = (int)pool->num_pages;
    a.page_shift = shift_of(pool->page_size), a.by_width = divisor(table_width);
    a.chunks = (int)blocks_of(table_width, 256);
    a.row_blocks = (int)blocks_of(children * a.chunks, kWaves), a.old_blocks = (int)blocks_of(batch * a.chunks, kWaves);
    a.copy_blocks = copy_blocks(a.pool, copies);
    const hipStream_t s = (hipStream_t)stream;
    if (few_fork(batch, children, table_width, pool->num_pages)) {
        hipLaunchKernelGGL(fork_few_kernel, dim3((unsigned)(1 + a.row_blocks + a.copy_blocks)), dim3(kThreads), 0, s, a);
        return launched("paged_fork");
    }
    const int64_t child_blocks = blocks_of(children, kThreads);
    a.list_blocks = (int)blocks_of(groups_of(pool->num_pages), kWaves);
    a.first = (int32_t*)workspace, a.born = a.first + batch, a.rank = a.born + batch, a.list = a.rank + children;
    a.copies = a.list + children, a.free = a.copies + child_blocks, a.counts = a.free + 1;
    hipLaunchKernelGGL(fork_count_kernel, dim3((unsigned)(1 + a.list_blocks)), dim3(kThreads), 0, s, a);
    if (children) hipLaunchKernelGGL(fork_list_kernel, dim3((unsigned)(a.list_blocks + child_blocks)), dim3(kThreads), 0, s, a);
    const int64_t blocks = a.row_blocks + a.old_blocks + a.copy_blocks;
    if (blocks) hipLaunchKernelGGL(fork_apply_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, s, a);
    return launched("paged_fork");
}

int64_t qwen2_paged_compact_workspace_bytes(int64_t batch, int64_t table_width, int64_t num_pages) {
    if (batch < 0 || table_width <= 0 || num_pages <= kFewPages) return 0;
    return 4 * (num_pages + groups_of(num_pages) + 2 * (num_pages / 2) + 1);
}

int qwen2_paged_compact(const qwen2_page_pool* pool, const int32_t* page_table, int64_t table_stride,
                        const int32_t* page_users, int32_t* new_table, int32_t* new_users, int32_t* moved_to, int64_t batch,
                        int64_t table_width, void* workspace, int64_t workspace_bytes, void* stream) {
    CompactArgs a{};
    int status = paged_compact_sizes(pool, batch, table_width);
    if (status) return status;
    pool_view("paged_compact", pool, &a.pool);
    if (!aligned4({page_users, new_users, moved_to}) || (batch && !aligned4({page_table, new_table})))
        return set_error(W4G64_STATUS_INVALID_VALUE, "paged_compact pointers must be non-null, 4-byte aligned device pointers");
    const int64_t pages = pool->num_pages;
    status = check_workspace("paged_compact", qwen2_paged_compact_workspace_bytes(batch, table_width, pages), workspace, workspace_bytes);
    if (status) return status;
    a.table = page_table, a.table_stride = table_stride, a.users = page_users;
    a.new_table = new_table, a.new_users = new_users, a.moved_to = moved_to;
    a.batch = (int)batch, a.width = (int)table_width, a.pages = (int)pages, a.by_width = divisor(table_width);
    const hipStream_t s = (hipStream_t)stream;
    const int64_t most = pages / 2 * 2 * pool->layers;  // copies that there can be
    if (pages <= kFewPages) {
        a.table_blocks = (int)std::min<int64_t>(blocks_of(batch * table_width, kThreads), 512);  // (each plans: as many as run at once)
        a.copy_blocks = copy_blocks(a.pool, most);
        hipLaunchKernelGGL(compact_few_kernel, dim3((unsigned)(1 + a.table_blocks + a.copy_blocks)), dim3(kThreads), 0, s, a);
        return launched("paged_compact");
    }
    a.fate = (int32_t*)workspace, a.counts = a.fate + pages, a.holes = a.counts + groups_of(pages);
    a.movers = a.holes + pages / 2, a.moves = a.movers + pages / 2;
    const unsigned lists = (unsigned)blocks_of(groups_of(pages), kWaves);
    hipLaunchKernelGGL(compact_count_kernel, dim3(lists), dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(compact_list_kernel, dim3(lists), dim3(kThreads), 0, s, a);
    a.copy_blocks = copy_blocks(a.pool, most);
    a.page_blocks = (int)blocks_of(pages, kThreads), a.table_blocks = (int)blocks_of(batch * table_width, kThreads);
    const int64_t blocks = a.page_blocks + a.table_blocks + a.copy_blocks;
    hipLaunchKernelGGL(compact_apply_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, s, a);
    return launched("paged_compact");
}

}  // extern "C"
