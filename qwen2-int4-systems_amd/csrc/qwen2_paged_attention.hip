// Attention over a paged cache, the batch's common prefix computed once
// (qwen2_paged_attention, include/qwen2_decode.h).
//
// Work.  A "row" here is a (packed row, query head) pair of one key/value head:
// row m of a segment is token m / group, head m % group.  Two kinds of segment
// share one launch:
//   prefix    all rows of the batch against the shared pages of the table's
//             first row: the keys are read once per tile of rows, not per sequence;
//   own       one sequence's rows against the rest of its pages.
// A workgroup of four waves takes a tile of a segment's rows and one of several
// splits of its keys, in one of two forms:
//   narrow    16 rows.  The waves take different 32-key blocks, straight from
//             memory into operands, and meet in LDS at the end: for few rows.
//   wide      128 rows, 32 of each wave.  The workgroup goes through 64-key tiles
//             in LDS, the next one on its way (direct loads) while the waves work
//             on this one: for many rows.
// A second launch joins the splits of both kinds of segment.
//
// What bounds it.  Narrow: the keys' and values' read (64 sequences of 1 K
// positions, 2 key/value heads of 128: 65 MB in 15.5 us, 4.2 TB/s) and, where that is
// little, 5-6 us of dependent loads, serial instructions and the join's 2-4.  Three
// workgroups a CU with one block in flight beat two with two (24 sequences of up
// to 2 K: 11.7 and 12.6 us).  Wide: matrix and vector unit, which overlap by a third
// only (two waves of a SIMD, 8 products and 32 additions each 64 and 70 ns alone, 100
// together; exponentials hide): 96 products and some 320 vector instructions a wave
// and tile.  1920 rows a key/value head over 16 K positions take 50 us beyond some 10
// for start and end, 640 TFLOP/s, at 1.9 to 2.0 GHz.  On the way, 64 x 5 rows, 12/2
// heads, 16 K shared and up to 1 K own positions, us per call: 160 narrow alone, 106 wide,
// 75 with values read transposed from LDS instead of permuted and masks in branches
// of their own, 69 with LDS reads issued ahead and the workgroups dealt out by time.
// Measured and dropped: 32-key wide tiles at three waves per SIMD (61 -> 64), wave
// priorities around the products and splits that keep a tile's keys on one XCD
// (no change), all keys in one workgroup of twelve waves instead of a join (1 x 576
// 8.7 -> 10.9; a CU draws some 60 GB/s).
//
// One pass over the keys: running maximum, sum and value sums per row.  MFMA
// layout (v_mfma_f32_16x16x32; lane l = 16 q + j supplies row j of A and column
// j of B with K slots 8 q .. 8 q + 7 and receives D[4 q + r][j]):
//   scores  A = 16 keys, B = 16 query rows: lane (j, q) gets row j's scores of
//           keys 4 q + r;
//   values  the lane's own 8 probabilities of a 32-key block are its 8 K slots;
//           A = the values transposed.  Narrow: lane (j, q) loads kVd = D / 16
//           dimensions from kVd j of its 8 keys and pairs keys up by v_perm;
//           dimension kVd j + dd is row j of the dd-th product.  Wide: LDS reads
//           that transpose; dimension 16 dd + j is row j of the dd-th product.
// A probability is kept as two 16-bit terms (16 bits or more of it): one term
// alone would be as coarse as the output.
//
// The sums are rescaled only once a score passes their reference by kLazy units
// of the base-2 exponent (from the floor on the first block); until then
// probabilities reach 2^kLazy times the reference's, which changes no relative
// rounding.
//
// Pages hold at least 16 positions, so that 16 aligned keys lie in one page and
// the page's number is the wave's, not the lane's.  Every loaded address lies in
// a page of the pool; what a block holds past the last visible key is replaced
// by zeros, scores there by -inf.
#include <math.h>

#include <type_traits>

#include "qwen2_attention.h"
#include "qwen2_paged_device.h"

namespace w4g64 {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kNarrowRows = 16;  // rows of a workgroup
constexpr int kWideRows = 128;
constexpr int kBlock = 32;       // keys of a narrow block
constexpr int kTileKeys = 64;    // keys of a wide tile
constexpr int kMaxSplits = 64;

struct PagedAttnArgs {
    PagedView c;
    const uint16_t* q;
    uint16_t* out;
    int64_t q_row, q_head, out_row, out_head;
    float* stats;         // [rows][heads][slots] (maximum, sum)
    float* partials;      // [rows][heads][slots][D]
    float scale2;         // |scale| * log2(e), above zero
    uint32_t query_sign;  // both signs of a word of queries where the scale is negative
    int rows, heads, group;
    int prefix;           // positions of the shared pages
    int prefix_tiles, prefix_splits, own_tiles, own_splits, slots;
    int prefix_wide, own_wide;
    int zero_rest;
    Divisor by_group, by_heads, by_kv_heads, by_prefix_splits, by_own_splits;
};

// The kernel's arguments, read anew: what only the end of a kernel needs is not
// held in scalar registers (and spilled) over its loop.
__device__ __forceinline__ PagedAttnArgs late_arguments() {
    typedef const __attribute__((address_space(4))) uint32_t* words_t;
    words_t p = (words_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    uint32_t w[sizeof(PagedAttnArgs) / 4];
#pragma unroll
    for (int i = 0; i < (int)(sizeof(w) / 4); ++i) w[i] = p[i];
    PagedAttnArgs a;
    static_assert(sizeof(w) == sizeof(a), "whole words");
    __builtin_memcpy(&a, w, sizeof(a));
    return a;
}

// An index array's entry at a wave's own index, through the scalar cache.
__device__ __forceinline__ int scalar_load(const int32_t* p, int64_t i) {
    return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)(p + i);
}

// Rows of a segment from which wide tiles are taken.  Main kernel, us, narrow /
// wide, 12/2 heads of 128: a prefix of 1 K by 96 rows 10.0 / 12.1, by 240 17.4 / 15.1,
// of 4 K by 96 17.3 / 22.3, by 192 16.0 / 15.2, by 240 31.0 / 25.0.  The bound is the
// prefix's.  Own segments go by it too, and lose by it between 128 and some 1000 rows
// a sequence (each form with its own splits, us per call): one sequence of 144 rows
// after 1 K positions 9.5 / 14.4, 240 11.8 / 15.5, 960 16.6 / 19.4; 2400 rows 15.0 / 17.7 after
// none, 35.0 / 27.7 after 1.6 K; 12000 rows 68.7 / 54.0 after none, 372 / 163 after 6 K; six
// sequences of 240 rows after 1 K 19.4 / 21.9, of 1200 after 700 36.5 / 30.9.
constexpr int kWideFrom = 128;
// Whether a sequence's own rows go by wide tiles, where the call has any.
__device__ __forceinline__ bool wide_rows(const PagedAttnArgs& a, int tokens) {
    return a.own_wide && tokens * a.group > kWideFrom;
}

// The sequence, its rows and the place of own tile `tile`: the tiles of every
// sequence counted up, 64 sequences at a time.  false: past the last one.
__device__ __forceinline__ bool find_tile(const PagedAttnArgs& a, int tile, int lane, int& sequence, int& local,
                                          SequenceRows& rows) {
    int before = 0;
    const int all = rows_end(a.c.cu_rows, a.c.batch, a.rows);
    for (int base = 0; base < a.c.batch; base += 64) {
        const int i = base + lane;
        SequenceRows s{0, 0, 0};
        if (i < a.c.batch) s = sequence_rows(a.c.cu_rows, a.c.lengths, i, all);
        const int tokens = s.end - s.begin;
        const int count = wide_rows(a, tokens) ? (tokens * a.group + kWideRows - 1) / kWideRows
                                               : (tokens * a.group + kNarrowRows - 1) / kNarrowRows;
        const int upto = before + running_sum(count);
        const uint64_t past = __ballot(upto > tile);
        if (past) {
            const int at = __ffsll((unsigned long long)past) - 1;
            sequence = base + at;
            local = tile - __builtin_amdgcn_readlane(upto - count, at);
            rows.begin = __builtin_amdgcn_readlane(s.begin, at);
            rows.end = __builtin_amdgcn_readlane(s.end, at);
            // (the length: at most 31 bits and a sign below the rows)
            rows.first = (int64_t)__builtin_amdgcn_readlane((int)(s.first + tokens), at) - (rows.end - rows.begin);
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// The sequence of a row by halving (cu_rows does not fall); batch if none.
__device__ __forceinline__ int sequence_by_halving(const int32_t* cu_rows, int batch, int row) {
    int lo = 0, hi = batch;  // the first sequence that ends past the row
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (cu_rows[mid + 1] <= row) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// What a workgroup works on.
struct Segment {
    bool shared, wide;
    bool sees_all;        // prefix: every row sees all of it
    int split, splits, kvh, tile;
    int first_token;
    int count;            // rows
    int64_t first;        // own: the first token's position
    int key_lo;
    int64_t key_end, held;
    const int32_t* table;
};

__device__ __forceinline__ bool find_segment(const PagedAttnArgs& a, int lane, Segment& s) {
    const int prefix_work = a.prefix_tiles * a.c.kv_heads * a.prefix_splits;
    s.shared = (int)blockIdx.x < prefix_work;
    const int work = s.shared ? (int)blockIdx.x : (int)blockIdx.x - prefix_work;
    s.splits = s.shared ? a.prefix_splits : a.own_splits;
    const int slot = s.shared ? a.by_prefix_splits(work) : a.by_own_splits(work);  // tile * kv_heads + kvh
    s.split = work - slot * s.splits;
    s.tile = a.by_kv_heads(slot);
    s.kvh = slot - s.tile * a.c.kv_heads;
    s.held = (int64_t)a.c.table_width << a.c.page_shift;
    s.sees_all = false;
    if (s.shared) {
        s.wide = a.prefix_wide;
        s.first_token = 0;
        // (rows behind the last sequence are not this kernel's to write)
        const int all = rows_end(a.c.cu_rows, a.c.batch, a.rows);
        s.count = all * a.group;
        if ((int64_t)s.tile * (s.wide ? kWideRows : kNarrowRows) >= s.count) return false;
        s.first = 0;
        s.key_lo = 0;
        s.key_end = a.prefix;
        s.table = a.c.table;
        // (the usual case, found out at once: all new positions lie behind the prefix)
        bool behind = a.own_splits > 0;
        for (int i = lane; i < a.c.batch; i += 64) {
            const SequenceRows r = sequence_rows(a.c.cu_rows, a.c.lengths, i, all);
            behind = behind && (r.end == r.begin || r.first >= a.prefix);
        }
        s.sees_all = __all(behind);
        return true;
    }
    int sequence;
    SequenceRows r;
    if (!find_tile(a, s.tile, lane, sequence, s.tile, r)) return false;
    s.wide = wide_rows(a, r.end - r.begin);
    s.first_token = r.begin;
    s.count = (r.end - r.begin) * a.group;
    s.first = r.first;
    s.key_lo = a.prefix;
    s.key_end = s.held;
    s.table = a.c.table + sequence * a.c.table_stride;
    return true;
}

// A row of a segment, as a lane holds it.
struct Row {
    int token, head;
    int limit;    // the last of the segment's keys that it sees, key_lo - 1 if none
    bool live;    // there is such a row
    bool beyond;  // it reaches past its table
};

__device__ __forceinline__ Row row_at(const PagedAttnArgs& a, const Segment& s, int m) {
    Row r;
    r.live = m < s.count;
    m = r.live ? m : s.count - 1;
    const int t = a.by_group(m);
    r.token = s.first_token + t;
    r.head = s.kvh * a.group + (m - t * a.group);
    r.beyond = false;
    if (s.sees_all) {
        r.limit = r.live ? (int)s.key_end - 1 : s.key_lo - 1;
        return r;
    }
    int64_t position = s.first + t;
    bool known = r.live;
    if (s.shared) {
        const int b = sequence_by_halving(a.c.cu_rows, a.c.batch, r.token);
        known = known && b < a.c.batch;
        if (known) {
            const SequenceRows q = sequence_rows(a.c.cu_rows, a.c.lengths, b, rows_end(a.c.cu_rows, a.c.batch, a.rows));
            known = r.token >= q.begin && r.token < q.end;
            position = q.first + (r.token - q.begin);
        }
    }
    if (!known) position = -1;  // (rows of no sequence see nothing)
    r.beyond = position >= s.held;
    r.limit = (int)max(min(position, s.key_end - 1), (int64_t)(s.key_lo - 1));
    return r;
}

// What the table says of a segment's 16 keys from t, the wave's own; keys that no
// row sees (t > most): any page.  (checked_page comes with the use, one round
// later: the load is not waited for here.)
__device__ __forceinline__ int table_entry(const PagedAttnArgs& a, const Segment& s, int t, int most) {
    return t > most ? 0 : scalar_load(s.table, t >> a.c.page_shift);  // (most lies in the table)
}

// Where a row's partial results of this workgroup's split go.
__device__ __forceinline__ int64_t slot_of(const PagedAttnArgs& a, const Segment& s, const Row& row) {
    return ((int64_t)row.token * a.heads + row.head) * a.slots + (s.shared ? 0 : a.prefix_splits) + s.split;
}

// One lane's part of kTiles 16-row tiles: the running softmax and value sums of
// row j of each, o[u][dd][r] over the dimensions kVd (4 q + r) + dd (narrow), or 16
// dd + 4 q + r (wide).
template <class E, int D, int kTiles>
struct Attend {
    static constexpr int kVd = D / 16;     // dimensions of a value per lane
    static constexpr int kVw = kVd / 2;    // words of them
    static constexpr int kSteps = D / 32;  // K steps of a score
    typedef uint32_t vword __attribute__((ext_vector_type(kVw)));

    float m_run[kTiles], l_run[kTiles];
    bool seen[kTiles];
    float4v o[kTiles][kVd];

    __device__ __forceinline__ void start() {
#pragma unroll
        for (int u = 0; u < kTiles; ++u) {
            m_run[u] = kScoreFloor, l_run[u] = 0.0f;
            seen[u] = false;
#pragma unroll
            for (int dd = 0; dd < kVd; ++dd) o[u][dd] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }

    // Before a lane's kCount scores of tile u become probabilities: the sums rescaled
    // where needed.
    template <int kCount>
    __device__ __forceinline__ void settle(int u, const float (&s)[kCount], float scale2) {
        float top = s[0];
#pragma unroll
        for (int e = 1; e < kCount; ++e) top = fmaxf(top, s[e]);
        const float mn = quarters_max(top) * scale2;
        if (__any(mn - m_run[u] > kLazy<E>)) {
            const float to = fmaxf(m_run[u], mn);
            const float alpha = __builtin_amdgcn_exp2f(m_run[u] - to);  // (1 where it is another row's turn)
            l_run[u] *= alpha;
#pragma unroll
            for (int dd = 0; dd < kVd; ++dd) o[u][dd] *= alpha;
            m_run[u] = to;
        }
    }

    // Eight scores of tile u as probabilities, in two 16-bit terms.
    template <int kCount>
    __device__ __forceinline__ void soften(int u, const float (&s)[kCount], int from, u32x4& ph, u32x4& pl,
                                           float scale2) {
        const float ref = kProbShift<E> - m_run[u];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[from + 2 * e], scale2, ref));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(s[from + 2 * e + 1], scale2, ref));
            l_run[u] += p0 + p1;
            ph[e] = E::pack(p0, p1);
            pl[e] = E::pack(p0 - E::lo(ph[e]), p1 - E::hi(ph[e]));
        }
    }

    // Eight of tile u's keys from t0 as ones where the row sees them.
    __device__ __forceinline__ static void show(int limit, int t0, int q, u32x4& ph, u32x4& pl) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int t = t0 + 16 * (e / 2) + 4 * q + 2 * (e % 2);
            ph[e] = (t <= limit ? E::kOne : 0u) | (t + 1 <= limit ? E::kOne << 16 : 0u);
            pl[e] = 0u;
        }
    }

    // Product dd of the value sums of 32 keys: vt holds, for the product's row j, the
    // values of the lane's keys 16 (e / 4) + 4 q + e % 4.
    __device__ __forceinline__ void gather(int dd, const u32x4& vt, const u32x4 (&ph)[kTiles], const u32x4 (&pl)[kTiles]) {
#pragma unroll
        for (int u = 0; u < kTiles; ++u) o[u][dd] = E::mfma(vt, ph[u], o[u][dd]);
#pragma unroll
        for (int u = 0; u < kTiles; ++u) o[u][dd] = E::mfma(vt, pl[u], o[u][dd]);
    }

    // After a counting pass: which sums are not zero, a bit each; and what they say.
    __device__ __forceinline__ uint64_t marks() const {
        uint64_t m = 0;
#pragma unroll
        for (int u = 0; u < kTiles; ++u)
#pragma unroll
            for (int dd = 0; dd < kVd; ++dd)
#pragma unroll
                for (int r = 0; r < 4; ++r) m |= (uint64_t)(o[u][dd][r] != 0.0f) << ((u * kVd + dd) * 4 + r);
        return m;
    }
    __device__ __forceinline__ void mark(uint64_t up, uint64_t down) {
#pragma unroll
        for (int u = 0; u < kTiles; ++u)
#pragma unroll
            for (int dd = 0; dd < kVd; ++dd)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int bit = (u * kVd + dd) * 4 + r;
                    const float plus = (up >> bit) & 1 ? INFINITY : 0.0f, minus = (down >> bit) & 1 ? INFINITY : 0.0f;
                    o[u][dd][r] += plus - minus;  // (both: NaN)
                }
    }

    __device__ __forceinline__ bool finite() const {
        bool fine = true;
#pragma unroll
        for (int u = 0; u < kTiles; ++u)
#pragma unroll
            for (int dd = 0; dd < kVd; ++dd)
#pragma unroll
                for (int r = 0; r < 4; ++r) fine = fine && fabsf(o[u][dd][r]) < INFINITY;
        return fine;
    }
};

// A value that a rare branch works with: keeps the compiler from running the
// branch's instructions always.
__device__ __forceinline__ int rare(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// The queries of a row as MFMA operand pieces.
template <int kSteps>
__device__ __forceinline__ void load_queries(const PagedAttnArgs& a, const Row& row, int q, u32x4 (&qf)[kSteps]) {
    const uint16_t* from = a.q + row.token * a.q_row + row.head * a.q_head + 8 * q;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qf[s] = *(const u32x4*)(from + 32 * s) ^ a.query_sign;
}

// Least and largest limit over rows m0 .. m0 + count - 1 of a segment (those that
// there are): an own segment's rise with the row; where a prefix is not all seen,
// the widest they can be.
__device__ __forceinline__ void limits(const PagedAttnArgs& a, const Segment& s, int m0, int count, int& least, int& most) {
    const int last = min(m0 + count, s.count) - 1;
    if (last < m0) {
        least = 0x7FFFFFFF, most = s.key_lo - 1;
    } else if (s.shared) {
        most = (int)s.key_end - 1;
        least = s.sees_all ? most : s.key_lo - 1;
    } else {
        const int64_t first = s.first + a.by_group(m0), end = s.first + a.by_group(last);
        least = (int)max(min(first, s.key_end - 1), (int64_t)(s.key_lo - 1));
        most = (int)max(min(end, s.key_end - 1), (int64_t)(s.key_lo - 1));
    }
}

// ---- narrow ----

template <class E, int D>
struct KeyBlock {
    u32x4 k[2][D / 32];                     // key 16 h + j, dimensions 32 s + 8 q ..
    typename Attend<E, D, 1>::vword v[8];   // value of key 16 (e / 4) + 4 q + e % 4, dimensions kVd j ..
    bool bad[2];
};

// A workgroup's 32-key blocks of its segment: begin, begin + step, ... below end.
struct KeyRange {
    int begin, step, end;
};

template <class E, int D>
__device__ __forceinline__ void narrow(const PagedAttnArgs& a, const Segment& s, int tile, const KeyRange& keys, int lane,
                                       int wave, unsigned char* meet0, unsigned char* meet1) {
    typedef Attend<E, D, 1> A;
    const int j = lane & 15;
    const int q = lane >> 4;
    int least, most;
    limits(a, s, tile * kNarrowRows, kNarrowRows, least, most);
    const int blocks = min(most >= s.key_lo ? (most - s.key_lo) / kBlock + 1 : 0, keys.end);
    const int first = keys.begin + keys.step * wave, stride = keys.step * kWaves;

    const uint16_t* kc = a.c.k + s.kvh * a.c.k_head;
    const uint16_t* vc = a.c.v + s.kvh * a.c.v_head;
    const int k_lane = j * (int)a.c.k_position + 8 * q;
    const int v_lane = 4 * q * (int)a.c.v_position + A::kVd * j;
    const int mask = (1 << a.c.page_shift) - 1;
    struct Pages {
        int p[2];
    };
    auto look = [&](int block) {
        const int t = s.key_lo + block * kBlock;
        return Pages{{table_entry(a, s, t, most), table_entry(a, s, t + 16, most)}};
    };
    auto load = [&](KeyBlock<E, D>& b, int block, const Pages& pages) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int t = s.key_lo + block * kBlock + 16 * h;
            const int entry = checked_page(pages.p[h], a.c.num_pages);
            b.bad[h] = entry < 0;
            const int64_t page = max(entry, 0);
            const uint16_t* kp = kc + page * a.c.k_page + (t & mask) * a.c.k_position;
            const uint16_t* vp = vc + page * a.c.v_page + (t & mask) * a.c.v_position;
#pragma unroll
            for (int i = 0; i < A::kSteps; ++i) b.k[h][i] = *(const u32x4*)(kp + k_lane + 32 * i);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                b.v[4 * h + r] = *(const typename A::vword*)(vp + v_lane + r * (int)a.c.v_position);
        }
    };
    // the first block is on its way before the rows and their queries are looked up
    KeyBlock<E, D> b;
    if (first < blocks) load(b, first, look(first));
    Pages next = look(first + stride);
    const Row row = row_at(a, s, tile * kNarrowRows + j);
    u32x4 qf[A::kSteps];
    load_queries(a, row, q, qf);
    A state;
    auto compute = [&](KeyBlock<E, D>& b, int block, auto ordinary, Pass pass) {
        const int t0 = s.key_lo + block * kBlock;
        float x[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < A::kSteps; ++i) acc = E::mfma(b.k[h][i], qf[i], acc);
#pragma unroll
            for (int r = 0; r < 4; ++r) x[4 * h + r] = acc[r];
        }
        if (t0 + kBlock - 1 > least) {
            const int sees = rare(row.limit - t0 - 4 * q), held = rare(most - t0 - 4 * q);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int t = 16 * (e / 4) + e % 4;
                if (t > sees) x[e] = -INFINITY;
                if (t > held) b.v[e] = typename A::vword{};
            }
        }
        state.seen[0] = state.seen[0] || t0 <= row.limit;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (b.bad[h] && t0 + 16 * h <= row.limit) state.l_run[0] = __builtin_nanf("");
        u32x4 h1[1], l1[1];
        if (ordinary || pass == kFinite) {
            state.settle(0, x, a.scale2);
            state.soften(0, x, 0, h1[0], l1[0], a.scale2);
        } else {
            A::show(row.limit, t0, q, h1[0], l1[0]);
        }
#pragma unroll
        for (int dd = 0; dd < A::kVd; ++dd) {
            const uint32_t sel = (dd & 1) ? 0x07060302u : 0x05040100u;  // high or low halves
            u32x4 vt;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                vt[e] = __builtin_amdgcn_perm(b.v[2 * e + 1][dd / 2], b.v[2 * e][dd / 2], sel);
                if constexpr (!ordinary) vt[e] = pass_word<E>(vt[e], pass);
            }
            state.gather(dd, vt, h1, l1);
        }
    };
    state.start();
    for (int block = first; block < blocks;) {
        compute(b, block, std::true_type{}, kOrdinary);
        block += stride;
        if (block < blocks) load(b, block, next);
        next = look(block + stride);
    }
    if (!__all(state.finite())) {  // (the wave's)
        uint64_t up = 0, down = 0;
#pragma unroll 1
        for (int pass = kCountUp; pass <= kFinite; ++pass) {
            state.start();
#pragma unroll 1
            for (int block = first; block < blocks; block += stride) {
                load(b, block, look(block));
                compute(b, block, std::false_type{}, (Pass)pass);
            }
            if (pass == kCountUp) up = state.marks();
            if (pass == kCountDown) down = state.marks();
        }
        state.mark(up, down);
    }

    // ---- the waves' results meet in LDS ----
    constexpr int kStride = D + 4;
    typedef float Line[kStride];  // a row's sums
    constexpr int kLines = 16 * kStride * (int)sizeof(float);
    auto lines = [&](int w) { return (Line*)((w < 2 ? meet0 : meet1) + (w & 1) * kLines); };
    auto stats = [&](int w) { return (float2v*)((w < 2 ? meet0 : meet1) + 2 * kLines + (w & 1) * 16 * sizeof(float2v)); };
    float l = quarters_sum(state.l_run[0]);
    if (row.beyond && s.split == 0) {
        l = __builtin_nanf("");
        state.seen[0] = true;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int dd = 0; dd < A::kVd; dd += 4)
            *(float4v*)&lines(wave)[j][A::kVd * (4 * q + r) + dd] =
                float4v{state.o[0][dd][r], state.o[0][dd + 1][r], state.o[0][dd + 2][r], state.o[0][dd + 3][r]};
    if (q == 0) stats(wave)[j] = float2v{state.seen[0] ? state.m_run[0] : -INFINITY, l};  // -inf: no key seen
    __syncthreads();
    // thread t: row t / 16, dimensions kVd (t % 16) ..
    const int tid = 64 * wave + lane;
    const int g = tid / 16;
    const int d0 = A::kVd * (tid % 16);
    const PagedAttnArgs late = late_arguments();
    const Row mine = row_at(late, s, tile * kNarrowRows + g);
    if (!mine.live) return;
    float2v st[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) st[w] = stats(w)[g];
    const float top = fmaxf(fmaxf(st[0][0], st[1][0]), fmaxf(st[2][0], st[3][0]));
    float sum[A::kVd] = {};
    l = 0.0f;
    if (top > -INFINITY) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(st[w][0] - top);
            if (f == 0.0f) {
                // no key, or keys of no weight beside the others': nothing, unless a value that
                // the row sees was not finite
                if (st[w][0] > -INFINITY) {
                    if (st[w][1] != st[w][1]) l = st[w][1];
#pragma unroll
                    for (int i = 0; i < A::kVd; ++i) add_odd(sum[i], lines(w)[g][d0 + i]);
                }
                continue;
            }
            l = fmaf(st[w][1], f, l);
#pragma unroll
            for (int i = 0; i < A::kVd; ++i) sum[i] = fmaf(lines(w)[g][d0 + i], f, sum[i]);
        }
    }
    if (late.slots == 1) {
        const float inv = top > -INFINITY ? 1.0f / l : 0.0f;
        typename A::vword x;
#pragma unroll
        for (int i = 0; i < A::kVw; ++i) x[i] = E::pack(sum[2 * i] * inv, sum[2 * i + 1] * inv);
        *(typename A::vword*)(late.out + mine.token * late.out_row + mine.head * late.out_head + d0) = x;
        return;
    }
    const int64_t slot = slot_of(late, s, mine);
    if (tid % 16 == 0) *(float2v*)(late.stats + 2 * slot) = float2v{top, l};
    if (top == -INFINITY) return;  // (the join does not read it)
#pragma unroll
    for (int i = 0; i < A::kVd; i += 4)
        *(float4v*)(late.partials + slot * D + d0 + i) = float4v{sum[i], sum[i + 1], sum[i + 2], sum[i + 3]};
}

// ---- wide ----

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v* lds_halves_t;

// This wave's loads into LDS have landed.
__device__ __forceinline__ void wait_loads() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((0x7 << 4) | (0xF << 8));  // vmcnt 0 (gfx9 encoding)
    asm volatile("" ::: "memory");
}
// All of this wave's loads into LDS and stores to it have landed, then all waves'.
__device__ __forceinline__ void all_landed() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x7 << 4);  // vmcnt 0, lgkmcnt 0 (gfx9 encoding)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A tile's keys or values in LDS: 64 rows of D elements in 16-byte pieces, piece
// c of row r in slot c ^ turn(r).  Keys are read one piece of 16 rows at a time:
// the turns are all different (D 64: where the rows' banks are the same).  Values
// are read transposed, 32 bytes of 4 rows by 16 lanes (ds_read_b64_tr_b16: lane t
// brings elements 4 (t % 4) .. of row t / 4 and gets element t of the four
// rows): there the pairs of pieces are turned.
template <int D>
struct Tile {
    static constexpr int kPieces = D / 8;
    static constexpr int kRowBytes = 2 * D;
    static constexpr int kBytes = kTileKeys * kRowBytes;
    static constexpr int kRowsPerLoad = 64 / kPieces;  // rows that a wave's 16-byte load fills
    static constexpr int kLoads = 16 / kRowsPerLoad;   // loads of 16 keys
    static __device__ __forceinline__ int key_turn(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
    static __device__ __forceinline__ int value_turn(int row) { return D == 128 ? 2 * (row & 7) : row & 6; }
};

// false, with nothing stored, where a value sum came out infinite or NaN: the
// rows are then left to narrow(), over the keys given back.
template <class E, int D>
__device__ __forceinline__ bool wide(const PagedAttnArgs& a, const Segment& s, int lane, int wave, unsigned char* k0,
                                     unsigned char* v0, unsigned char* k1, unsigned char* v1, int (*bad)[kWaves],
                                     int* odd, KeyRange& keys) {
    typedef Attend<E, D, 2> A;
    typedef Tile<D> T;
    const int j = lane & 15;
    const int q = lane >> 4;
    const int m0 = s.tile * kWideRows + 32 * wave;
    // the wave's rows, then the workgroup's
    int least, most, all_least, all_most;
    limits(a, s, m0, 32, least, most);
    limits(a, s, s.tile * kWideRows, kWideRows, all_least, all_most);
    const int tiles = all_most >= s.key_lo ? (all_most - s.key_lo) / kTileKeys + 1 : 0;
    const int per = (tiles + s.splits - 1) / s.splits;
    const int begin = s.split * per;
    const int end = min(tiles, begin + per);

    // wave w brings keys 16 w .. 16 w + 15 of a tile
    const uint16_t* kc = a.c.k + s.kvh * a.c.k_head;
    const uint16_t* vc = a.c.v + s.kvh * a.c.v_head;
    const int mask = (1 << a.c.page_shift) - 1;
    int k_at[T::kLoads], v_at[T::kLoads];
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) {
        const int r = T::kRowsPerLoad * i + lane / T::kPieces;
        k_at[i] = 2 * r * (int)a.c.k_position + 16 * ((lane % T::kPieces) ^ T::key_turn(r));
        v_at[i] = 2 * r * (int)a.c.v_position + 16 * ((lane % T::kPieces) ^ T::value_turn(r));
    }
    auto look = [&](int tile) { return table_entry(a, s, s.key_lo + tile * kTileKeys + 16 * wave, all_most); };
    auto stage = [&](int tile, int entry, unsigned char* keys, unsigned char* values, int* flags) {
        const int page = checked_page(entry, a.c.num_pages);
        const int t = s.key_lo + tile * kTileKeys + 16 * wave;
        if (lane == 0) flags[wave] = page < 0;
        const int64_t p = max(page, 0);
        const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(kc + p * a.c.k_page + (t & mask) * a.c.k_position), 0, (15 * (int)a.c.k_position + D) * 2, 0x00020000);
        const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(vc + p * a.c.v_page + (t & mask) * a.c.v_position), 0, (15 * (int)a.c.v_position + D) * 2, 0x00020000);
#pragma unroll
        for (int i = 0; i < T::kLoads; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_ptr_t)(keys + 16 * wave * T::kRowBytes + 1024 * i), 16, k_at[i],
                                                     0, 0, 0);
#pragma unroll
        for (int i = 0; i < T::kLoads; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_ptr_t)(values + 16 * wave * T::kRowBytes + 1024 * i), 16,
                                                     v_at[i], 0, 0, 0);
    };
    // Before the barrier: values past the last visible key become zeros (their
    // probabilities are, but what lies there may not be finite).
    auto settle = [&](int tile, unsigned char* values) {
        const int held = all_most - (s.key_lo + tile * kTileKeys + 16 * wave);  // last of the wave's 16 keys
        if (held >= 15) return;
        wait_loads();
#pragma unroll
        for (int i = 0; i < T::kLoads; ++i) {
            const int r = T::kRowsPerLoad * i + lane / T::kPieces;
            if (r > held)
                *(u32x4*)(values + (16 * wave + r) * T::kRowBytes + 16 * (lane % T::kPieces)) = u32x4{0u, 0u, 0u, 0u};
        }
    };
    // the first tile is on its way before the rows and their queries are looked up
    if (begin < end) stage(begin, look(begin), k0, v0, bad[0]);
    int next = look(begin + 1);
    u32x4 qf[2][A::kSteps];
    int limit[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const Row row = row_at(a, s, m0 + 16 * u + j);
        limit[u] = row.limit;
        load_queries(a, row, q, qf[u]);
    }
    A state;
    auto compute = [&](int tile, const unsigned char* keys, const unsigned char* values, const int* flags) {
        const int t0 = s.key_lo + tile * kTileKeys;
        if (t0 > most) return;  // (the wave's)
        float x[2][16];
        // keys of the next product on their way while this one's are used
        u32x4 kf[2][A::kSteps];
        auto load_keys = [&](int h) {
#pragma unroll
            for (int i = 0; i < A::kSteps; ++i)
                kf[h & 1][i] = *(const u32x4*)(keys + (16 * h + j) * T::kRowBytes + 16 * ((4 * i + q) ^ T::key_turn(j)));
        };
        load_keys(0);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            if (h < 3) load_keys(h + 1);
            __builtin_amdgcn_sched_barrier(0);
            float4v acc[2] = {};
#pragma unroll
            for (int i = 0; i < A::kSteps; ++i)
#pragma unroll
                for (int u = 0; u < 2; ++u) acc[u] = E::mfma(kf[h & 1][i], qf[u][i], acc[u]);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) x[u][4 * h + r] = acc[u][r];
        }
        if (t0 + kTileKeys - 1 > least) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int sees = rare(limit[u] - t0 - 4 * q);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (16 * (e / 4) + e % 4 > sees) x[u][e] = -INFINITY;
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) state.seen[u] = state.seen[u] || t0 <= limit[u];
        if (__builtin_amdgcn_readfirstlane(flags[0] | flags[1] | flags[2] | flags[3])) {
#pragma unroll
            for (int h = 0; h < 4; ++h)
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    if (flags[h] && t0 + 16 * h <= limit[u]) state.l_run[u] = __builtin_nanf("");
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) state.settle(u, x[u], a.scale2);
        // the lane's part of the four rows 4 q ..: row 4 q + j / 4, elements 4 (j % 4) ..
        u32x4 vt[2];
        auto load_values = [&](int i, int dd) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {  // (rows 16 apart turn alike)
                const int r = 4 * q + j / 4;
                const unsigned char* at = values + r * T::kRowBytes +
                                          16 * ((2 * dd + (j & 3) / 2) ^ T::value_turn(r)) + 8 * (j & 1) +
                                          (32 * i + 16 * g) * T::kRowBytes;
                const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_halves_t)at));
                vt[dd & 1][2 * g] = w[0], vt[dd & 1][2 * g + 1] = w[1];
            }
        };
        load_values(0, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            u32x4 ph[2], pl[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) state.soften(u, x[u], 8 * i, ph[u], pl[u], a.scale2);
#pragma unroll
            for (int dd = 0; dd < A::kVd; ++dd) {
                if (dd + 1 < A::kVd) load_values(i, dd + 1);
                else if (i == 0) load_values(1, 0);
                __builtin_amdgcn_sched_barrier(0x7);  // (no LDS read past this; arithmetic as it likes)
                state.gather(dd, vt[dd & 1], ph, pl);
            }
        }
    };
    // The next tile on its way while this one is worked on: its buffer was read
    // before the barrier.
    state.start();
    if (begin < end) {
        for (int tile = begin;;) {
            settle(tile, v0);
            all_landed();
            if (tile + 1 < end) stage(tile + 1, next, k1, v1, bad[1]);
            next = look(tile + 2);
            compute(tile, k0, v0, bad[0]);
            if (++tile >= end) break;
            settle(tile, v1);
            all_landed();
            if (tile + 1 < end) stage(tile + 1, next, k0, v0, bad[0]);
            next = look(tile + 2);
            compute(tile, k1, v1, bad[1]);
            if (++tile >= end) break;
        }
    }
    if (lane == 0) odd[wave] = 0;
    if (!__all(state.finite()) && lane == 0) odd[wave] = 1;
    __syncthreads();
    if (odd[0] | odd[1] | odd[2] | odd[3]) {
        __syncthreads();  // (LDS is free)
        keys = KeyRange{kTileKeys / kBlock * begin, 1, kTileKeys / kBlock * end};
        return false;
    }
    const PagedAttnArgs late = late_arguments();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        float l = quarters_sum(state.l_run[u]);
        float m = state.seen[u] ? state.m_run[u] : -INFINITY;
        const Row row = row_at(late, s, rare(m0 + 16 * u + j));  // (again: not kept in registers over the keys)
        if (!row.live) continue;
        if (row.beyond && s.split == 0) {
            l = __builtin_nanf("");
            m = fmaxf(m, kScoreFloor);
        }
        if (late.slots == 1) {
            const float inv = m > -INFINITY ? 1.0f / l : 0.0f;
            uint16_t* to = late.out + row.token * late.out_row + row.head * late.out_head + 4 * q;
#pragma unroll
            for (int dd = 0; dd < A::kVd; ++dd) {
                const float4v x = state.o[u][dd];
                *(u32x2*)(to + 16 * dd) = u32x2{E::pack(x[0] * inv, x[1] * inv), E::pack(x[2] * inv, x[3] * inv)};
            }
            continue;
        }
        const int64_t slot = slot_of(late, s, row);
        if (q == 0) *(float2v*)(late.stats + 2 * slot) = float2v{m, l};
        if (m == -INFINITY) continue;  // (the join does not read it)
        float* to = late.partials + slot * D + 4 * q;
#pragma unroll
        for (int dd = 0; dd < A::kVd; ++dd) *(float4v*)(to + 16 * dd) = state.o[u][dd];
    }
    return true;
}

// kWide: the prefix or the own segments go by wide tiles.
template <class E, int D, bool kWide>
__global__ __launch_bounds__(kThreads, kWide ? 2 : 3) void paged_attention_kernel(PagedAttnArgs a) {
    constexpr int kMeet = 2 * 16 * (4 * (D + 4) + 8);  // two narrow waves' sums and statistics
    static_assert(kMeet >= Tile<D>::kBytes, "or a wide tile's keys");
    __shared__ __attribute__((aligned(16))) unsigned char k0[kMeet], k1[kMeet];
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // rows behind the last sequence, where no second launch sees to them
    if (a.slots == 1 && a.zero_rest) {
        for (int64_t r = rest_row(a.c.cu_rows, a.c.batch, a.rows, blockIdx.x); r < a.rows; r += gridDim.x)
            for (int d = 8 * tid; d < a.heads * D; d += 8 * kThreads)
                *(u32x4*)(a.out + r * a.out_row + (d / D) * a.out_head + d % D) = u32x4{0u, 0u, 0u, 0u};
    }
    Segment s;
    if (!find_segment(a, lane, s)) return;
    int tile = s.tile, past = tile + 1;
    KeyRange keys{s.split, s.splits, 0x7FFFFFFF};
    if constexpr (kWide) {
        // (objects of their own: a read of one does not wait for loads into another)
        __shared__ __attribute__((aligned(16))) unsigned char v0[Tile<D>::kBytes], v1[Tile<D>::kBytes];
        __shared__ int bad[2][kWaves], odd[kWaves];
        if (s.wide) {
            if (wide<E, D>(a, s, lane, wave, k0, v0, k1, v1, bad, odd, keys)) return;
            tile *= kWideRows / kNarrowRows;
            past = tile + kWideRows / kNarrowRows;
        }
    }
    while (true) {
        narrow<E, D>(a, s, tile, keys, lane, wave, k0, k1);
        if (++tile >= past) break;
        __syncthreads();  // (LDS is free again)
    }
}

// One wave per (packed row, query head): lane l's D / 32 dimensions of the slots
// l / 32, l / 32 + 2, ...; the halves are added at the end.
template <class E, int D>
__global__ __launch_bounds__(kThreads) void paged_join_kernel(PagedAttnArgs a) {
    constexpr int kPer = D / 32;
    typedef float fvec __attribute__((ext_vector_type(kPer)));
    const int lane = threadIdx.x & 63;
    const int index = (int)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (index >= a.rows * a.heads) return;
    const int row = a.by_heads(index);
    const int head = index - row * a.heads;
    const int64_t at = index;
    uint16_t* to = a.out + row * a.out_row + head * a.out_head;
    const float* stats = a.stats + 2 * at * a.slots;
    const bool has = lane < a.slots;
    float sum[kPer] = {};
    const float* part = a.partials + at * a.slots * D + kPer * (lane % 32);
    const int half = lane / 32;
    // Eight slots' loads at once, the first ones before the statistics arrive: a slot
    // that nobody wrote has a factor of zero and is left out, whatever it holds.
    fvec x[4];
    auto load = [&](int first) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *(const fvec*)(part + min(first + 2 * i + half, a.slots - 1) * D);
    };
    load(0);
    const float m = has ? stats[2 * lane] : -INFINITY;
    const float sum_l = has ? stats[2 * lane + 1] : 0.0f;
    if (row >= scalar_load(a.c.cu_rows, a.c.batch)) {  // behind the last sequence
        if (a.zero_rest && lane < D / 8) *(u32x4*)(to + 8 * lane) = u32x4{0u, 0u, 0u, 0u};
        return;
    }
    const float top = wave_max64(m);
    const float f = m > -INFINITY ? __builtin_amdgcn_exp2f(m - top) : 0.0f;
    const float l = wave_sum64(f != 0.0f || sum_l != sum_l ? sum_l * f : 0.0f);  // (NaN: a page that was not there)
    for (int first = 0; first < a.slots; first += 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float fs = __shfl(f, min(first + 2 * i + half, 63));  // (0 past the slots)
#pragma unroll
            for (int e = 0; e < kPer; ++e) sum[e] = fs != 0.0f ? fmaf(x[i][e], fs, sum[e]) : sum[e];
        }
        if (first + 8 < a.slots) load(first + 8);
    }
    // slots of no weight beside the others': their values that were not finite
    for (uint64_t low = __ballot(m > -INFINITY && f == 0.0f); low; low &= low - 1) {
        const fvec odd = *(const fvec*)(part + (__ffsll((unsigned long long)low) - 1) * D);
        if (half == 0)
#pragma unroll
            for (int e = 0; e < kPer; ++e) add_odd(sum[e], odd[e]);
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) sum[e] += __shfl_xor(sum[e], 32);
    if (lane >= 32) return;
    const float inv = top > -INFINITY ? 1.0f / l : 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; e += 2)
        *(uint32_t*)(to + kPer * lane + e) = E::pack(sum[e] * inv, sum[e + 1] * inv);
}

// How a call is cut up; the same from the same sizes, whatever the device holds.
struct PagedPlan {
    int64_t prefix, prefix_tiles, prefix_splits, own_tiles, own_splits, slots;
    bool prefix_wide, own_wide;
};

PagedPlan paged_plan(const PagedView& c, int64_t rows, int64_t heads, int64_t head_dim, int64_t shared_pages) {
    PagedPlan p{};
    const int64_t group = heads / c.kv_heads;
    const int64_t sequences = c.batch < rows ? c.batch : rows;
    p.prefix = shared_pages << c.page_shift;
    const int64_t own = ((int64_t)c.table_width - shared_pages) << c.page_shift;
    // (own: on the average; the sequences with few rows among them go by narrow tiles
    // all the same, at most eight each)
    p.prefix_wide = p.prefix > 0 && rows * group > kWideFrom;
    p.own_wide = own > 0 && rows * group > kWideFrom * sequences;
    const int64_t prefix_tile = p.prefix_wide ? kWideRows : kNarrowRows, own_tile = p.own_wide ? kWideRows : kNarrowRows;
    int64_t usual = 0;  // own tiles if all sequences have the average rows
    if (p.prefix > 0) p.prefix_tiles = (rows * group + prefix_tile - 1) / prefix_tile;
    if (own > 0) {
        usual = sequences * ((rows * group + sequences * own_tile - 1) / (sequences * own_tile));
        p.own_tiles = p.own_wide ? rows * group / kWideRows + kWideFrom / kNarrowRows * sequences
                                 : rows * group / kNarrowRows + sequences;
    }
    // Splits: as many workgroups as the chip holds at once, dealt out by the time that
    // the two kinds of segment take (a key costs a wide tile some four times a narrow
    // one's; tables are half full), but no more than leave a block for each wave.
    const bool wide = p.prefix_wide || p.own_wide;
    const int64_t hold = 256 * (head_dim == 64 ? (wide ? 3 : 5) : (wide ? 2 : 3));
    const double prefix_time = (double)p.prefix_tiles * p.prefix * (p.prefix_wide ? 4 : 1);
    const double own_time = (double)usual * own / 2 * (p.own_wide ? 4 : 1);
    const int64_t prefix_hold = (int64_t)(hold * (prefix_time / (prefix_time + own_time)));
    auto splits = [&](int64_t hold, int64_t tiles, int64_t keys) {
        const int64_t workgroups = tiles * c.kv_heads, most = (keys + kBlock * kWaves - 1) / (kBlock * kWaves);
        int64_t s = hold > workgroups ? hold / workgroups : 1;
        s = s < most ? s : most;
        return s < kMaxSplits / 2 ? s : kMaxSplits / 2;
    };
    if (p.prefix > 0) p.prefix_splits = splits(prefix_hold, p.prefix_tiles, p.prefix);
    if (own > 0) p.own_splits = splits(hold - prefix_hold, usual, own);
    p.slots = p.prefix_splits + p.own_splits;
    return p;
}

template <class E, int D>
hipError_t launch_paged_attention(const PagedAttnArgs& a, int64_t workgroups, hipStream_t stream) {
    if (a.prefix_wide || a.own_wide)
        hipLaunchKernelGGL((paged_attention_kernel<E, D, true>), dim3((unsigned)workgroups), dim3(kThreads), 0, stream, a);
    else
        hipLaunchKernelGGL((paged_attention_kernel<E, D, false>), dim3((unsigned)workgroups), dim3(kThreads), 0, stream, a);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess || a.slots == 1) return err;
    const int64_t joins = ((int64_t)a.rows * a.heads + kWaves - 1) / kWaves;
    hipLaunchKernelGGL((paged_join_kernel<E, D>), dim3((unsigned)joins), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

// The sizes of a call that both entry points go by.
int attention_sizes(const qwen2_paged_cache* cache, PagedView* view, int64_t rows, int64_t heads, int64_t shared_pages) {
    const int status = paged_view(cache, view);
    if (status) return status;
    if (cache->head_dim != 64 && cache->head_dim != 128)
        return set_error(W4G64_STATUS_UNSUPPORTED, "paged_attention needs a head_dim of 64 or 128, got %lld",
                         (long long)cache->head_dim);
    if (heads <= 0 || heads % cache->kv_heads || heads > 0xFFFF)
        return set_error(W4G64_STATUS_INVALID_VALUE, "paged_attention heads must be a positive multiple of kv_heads, got %lld and %lld",
                         (long long)heads, (long long)cache->kv_heads);
    if (rows < 0 || rows > 0x7FFFFFF)
        return set_error(W4G64_STATUS_INVALID_VALUE, "paged_attention rows must be in [0, 2^27), got %lld", (long long)rows);
    if (shared_pages < 0 || shared_pages > cache->table_width)
        return set_error(W4G64_STATUS_INVALID_VALUE, "shared_pages must be in [0, table_width = %lld], got %lld",
                         (long long)cache->table_width, (long long)shared_pages);
    if ((cache->table_width << view->page_shift) > 0x7FF00000)
        return set_error(W4G64_STATUS_UNSUPPORTED, "paged_attention tables must hold at most 2^31 - 2^20 positions");
    return W4G64_STATUS_OK;
}

}  // namespace
}  // namespace w4g64

using namespace w4g64;

extern "C" {

int64_t qwen2_paged_attention_workspace_bytes(const qwen2_paged_cache* cache, int64_t rows, int64_t heads,
                                              int64_t shared_pages) {
    PagedView view{};
    if (attention_sizes(cache, &view, rows, heads, shared_pages) || rows == 0) return 0;
    const PagedPlan p = paged_plan(view, rows, heads, cache->head_dim, shared_pages);
    return p.slots == 1 ? 0 : rows * heads * p.slots * (cache->head_dim + 2) * (int64_t)sizeof(float) + 16;
}

int qwen2_paged_attention(const qwen2_paged_cache* cache, const qwen2_rows* q, const qwen2_rows* out, int64_t rows,
                          int64_t heads, int64_t shared_pages, float scale, int zero_rest, void* workspace,
                          int64_t workspace_bytes, void* stream) {
    PagedAttnArgs a{};
    const int status = attention_sizes(cache, &a.c, rows, heads, shared_pages);
    if (status) return status;
    if (!isfinite(scale)) return set_error(W4G64_STATUS_INVALID_VALUE, "paged_attention scale must be finite");
    if (rows == 0) return clear_error();
    for (const qwen2_rows* r : {q, out})
        if (!r || !r->data || ((uintptr_t)r->data & 15) || r->row % 8 || r->head % 8)
            return set_error(W4G64_STATUS_INVALID_VALUE,
                             "q and out must be non-null, 16-byte aligned, with strides that are multiples of 8 elements");
    const PagedPlan p = paged_plan(a.c, rows, heads, cache->head_dim, shared_pages);
    const int64_t need = qwen2_paged_attention_workspace_bytes(cache, rows, heads, shared_pages);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
        return set_error(W4G64_STATUS_WORKSPACE, "paged_attention needs %lld workspace bytes, 16-byte aligned, got %lld",
                         (long long)need, (long long)(workspace ? workspace_bytes : 0));
    const int64_t workgroups =
        (p.prefix_tiles * p.prefix_splits + p.own_tiles * p.own_splits) * cache->kv_heads;
    if (workgroups > 0x7FFFFFFF || rows * heads > 0x7FF00000)
        return set_error(W4G64_STATUS_UNSUPPORTED, "paged_attention call is too large: %lld workgroups", (long long)workgroups);
    a.q = (const uint16_t*)q->data, a.q_row = q->row, a.q_head = q->head;
    a.out = (uint16_t*)out->data, a.out_row = out->row, a.out_head = out->head;
    a.partials = (float*)workspace;  // (D floats per slot: 16-byte aligned)
    a.stats = a.partials + rows * heads * p.slots * cache->head_dim;
    // (a scale of zero: as small as there is, so that a hidden key's -inf stays -inf)
    const float scale2 = fabsf(scale) * 1.44269504088896340736f;
    a.scale2 = scale2 > 0.0f ? fminf(scale2, 3.402823466e+38f) : 1.401298464324817e-45f;
    a.query_sign = scale < 0.0f ? 0x80008000u : 0u;
    a.rows = (int)rows, a.heads = (int)heads, a.group = (int)(heads / cache->kv_heads);
    a.prefix = (int)p.prefix;
    a.prefix_tiles = (int)p.prefix_tiles, a.prefix_splits = (int)p.prefix_splits;
    a.own_tiles = (int)p.own_tiles, a.own_splits = (int)p.own_splits, a.slots = (int)p.slots;
    a.prefix_wide = p.prefix_wide, a.own_wide = p.own_wide;
    a.by_group = divisor(a.group), a.by_heads = divisor(heads), a.by_kv_heads = divisor(cache->kv_heads);
    a.by_prefix_splits = divisor(p.prefix_splits), a.by_own_splits = divisor(p.own_splits);
    a.zero_rest = zero_rest;
    const hipStream_t s = (hipStream_t)stream;
    hipError_t err;
    if (cache->dtype == W4G64_DTYPE_BF16)
        err = cache->head_dim == 128 ? launch_paged_attention<Bf16, 128>(a, workgroups, s)
                                     : launch_paged_attention<Bf16, 64>(a, workgroups, s);
    else
        err = cache->head_dim == 128 ? launch_paged_attention<F16, 128>(a, workgroups, s)
                                     : launch_paged_attention<F16, 64>(a, workgroups, s);
    if (err != hipSuccess)
        return set_error(W4G64_STATUS_HIP_ERROR, "paged_attention launch failed: %s", hipGetErrorString(err));
    return clear_error();
}

}  // extern "C"
