// Causal attention over whole prompts of different lengths, packed
// (qwen2_packed_attention, include/qwen2_decode.h).
//
// Work.  A "row" here is a (token, query head) pair of one sequence and key/value
// head: row m is token m / group, head m % group of the group, so that heads that
// share keys fill a tile together and a short prompt's tile is not mostly empty.  A
// workgroup goes through tiles of keys in LDS, the next one on its way (direct loads)
// while the waves work on this one.  kSplit waves share 32 rows, each with kBlocks * 32
// of every tile's keys, and meet in LDS at the end.
//
// One pass over the keys: running maximum, sum and value sums per row.  MFMA layout
// (v_mfma_f32_32x32x16; lane l = 32 h + j supplies row j of A and column j of B with K
// slots 8 h .. 8 h + 7 and receives D[8 (i / 4) + 4 h + i % 4][j] in register i):
//   scores  A = 32 keys, B = 32 query rows: a lane holds 16 of its row's 32 scores,
//           the lane 32 further the others;
//   values  the lane's scores as they are, eight by eight, are its K slots of B: slot e
//           is key 8 (e / 4) + 4 h + e % 4 of 16.  A = the values in that order of the
//           keys, by LDS reads that transpose; dimension 32 dd + j is row j of the dd-th
//           product.
//
// A probability is rounded once, to the tensors' type, before it meets its value: half
// a step of it (2^-9 of its size in bf16) for each key, which the result's own rounding
// matches; the sum that divides adds up the rounded ones, so that what all values have
// in common is not moved.  Scores, maxima and sums are fp32.
//
// The sums are rescaled only once a score passes their reference by kLazy units of the
// base-2 exponent; until then probabilities reach 2^kLazy times the reference's, which
// changes no relative rounding.
//
// What bounds it.  Long prompts: a SIMD's matrix unit and its vector unit, which share the
// time of two waves and overlap only in part.  64 keys by 32 rows of 128 dimensions are
// 32 products (535 ns) and, a lane, 32 exponentials (164 ns) with some 96 other vector
// instructions (236 ns); alone a wave takes 1.2 us for such a tile, two waves 2.0.  12/2
// heads of 128, bf16: one prompt of 16384 tokens 759 to 830 us (by the card; 1090 to 1000
// TFLOP/s, a product of 8192^3 reaching 1206; on the slowest one the matrix unit is busy for
// 55 % of the shader engines' cycles, the vector unit for 44 %, no LDS bank conflicts); three
// of 1003, 4001 and 6999, 32/8 heads, fp16, 559 to 601 (967 to 900).  Heads of 64, half the
// products for the same exponentials: 16384 tokens, 16/16 heads, 645 (852).  Eight of 400 to
// 1600: 46 us (620): the longest prompt's last tiles.  Short ones: loads that depend on each
// other (bounds, then rows, then the output) and the launch: 37 tokens 5.1 to 5.4, 512 10.6.
// What else was measured, us for 16384 tokens against 780: products of the next tile
// between the exponentials of this one by hand 970 to 1300 (registers); a ring of 32-key
// tiles 975 to 1050; one wave a SIMD with more rows 970 to 1240; two groups of waves in
// turns at 256 rows 786 to 801 (a prompt of 4096 100 against 69); wave priorities the
// same.  Eight prompts of 1000 tokens, 44 then: eight waves on 128 rows, two a row, 56;
// tiles of 16 rows straight from memory 158.  The rounded probabilities unpacked and
// added one by one, in place of add_pair(), cost 2.6 %.
#include <math.h>

#include <type_traits>

#include "qwen2_attention.h"
#include "qwen2_packed.h"
#include "qwen2_paged_device.h"
#include "serving_sizes.h"

namespace w4g64 {
namespace {

constexpr int kWaveRows = 32;

struct PackedArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
    const int32_t* cu_rows;
    float scale2;         // |scale| * log2(e), above zero
    uint32_t query_sign;  // both signs of a word of queries where the scale is negative
    int batch, rows, heads, kv_heads, group;
    int zero_rest;
    Divisor by_group, by_kv_heads;
};

template <class E> __device__ __forceinline__ float16v mfma32(const u32x4& a, const u32x4& b, const float16v& c);
template <> __device__ __forceinline__ float16v mfma32<Bf16>(const u32x4& a, const u32x4& b, const float16v& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ float16v mfma32<F16>(const u32x4& a, const u32x4& b, const float16v& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// c plus both halves of a word, in one instruction.  It cuts sums off where an addition
// rounds them (2^-24 of the sum at a time, always down), so it adds up a tile's
// probabilities, not all of them.
template <class E> __device__ __forceinline__ float add_pair(uint32_t w, float c);
template <> __device__ __forceinline__ float add_pair<Bf16>(uint32_t w, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, w), __builtin_bit_cast(bf16x2v, 0x3F803F80u), c, false);
}
template <> __device__ __forceinline__ float add_pair<F16>(uint32_t w, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, w), __builtin_bit_cast(half2v, 0x3C003C00u), c, false);
}

// Over the two lanes j, j + 32.
__device__ __forceinline__ float halves_max(float v) {
    const float2v r = swap32(v);
    return fmaxf(r[0], r[1]);
}
__device__ __forceinline__ float halves_sum(float v) {
    const float2v r = swap32(v);
    return r[0] + r[1];
}

// A value that a rare branch works with: keeps the compiler from running the
// branch's instructions always.
__device__ __forceinline__ int rare(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// What a workgroup works on: a tile of one sequence's rows.
struct Piece {
    int begin;   // the sequence's first row of the tensors
    int count;   // its (token, head) rows
    int tile;
    int kvh;
};

// The piece of workgroup `item`, up to 64 sequences: tiles in the order of their keys'
// number, the most first (a tile's place in its sequence goes by it), so that no
// workgroup begins a long one when the others are done; with kPairs, where a CU holds two
// workgroups, the second one of each of the 256 CUs takes the shortest, as the longest
// tiles are what a call waits for and two of them on a CU slow each other (eight prompts
// of 1000 tokens 44.3 us in order, 41.3 so; one workgroup a CU, a prompt of 2048 31.8 and
// 36.3).
template <int kRows, bool kPairs>
__device__ __forceinline__ bool find_longest(const PackedArgs& a, int item, int lane, Piece& s) {
    // (both bounds and the last one on their way together)
    const int b = min(lane, a.batch - 1);
    const int end = rows_end(a.cu_rows, a.batch, a.rows);
    const PackedRows r = packed_rows(a.cu_rows[b], a.cu_rows[b + 1], end);
    const int count = lane < a.batch ? (r.end - r.begin) * a.group : 0;
    const int tiles = (count + kRows - 1) / kRows;
    const int sum = a.batch == 1 ? __builtin_amdgcn_readfirstlane(tiles) : __builtin_amdgcn_readlane(running_sum(tiles), 63);
    constexpr int kCUs = 256;
    const int all = sum * a.kv_heads, seconds = min(kCUs, all - kCUs);
    if (item >= all) return false;
    if (kPairs && item >= kCUs) item = item < kCUs + seconds ? all - 1 - (item - kCUs) : item - seconds;
    const int index = a.by_kv_heads(item);
    s.kvh = item - index * a.kv_heads;
    int at = 0;
    if (a.batch == 1) {
        s.tile = sum - 1 - index;
    } else {
        // more than `index` tiles have the place `low` in their sequence or a later one,
        // `fewer`, and not more, the place `high`
        int low = 0, high = (a.rows * a.group + kRows - 1) / kRows, fewer = 0;
        while (high - low > 1) {
            const int mid = (low + high) / 2;
            const int from = __builtin_amdgcn_readlane(running_sum(max(tiles - mid, 0)), 63);
            if (from > index) low = mid;
            else high = mid, fewer = from;
        }
        s.tile = low;
        const int has = tiles > low, rank = running_sum(has);  // (of all lanes)
        at = __ffsll((unsigned long long)__ballot(has && rank == index - fewer + 1)) - 1;
    }
    s.begin = __builtin_amdgcn_readlane(r.begin, at);
    s.count = __builtin_amdgcn_readlane(count, at);
    return true;
}

// More sequences: one after the other, the last tile first; 256 are looked through at a
// time, four of a lane.
template <int kRows>
__device__ __forceinline__ bool find_in_turn(const PackedArgs& a, int item, int lane, Piece& s) {
    const int end = rows_end(a.cu_rows, a.batch, a.rows);
    const int index = a.by_kv_heads(item);
    s.kvh = item - index * a.kv_heads;
    int before = 0, next[5];
    auto load = [&](int base) {
#pragma unroll
        for (int i = 0; i < 5; ++i) next[i] = a.cu_rows[min(base + 4 * lane + i, a.batch)];
    };
    load(0);
    for (int base = 0; base < a.batch; base += 256) {
        int bound[5], count[4], tiles[4];
#pragma unroll
        for (int i = 0; i < 5; ++i) bound[i] = next[i];
        load(base + 256);  // (its end over and over, past it)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const PackedRows r = packed_rows(bound[i], bound[i + 1], end);
            bound[i] = r.begin, count[i] = base + 4 * lane + i < a.batch ? (r.end - r.begin) * a.group : 0;
            tiles[i] = (count[i] + kRows - 1) / kRows;
        }
        const int mine = tiles[0] + tiles[1] + tiles[2] + tiles[3];
        const int upto = running_sum(mine), sum = __builtin_amdgcn_readlane(upto, 63);
        if (index >= before + sum) {
            before += sum;
            continue;
        }
        const int at = __ffsll((unsigned long long)__ballot(before + upto > index)) - 1;
        int left = index - (before + __builtin_amdgcn_readlane(upto - mine, at));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int here = __builtin_amdgcn_readlane(tiles[i], at);
            if (left >= 0 && left < here) {
                s.begin = __builtin_amdgcn_readlane(bound[i], at);
                s.count = __builtin_amdgcn_readlane(count[i], at);
                s.tile = here - 1 - left;
            }
            left -= here;
        }
        return true;
    }
    return false;
}

// A row of a tile, as a lane holds it.
struct Row {
    int token;  // of the sequence: the last key that it sees
    int head;
    bool live;  // there is such a row
};
__device__ __forceinline__ Row row_at(const PackedArgs& a, const Piece& s, int m) {
    Row r;
    r.live = m < s.count;
    m = r.live ? m : s.count - 1;
    r.token = a.by_group(m);
    r.head = s.kvh * a.group + (m - r.token * a.group);
    return r;
}

template <int kSteps>
__device__ __forceinline__ void load_queries(const PackedArgs& a, const Piece& s, const Row& row, int h,
                                             u32x4 (&qf)[kSteps]) {
    const uint16_t* from = a.q + (int64_t)(s.begin + row.token) * a.q_row + row.head * a.q_head + 8 * h;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) qf[i] = *(const u32x4*)(from + 16 * i) ^ a.query_sign;
}

// One lane's part of 32 rows: the running softmax and value sums of row j; o[dd][i] is
// dimension 32 dd + 8 (i / 4) + 4 h + i % 4.
template <class E, int D>
struct Attend {
    static constexpr int kVd = D / 32;     // products of the values
    static constexpr int kSteps = D / 16;  // K steps of a score

    float m_run, l_run;
    float16v o[kVd];

    __device__ __forceinline__ void start() {
        m_run = kScoreFloor, l_run = 0.0f;
#pragma unroll
        for (int dd = 0; dd < kVd; ++dd) o[dd] = float16v{};
    }

    // Before a lane's scores become probabilities: the sums rescaled where needed.
    template <int kCount>
    __device__ __forceinline__ void settle(const float (&s)[kCount], float scale2) {
        float top = s[0];
#pragma unroll
        for (int e = 1; e < kCount; ++e) top = fmaxf(top, s[e]);
        const float mn = halves_max(top) * scale2;
        if (__any(mn - m_run > kLazy<E>)) {
            const float to = fmaxf(m_run, mn);
            const float alpha = __builtin_amdgcn_exp2f(m_run - to);  // (1 where it is another row's turn)
            l_run *= alpha;
#pragma unroll
            for (int dd = 0; dd < kVd; ++dd) o[dd] *= alpha;
            m_run = to;
        }
    }

    // Eight scores as probabilities, which `sum` adds up.
    template <int kCount>
    __device__ __forceinline__ u32x4 soften(const float (&s)[kCount], int from, float scale2, float& sum) const {
        const float ref = kProbShift<E> - m_run;
        u32x4 p;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            p[e] = E::pack(__builtin_amdgcn_exp2f(fmaf(s[from + 2 * e], scale2, ref)),
                           __builtin_amdgcn_exp2f(fmaf(s[from + 2 * e + 1], scale2, ref)));
            sum = add_pair<E>(p[e], sum);
        }
        return p;
    }

    // After a counting pass: which sums are not zero, a bit each; and what they say.
    __device__ __forceinline__ uint64_t marks() const {
        uint64_t m = 0;
#pragma unroll
        for (int dd = 0; dd < kVd; ++dd)
#pragma unroll
            for (int i = 0; i < 16; ++i) m |= (uint64_t)(o[dd][i] != 0.0f) << (16 * dd + i);
        return m;
    }
    __device__ __forceinline__ void mark(uint64_t up, uint64_t down) {
#pragma unroll
        for (int dd = 0; dd < kVd; ++dd)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int bit = 16 * dd + i;
                const float plus = (up >> bit) & 1 ? INFINITY : 0.0f, minus = (down >> bit) & 1 ? INFINITY : 0.0f;
                o[dd][i] += plus - minus;  // (both: NaN)
            }
    }
    __device__ __forceinline__ bool finite() const {
        float nothing[4] = {};  // 0 times what is not finite is NaN
#pragma unroll
        for (int dd = 0; dd < kVd; ++dd)
#pragma unroll
            for (int i = 0; i < 16; ++i) nothing[i % 4] = fmaf(o[dd][i], 0.0f, nothing[i % 4]);
        return (nothing[0] + nothing[1]) + (nothing[2] + nothing[3]) == 0.0f;
    }
};

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v* lds_halves_t;

// All of this wave's loads into LDS have landed, then all waves'.
__device__ __forceinline__ void all_landed() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x7 << 4);  // vmcnt 0, lgkmcnt 0 (gfx9 encoding)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A tile's keys or values in LDS: kKeys rows of D elements in 16-byte pieces, piece c of
// row r in slot c ^ turn(r).  Keys are read one piece of 32 rows at a time: the turns of
// 16 rows are all different (D 64: where the rows' banks are the same).  Values are read
// transposed (ds_read_b64_tr_b16: of 16 lanes, lane t brings elements 4 (t % 4) .. of
// row t / 4 and gets element t of the four rows), 64 bytes of 4 rows by 32 lanes: there
// the groups of four pieces are turned.
template <int D, int kWaves, int kKeys>
struct Tile {
    static constexpr int kPieces = D / 8;
    static constexpr int kRowBytes = 2 * D;
    static constexpr int kBytes = kKeys * kRowBytes;
    static constexpr int kWaveKeys = kKeys / kWaves;       // that a wave brings
    static constexpr int kRowsPerLoad = 64 / kPieces;      // rows that a wave's 16-byte load fills
    static constexpr int kLoads = kWaveKeys / kRowsPerLoad;
    static __device__ __forceinline__ int key_turn(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
    static __device__ __forceinline__ int value_turn(int row) { return D == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }
};

template <class E, int D, int kWaves, int kSplit, int kBlocks>
__device__ __forceinline__ void attend_piece(const PackedArgs& a) {
    constexpr int kThreads = 64 * kWaves, kKeys = 32 * kBlocks * kSplit;
    typedef Attend<E, D> A;
    typedef Tile<D, kWaves, kKeys> T;
    constexpr int kRows = kWaves / kSplit * kWaveRows;  // of the workgroup
    // (objects of their own: a read of one does not wait for loads into another)
    __shared__ __attribute__((aligned(16))) unsigned char k0[T::kBytes], v0[T::kBytes], k1[T::kBytes], v1[T::kBytes];
    __shared__ float2v stats[kWaves][64];
    __shared__ int odd;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31;
    const int h = lane >> 5;
    if (a.zero_rest) {
        const FreeRows rest = free_rows(a.cu_rows, a.batch, a.rows);
        for (int64_t i = blockIdx.x, n = free_count(rest, a.rows); i < n; i += gridDim.x) {
            const int64_t r = free_row(rest, (int)i);
            for (int d = 8 * tid; d < a.heads * D; d += 8 * kThreads)
                *(u32x4*)(a.out + r * a.out_row + (d / D) * a.out_head + d % D) = u32x4{0u, 0u, 0u, 0u};
        }
    }
    Piece s;
    constexpr bool kPairs = kWaves == 4 && 4 * T::kBytes <= 80 << 10;  // two workgroups a CU
    if (a.batch <= 64 ? !find_longest<kRows, kPairs>(a, (int)blockIdx.x, lane, s) : !find_in_turn<kRows>(a, (int)blockIdx.x, lane, s))
        return;

    const int part = wave % kSplit;  // of every tile's keys
    const int m0 = s.tile * kRows + kWaveRows * (wave / kSplit);
    // the wave's rows, then the workgroup's (rows past the last one are that one again)
    const int least = a.by_group(min(m0, s.count - 1));
    const int most = m0 < s.count ? a.by_group(min(m0 + kWaveRows, s.count) - 1) : -1;  // (a wave without rows has no keys)
    const int all_most = a.by_group(min((s.tile + 1) * kRows, s.count) - 1);
    const int tiles = all_most / kKeys + 1;

    const uint16_t* kc = a.k + s.begin * a.k_row + s.kvh * a.k_head;
    const uint16_t* vc = a.v + s.begin * a.v_row + s.kvh * a.v_head;
    int k_at[T::kLoads], v_at[T::kLoads];
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) {
        const int r = T::kRowsPerLoad * i + lane / T::kPieces;
        k_at[i] = 2 * r * (int)a.k_row + 16 * ((lane % T::kPieces) ^ T::key_turn(r));
        v_at[i] = 2 * r * (int)a.v_row + 16 * ((lane % T::kPieces) ^ T::value_turn(r));
    }
    auto stage = [&](int tile, unsigned char* keys, unsigned char* values) {
        // (a key past the last visible one: that one again, of no weight)
        const int t = min(tile * kKeys + T::kWaveKeys * wave, all_most), past = min(all_most - t, T::kWaveKeys - 1);
        const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((void*)(kc + t * a.k_row), 0,
                                                                            (past * (int)a.k_row + D) * 2, 0x00020000);
        const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((void*)(vc + t * a.v_row), 0,
                                                                            (past * (int)a.v_row + D) * 2, 0x00020000);
        unsigned char* k_to = keys + T::kWaveKeys * wave * T::kRowBytes;
        unsigned char* v_to = values + T::kWaveKeys * wave * T::kRowBytes;
        if (past < T::kWaveKeys - 1) {
#pragma unroll
            for (int i = 0; i < T::kLoads; ++i) {
                const int r = rare(T::kRowsPerLoad * i + lane / T::kPieces), back = max(r - past, 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_ptr_t)(k_to + 1024 * i), 16,
                                                         k_at[i] - 2 * back * (int)a.k_row, 0, 0, 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_ptr_t)(v_to + 1024 * i), 16,
                                                         v_at[i] - 2 * back * (int)a.v_row, 0, 0, 0);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < T::kLoads; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_ptr_t)(k_to + 1024 * i), 16, k_at[i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < T::kLoads; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_ptr_t)(v_to + 1024 * i), 16, v_at[i], 0, 0, 0);
    };
    if (tid == 0) odd = 0;
    stage(0, k0, v0);
    const Row row = row_at(a, s, m0 + j);
    u32x4 qf[A::kSteps];
    load_queries(a, s, row, h, qf);
    A state;
    auto compute = [&](int tile, const unsigned char* keys, const unsigned char* values, auto ordinary, Pass pass) {
        const int t0 = tile * kKeys + 32 * kBlocks * part;
        if (t0 > most) return;  // (the wave's)
        float x[16 * kBlocks];
        u32x4 kf[2][A::kSteps];
        auto load_keys = [&](int b) {
#pragma unroll
            for (int i = 0; i < A::kSteps; ++i)
                kf[b & 1][i] = *(const u32x4*)(keys + (32 * (kBlocks * part + b) + j) * T::kRowBytes + 16 * ((2 * i + h) ^ T::key_turn(j)));
        };
        load_keys(0);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            if (b + 1 < kBlocks) load_keys(b + 1);
            __builtin_amdgcn_sched_barrier(0);
            float16v acc = {};
#pragma unroll
            for (int i = 0; i < A::kSteps; ++i) acc = mfma32<E>(kf[b & 1][i], qf[i], acc);
#pragma unroll
            for (int e = 0; e < 16; ++e) x[16 * b + e] = acc[e];
        }
        if (t0 + 32 * kBlocks - 1 > least) {
            const int sees = rare(row.token - t0 - 4 * h);
#pragma unroll
            for (int e = 0; e < 16 * kBlocks; ++e)
                if (8 * (e / 4) + e % 4 > sees) x[e] = -INFINITY;
        }
        if (ordinary || pass == kFinite) state.settle(x, a.scale2);
        const int t = lane & 15, block = (lane >> 4) & 1;
        float sum = 0.0f;
        u32x4 vt[2];
        auto load_values = [&](int half, int dd) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int r = 32 * kBlocks * part + 16 * half + 8 * g + 4 * h + t / 4;
                const unsigned char* at = values + r * T::kRowBytes +
                                          16 * ((4 * dd + 2 * block + (t & 3) / 2) ^ T::value_turn(t / 4)) + 8 * (t & 1);
                const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_halves_t)at));
                vt[dd & 1][2 * g] = w[0], vt[dd & 1][2 * g + 1] = w[1];
            }
        };
        load_values(0, 0);
#pragma unroll
        for (int half = 0; half < 2 * kBlocks; ++half) {
            u32x4 p;
            if (ordinary || pass == kFinite) {
                p = state.soften(x, 8 * half, a.scale2, sum);
            } else {  // ones where the row sees the keys
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = t0 + 16 * half + 8 * (e / 2) + 4 * h + 2 * (e % 2);
                    p[e] = (key <= row.token ? E::kOne : 0u) | (key + 1 <= row.token ? E::kOne << 16 : 0u);
                }
            }
#pragma unroll
            for (int dd = 0; dd < A::kVd; ++dd) {
                if (dd + 1 < A::kVd) load_values(half, dd + 1);
                else if (half + 1 < 2 * kBlocks) load_values(half + 1, 0);
                __builtin_amdgcn_sched_barrier(0x7);
                u32x4 w = vt[dd & 1];
                if constexpr (!ordinary)
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = pass_word<E>(w[e], pass);
                state.o[dd] = mfma32<E>(w, p, state.o[dd]);
            }
        }
        state.l_run += sum;
    };
    // The next tile on its way while this one is worked on: its buffer was read before
    // the barrier.
    state.start();
    for (int tile = 0;;) {
        all_landed();
        if (tile + 1 < tiles) stage(tile + 1, k1, v1);
        compute(tile, k0, v0, std::true_type{}, kOrdinary);
        if (++tile >= tiles) break;
        all_landed();
        if (tile + 1 < tiles) stage(tile + 1, k0, v0);
        compute(tile, k1, v1, std::true_type{}, kOrdinary);
        if (++tile >= tiles) break;
    }
    const bool fine = __all(state.finite());
    if (!fine && lane == 0) odd = 1;
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(odd)) {
        uint64_t up = 0, down = 0;
#pragma unroll 1
        for (int pass = kCountUp; pass <= kFinite; ++pass) {
            state.start();
#pragma unroll 1
            for (int tile = 0; tile < tiles; ++tile) {
                stage(tile, k0, v0);
                all_landed();
                compute(tile, k0, v0, std::false_type{}, (Pass)pass);
                __syncthreads();
            }
            if (pass == kCountUp) up = state.marks();
            if (pass == kCountDown) down = state.marks();
        }
        state.mark(up, down);
    }

    const float l_wave = halves_sum(state.l_run);
    uint16_t* to = a.out + (int64_t)(s.begin + row.token) * a.out_row + row.head * a.out_head + 4 * h;
    if constexpr (kSplit == 1) {
        if (!row.live) return;
        const float inv = 1.0f / l_wave;
#pragma unroll
        for (int dd = 0; dd < A::kVd; ++dd)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *(u32x2*)(to + 32 * dd + 2 * i) = u32x2{E::pack(state.o[dd][i] * inv, state.o[dd][i + 1] * inv),
                                                        E::pack(state.o[dd][i + 2] * inv, state.o[dd][i + 3] * inv)};
    } else {
        // The waves' sums meet in LDS, register i of product dd at (16 dd + i) * 64 + lane,
        // and each wave adds up 16 / kSplit registers of every product.
        constexpr int kSums = 64 * 16 * A::kVd, kEach = kWaves / 4;  // floats of a wave; waves in a buffer
        static_assert(T::kBytes >= kEach * kSums * (int)sizeof(float), "the waves' sums fit the tiles");
        auto sums_of = [&](int w) {
            const int at = w / kEach;
            return (float*)(at < 2 ? (at ? v0 : k0) : (at > 2 ? v1 : k1)) + w % kEach * kSums;
        };
#pragma unroll
        for (int dd = 0; dd < A::kVd; ++dd)
#pragma unroll
            for (int i = 0; i < 16; ++i) sums_of(wave)[(16 * dd + i) * 64 + lane] = state.o[dd][i];
        // (-inf: no key in the wave's parts)
        stats[wave][lane] = float2v{row.token >= 32 * kBlocks * part ? state.m_run : -INFINITY, l_wave};
        __syncthreads();
        if (!row.live) return;
        const int first = wave - part;
        float top = -INFINITY, l = 0.0f, sum[16 / kSplit][A::kVd] = {};
#pragma unroll
        for (int w = 0; w < kSplit; ++w) top = fmaxf(top, stats[first + w][lane][0]);
#pragma unroll
        for (int w = 0; w < kSplit; ++w) {
            const float2v st = stats[first + w][lane];
            const float f = __builtin_amdgcn_exp2f(st[0] - top);
            const float* from = sums_of(first + w) + 16 / kSplit * part * 64 + lane;
            if (f != 0.0f) {
                l = fmaf(st[1], f, l);
#pragma unroll
                for (int i = 0; i < 16 / kSplit; ++i)
#pragma unroll
                    for (int dd = 0; dd < A::kVd; ++dd) sum[i][dd] = fmaf(from[(16 * dd + i) * 64], f, sum[i][dd]);
            } else if (st[0] > -INFINITY) {
                // keys of no weight beside the others': nothing, unless a value that the row
                // sees was not finite
                if (st[1] != st[1]) l = st[1];
#pragma unroll
                for (int i = 0; i < 16 / kSplit; ++i)
#pragma unroll
                    for (int dd = 0; dd < A::kVd; ++dd) add_odd(sum[i][dd], from[(16 * dd + i) * 64]);
            }
        }
        const float inv = 1.0f / l;
        to += 2 * (16 / kSplit) * part;
#pragma unroll
        for (int dd = 0; dd < A::kVd; ++dd)
#pragma unroll
            for (int i = 0; i < 16 / kSplit; i += 4)
                *(u32x2*)(to + 32 * dd + 2 * i) = u32x2{E::pack(sum[i][dd] * inv, sum[i + 1][dd] * inv),
                                                        E::pack(sum[i + 2][dd] * inv, sum[i + 3][dd] * inv)};
    }
}

// (waves per SIMD: two with 256 registers each, where LDS holds as much; short prompts of
// 64 dimensions four, for which nine registers are put away during the counting passes
// alone: 200 of 30 15.1 -> 13.4 us, 32 of 200 17.6 -> 16.2, 96 of 1 to 119 14.0 -> 14.3)
template <class E, int D, int kWaves, int kSplit, int kBlocks>
__global__ __launch_bounds__(64 * kWaves, kWaves == 4 && kSplit == 4 && D == 128 ? 1 : kWaves == 2 && D == 64 ? 4 : 2)
void packed_attention_kernel(PackedArgs a) {
    attend_piece<E, D, kWaves, kSplit, kBlocks>(a);
}

// The forms of a call's workgroups.
enum Form { kShort, kLong, kSplit2, kSplit4, kSplit4Tall };
int tile_rows(Form f) { return f == kLong ? 128 : f == kSplit4 ? 32 : 64; }

template <class E, int D>
hipError_t launch_packed_attention(const PackedArgs& a, Form form, int64_t workgroups, hipStream_t stream) {
    const dim3 grid((unsigned)workgroups);
    if (form == kShort) hipLaunchKernelGGL((packed_attention_kernel<E, D, 2, 1, 1>), grid, dim3(128), 0, stream, a);
    else if (form == kLong) hipLaunchKernelGGL((packed_attention_kernel<E, D, 4, 1, 2>), grid, dim3(256), 0, stream, a);
    else if (form == kSplit2) hipLaunchKernelGGL((packed_attention_kernel<E, D, 4, 2, 1>), grid, dim3(256), 0, stream, a);
    else if (form == kSplit4) hipLaunchKernelGGL((packed_attention_kernel<E, D, 4, 4, 1>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((packed_attention_kernel<E, D, 8, 4, 1>), grid, dim3(512), 0, stream, a);
    return hipGetLastError();
}

// The form of a call.  Prompts of a tile or two want small workgroups, of which a CU holds
// many (kShort, tiles of 32 keys).  A longer one's time is that of its keys one tile
// after the other, so long as the chip holds all workgroups at once; then what counts is
// the products' rate, which the fewest waves per row give.  The lengths are on the GPU: it
// goes by the sequences' average.
// us a call, 12/2 heads of 128, kShort / best of the others: one prompt of 16 tokens
// 5.3 / 6.7, 64 6.1 / 7.1, 128 7.4 / 7.6, 256 10.1 / 8.7; 96 of 10 6.1 / 6.8; sixteen of
// 128 10.4 / 11.3, 200 13.2 / 14.1, 300 17.6 / 17.6; 32 of 200 20.4 / 23.6, 500 55.9 /
// 50.4; 16/16 heads of 64, 200 of 30 15.4 / 21.7; four of 200 7.6 / 7.1, 16 of 200 10.4 / 11.7; one
// prompt of 2000 among 40 of 16 tokens, on the other hand, 49 / 33.
// kLong / kSplit2 / kSplit4 / kSplit4Tall: one of 512 15.3 / 12.3 / 11.1 / 12.1, 1024 24.6 / 19.2 /
// 19.6 / 17.3, 2048 43 / 34 / 50 / 30, 3000 62 / 50 / 94 / 58, 16384 795 / 908 / 1991 / 1019;
// four of 512 16.9 / 15.5 / 28 / 21, eight 20 / 24 / 54 / 33; 16/16 heads of 64: one of 1000 17.1 /
// 13.4 / 10.6 / 11.8, two 18.4 / 15.4 / 19.5 / 18.1.
Form form_of(int64_t rows, int64_t sequences, int64_t group, int64_t kv_heads, int64_t head_dim) {
    const int64_t usual = rows / sequences, few = head_dim == 128 ? 288 : 576, half = head_dim == 128 ? 256 : 512;
    auto tiles = [&](int64_t size) { return sequences * ((usual * group + size - 1) / size) * kv_heads; };
    if (usual <= 128 || (usual <= 256 && tiles(64) > 512)) return kShort;
    if (tiles(32) <= few) return kSplit4;
    if (tiles(64) <= 256 || (tiles(64) <= half * 3 / 2 && usual >= 1024)) return kSplit4Tall;
    return tiles(64) <= 512 || (tiles(64) <= 800 && usual >= 2048) ? kSplit2 : kLong;
}

// How a call is cut up, if its sizes are any (a status if not).
struct PackedPlan {
    Form form;
    int64_t group, workgroups;
};
int packed_plan(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t k_row, int64_t v_row,
                int dtype, float scale, PackedPlan* plan) {
    if (dtype != W4G64_DTYPE_BF16 && dtype != W4G64_DTYPE_F16)
        return set_error(W4G64_STATUS_INVALID_DTYPE, "packed_attention dtype must be bf16 or fp16, got code %d", dtype);
    if (head_dim != 64 && head_dim != 128)
        return set_error(W4G64_STATUS_UNSUPPORTED, "packed_attention needs a head_dim of 64 or 128, got %lld", (long long)head_dim);
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads || heads > 0xFFFF)
        return set_error(W4G64_STATUS_INVALID_VALUE, "packed_attention heads must be a positive multiple of kv_heads, got %lld and %lld",
                         (long long)heads, (long long)kv_heads);
    if (rows < 0 || rows > 0x7FFFFFF || batch < 0 || batch > 0x7FFFFFF)
        return set_error(W4G64_STATUS_INVALID_VALUE, "packed_attention rows and batch must be in [0, 2^27), got %lld and %lld",
                         (long long)rows, (long long)batch);
    if (!isfinite(scale)) return set_error(W4G64_STATUS_INVALID_VALUE, "packed_attention scale must be finite");
    if (rows == 0 || batch == 0) return clear_error();
    if (k_row > (1 << 24) || v_row > (1 << 24) || k_row < 0 || v_row < 0)
        return set_error(W4G64_STATUS_UNSUPPORTED, "k and v rows must be at most 2^24 elements apart");
    const int64_t group = heads / kv_heads, sequences = batch < rows ? batch : rows;
    const Form form = form_of(rows, sequences, group, kv_heads, head_dim);
    // (every sequence may end inside a tile; the empty ones have none)
    const int64_t workgroups = (rows * group / tile_rows(form) + sequences) * kv_heads;
    if (rows * heads > 0x7FF00000 || workgroups > 0xFFFFFF)
        return set_error(W4G64_STATUS_UNSUPPORTED, "packed_attention call is too large: %lld workgroups", (long long)workgroups);
    *plan = PackedPlan{form, group, workgroups};
    return clear_error();
}

}  // namespace

int packed_attention_sizes(int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t k_row,
                           int64_t v_row, int dtype, float scale) {
    PackedPlan plan;
    return packed_plan(batch, rows, heads, kv_heads, head_dim, k_row, v_row, dtype, scale, &plan);
}

}  // namespace w4g64

using namespace w4g64;

extern "C" int qwen2_packed_attention(const qwen2_rows* q, const qwen2_rows* k, const qwen2_rows* v, const qwen2_rows* out,
                                      const int32_t* cu_rows, int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads,
                                      int64_t head_dim, int dtype, float scale, int zero_rest, void* stream) {
    PackedPlan plan;
    const int status = packed_plan(batch, rows, heads, kv_heads, head_dim, k ? k->row : 0, v ? v->row : 0, dtype, scale, &plan);
    if (status || rows == 0 || batch == 0) return status;
    for (const qwen2_rows* r : {q, k, v, out})
        if (!r || !r->data || ((uintptr_t)r->data & 15) || r->row % 8 || r->head % 8)
            return set_error(W4G64_STATUS_INVALID_VALUE,
                             "q, k, v and out must be non-null, 16-byte aligned, with strides that are multiples of 8 elements");
    if (!cu_rows || ((uintptr_t)cu_rows & 3))
        return set_error(W4G64_STATUS_INVALID_VALUE, "cu_rows must be a non-null, 4-byte aligned device pointer");
    const auto [form, group, workgroups] = plan;
    PackedArgs a{};
    a.q = (const uint16_t*)q->data, a.q_row = q->row, a.q_head = q->head;
    a.k = (const uint16_t*)k->data, a.k_row = k->row, a.k_head = k->head;
    a.v = (const uint16_t*)v->data, a.v_row = v->row, a.v_head = v->head;
    a.out = (uint16_t*)out->data, a.out_row = out->row, a.out_head = out->head;
    a.cu_rows = cu_rows;
    // (a scale of zero: as small as there is, so that a hidden key's -inf stays -inf)
    const float scale2 = fabsf(scale) * 1.44269504088896340736f;
    a.scale2 = scale2 > 0.0f ? fminf(scale2, 3.402823466e+38f) : 1.401298464324817e-45f;
    a.query_sign = scale < 0.0f ? 0x80008000u : 0u;
    a.batch = (int)batch, a.rows = (int)rows, a.heads = (int)heads, a.kv_heads = (int)kv_heads, a.group = (int)group;
    a.zero_rest = zero_rest;
    a.by_group = divisor(group), a.by_kv_heads = divisor(kv_heads);
    const hipStream_t s = (hipStream_t)stream;
    hipError_t err;
    if (dtype == W4G64_DTYPE_BF16)
        err = head_dim == 128 ? launch_packed_attention<Bf16, 128>(a, form, workgroups, s) : launch_packed_attention<Bf16, 64>(a, form, workgroups, s);
    else
        err = head_dim == 128 ? launch_packed_attention<F16, 128>(a, form, workgroups, s) : launch_packed_attention<F16, 64>(a, form, workgroups, s);
    if (err != hipSuccess) return set_error(W4G64_STATUS_HIP_ERROR, "packed_attention launch failed: %s", hipGetErrorString(err));
    return clear_error();
}
