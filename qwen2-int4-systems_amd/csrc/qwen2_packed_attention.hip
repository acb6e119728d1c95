// Causal attention over whole prompts of different lengths, packed
// (qwen2_packed_attention, include/qwen2_decode.h).
//
// Work.  A "row" here is a (token, query head) pair of one sequence and key/value
// head: row m is token m / group, head m % group of the group, so that heads that
// share keys fill a tile together and a short prompt's tile is not mostly empty.  A
// workgroup of four waves takes a tile of rows in one of two forms:
//   narrow    32 rows.  The waves take different 32-key blocks, straight from memory
//             into operands, and meet in LDS at the end.
//   wide      128 rows, 32 of each wave.  The workgroup goes through 64-key tiles in
//             LDS, the next one on its way (direct loads) while the waves work on this
//             one.
//
// One pass over the keys: running maximum, sum and value sums per row.  MFMA layout
// (v_mfma_f32_32x32x16; lane l = 32 h + j supplies row j of A and column j of B with K
// slots 8 h .. 8 h + 7 and receives D[8 (i / 4) + 4 h + i % 4][j] in register i):
//   scores  A = 32 keys, B = 32 query rows: a lane holds 16 of its row's 32 scores,
//           the lane 32 further the others;
//   values  the lane's scores as they are, eight by eight, are its K slots of B: slot e
//           is key 8 (e / 4) + 4 h + e % 4 of 16.  A = the values transposed, in that
//           order of the keys.  Narrow: lane (j, h) loads kVd = D / 32 dimensions from
//           kVd j of its keys and pairs keys up by v_perm; dimension kVd j + dd is row
//           j of the dd-th product.  Wide: LDS reads that transpose; dimension 32 dd +
//           j is row j of the dd-th product.
//
// A probability is rounded once, to the tensors' type, before it meets its value: half
// a step of it (2^-9 of its size in bf16) for each key, which the result's own rounding
// matches; the sum that divides adds up the rounded ones, so that what all values have
// in common is not moved.  Scores, maxima and sums are fp32.
//
// The sums are rescaled only once a score passes their reference by kLazy units of the
// base-2 exponent; until then probabilities reach 2^kLazy times the reference's, which
// changes no relative rounding.
#include <math.h>

#include <type_traits>

#include "qwen2_attention.h"
#include "qwen2_packed.h"
#include "qwen2_paged_device.h"

namespace w4g64 {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kNarrowRows = 32;
constexpr int kBlock = 32;     // keys of a narrow block

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

// c plus both halves of a word.
template <class E> __device__ __forceinline__ float add_pair(uint32_t w, float c) {
    return c + (E::lo(w) + E::hi(w));
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

// Tile `index`: the tiles of every sequence counted up, 64 sequences at a time; those
// of a sequence from its end, where the most keys are.
template <int kRows>
__device__ __forceinline__ bool find_piece(const PackedArgs& a, int index, int lane, Piece& s) {
    int before = 0;
    const int all = rows_end(a.cu_rows, a.batch, a.rows);
    for (int base = 0; base < a.batch; base += 64) {
        const int b = base + lane;
        PackedRows r{0, 0};
        if (b < a.batch) r = packed_rows(a.cu_rows, b, all);
        const int count = (r.end - r.begin) * a.group;
        const int tiles = (count + kRows - 1) / kRows;
        int upto = tiles;
        for (int d = 1; d < 64; d <<= 1) {
            const int other = __shfl_up(upto, d);
            if (lane >= d) upto += other;
        }
        const uint64_t past = __ballot(before + upto > index);
        if (past) {
            const int at = __ffsll((unsigned long long)past) - 1;
            s.begin = __builtin_amdgcn_readlane(r.begin, at);
            s.count = __builtin_amdgcn_readlane(count, at);
            s.tile = before + __builtin_amdgcn_readlane(upto, at) - 1 - index;
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
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
__device__ __forceinline__ void load_queries(const PackedArgs& a, const Piece& s, const Row& row, int h, u32x4 (&qf)[kSteps]) {
    const uint16_t* from = a.q + (int64_t)(s.begin + row.token) * a.q_row + row.head * a.q_head + 8 * h;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) qf[i] = *(const u32x4*)(from + 16 * i) ^ a.query_sign;
}

// One lane's part of 32 rows: the running softmax and value sums of row j; o[dd][i]
// is row 8 (i / 4) + 4 h + i % 4 of the dd-th product.
template <class E, int D>
struct Attend {
    static constexpr int kVd = D / 32;
    static constexpr int kVw = kVd / 2;
    static constexpr int kSteps = D / 16;  // K steps of a score
    typedef uint32_t vword __attribute__((ext_vector_type(kVw)));

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

    // Eight scores as probabilities.
    template <int kCount>
    __device__ __forceinline__ u32x4 soften(const float (&s)[kCount], int from, float scale2) {
        const float ref = kProbShift<E> - m_run;
        u32x4 p;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            p[e] = E::pack(__builtin_amdgcn_exp2f(fmaf(s[from + 2 * e], scale2, ref)),
                           __builtin_amdgcn_exp2f(fmaf(s[from + 2 * e + 1], scale2, ref)));
            l_run = add_pair<E>(p[e], l_run);
        }
        return p;
    }

    // Eight keys' ones where the row sees them (keys 8 (e / 4) + 4 h + e % 4 from t0).
    static __device__ __forceinline__ u32x4 show(int limit, int t0, int h) {
        u32x4 p;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int t = t0 + 8 * (e / 2) + 4 * h + 2 * (e % 2);
            p[e] = (t <= limit ? E::kOne : 0u) | (t + 1 <= limit ? E::kOne << 16 : 0u);
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
        bool fine = true;
#pragma unroll
        for (int dd = 0; dd < kVd; ++dd)
#pragma unroll
            for (int i = 0; i < 16; ++i) fine = fine && fabsf(o[dd][i]) < INFINITY;
        return fine;
    }
};

// ---- narrow ----

template <class E, int D>
struct KeyBlock {
    u32x4 k[D / 16];                    // key j, dimensions 16 i + 8 h ..
    typename Attend<E, D>::vword v[16];  // value of key 16 (e / 8) + 8 (e % 8 / 4) + 4 h + e % 4, dimensions kVd j ..
};

// The lane's value sums of each wave in LDS: 64 lanes of 16 D / 32 floats, so that a
// wave's piece is one tile of 64 keys.
template <int D> constexpr int kMeetBytes = 64 * 16 * (D / 32) * (int)sizeof(float);

template <class E, int D>
__device__ __forceinline__ void narrow(const PackedArgs& a, const Piece& s, int tile, int lane, int wave,
                                       unsigned char* meet0, unsigned char* meet1, unsigned char* meet2,
                                       unsigned char* meet3, float2v (*stats)[64]) {
    typedef Attend<E, D> A;
    const int j = lane & 31;
    const int h = lane >> 5;
    const int m0 = tile * kNarrowRows;
    const int least = a.by_group(m0), most = a.by_group(min(m0 + kNarrowRows, s.count) - 1);
    const int blocks = most / kBlock + 1;
    const uint16_t* kc = a.k + s.begin * a.k_row + s.kvh * a.k_head + 8 * h;
    const uint16_t* vc = a.v + s.begin * a.v_row + s.kvh * a.v_head + A::kVd * j;
    // (a key past the last visible one: that one again, of no weight)
    auto load = [&](KeyBlock<E, D>& b, int block) {
        const int t0 = block * kBlock;
        const uint16_t* kp = kc + (int64_t)min(t0 + j, most) * a.k_row;
#pragma unroll
        for (int i = 0; i < A::kSteps; ++i) b.k[i] = *(const u32x4*)(kp + 16 * i);
#pragma unroll
        for (int e = 0; e < 16; ++e)
            b.v[e] = *(const typename A::vword*)(vc + (int64_t)min(t0 + 8 * (e / 4) + 4 * h + e % 4, most) * a.v_row);
    };
    KeyBlock<E, D> b;
    if (wave < blocks) load(b, wave);
    const Row row = row_at(a, s, m0 + j);
    u32x4 qf[A::kSteps];
    load_queries(a, s, row, h, qf);
    A state;
    auto compute = [&](const KeyBlock<E, D>& b, int block, auto ordinary, Pass pass) {
        const int t0 = block * kBlock;
        float16v acc = {};
#pragma unroll
        for (int i = 0; i < A::kSteps; ++i) acc = mfma32<E>(b.k[i], qf[i], acc);
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = acc[e];
        if (t0 + kBlock - 1 > least) {
            const int sees = rare(row.token - t0 - 4 * h);
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (8 * (e / 4) + e % 4 > sees) x[e] = -INFINITY;
        }
        if (ordinary || pass == kFinite) state.settle(x, a.scale2);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const u32x4 p = ordinary || pass == kFinite ? state.soften(x, 8 * half, a.scale2)
                                                        : A::show(row.token, t0 + 16 * half, h);
#pragma unroll
            for (int dd = 0; dd < A::kVd; ++dd) {
                const uint32_t select = (dd & 1) ? 0x07060302u : 0x05040100u;  // high or low halves
                u32x4 vt;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    vt[e] = __builtin_amdgcn_perm(b.v[8 * half + 2 * e + 1][dd / 2], b.v[8 * half + 2 * e][dd / 2], select);
                    if constexpr (!ordinary) vt[e] = pass_word<E>(vt[e], pass);
                }
                state.o[dd] = mfma32<E>(vt, p, state.o[dd]);
            }
        }
    };
    state.start();
    for (int block = wave; block < blocks;) {
        compute(b, block, std::true_type{}, kOrdinary);
        block += kWaves;
        if (block < blocks) load(b, block);
    }
    if (!__all(state.finite())) {  // (the wave's)
        uint64_t up = 0, down = 0;
#pragma unroll 1
        for (int pass = kCountUp; pass <= kFinite; ++pass) {
            state.start();
#pragma unroll 1
            for (int block = wave; block < blocks; block += kWaves) {
                load(b, block);
                compute(b, block, std::false_type{}, (Pass)pass);
            }
            if (pass == kCountUp) up = state.marks();
            if (pass == kCountDown) down = state.marks();
        }
        state.mark(up, down);
    }

    // ---- the waves' results meet in LDS: register i of product dd at (16 dd + i) * 64 + lane ----
    auto meet = [&](int w) { return (float*)(w < 2 ? (w ? meet1 : meet0) : (w > 2 ? meet3 : meet2)); };
#pragma unroll
    for (int dd = 0; dd < A::kVd; ++dd)
#pragma unroll
        for (int i = 0; i < 16; ++i) meet(wave)[(16 * dd + i) * 64 + lane] = state.o[dd][i];
    // (-inf: no key in the wave's blocks)
    stats[wave][lane] = float2v{row.token >= wave * kBlock ? state.m_run : -INFINITY, halves_sum(state.l_run)};
    __syncthreads();
    // this wave's registers 4 wave .. 4 wave + 3 of every product
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w][lane][0]);
    float l = 0.0f, sum[4][A::kVd] = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const float2v st = stats[w][lane];
        const float f = __builtin_amdgcn_exp2f(st[0] - top);
        const float* from = meet(w) + (4 * wave) * 64 + lane;
        if (f != 0.0f) {
            l = fmaf(st[1], f, l);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int dd = 0; dd < A::kVd; ++dd) sum[i][dd] = fmaf(from[(16 * dd + i) * 64], f, sum[i][dd]);
        } else if (st[0] > -INFINITY) {
            // keys of no weight beside the others': nothing, unless a value that the row
            // sees was not finite
            if (st[1] != st[1]) l = st[1];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int dd = 0; dd < A::kVd; ++dd) add_odd(sum[i][dd], from[(16 * dd + i) * 64]);
        }
    }
    if (!row.live) return;
    const float inv = 1.0f / l;
    uint16_t* to = a.out + (int64_t)(s.begin + row.token) * a.out_row + row.head * a.out_head + A::kVd * (8 * wave + 4 * h);
    uint32_t word[2 * A::kVd];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int dd = 0; dd < A::kVd; dd += 2) word[(A::kVd * i + dd) / 2] = E::pack(sum[i][dd] * inv, sum[i][dd + 1] * inv);
#pragma unroll
    for (int i = 0; i < 2 * A::kVd; i += 4) *(u32x4*)(to + 2 * i) = u32x4{word[i], word[i + 1], word[i + 2], word[i + 3]};
}

template <class E, int D>
__global__ __launch_bounds__(kThreads, 2) void packed_attention_kernel(PackedArgs a) {
    __shared__ __attribute__((aligned(16))) unsigned char k0[kMeetBytes<D>], v0[kMeetBytes<D>], k1[kMeetBytes<D>], v1[kMeetBytes<D>];
    __shared__ float2v stats[kWaves][64];
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (a.zero_rest) {
        for (int64_t r = rest_row(a.cu_rows, a.batch, a.rows, blockIdx.x); r < a.rows; r += gridDim.x)
            for (int d = 8 * tid; d < a.heads * D; d += 8 * kThreads)
                *(u32x4*)(a.out + r * a.out_row + (d / D) * a.out_head + d % D) = u32x4{0u, 0u, 0u, 0u};
    }
    Piece s;
    const int index = a.by_kv_heads((int)blockIdx.x);
    s.kvh = (int)blockIdx.x - index * a.kv_heads;
    if (!find_piece<kNarrowRows>(a, index, lane, s)) return;
    narrow<E, D>(a, s, s.tile, lane, wave, k0, v0, k1, v1, stats);
}

template <class E, int D>
hipError_t launch_packed_attention(const PackedArgs& a, int64_t workgroups, hipStream_t stream) {
    hipLaunchKernelGGL((packed_attention_kernel<E, D>), dim3((unsigned)workgroups), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace
}  // namespace w4g64

using namespace w4g64;

extern "C" int qwen2_packed_attention(const qwen2_rows* q, const qwen2_rows* k, const qwen2_rows* v, const qwen2_rows* out,
                                      const int32_t* cu_rows, int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads,
                                      int64_t head_dim, int dtype, float scale, int zero_rest, void* stream) {
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
    for (const qwen2_rows* r : {q, k, v, out})
        if (!r || !r->data || ((uintptr_t)r->data & 15) || r->row % 8 || r->head % 8)
            return set_error(W4G64_STATUS_INVALID_VALUE,
                             "q, k, v and out must be non-null, 16-byte aligned, with strides that are multiples of 8 elements");
    if (!cu_rows || ((uintptr_t)cu_rows & 3))
        return set_error(W4G64_STATUS_INVALID_VALUE, "cu_rows must be a non-null, 4-byte aligned device pointer");
    const int64_t group = heads / kv_heads, sequences = batch < rows ? batch : rows;
    // (every sequence may end inside a tile; the empty ones have none)
    const int64_t workgroups = (rows * group / kNarrowRows + sequences) * kv_heads;
    if (rows * heads > 0x7FF00000 || workgroups > 0xFFFFFF)
        return set_error(W4G64_STATUS_UNSUPPORTED, "packed_attention call is too large: %lld workgroups", (long long)workgroups);
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
        err = head_dim == 128 ? launch_packed_attention<Bf16, 128>(a, workgroups, s) : launch_packed_attention<Bf16, 64>(a, workgroups, s);
    else
        err = head_dim == 128 ? launch_packed_attention<F16, 128>(a, workgroups, s) : launch_packed_attention<F16, 64>(a, workgroups, s);
    if (err != hipSuccess) return set_error(W4G64_STATUS_HIP_ERROR, "packed_attention launch failed: %s", hipGetErrorString(err));
    return clear_error();
}
