// Attention over a paged cache, the batch's common prefix computed once
// (qwen2_paged_attention, include/qwen2_decode.h).
//
// Work.  A "row" here is a (packed row, query head) pair of one key/value head:
// row m of a segment is token m / group, head m % group.  Two kinds of segment
// share one launch:
//   prefix    all rows of the batch against the shared pages of the table's
//             first row: the keys are read once per 16 rows, not per sequence;
//   own       one sequence's rows against the rest of its pages.
// A workgroup takes 16 rows of a segment and one of several splits of its keys;
// 32-key blocks are dealt round robin to the splits, then to the workgroup's
// four waves, which work alone and meet in LDS at the end.  A second launch
// joins the splits of both kinds.
//
// One pass over the keys: running maximum, sum and value sums per row.  MFMA
// layout (v_mfma_f32_16x16x32; lane l = 16 q + j supplies row j of A and column
// j of B with K slots 8 q .. 8 q + 7 and receives D[4 q + r][j]):
//   scores  A = 16 keys, B = the 16 query rows: lane (j, q) gets row j's scores
//           of keys 4 q + r;
//   values  the lane's own 8 probabilities of a 32-key block are its 8 K slots;
//           A = the values transposed: lane (j, q) loads kVd = D / 16 dimensions
//           from kVd j of its 8 keys and pairs keys up by v_perm; dimension
//           kVd j + dd is row j of the dd-th product.
// A probability is kept as two 16-bit terms (16 bits or more of it): one term
// alone would be as coarse as the output.
//
// Pages hold at least 16 positions, so that 16 aligned keys lie in one page and
// the page's number is the wave's, not the lane's.  Every loaded address lies in
// a page of the pool; what a block holds past the last visible key is replaced
// by zeros, scores there by -inf.
#include <math.h>

#include "qwen2_attention.h"
#include "qwen2_paged_device.h"

namespace w4g64 {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kTile = 16;   // rows of a workgroup
constexpr int kBlock = 32;  // keys of a block
constexpr int kMaxSplits = 64;

struct PagedAttnArgs {
    PagedView c;
    const uint16_t* q;
    uint16_t* out;
    int64_t q_row, q_head, out_row, out_head;
    float* stats;     // [rows][heads][slots] (maximum, sum)
    float* partials;  // [rows][heads][slots][D]
    float scale2;     // scale * log2(e)
    int rows, heads, group;
    int prefix;       // positions of the shared pages
    int prefix_tiles, prefix_splits, own_tiles, own_splits, slots;
    int zero_rest;
};

// Shift of the probabilities' exponent: fp16 ends at 2^-24, and a key far below
// its row's maximum still counts if there are many; with 2^14 for the maximum
// the terms reach down to 2^-38 of it.
template <class E> constexpr float kProbShift = 0.0f;
template <> constexpr float kProbShift<F16> = 14.0f;

__device__ __forceinline__ uint32_t keep_halves(uint32_t w, bool lo, bool hi) {
    return w & ((lo ? 0x0000FFFFu : 0u) | (hi ? 0xFFFF0000u : 0u));
}
template <class E> __device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
    return keep_halves(w, (w & E::kExponent) != E::kExponent, ((w >> 16) & E::kExponent) != E::kExponent);
}

// The sequence and place of own tile `tile` of 16 rows: the tiles of every
// sequence counted up, 64 sequences at a time.  false: past the last one.
__device__ __forceinline__ bool find_tile(const PagedAttnArgs& a, int tile, int lane, int& sequence, int& local) {
    int before = 0;
    for (int base = 0; base < a.c.batch; base += 64) {
        const int i = base + lane;
        int count = 0;
        if (i < a.c.batch) {
            const SequenceRows s = sequence_rows(a.c.cu_rows, a.c.lengths, i, a.rows);
            count = (int)(((int64_t)(s.end - s.begin) * a.group + kTile - 1) / kTile);
        }
        int upto = count;
#pragma unroll
        for (int step = 1; step < 64; step *= 2) {
            const int other = __shfl_up(upto, step);
            if (lane >= step) upto += other;
        }
        const uint64_t past = __ballot(before + upto > tile);
        if (past) {
            const int at = __ffsll((unsigned long long)past) - 1;
            sequence = base + at;
            local = tile - before - __shfl(upto - count, at);
            return true;
        }
        before += __shfl(upto, 63);
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

template <class E, int D>
__global__ __launch_bounds__(kThreads, 2) void paged_attention_kernel(PagedAttnArgs a) {
    constexpr int kVd = D / 16;           // dimensions of a value per lane
    constexpr int kVw = kVd / 2;          // words of them
    constexpr int kSteps = D / 32;        // K steps of a score
    constexpr int kStride = D + 4;
    typedef uint32_t vword __attribute__((ext_vector_type(kVw)));
    __shared__ __attribute__((aligned(16))) float so[kWaves][kTile][kStride];
    __shared__ float sm[kWaves][kTile];
    __shared__ float sl[kWaves][kTile];
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 15;
    const int q = lane >> 4;

    // rows behind the last sequence, where no second launch sees to them
    if (a.slots == 1 && a.zero_rest) {
        for (int r = max(a.c.cu_rows[a.c.batch], 0) + (int)blockIdx.x; r < a.rows; r += (int)gridDim.x)
            for (int d = 8 * tid; d < a.heads * D; d += 8 * kThreads)
                *(u32x4*)(a.out + r * a.out_row + (d / D) * a.out_head + d % D) = u32x4{0u, 0u, 0u, 0u};
    }

    // ---- which rows, which keys ----
    const int prefix_work = a.prefix_tiles * a.c.kv_heads * a.prefix_splits;
    const bool shared = (int)blockIdx.x < prefix_work;
    const int work = shared ? (int)blockIdx.x : (int)blockIdx.x - prefix_work;
    const int splits = shared ? a.prefix_splits : a.own_splits;
    const int split = work % splits;
    const int kvh = work / splits % a.c.kv_heads;
    int tile = work / splits / a.c.kv_heads;
    int first_token = 0, tokens = a.rows, sequence = 0;
    if (!shared) {
        int local;
        if (!find_tile(a, tile, lane, sequence, local)) return;
        sequence = __builtin_amdgcn_readfirstlane(sequence);
        tile = __builtin_amdgcn_readfirstlane(local);
        const SequenceRows s = sequence_rows(a.c.cu_rows, a.c.lengths, sequence, a.rows);
        first_token = s.begin;
        tokens = s.end - s.begin;
    }
    const int64_t m = (int64_t)tile * kTile + j;  // this lane's row
    const bool live = m < (int64_t)tokens * a.group;
    const int64_t mc = live ? m : (int64_t)tokens * a.group - 1;
    const int token = first_token + (int)(mc / a.group);
    const int head = kvh * a.group + (int)(mc % a.group);
    // the row's position; rows that no sequence has see nothing
    int64_t position = -1;
    bool known = live;
    if (shared) {
        const int b = sequence_by_halving(a.c.cu_rows, a.c.batch, token);
        known = known && b < a.c.batch;
        if (known) {
            const SequenceRows s = sequence_rows(a.c.cu_rows, a.c.lengths, b, a.rows);
            known = token >= s.begin && token < s.end;
            position = s.first + (token - s.begin);
        }
    } else {
        const SequenceRows s = sequence_rows(a.c.cu_rows, a.c.lengths, sequence, a.rows);
        position = s.first + (token - s.begin);
    }
    if (!known) position = -1;
    const int64_t held = (int64_t)a.c.table_width << a.c.page_shift;
    const bool beyond = position >= held;  // reaches past its table
    // last key of this segment that the row sees, below the segment's first if none
    const int key_lo = shared ? 0 : a.prefix;
    const int64_t key_end = shared ? a.prefix : held;
    const int limit = (int)max(min(position, key_end - 1), (int64_t)(key_lo - 1));
    int most = live ? limit : key_lo - 1, least = live ? limit : 0x7FFFFFFF;
#pragma unroll
    for (int step = 1; step < 16; step *= 2) {
        most = max(most, __shfl_xor(most, step));
        least = min(least, __shfl_xor(least, step));
    }
    most = __builtin_amdgcn_readfirstlane(most);
    least = __builtin_amdgcn_readfirstlane(least);
    const int blocks = (most - key_lo) / kBlock + (most >= key_lo ? 1 : 0);

    const int32_t* table = a.c.table + (shared ? 0 : sequence * a.c.table_stride);
    const uint16_t* kc = a.c.k + kvh * a.c.k_head;
    const uint16_t* vc = a.c.v + kvh * a.c.v_head;

    u32x4 qf[kSteps];
    {
        const uint16_t* from = a.q + token * a.q_row + head * a.q_head + 8 * q;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) qf[s] = *(const u32x4*)(from + 32 * s);
    }

    float m_run = kScoreFloor, l_run = 0.0f;
    bool seen = false;
    float4v o[kVd];
    u32x4 k[2][kSteps];
    vword v[8];
    int bad[2];

    const int k_lane = j * (int)a.c.k_position + 8 * q;
    const int v_lane = 4 * q * (int)a.c.v_position + kVd * j;
    const int mask = (1 << a.c.page_shift) - 1;
    auto load = [&](int block) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int t = key_lo + block * kBlock + 16 * h;
            // (16 keys that no row sees: any page)
            int page = t > most ? 0 : page_of(table, a.c.table_width, a.c.page_shift, a.c.num_pages, t);
            bad[h] = page < 0;
            page = max(page, 0);
            const uint16_t* kp = kc + page * a.c.k_page + (t & mask) * a.c.k_position;
            const uint16_t* vp = vc + page * a.c.v_page + (t & mask) * a.c.v_position;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) k[h][s] = *(const u32x4*)(kp + k_lane + 32 * s);
#pragma unroll
            for (int r = 0; r < 4; ++r) v[4 * h + r] = *(const vword*)(vp + v_lane + r * (int)a.c.v_position);
        }
    };
    auto compute = [&](int block, bool careful) {
        const int t0 = key_lo + block * kBlock;
        const bool edge = t0 + kBlock - 1 > least;
        float s[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < kSteps; ++u) acc = E::mfma(k[h][u], qf[u], acc);
#pragma unroll
            for (int r = 0; r < 4; ++r) s[4 * h + r] = acc[r] * a.scale2;
        }
        if (edge) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int t = t0 + 16 * (e / 4) + 4 * q + e % 4;
                if (t > limit) s[e] = -INFINITY;
                if (t > most) v[e] = vword{};
            }
        }
        seen = seen || t0 <= limit;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (bad[h] && t0 + 16 * h <= limit) l_run = __builtin_nanf("");
        float top = s[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = fmaxf(top, s[e]);
        const float to = fmaxf(m_run, quarters_max(top));
        if (__any(to != m_run)) {
            const float alpha = __builtin_amdgcn_exp2f(m_run - to);
            l_run *= alpha;
#pragma unroll
            for (int dd = 0; dd < kVd; ++dd) o[dd] *= alpha;
            m_run = to;
        }
        u32x4 ph, pl;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float p0 = __builtin_amdgcn_exp2f(s[2 * e] - to + kProbShift<E>);
            const float p1 = __builtin_amdgcn_exp2f(s[2 * e + 1] - to + kProbShift<E>);
            l_run += p0 + p1;
            ph[e] = E::pack(p0, p1);
            pl[e] = E::pack(p0 - E::lo(ph[e]), p1 - E::hi(ph[e]));
        }
#pragma unroll
        for (int dd = 0; dd < kVd; ++dd) {
            const uint32_t sel = (dd & 1) ? 0x07060302u : 0x05040100u;  // high or low halves
            u32x4 vt;
#pragma unroll
            for (int e = 0; e < 4; ++e) vt[e] = __builtin_amdgcn_perm(v[2 * e + 1][dd / 2], v[2 * e][dd / 2], sel);
            if (!careful) {
                o[dd] = E::mfma(vt, ph, o[dd]);
                o[dd] = E::mfma(vt, pl, o[dd]);
                continue;
            }
            // A value that is not finite must reach only the rows that see its key
            // (0 * inf is NaN): the finite ones as always, the others column by
            // column with what the column does not see at zero.
            u32x4 plain, odd;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                plain[e] = finite_halves<E>(vt[e]);
                odd[e] = vt[e] & ~plain[e];
            }
            o[dd] = E::mfma(plain, ph, o[dd]);
            o[dd] = E::mfma(plain, pl, o[dd]);
            for (int c = 0; c < kTile; ++c) {
                const int sees = __builtin_amdgcn_readlane(limit, c);
                u32x4 part;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = t0 + 16 * (e / 2) + 4 * q + 2 * (e % 2);
                    part[e] = keep_halves(odd[e], t <= sees, t + 1 <= sees);
                }
                const float4v more = E::mfma(part, ph, float4v{0.0f, 0.0f, 0.0f, 0.0f});
                if (j == c) o[dd] += more;
            }
        }
    };
    // The second pass is for value sums that came out infinite or NaN.
    for (int pass = 0; pass < 2; ++pass) {
        m_run = kScoreFloor, l_run = 0.0f;
        seen = false;
#pragma unroll
        for (int dd = 0; dd < kVd; ++dd) o[dd] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
        for (int block = split + splits * wave; block < blocks; block += splits * kWaves) {
            load(block);
            compute(block, pass != 0);
        }
        bool fine = true;
#pragma unroll
        for (int dd = 0; dd < kVd; ++dd)
#pragma unroll
            for (int r = 0; r < 4; ++r) fine = fine && fabsf(o[dd][r]) < INFINITY;
        if (__all(fine)) break;
    }

    // ---- the waves' results meet in LDS ----
    float l_all = quarters_sum(l_run);
    if (beyond && split == 0) {
        l_all = __builtin_nanf("");
        seen = true;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int dd = 0; dd < kVd; dd += 4)
            *(float4v*)&so[wave][j][kVd * (4 * q + r) + dd] = float4v{o[dd][r], o[dd + 1][r], o[dd + 2][r], o[dd + 3][r]};
    if (q == 0) {
        sm[wave][j] = seen ? m_run : -INFINITY;  // -inf: no key seen
        sl[wave][j] = l_all;
    }
    __syncthreads();
    // thread t: row t / 16, dimensions kVd (t % 16) ..
    const int g = tid / 16;
    const int d0 = kVd * (tid % 16);
    const int64_t mg = (int64_t)tile * kTile + g;
    if (mg >= (int64_t)tokens * a.group) return;
    float top = sm[0][g];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, sm[w][g]);
    float sum[kVd] = {};
    float l = 0.0f;
    if (top > -INFINITY) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(sm[w][g] - top);
            if (f == 0.0f && sl[w][g] == sl[w][g]) continue;  // (no key, or none that counts; its sums may be infinite)
            l = fmaf(sl[w][g], f, l);
#pragma unroll
            for (int i = 0; i < kVd; ++i) sum[i] = fmaf(so[w][g][d0 + i], f, sum[i]);
        }
    }
    const int tg = first_token + (int)(mg / a.group);
    const int hg = kvh * a.group + (int)(mg % a.group);
    if (a.slots == 1) {
        const float inv = top > -INFINITY ? 1.0f / l : 0.0f;
        uint16_t* to = a.out + tg * a.out_row + hg * a.out_head + d0;
#pragma unroll
        for (int i = 0; i < kVd; i += 4)
            *(u32x2*)(to + i) = u32x2{E::pack(sum[i] * inv, sum[i + 1] * inv), E::pack(sum[i + 2] * inv, sum[i + 3] * inv)};
        return;
    }
    const int64_t slot = ((int64_t)tg * a.heads + hg) * a.slots + (shared ? split : a.prefix_splits * (a.prefix > 0) + split);
    if (tid % 16 == 0) *(float2v*)(a.stats + 2 * slot) = float2v{top, l};
    if (top == -INFINITY) return;  // (the join does not read it)
#pragma unroll
    for (int i = 0; i < kVd; i += 4)
        *(float4v*)(a.partials + slot * D + d0 + i) = float4v{sum[i], sum[i + 1], sum[i + 2], sum[i + 3]};
}

// One wave per (packed row, query head): lane l's D / 32 dimensions of the slots
// l / 32, l / 32 + 2, ...; the halves are added at the end.
template <class E, int D>
__global__ __launch_bounds__(kThreads) void paged_join_kernel(PagedAttnArgs a) {
    constexpr int kPer = D / 32;
    const int lane = threadIdx.x & 63;
    const int64_t at = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (at >= (int64_t)a.rows * a.heads) return;
    const int row = (int)(at / a.heads);
    const int head = (int)(at - (int64_t)row * a.heads);
    uint16_t* to = a.out + row * a.out_row + head * a.out_head;
    if (row >= a.c.cu_rows[a.c.batch]) {  // behind the last sequence
        if (a.zero_rest && lane < D / 8) *(u32x4*)(to + 8 * lane) = u32x4{0u, 0u, 0u, 0u};
        return;
    }
    const float* stats = a.stats + 2 * at * a.slots;
    const bool has = lane < a.slots;
    const float m = has ? stats[2 * lane] : -INFINITY;
    const float sum_l = has ? stats[2 * lane + 1] : 0.0f;
    const float top = wave_max64(m);
    const float f = m > -INFINITY ? __builtin_amdgcn_exp2f(m - top) : 0.0f;
    const float l = wave_sum64(f != 0.0f || sum_l != sum_l ? sum_l * f : 0.0f);  // (NaN: a page that was not there)
    float sum[kPer] = {};
    for (int i = 0; i < a.slots; i += 2) {
        const int s = min(i + lane / 32, a.slots - 1);
        float fs = __shfl(f, s);
        if (i + lane / 32 >= a.slots) fs = 0.0f;
        if (fs == 0.0f) continue;
        const float* part = a.partials + (at * a.slots + s) * D + kPer * (lane % 32);
#pragma unroll
        for (int e = 0; e < kPer; ++e) sum[e] = fmaf(part[e], fs, sum[e]);
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
};

PagedPlan paged_plan(const PagedView& c, int64_t rows, int64_t heads, int64_t shared_pages) {
    PagedPlan p{};
    const int64_t group = heads / c.kv_heads;
    p.prefix = shared_pages << c.page_shift;
    const int64_t own = ((int64_t)c.table_width - shared_pages) << c.page_shift;
    auto splits = [&](int64_t workgroups, int64_t keys) {
        const int64_t most = (keys + kBlock * kWaves - 1) / (kBlock * kWaves);  // a block per wave
        int64_t s = (512 + workgroups - 1) / workgroups;
        s = s < most ? s : most;
        return s < kMaxSplits / 2 ? s : kMaxSplits / 2;
    };
    if (p.prefix > 0) {
        p.prefix_tiles = (rows * group + kTile - 1) / kTile;
        p.prefix_splits = splits(p.prefix_tiles * c.kv_heads, p.prefix);
    }
    if (own > 0) {
        p.own_tiles = rows * group / kTile + (c.batch < rows ? c.batch : rows);
        p.own_splits = splits(p.own_tiles * c.kv_heads, own);
    }
    p.slots = p.prefix_splits + p.own_splits;
    return p;
}

template <class E, int D>
hipError_t launch_paged_attention(const PagedAttnArgs& a, int64_t workgroups, hipStream_t stream) {
    hipLaunchKernelGGL((paged_attention_kernel<E, D>), dim3((unsigned)workgroups), dim3(kThreads), 0, stream, a);
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
    if ((cache->table_width << view->page_shift) > 0x7FFFFF00)
        return set_error(W4G64_STATUS_UNSUPPORTED, "paged_attention tables must hold fewer than 2^31 - 256 positions");
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
    const PagedPlan p = paged_plan(view, rows, heads, shared_pages);
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
    const PagedPlan p = paged_plan(a.c, rows, heads, shared_pages);
    const int64_t need = qwen2_paged_attention_workspace_bytes(cache, rows, heads, shared_pages);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
        return set_error(W4G64_STATUS_WORKSPACE, "paged_attention needs %lld workspace bytes, 16-byte aligned, got %lld",
                         (long long)need, (long long)(workspace ? workspace_bytes : 0));
    const int64_t workgroups =
        (p.prefix_tiles * p.prefix_splits + p.own_tiles * p.own_splits) * cache->kv_heads;
    if (workgroups > 0x7FFFFFFF || rows * heads > 0x7FFFFFFF)
        return set_error(W4G64_STATUS_UNSUPPORTED, "paged_attention call is too large: %lld workgroups", (long long)workgroups);
    a.q = (const uint16_t*)q->data, a.q_row = q->row, a.q_head = q->head;
    a.out = (uint16_t*)out->data, a.out_row = out->row, a.out_head = out->head;
    a.partials = (float*)workspace;  // (D floats per slot: 16-byte aligned)
    a.stats = a.partials + rows * heads * p.slots * cache->head_dim;
    a.scale2 = scale * 1.44269504088896340736f;
    a.rows = (int)rows, a.heads = (int)heads, a.group = (int)(heads / cache->kv_heads);
    a.prefix = (int)p.prefix;
    a.prefix_tiles = (int)p.prefix_tiles, a.prefix_splits = (int)p.prefix_splits;
    a.own_tiles = (int)p.own_tiles, a.own_splits = (int)p.own_splits, a.slots = (int)p.slots;
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
