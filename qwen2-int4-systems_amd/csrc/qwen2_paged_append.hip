// Rotary step and paged cache write of the new positions
// (qwen2_paged_append, include/qwen2_decode.h).
//
// One wave per packed row, or per part of a row's heads where there are few
// rows.  Its lanes first form the row's angles, one frequency each (64 at head
// dimension 128: one sine and cosine per lane), and leave cosine and sine in
// the wave's own LDS; then each lane takes units of 32 bytes of a head, which
// hold eight pairs in either layout: pieces 8 u and rotary/2 + 8 u of the half
// layout, 16 u and 16 u + 8 of the interleaved one.  A unit past the rotary
// dimensions, or of a value, is copied.
//
// The angle is position * frequency in turns, in 64 bits, less its whole
// turns: in 32 bits a position of a million is off by 0.06 radians.  What is
// left goes through fp32 (1e-7 radians), the products are fp32, the only
// rounding to 16 bits is the result's.
//
// Bound by memory for prompts (8 K rows of 12/2 heads of 128: 67 MB in 13 us, 5.2
// TB/s) and by its chain of loads (cu_rows, lengths, page) for a decode step: one
// row 2.7 us, 64 x 5 rows of 32/8 heads 4.7, under a call of 5 to 6 us, most of it the
// host's launch.
#include <hip/hip_runtime.h>
#include <math.h>

#include "qwen2_decode.h"
#include "qwen2_paged_device.h"
#include "w4g64_internal.h"

namespace w4g64 {
namespace {

constexpr int kWaves = 4;
constexpr int kMaxPairs = 128;  // head dimension 256

struct AppendArgs {
    PagedView c;
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
    const float* inv_freq;
    float scale;
    int rows, heads, head_dim, rotary, zero_rest;
    int parts;  // waves per row
};

// The sequence of a row: how many end at or before it (64 at a time).
__device__ __forceinline__ int sequence_of(const int32_t* cu_rows, int batch, int row, int lane) {
    int count = 0;
    for (int base = 0; base < batch; base += 64) {
        const int i = base + lane;
        const int n = __popcll(__ballot(i < batch && cu_rows[i + 1] <= row));
        count += n;
        if (n < 64) break;
    }
    return count;
}

template <class E, bool kInterleaved>
__global__ __launch_bounds__(64 * kWaves) void paged_append_kernel(AppendArgs a) {
    __shared__ float cs[kWaves][kMaxPairs];
    __shared__ float sn[kWaves][kMaxPairs];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t at = (int64_t)blockIdx.x * kWaves + wave;
    if (at >= (int64_t)a.rows * a.parts) return;
    const int row = (int)(at / a.parts);
    const int part = (int)(at - (int64_t)row * a.parts);
    const int per = a.head_dim / 16;  // units of a head
    const int units = (a.heads + 2 * a.c.kv_heads) * per;
    const int seq = sequence_of(a.c.cu_rows, a.c.batch, row, lane);
    SequenceRows s{0, 0, 0};
    if (seq < a.c.batch) s = sequence_rows(a.c.cu_rows, a.c.lengths, seq, rows_end(a.c.cu_rows, a.c.batch, a.rows));
    if (row < s.begin || row >= s.end) {  // no sequence's row
        if (!a.zero_rest) return;
        for (int u = 64 * part + lane; u < a.heads * per; u += 64 * a.parts) {
            uint16_t* to = a.out + row * a.out_row + (u / per) * a.out_head + 16 * (u % per);
            *(u32x4*)to = u32x4{0u, 0u, 0u, 0u};
            *(u32x4*)(to + 8) = u32x4{0u, 0u, 0u, 0u};
        }
        return;
    }
    const int64_t position = s.first + (row - s.begin);
    const int page = page_of(a.c.table + seq * a.c.table_stride, a.c.table_width, a.c.page_shift, a.c.num_pages,
                             position);
    const int64_t place = position & ((1 << a.c.page_shift) - 1);
    for (int i = lane; i < a.rotary / 2; i += 64) {
        constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)
        const double turns = (double)position * ((double)a.inv_freq[i] * kTurn);
        const float left = (float)(2.0 * (turns - rint(turns)));  // half turns, in [-1, 1]
        float sine, cosine;
        sincospif(left, &sine, &cosine);
        cs[wave][i] = cosine * a.scale;
        sn[wave][i] = sine * a.scale;
    }
    // (the wave's own LDS: its stores before its loads)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    for (int u = 64 * part + lane; u < units; u += 64 * a.parts) {
        const int head = u / per;
        const int r = u - head * per;
        const uint16_t* from;
        uint16_t* to;
        bool turn = r < a.rotary / 16;
        if (head < a.heads) {
            from = a.q + row * a.q_row + head * a.q_head;
            to = a.out + row * a.out_row + head * a.out_head;
        } else if (head < a.heads + a.c.kv_heads) {
            const int h = head - a.heads;
            from = a.k + row * a.k_row + h * a.k_head;
            to = page < 0 ? nullptr : a.c.k + page * a.c.k_page + h * a.c.k_head + place * a.c.k_position;
        } else {
            const int h = head - a.heads - a.c.kv_heads;
            from = a.v + row * a.v_row + h * a.v_head;
            to = page < 0 ? nullptr : a.c.v + page * a.c.v_page + h * a.c.v_head + place * a.c.v_position;
            turn = false;
        }
        if (!to) continue;
        const int d0 = !kInterleaved && turn ? 8 * r : 16 * r;
        const int d1 = !kInterleaved && turn ? 8 * r + a.rotary / 2 : 16 * r + 8;
        u32x4 x = *(const u32x4*)(from + d0), y = *(const u32x4*)(from + d1);
        if (turn) {
            const float* c = &cs[wave][8 * r];
            const float* n = &sn[wave][8 * r];
            if constexpr (kInterleaved) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float xa = E::lo(x[e]), xb = E::hi(x[e]), ya = E::lo(y[e]), yb = E::hi(y[e]);
                    x[e] = E::pack(fmaf(xa, c[e], -xb * n[e]), fmaf(xb, c[e], xa * n[e]));
                    y[e] = E::pack(fmaf(ya, c[4 + e], -yb * n[4 + e]), fmaf(yb, c[4 + e], ya * n[4 + e]));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float xa = E::lo(x[e]), xb = E::hi(x[e]), ya = E::lo(y[e]), yb = E::hi(y[e]);
                    x[e] = E::pack(fmaf(xa, c[2 * e], -ya * n[2 * e]), fmaf(xb, c[2 * e + 1], -yb * n[2 * e + 1]));
                    y[e] = E::pack(fmaf(ya, c[2 * e], xa * n[2 * e]), fmaf(yb, c[2 * e + 1], xb * n[2 * e + 1]));
                }
            }
        }
        *(u32x4*)(to + d0) = x;
        *(u32x4*)(to + d1) = y;
    }
}

// Waves per row: one where the rows alone give every SIMD two waves, else as many
// as that takes, up to what a row's units fill (64 each): a row is two to ten
// rounds of a wave, which the waves of a decode step do side by side.
int append_parts(int64_t rows, int64_t units) {
    const int64_t most = (units + 63) / 64;
    const int64_t want = (2048 + rows - 1) / rows;
    return (int)(want < most ? want : most);
}

template <class E>
void launch_append(const AppendArgs& a, bool interleaved, hipStream_t stream) {
    const dim3 grid((unsigned)(((int64_t)a.rows * a.parts + kWaves - 1) / kWaves));
    if (interleaved)
        hipLaunchKernelGGL((paged_append_kernel<E, true>), grid, dim3(64 * kWaves), 0, stream, a);
    else
        hipLaunchKernelGGL((paged_append_kernel<E, false>), grid, dim3(64 * kWaves), 0, stream, a);
}

bool rows_usable(const qwen2_rows* r) {
    return r && r->data && !((uintptr_t)r->data & 15) && r->row % 8 == 0 && r->head % 8 == 0;
}

}  // namespace

int paged_view(const qwen2_paged_cache* c, PagedView* view) {
    if (!c) return set_error(W4G64_STATUS_INVALID_VALUE, "paged cache must not be null");
    if (c->dtype != W4G64_DTYPE_BF16 && c->dtype != W4G64_DTYPE_F16)
        return set_error(W4G64_STATUS_INVALID_DTYPE, "paged cache dtype must be bf16 or fp16, got code %d", c->dtype);
    int shift = 4;
    while (shift < 20 && (int64_t(1) << shift) < c->page_size) ++shift;
    if (c->page_size != int64_t(1) << shift)
        return set_error(W4G64_STATUS_INVALID_VALUE, "page_size must be a power of two in [16, 2^20], got %lld",
                         (long long)c->page_size);
    if (c->batch <= 0 || c->kv_heads <= 0 || c->batch > 0x7FFFFFFE || c->kv_heads > 0xFFFF)
        return set_error(W4G64_STATUS_INVALID_VALUE, "paged cache batch and kv_heads must be positive, got %lld and %lld",
                         (long long)c->batch, (long long)c->kv_heads);
    if (c->num_pages <= 0 || c->num_pages > 0x7FFFFFFF || c->table_width <= 0 || c->table_width > 0x7FFFFFFF)
        return set_error(W4G64_STATUS_INVALID_VALUE,
                         "paged cache needs num_pages and table_width in [1, 2^31), got %lld and %lld",
                         (long long)c->num_pages, (long long)c->table_width);
    if (!c->k || !c->v || !c->page_table || !c->cu_rows || !c->lengths)
        return set_error(W4G64_STATUS_INVALID_VALUE, "paged cache pointers must be non-null device pointers");
    const int64_t strides[6] = {c->k_page, c->k_head, c->k_position, c->v_page, c->v_head, c->v_position};
    bool aligned = !(((uintptr_t)c->k | (uintptr_t)c->v) & 15);
    for (int64_t s : strides) aligned = aligned && s >= 0 && s % 8 == 0;
    if (!aligned)
        return set_error(W4G64_STATUS_INVALID_VALUE,
                         "paged cache must be 16-byte aligned with strides that are multiples of 8 elements");
    if (((uintptr_t)c->page_table | (uintptr_t)c->cu_rows | (uintptr_t)c->lengths) & 3)
        return set_error(W4G64_STATUS_INVALID_VALUE, "page_table, cu_rows and lengths must be 4-byte aligned");
    if (c->k_position > (1 << 24) || c->v_position > (1 << 24))
        return set_error(W4G64_STATUS_UNSUPPORTED, "paged cache position strides must be at most 2^24 elements");
    *view = PagedView{(uint16_t*)c->k, (uint16_t*)c->v, c->k_page,      c->k_head,   c->k_position,    c->v_page,
                      c->v_head,       c->v_position,   c->page_table,  c->table_stride, c->cu_rows,   c->lengths,
                      (int)c->batch,   (int)c->kv_heads, (int)c->num_pages, shift,    (int)c->table_width};
    return W4G64_STATUS_OK;
}

}  // namespace w4g64

using namespace w4g64;

extern "C" int qwen2_paged_append(const qwen2_paged_cache* cache, const qwen2_rows* q, const qwen2_rows* k,
                                  const qwen2_rows* v, const qwen2_rows* out, const float* inv_freq,
                                  int64_t rotary_dim, int interleaved, float rotary_scale, int64_t rows, int64_t heads,
                                  int zero_rest, void* stream) {
    AppendArgs a{};
    const int status = paged_view(cache, &a.c);
    if (status) return status;
    if (cache->head_dim <= 0 || cache->head_dim % 16 || cache->head_dim > 2 * kMaxPairs)
        return set_error(W4G64_STATUS_UNSUPPORTED, "paged_append needs a head_dim that is a multiple of 16 up to %d, got %lld",
                         2 * kMaxPairs, (long long)cache->head_dim);
    if (rotary_dim < 0 || rotary_dim % 16 || rotary_dim > cache->head_dim)
        return set_error(W4G64_STATUS_INVALID_VALUE,
                         "rotary_dim must be a multiple of 16 in [0, head_dim = %lld], got %lld",
                         (long long)cache->head_dim, (long long)rotary_dim);
    if (rows < 0 || rows > 0x7FFFFFF || heads <= 0 || heads > 0xFFFF)
        return set_error(W4G64_STATUS_INVALID_VALUE, "paged_append rows must be in [0, 2^27) and heads in [1, 2^16), got %lld and %lld",
                         (long long)rows, (long long)heads);
    if (!isfinite(rotary_scale)) return set_error(W4G64_STATUS_INVALID_VALUE, "rotary_scale must be finite");
    if (rows == 0) return clear_error();
    if (!rows_usable(q) || !rows_usable(k) || !rows_usable(v) || !rows_usable(out))
        return set_error(W4G64_STATUS_INVALID_VALUE,
                         "q, k, v and out must be non-null, 16-byte aligned, with strides that are multiples of 8 elements");
    if (rotary_dim && (!inv_freq || ((uintptr_t)inv_freq & 3)))
        return set_error(W4G64_STATUS_INVALID_VALUE, "inv_freq must be a non-null, 4-byte aligned device pointer");
    a.q = (const uint16_t*)q->data, a.q_row = q->row, a.q_head = q->head;
    a.k = (const uint16_t*)k->data, a.k_row = k->row, a.k_head = k->head;
    a.v = (const uint16_t*)v->data, a.v_row = v->row, a.v_head = v->head;
    a.out = (uint16_t*)out->data, a.out_row = out->row, a.out_head = out->head;
    a.inv_freq = inv_freq;
    a.scale = rotary_scale;
    a.rows = (int)rows, a.heads = (int)heads, a.head_dim = (int)cache->head_dim, a.rotary = (int)rotary_dim;
    a.zero_rest = zero_rest;
    a.parts = append_parts(rows, (heads + 2 * cache->kv_heads) * (cache->head_dim / 16));
    if (cache->dtype == W4G64_DTYPE_BF16)
        launch_append<Bf16>(a, interleaved != 0, (hipStream_t)stream);
    else
        launch_append<F16>(a, interleaved != 0, (hipStream_t)stream);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess)
        return set_error(W4G64_STATUS_HIP_ERROR, "paged_append launch failed: %s", hipGetErrorString(err));
    return clear_error();
}
