// Verification of drafted tokens (qwen2_verify_drafts, include/qwen2_decode.h).
//
//   verify_one_kernel   one workgroup per sequence does all of what follows;
//   verify_sum_kernel   one wave per (sequence, span of 1024 entries of the
//                       vocabulary): finds how many drafts stand (every wave
//                       for itself: a few loads), then adds up its entries'
//                       weights;
//   verify_pick_kernel  one wave per sequence: the span in which the
//                       running sum passes uniform * total, then the entry.
// Where max(p - q, 0) is zero everywhere, the picking wave goes through the
// target's row by itself.
//
// Only one row of the target's (and the draft's) probabilities is read per
// sequence, 16 bytes a lane.  A weight is a difference of two 24-bit numbers and
// the sums run over the vocabulary, so they are held in 64 bits, in one fixed
// order: the chosen entry is the definition's unless the uniform's share of the
// total lies within roundings of 2^-53 of a border between two entries (then it
// may be a neighbour of weight), and never one without weight.
//
// Bound by the rows' read from memory (64 x 4 drafts of 151936 fp32: 77.8 MB in
// 14.1 us of the sums, 17.5 the call), and for few sequences by its chain of round
// trips (drafted id, its probabilities, the row) and the host's launches, some 4 us
// each.  First forms, us: 64 x 4 147 with single entries per lane and both sums in
// every workgroup, 19.6 with 16-byte loads and the pick by one wave.
#include <hip/hip_runtime.h>

#include "qwen2_decode.h"
#include "w4g64_device.h"
#include "w4g64_internal.h"

namespace w4g64 {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kSpan = 1024;   // entries of a sum, 16 of a lane
constexpr int kMargin = 4096; // vocabularies end so far below 2^31

struct VerifyArgs {
    const void* target;
    const void* draft;
    int64_t target_batch, target_row, draft_batch, draft_row;
    const int64_t* draft_tokens;
    const int32_t* draft_lengths;
    const float* uniforms;
    int64_t* tokens;
    int32_t* accepted;
    double* sums;      // [batch][spans]
    int32_t* standing; // [batch]
    int batch, drafts, vocab, spans;
};

template <int XK>
__device__ __forceinline__ double value(const void* p, int64_t i) {
    if constexpr (XK == kF32) return (double)((const float*)p)[i];
    if constexpr (XK == kBF16) return (double)bf16_bits_to_float(((const uint16_t*)p)[i]);
    return (double)half_bits_to_float(((const uint16_t*)p)[i]);
}

// How many drafts of the sequence stand; `count` is how many there are.
template <int XK>
__device__ __forceinline__ int standing(const VerifyArgs& a, int b, int lane, int& count) {
    count = a.drafts;
    if (a.draft_lengths) count = min(max(a.draft_lengths[b], 0), a.drafts);
    for (int base = 0; base < count; base += 64) {
        const int i = base + lane;
        bool stands = i >= count;  // (lanes past the end do not stop the run)
        if (i < count) {
            const int64_t x = a.draft_tokens[(int64_t)b * a.drafts + i];
            if (x >= 0 && x < a.vocab) {
                const double p = value<XK>(a.target, b * a.target_batch + i * a.target_row + x);
                const double q = a.draft ? value<XK>(a.draft, b * a.draft_batch + i * a.draft_row + x) : 1.0;
                stands = (double)a.uniforms[(int64_t)b * (a.drafts + 1) + i] * q < p;
            }
        }
        const uint64_t fall = ~__ballot(stands);
        if (fall) return base + __ffsll((unsigned long long)fall) - 1;
    }
    return count;
}

// Where a row's weights come from.
struct Weights {
    const void* target;
    const void* draft;  // null: none, or one at `hot`
    int64_t target_at, draft_at;
    int64_t hot;        // -1: none
};
__device__ __forceinline__ Weights weights_of(const VerifyArgs& a, int b, int n, int count) {
    Weights w{a.target, nullptr, b * a.target_batch + n * a.target_row, 0, -1};
    if (n < count) {
        if (a.draft) {
            w.draft = a.draft;
            w.draft_at = b * a.draft_batch + n * a.draft_row;
        } else {
            w.hot = a.draft_tokens[(int64_t)b * a.drafts + n];
        }
    }
    return w;
}

// Loads at an entry's alignment: one access, the target takes unaligned ones.
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));

// kCount (4 or 8) entries v .. of a row, zero past its end.
template <int XK, int kCount>
__device__ __forceinline__ void entries(const void* p, int64_t at, int v, int vocab, float (&x)[kCount]) {
    if (v + kCount > vocab) {
#pragma unroll
        for (int e = 0; e < kCount; ++e) x[e] = v + e < vocab ? (float)value<XK>(p, at + v + e) : 0.0f;
    } else if constexpr (XK == kF32) {
#pragma unroll
        for (int i = 0; i < kCount; i += 4) {
            // (bit cast as a whole: that of one element compiles to element 0 with this compiler)
            const float4v w = __builtin_bit_cast(float4v, *(const u32x4_any*)((const float*)p + at + v + i));
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i + e] = w[e];
        }
    } else {
        uint32_t w[kCount / 2];
        if constexpr (kCount == 8) {
            const u32x4 l = *(const u32x4_any*)((const uint16_t*)p + at + v);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = l[e];
        } else {
            const u32x2 l = *(const u32x2_any*)((const uint16_t*)p + at + v);
            w[0] = l[0], w[1] = l[1];
        }
#pragma unroll
        for (int e = 0; e < kCount; ++e) {
            const uint16_t h = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
            x[e] = XK == kBF16 ? bf16_bits_to_float(h) : half_bits_to_float(h);
        }
    }
}

// How a span's weights come about: the target alone, less the draft's, or less one
// at `hot` (the one span that holds it).
enum Less { kNothing, kDraft, kHot };

// The weight max(p - q, 0) of an entry; `odd` remembers a NaN, which the maximum
// drops.
template <int kLess>
__device__ __forceinline__ double weight(const Weights& w, int v, float p, float q, bool& odd) {
    double x = (double)p;
    if constexpr (kLess == kDraft) x -= (double)q;
    if constexpr (kLess == kHot) x -= v == w.hot ? 1.0 : 0.0;
    odd = odd || x != x;
    return __builtin_fmax(x, 0.0);
}

__device__ __forceinline__ double shfl_xor_f64(double v, int mask) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __shfl_xor((uint32_t)u, mask), hi = __shfl_xor((uint32_t)(u >> 32), mask);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// The sum of one span's weights, in every lane; NaN if one of them is.
template <int XK, int kLess>
__device__ __forceinline__ double span_sum(const Weights& w, int vocab, int span, int lane) {
    constexpr int kLoad = XK == kF32 ? 4 : 8;         // entries of a lane's load
    constexpr int kLoads = kSpan / (64 * kLoad);
    float p[kLoads][kLoad], q[kLoads][kLoad];
    const int v0 = span * kSpan + kLoad * lane;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) entries<XK>(w.target, w.target_at, v0 + 64 * kLoad * i, vocab, p[i]);
    if constexpr (kLess == kDraft) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) entries<XK>(w.draft, w.draft_at, v0 + 64 * kLoad * i, vocab, q[i]);
    }
    double sum = 0.0;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
        for (int e = 0; e < kLoad; ++e)
            sum += weight<kLess>(w, v0 + 64 * kLoad * i + e, p[i][e], kLess == kDraft ? q[i][e] : 0.0f, odd);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) sum += shfl_xor_f64(sum, m);
    return __any(odd) ? __builtin_nan("") : sum;
}
template <int XK>
__device__ __forceinline__ double span_sum(const Weights& w, int vocab, int span, int lane) {
    if (w.draft) return span_sum<XK, kDraft>(w, vocab, span, lane);
    if (w.hot >= 0 && w.hot / kSpan == span) return span_sum<XK, kHot>(w, vocab, span, lane);
    return span_sum<XK, kNothing>(w, vocab, span, lane);
}

template <int XK>
__global__ __launch_bounds__(kThreads) void verify_sum_kernel(VerifyArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t at = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (at >= (int64_t)a.batch * a.spans) return;
    const int b = (int)(at / a.spans);
    const int span = (int)(at - (int64_t)b * a.spans);
    int count;
    const int n = standing<XK>(a, b, lane, count);
    if (span == 0 && lane == 0) a.standing[b] = n;
    const double sum = span_sum<XK>(weights_of(a, b, n, count), a.vocab, span, lane);
    if (lane == 0) a.sums[at] = sum;
}

// Running sums over the wave's lanes, each lane's own value counted: within rows
// of 16 lanes by shifts, then rows 1 and 3, then 2 and 3 take the last lane
// before them.  (Lanes without a source receive 0.)
template <int kControl, int kRows>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, kControl, kRows, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), kControl, kRows, 0xF, false);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double running_sum(double v) {
    v += dpp_f64<0x111, 0xF>(v);
    v += dpp_f64<0x112, 0xF>(v);
    v += dpp_f64<0x114, 0xF>(v);
    v += dpp_f64<0x118, 0xF>(v);
    v += dpp_f64<0x142, 0xA>(v);
    v += dpp_f64<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// The choice of sequence b by one wave, no barrier: lane l has spans per l .. per l +
// per - 1, then entries 16 l .. 16 l + 15 of the span.  (A workgroup of four waves
// over LDS, with shuffles for its scans, took 10 us for any batch.)
template <int XK>
__device__ __forceinline__ void pick(const VerifyArgs& a, int b, int lane, const double* sums, int n, int count) {
    constexpr int kOwn = kSpan / 64;
    const int per = (a.spans + 63) / 64;
    const int first = per * lane;
    // (the usual vocabulary's spans of a lane are held: their loads go out together)
    constexpr int kHeld = 3;
    const int mine_spans = min(per, a.spans - first);
    double held[kHeld], own = 0.0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = i < mine_spans ? sums[first + i] : 0.0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) own += held[i];
    for (int i = kHeld; i < mine_spans; ++i) own += sums[first + i];
    float u = a.uniforms[(int64_t)b * (a.drafts + 1) + a.drafts];
    Weights w = weights_of(a, b, n, count);
    constexpr float kBelowOne = 0.999999940395355224609375f;  // 1 - 2^-24
    if (u > kBelowOne) u = kBelowOne;
    if (u < 0.0f) u = 0.0f;
    const double end = running_sum(own);
    double total = lane_f64(end, 63), run = 0.0, goal;
    int span = 0;
    if (total != 0.0) {
        // every lane goes through its own spans from where the lanes before it end: the
        // first span of any weight at which the running sum passes the goal, of the first
        // lane that has one; if all stay a rounding below, the last span of any weight
        // (the lanes' ends are added up in different orders: one can lie above the one
        // before it though its spans are empty, so that it alone does not choose)
        goal = (double)u * total;
        const double up = __shfl_up(end, 1);  // (by every lane: one that is off gives nothing)
        double sum = lane ? up : 0.0, before = 0.0;
        int found = -1, some = -1;
        auto pass = [&](int i, double weight) {
            if (found >= 0 || !(weight > 0.0)) return;
            some = first + i, before = sum;
            sum += weight;
            if (sum > goal) found = some;
        };
#pragma unroll
        for (int i = 0; i < kHeld; ++i) pass(i, held[i]);
        for (int i = kHeld; i < mine_spans; ++i) pass(i, sums[first + i]);
        const uint64_t passed = __ballot(found >= 0), any = __ballot(some >= 0);
        if (passed | any) {
            const int at = passed ? __ffsll((unsigned long long)passed) - 1 : 63 - __clzll((unsigned long long)any);
            span = __builtin_amdgcn_readlane(some, at);  // (where one was found, the walk ended at it)
            run = lane_f64(before, at);
        }
    } else {
        // the draft falls short of the target nowhere: the target alone, by this wave
        w.draft = nullptr, w.hot = -1;
        for (int i = 0; i < a.spans; ++i) total += span_sum<XK>(w, a.vocab, i, lane);
        goal = (double)u * total;
        for (; span + 1 < a.spans; ++span) {
            const double next = run + span_sum<XK>(w, a.vocab, span, lane);
            if (next > goal) break;
            run = next;
        }
    }
    int64_t token = -1;
    if (total > 0.0 && total < __builtin_inf() && u == u) {  // (the same in every lane)
        const int v0 = span * kSpan + kOwn * lane;
        float p[kOwn / 4][4], q[kOwn / 4][4] = {};
#pragma unroll
        for (int i = 0; i < kOwn / 4; ++i) entries<XK>(w.target, w.target_at, v0 + 4 * i, a.vocab, p[i]);
        if (w.draft)
#pragma unroll
            for (int i = 0; i < kOwn / 4; ++i) entries<XK>(w.draft, w.draft_at, v0 + 4 * i, a.vocab, q[i]);
        double each[kOwn], mine = 0.0;
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
            // (of the two, one is not there and takes nothing off)
            const double less = (double)q[e / 4][e % 4] + (v0 + e == w.hot ? 1.0 : 0.0);
            each[e] = __builtin_fmax((double)p[e / 4][e % 4] - less, 0.0);
            mine += each[e];
        }
        const double upto = running_sum(mine);
        const double before = __shfl_up(upto, 1);  // (by every lane: one that is off gives nothing)
        double sum = run + (lane ? before : 0.0);
        int found = -1, some = -1;
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
            sum += each[e];
            if (each[e] > 0.0) {
                some = v0 + e;
                if (sum > goal && found < 0) found = v0 + e;
            }
        }
        // the first entry to pass; if all stay a rounding below, the last of any weight
        const uint64_t passed = __ballot(found >= 0), any = __ballot(some >= 0);
        if (passed) token = __shfl(found, __ffsll((unsigned long long)passed) - 1);
        else if (any) token = __shfl(some, 63 - __clzll((unsigned long long)any));
    }
    for (int i = lane; i <= a.drafts; i += 64) {
        const int64_t to = (int64_t)b * (a.drafts + 1) + i;
        a.tokens[to] = i < n ? a.draft_tokens[(int64_t)b * a.drafts + i] : (i == n ? token : -1);
    }
    if (lane == 0) a.accepted[b] = n;
}

template <int XK>
__global__ __launch_bounds__(64) void verify_pick_kernel(VerifyArgs a) {
    const int b = blockIdx.x;
    int count = a.drafts;
    if (a.draft_lengths) count = min(max(a.draft_lengths[b], 0), a.drafts);
    pick<XK>(a, b, threadIdx.x, a.sums + (int64_t)b * a.spans, a.standing[b], count);
}

// Both in one launch, a workgroup of 16 waves per sequence: the spans' sums meet in
// LDS.
constexpr int kOneWaves = 16;
constexpr int kOneSpans = 512;
template <int XK>
__global__ __launch_bounds__(64 * kOneWaves) void verify_one_kernel(VerifyArgs a) {
    __shared__ double sums[kOneSpans];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.x;
    int count;
    const int n = standing<XK>(a, b, lane, count);
    const Weights w = weights_of(a, b, n, count);
    for (int span = wave; span < a.spans; span += kOneWaves) {
        const double sum = span_sum<XK>(w, a.vocab, span, lane);
        if (lane == 0) sums[span] = sum;
    }
    __syncthreads();
    if (wave == 0) pick<XK>(a, b, lane, sums, n, count);
}

// One launch where its workgroup has two spans a wave at most, or where there are
// sequences for every CU.  us per call, one launch / two: 1 x 8000 fp32 with a
// draft model 6.5 / 8.5, 1 x 32000 7.4 / 8.5, 96 x 32000 9.3 / 10.8, 1 x 50257 8.4 /
// 8.5, its bf16 9.7 / 8.5, 96 x 50257 bf16 13.4 / 11.6, 1 x 151936 bf16 19.8 / 8.4,
// but 256 x 50257 15.0 / 17.4 and 256 x 151936 35.8 / 39.7.
bool verify_in_one(const VerifyArgs& a) {
    return a.spans <= 2 * kOneWaves || (a.spans <= kOneSpans && a.batch >= 256);
}

template <int XK>
hipError_t launch_verify(const VerifyArgs& a, int64_t batch, hipStream_t stream) {
    if (verify_in_one(a)) {
        hipLaunchKernelGGL(verify_one_kernel<XK>, dim3((unsigned)batch), dim3(64 * kOneWaves), 0, stream, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(verify_sum_kernel<XK>, dim3((unsigned)((batch * a.spans + kWaves - 1) / kWaves)), dim3(kThreads), 0, stream, a);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    hipLaunchKernelGGL(verify_pick_kernel<XK>, dim3((unsigned)batch), dim3(64), 0, stream, a);
    return hipGetLastError();
}

int64_t verify_spans(int64_t vocab) { return (vocab + kSpan - 1) / kSpan; }

}  // namespace
}  // namespace w4g64

using namespace w4g64;

extern "C" {

int64_t qwen2_verify_drafts_workspace_bytes(int64_t batch, int64_t drafts, int64_t vocab) {
    if (batch <= 0 || drafts < 0 || vocab <= 0 || vocab > 0x7FFFFFFF - kMargin || batch > 0x7FFFFFFF / verify_spans(vocab))
        return 0;
    return batch * verify_spans(vocab) * (int64_t)sizeof(double) + batch * (int64_t)sizeof(int32_t);
}

int qwen2_verify_drafts(const void* target, int64_t target_batch, int64_t target_row, const void* draft,
                        int64_t draft_batch, int64_t draft_row, int dtype, const int64_t* draft_tokens,
                        const int32_t* draft_lengths, const float* uniforms, int64_t* tokens, int32_t* accepted,
                        int64_t batch, int64_t drafts, int64_t vocab, void* workspace, int64_t workspace_bytes,
                        void* stream) {
    if (dtype != W4G64_DTYPE_F32 && dtype != W4G64_DTYPE_BF16 && dtype != W4G64_DTYPE_F16)
        return set_error(W4G64_STATUS_INVALID_DTYPE, "verify_drafts probabilities must be fp32, bf16 or fp16, got code %d", dtype);
    if (batch < 0 || drafts < 0 || drafts > 0xFFFF || vocab <= 0 || vocab > 0x7FFFFFFF - kMargin)
        return set_error(W4G64_STATUS_INVALID_VALUE,
                         "verify_drafts needs drafts in [0, 2^16) and vocab in [1, 2^31 - 4096), got %lld and %lld",
                         (long long)drafts, (long long)vocab);
    if (batch == 0) return clear_error();
    const int64_t need = qwen2_verify_drafts_workspace_bytes(batch, drafts, vocab);
    if (!need) return set_error(W4G64_STATUS_UNSUPPORTED, "verify_drafts call is too large: batch %lld", (long long)batch);
    const int align = dtype == W4G64_DTYPE_F32 ? 3 : 1;
    if (!target || !uniforms || !tokens || !accepted || (drafts && !draft_tokens) ||
        (((uintptr_t)target | (uintptr_t)draft) & align) || (((uintptr_t)uniforms | (uintptr_t)accepted) & 3) ||
        (((uintptr_t)tokens | (uintptr_t)draft_tokens) & 7) || ((uintptr_t)draft_lengths & 3))
        return set_error(W4G64_STATUS_INVALID_VALUE, "verify_drafts needs non-null, element-aligned pointers");
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 7))
        return set_error(W4G64_STATUS_WORKSPACE, "verify_drafts needs %lld workspace bytes, 8-byte aligned, got %lld",
                         (long long)need, (long long)(workspace ? workspace_bytes : 0));
    VerifyArgs a{target, draft, target_batch, target_row, draft_batch, draft_row, draft_tokens, draft_lengths, uniforms,
                 tokens, accepted, (double*)workspace, nullptr, (int)batch, (int)drafts, (int)vocab, (int)verify_spans(vocab)};
    a.standing = (int32_t*)(a.sums + batch * a.spans);
    const hipStream_t s = (hipStream_t)stream;
    const hipError_t err = dtype == W4G64_DTYPE_F32    ? launch_verify<kF32>(a, batch, s)
                           : dtype == W4G64_DTYPE_BF16 ? launch_verify<kBF16>(a, batch, s)
                                                       : launch_verify<kF16>(a, batch, s);
    if (err != hipSuccess)
        return set_error(W4G64_STATUS_HIP_ERROR, "verify_drafts launch failed: %s", hipGetErrorString(err));
    return clear_error();
}

}  // extern "C"
