// Verification of drafted tokens (qwen2_verify_drafts, include/qwen2_decode.h).
//
//   verify_sum_kernel   one workgroup per (sequence, 4096 entries of the
//                       vocabulary): finds how many drafts stand (every
//                       workgroup for itself: a few loads), then adds up its
//                       entries' weights;
//   verify_pick_kernel  one workgroup per sequence: the chunk in which the
//                       running sum passes uniform * total, then the entry.
//
// Only one row of the target's (and the draft's) probabilities is read per
// sequence.  A weight is a difference of two 24-bit numbers and the sums run
// over the vocabulary, so they are held in 64 bits: the chosen entry is then
// the definition's, not the summation order's.  Sums have one fixed order: 16
// entries of a thread, the wave's threads pairwise, the waves, the chunks.
//
// Bound by the rows' read from memory, and for few sequences by two launches.
#include <hip/hip_runtime.h>

#include "qwen2_decode.h"
#include "w4g64_device.h"
#include "w4g64_internal.h"

namespace w4g64 {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 16;  // entries of a thread
constexpr int kChunk = kThreads * kPer;

struct VerifyArgs {
    const void* target;
    const void* draft;
    int64_t target_batch, target_row, draft_batch, draft_row;
    const int64_t* draft_tokens;
    const int32_t* draft_lengths;
    const float* uniforms;
    int64_t* tokens;
    int32_t* accepted;
    double* sums;  // [batch][chunks][2]: of the weights, and of the target alone
    int drafts, vocab, chunks;
};

template <int XK>
__device__ __forceinline__ double value(const void* p, int64_t i) {
    if constexpr (XK == kF32) return (double)((const float*)p)[i];
    if constexpr (XK == kBF16) return (double)bf16_bits_to_float(((const uint16_t*)p)[i]);
    return (double)half_bits_to_float(((const uint16_t*)p)[i]);
}

// max(x, 0), NaN kept.
__device__ __forceinline__ double positive(double x) { return x > 0.0 || x != x ? x : 0.0; }

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

// The thread's entries chunk * 4096 + 16 tid .. + 15 (zero past the vocabulary).
template <int XK>
__device__ __forceinline__ void thread_weights(const Weights& w, int vocab, int chunk, int tid, double (&less)[kPer],
                                               double (&plain)[kPer]) {
    const int v0 = chunk * kChunk + kPer * tid;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const int v = v0 + e;
        const bool in = v < vocab;
        const double p = in ? value<XK>(w.target, w.target_at + v) : 0.0;
        double q = v == w.hot ? 1.0 : 0.0;
        if (w.draft && in) q = value<XK>(w.draft, w.draft_at + v);
        plain[e] = positive(p);
        less[e] = positive(p - q);
    }
}

__device__ __forceinline__ double shfl_xor_f64(double v, int mask) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __shfl_xor((uint32_t)u, mask), hi = __shfl_xor((uint32_t)(u >> 32), mask);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

template <int XK>
__global__ __launch_bounds__(kThreads) void verify_sum_kernel(VerifyArgs a) {
    __shared__ double part[2][kThreads / 64];
    const int tid = threadIdx.x;
    const int b = blockIdx.x / a.chunks;
    const int chunk = blockIdx.x - b * a.chunks;
    int count;
    const int n = standing<XK>(a, b, tid & 63, count);
    const Weights w = weights_of(a, b, n, count);
    double less[kPer], plain[kPer];
    thread_weights<XK>(w, a.vocab, chunk, tid, less, plain);
    double sl = 0.0, sp = 0.0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        sl += less[e];
        sp += plain[e];
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        sl += shfl_xor_f64(sl, m);
        sp += shfl_xor_f64(sp, m);
    }
    if ((tid & 63) == 0) {
        part[0][tid >> 6] = sl;
        part[1][tid >> 6] = sp;
    }
    __syncthreads();
    if (tid < 2) {
        double s = part[tid][0];
        for (int i = 1; i < kThreads / 64; ++i) s += part[tid][i];
        a.sums[2 * (int64_t)blockIdx.x + tid] = s;
    }
}

// Sum of the values of the lower threads, in a workgroup of four waves.
__device__ __forceinline__ double sum_before(double own, int tid, double* shared) {
    const int lane = tid & 63;
    double upto = own;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const uint64_t u = __builtin_bit_cast(uint64_t, upto);
        const uint32_t lo = __shfl_up((uint32_t)u, step), hi = __shfl_up((uint32_t)(u >> 32), step);
        if (lane >= step) upto += __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
    }
    if (lane == 63) shared[tid >> 6] = upto;
    __syncthreads();
    double before = 0.0;
    for (int i = 0; i < (tid >> 6); ++i) before += shared[i];
    const uint64_t u = __builtin_bit_cast(uint64_t, upto);
    const uint32_t lo = __shfl_up((uint32_t)u, 1), hi = __shfl_up((uint32_t)(u >> 32), 1);
    if (lane) before += __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
    return before;
}

template <int XK>
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerifyArgs a) {
    __shared__ double totals[2];
    __shared__ double shared[kThreads / 64];
    __shared__ double base;
    __shared__ int chosen_chunk, chosen, last;
    const int tid = threadIdx.x;
    const int b = blockIdx.x;
    int count;
    const int n = standing<XK>(a, b, tid & 63, count);
    const Weights w = weights_of(a, b, n, count);
    const double* sums = a.sums + 2 * (int64_t)b * a.chunks;
    if (tid < 2) {
        double s = 0.0;
        for (int c = 0; c < a.chunks; ++c) s += sums[2 * c + tid];
        totals[tid] = s;
    }
    if (tid == 0) chosen = 0x7FFFFFFF, last = -1;
    __syncthreads();
    // no entry where the draft falls short of the target: the target alone
    const int which = totals[0] == 0.0;
    const double total = totals[which];
    float u = a.uniforms[(int64_t)b * (a.drafts + 1) + a.drafts];
    constexpr float kBelowOne = 0.999999940395355224609375f;  // 1 - 2^-24
    if (u > kBelowOne) u = kBelowOne;
    if (u < 0.0f) u = 0.0f;
    const double goal = (double)u * total;
    const bool usable = total > 0.0 && total < __builtin_inf() && u == u;  // (uniform)
    if (usable) {
        if (tid == 0) {
            double run = 0.0, at = 0.0;
            int c = -1;  // the first chunk whose end passes the goal
            for (int i = 0; i < a.chunks; ++i) {
                const double next = run + sums[2 * i + which];
                if (next > goal) {
                    c = i, at = run;
                    break;
                }
                run = next;
            }
            chosen_chunk = max(c, 0), base = at;  // (the last end is the total, past the goal)
        }
        __syncthreads();
        const int chunk = chosen_chunk;
        double less[kPer], plain[kPer], own = 0.0;
        thread_weights<XK>(w, a.vocab, chunk, tid, less, plain);
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            less[e] = which ? plain[e] : less[e];
            own += less[e];
        }
        double run = base + sum_before(own, tid, shared);
        int found = 0x7FFFFFFF, some = -1;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            run += less[e];
            const int v = chunk * kChunk + kPer * tid + e;
            if (less[e] > 0.0) {
                some = v;
                if (run > goal && found == 0x7FFFFFFF) found = v;
            }
        }
        if (found != 0x7FFFFFFF) atomicMin(&chosen, found);
        if (some >= 0) atomicMax(&last, some);
        __syncthreads();
    }
    // (the chunk's sum passes the goal; where its entries, added in another order,
    // stay a rounding below, it is the last of them)
    const int64_t token = !usable ? -1 : (chosen != 0x7FFFFFFF ? chosen : last);
    for (int i = tid; i <= a.drafts; i += kThreads) {
        const int64_t at = (int64_t)b * (a.drafts + 1) + i;
        a.tokens[at] = i < n ? a.draft_tokens[(int64_t)b * a.drafts + i] : (i == n ? token : -1);
    }
    if (tid == 0) a.accepted[b] = n;
}

template <int XK>
hipError_t launch_verify(const VerifyArgs& a, int64_t batch, hipStream_t stream) {
    hipLaunchKernelGGL(verify_sum_kernel<XK>, dim3((unsigned)(batch * a.chunks)), dim3(kThreads), 0, stream, a);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    hipLaunchKernelGGL(verify_pick_kernel<XK>, dim3((unsigned)batch), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

int64_t verify_chunks(int64_t vocab) { return (vocab + kChunk - 1) / kChunk; }

}  // namespace
}  // namespace w4g64

using namespace w4g64;

extern "C" {

int64_t qwen2_verify_drafts_workspace_bytes(int64_t batch, int64_t drafts, int64_t vocab) {
    if (batch <= 0 || drafts < 0 || vocab <= 0 || vocab > 0x7FFFFFFF - kChunk || batch > 0x7FFFFFFF / verify_chunks(vocab))
        return 0;
    return batch * verify_chunks(vocab) * 2 * (int64_t)sizeof(double);
}

int qwen2_verify_drafts(const void* target, int64_t target_batch, int64_t target_row, const void* draft,
                        int64_t draft_batch, int64_t draft_row, int dtype, const int64_t* draft_tokens,
                        const int32_t* draft_lengths, const float* uniforms, int64_t* tokens, int32_t* accepted,
                        int64_t batch, int64_t drafts, int64_t vocab, void* workspace, int64_t workspace_bytes,
                        void* stream) {
    if (dtype != W4G64_DTYPE_F32 && dtype != W4G64_DTYPE_BF16 && dtype != W4G64_DTYPE_F16)
        return set_error(W4G64_STATUS_INVALID_DTYPE, "verify_drafts probabilities must be fp32, bf16 or fp16, got code %d", dtype);
    if (batch < 0 || drafts < 0 || drafts > 0xFFFF || vocab <= 0 || vocab > 0x7FFFFFFF - kChunk)
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
                 tokens, accepted, (double*)workspace, (int)drafts, (int)vocab, (int)verify_chunks(vocab)};
    const hipStream_t s = (hipStream_t)stream;
    const hipError_t err = dtype == W4G64_DTYPE_F32    ? launch_verify<kF32>(a, batch, s)
                           : dtype == W4G64_DTYPE_BF16 ? launch_verify<kBF16>(a, batch, s)
                                                       : launch_verify<kF16>(a, batch, s);
    if (err != hipSuccess)
        return set_error(W4G64_STATUS_HIP_ERROR, "verify_drafts launch failed: %s", hipGetErrorString(err));
    return clear_error();
}

}  // extern "C"
