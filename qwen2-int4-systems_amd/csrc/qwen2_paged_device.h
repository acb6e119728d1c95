// What the kernels of packed rows share: the two 16-bit element types as pairs in
// a word, division by numbers that the host knows, the exponents of probabilities,
// values that are not finite, and the paged cache as its entry points check it.
#pragma once

#include <hip/hip_runtime.h>

#include "qwen2_decode.h"
#include "qwen2_paged.h"
#include "w4g64_device.h"

namespace w4g64 {

struct Bf16 {
    static __device__ __forceinline__ float lo(uint32_t w) { return bf16_lo(w); }
    static __device__ __forceinline__ float hi(uint32_t w) { return bf16_hi(w); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
    static constexpr uint32_t kExponent = 0x7F80u;  // all ones: an infinity or NaN
    static constexpr uint32_t kOne = 0x3F80u;
    static __device__ __forceinline__ float4v mfma(const u32x4& a, const u32x4& b, const float4v& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
};

struct F16 {
    static __device__ __forceinline__ float lo(uint32_t w) { return (float)__builtin_bit_cast(half2v, w)[0]; }
    static __device__ __forceinline__ float hi(uint32_t w) { return (float)__builtin_bit_cast(half2v, w)[1]; }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2v{a, b}, half2v));
    }
    static constexpr uint32_t kExponent = 0x7C00u;
    static constexpr uint32_t kOne = 0x3C00u;
    static __device__ __forceinline__ float4v mfma(const u32x4& a, const u32x4& b, const float4v& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0,
                                                      0, 0);
    }
};

// Division of numbers below 2^31 by a divisor that the host knows: the usual
// multiplication by 2^(32 + shift) / divisor, less its leading one.
struct Divisor {
    uint32_t magic, shift;
    __device__ __forceinline__ int operator()(int n) const {
        return (int)((__umulhi((uint32_t)n, magic) + (uint32_t)n) >> shift);
    }
};
inline Divisor divisor(int64_t d) {
    Divisor r{0, 0};
    d = d > 0 ? d : 1;
    while ((int64_t(1) << r.shift) < d) ++r.shift;
    r.magic = (uint32_t)((((uint64_t(1) << r.shift) - (uint64_t)d) << 32) / (uint64_t)d + (r.shift ? 1 : 0));
    return r;
}

// Running sums over the wave (shifts within rows of 16 lanes, then their last lanes
// passed on).
__device__ __forceinline__ int running_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// Exponents of probabilities.  bf16: they reach 2^kLazy before the sums are
// rescaled, and stay at one or below with 2^-kLazy for the reference, so that values
// add up as far as fp32 holds the keys' number times their size.  fp16 ends at
// 2^-24 and at 2^16, and a key far below its row's maximum still counts if there are
// many; with 2^11 for the reference the terms reach down to 2^-35 of it (and its
// values times their number stay far inside fp32).
template <class E> inline constexpr float kProbShift = -8.0f;
template <> inline constexpr float kProbShift<F16> = 11.0f;
template <class E> inline constexpr float kLazy = 8.0f;
template <> inline constexpr float kLazy<F16> = 4.0f;

// Values that are not finite (an infinity or a NaN, met in the sums of a first
// pass) must reach the rows that see their keys and no others, where a product
// with a probability of zero would give NaN.  Three more passes tell: two that
// count, for every row and dimension, the visible keys with +inf or NaN and with
// -inf or NaN (ones in place of probabilities and of such values), and one over
// the finite values alone.
enum Pass { kOrdinary, kCountUp, kCountDown, kFinite };
template <class E> __device__ __forceinline__ uint32_t pass_half(uint32_t h, Pass pass) {
    const bool odd = (h & E::kExponent) == E::kExponent;
    if (pass == kFinite) return odd ? 0u : h;
    const bool nan = (h & 0x7FFFu) > E::kExponent, down = (h & 0x8000u) != 0;
    return odd && (nan || down == (pass == kCountDown)) ? E::kOne : 0u;
}
template <class E> __device__ __forceinline__ uint32_t pass_word(uint32_t w, Pass pass) {
    return pass_half<E>(w & 0xFFFFu, pass) | (pass_half<E>(w >> 16, pass) << 16);
}

// What sums whose weight came out as zero still say: infinities and NaN, which the
// formula's weight, small as it is, does not take away.
__device__ __forceinline__ void add_odd(float& sum, float x) {
    if (!(fabsf(x) < INFINITY)) sum += x;
}

// The cache of a call, checked (the status of set_error where it cannot be used).
int paged_view(const qwen2_paged_cache* cache, PagedView* view);

}  // namespace w4g64
