// What the paged kernels share: the two 16-bit element types as pairs in a
// word, and the cache as their entry points check it.
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

// The cache of a call, checked (the status of set_error where it cannot be used).
int paged_view(const qwen2_paged_cache* cache, PagedView* view);

}  // namespace w4g64
