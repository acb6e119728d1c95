// What the kernels of packed prompts and of pages need besides tests/lanes, read
// before their sources: 32 x 32 matrix instructions and whole-number atomics.
#pragma once

#include <hip/hip_runtime.h>

#include <initializer_list>

namespace lanes {

// D = A B + C of 32 x 32 x 16: lane 32 h + j holds K slots 8 h .. of row j of A and
// column j of B, and rows 8 (i / 4) + 4 h + i % 4 of column j of C and D in place i.
typedef float float16 __attribute__((ext_vector_type(16)));
template <bool kBf16, class V>
float16 product32(const V& a, const V& b, const float16& c) {
    if (skip_products) return c;
    struct Operands {
        Eight a, b;
    };
    const Values& all = exchange(Operands{__builtin_bit_cast(Eight, a), __builtin_bit_cast(Eight, b)});
    const int h = lane() / 32, j = lane() % 32;
    float16 d = c;
    for (int g = 0; g < 2; ++g) {
        const Eight y = all.at<Operands>(32 * g + j).b;
        for (int i = 0; i < 16; ++i) {
            const Eight x = all.at<Operands>(32 * g + 8 * (i / 4) + 4 * h + i % 4).a;
            for (int e = 0; e < 8; ++e) d[i] += as_float(x.h[e], kBf16) * as_float(y.h[e], kBf16);
        }
    }
    return d;
}

// c plus both halves (the second operand is ones).
template <bool kBf16>
float pair_sum(uint32_t w, float c) {
    return c + (as_float((uint16_t)w, kBf16) + as_float((uint16_t)(w >> 16), kBf16));
}

}  // namespace lanes

#define __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, x, y, z) lanes::product32<true>(a, b, c)
#define __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, x, y, z) lanes::product32<false>(a, b, c)
#define __builtin_amdgcn_fdot2_f32_bf16(a, b, c, clamp) lanes::pair_sum<true>(__builtin_bit_cast(uint32_t, a), c)
#define __builtin_amdgcn_fdot2(a, b, c, clamp) lanes::pair_sum<false>(__builtin_bit_cast(uint32_t, a), c)
#define __builtin_amdgcn_mbcnt_lo(mask, base) ((base) + __builtin_popcount((mask) & (lanes::lane() < 32 ? (1u << lanes::lane()) - 1 : ~0u)))
#define __builtin_amdgcn_mbcnt_hi(mask, base) ((base) + __builtin_popcount((mask) & (lanes::lane() < 32 ? 0u : (1u << (lanes::lane() - 32)) - 1)))

// (one lane runs at a time)
inline int atomicAdd(int* p, int v) {
    const int old = *p;
    *p = old + v;
    return old;
}
inline int atomicMin(int* p, int v) {
    const int old = *p;
    *p = old < v ? old : v;
    return old;
}
