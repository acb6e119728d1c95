// Stands in for HIP's header where a test compiles kernels for the CPU: a
// workgroup's lanes run as coroutines (lanes.cpp), and what needs the other lanes of
// a wave (shuffles, ballots, matrix instructions, barriers) waits for them.  Loads
// and stores are the CPU's own, so that one outside its buffer ends the process.
// Only what the paged kernels use is here.
#pragma once

#include <math.h>
#include <stddef.h>
#include <stdint.h>
#include <string.h>

#include <functional>

#define __global__
#define __device__
#define __host__
#define __forceinline__ inline
#define __shared__ static  // one workgroup at a time
#define __launch_bounds__(...)

typedef void* hipStream_t;
typedef int hipError_t;
constexpr hipError_t hipSuccess = 0;
inline hipError_t hipGetLastError() { return hipSuccess; }
inline const char* hipGetErrorString(hipError_t) { return ""; }
struct dim3 {
    unsigned x;
    explicit dim3(unsigned x = 1) : x(x) {}
};

namespace lanes {

extern dim3 thread, block, grid;
extern bool skip_products;  // matrix products leave their sums as they are
void wave_sync();
void block_sync();
[[noreturn]] void fail(const char* what);
void launch(dim3 blocks, dim3 threads, const void* arguments, const std::function<void()>& kernel);
const void* arguments();
uint64_t alive();  // the wave's lanes that have not returned

// Every lane's value, good until the next exchange but one.
struct Values {
    unsigned char of[64][32];
    template <class T>
    T at(int lane) const {
        T t;
        memcpy(&t, of[lane & 63], sizeof(T));
        return t;
    }
};
const Values& exchange(const void* value, size_t bytes);
template <class T>
const Values& exchange(const T& v) {
    static_assert(sizeof(T) <= 32, "a lane's slot");
    return exchange(&v, sizeof(T));
}
inline int lane() { return (int)(thread.x & 63); }
inline int first() { return __builtin_ctzll(alive()); }
template <class T>
T read_lane(T v, int from) {
    return exchange(v).template at<T>(from);
}

inline int dpp(int old, int value, int control, int rows, int banks) {
    const Values& all = exchange(value);
    const int l = lane(), row = l / 16, at = l % 16;
    int from = -1;
    if (control < 0x100) from = (l & ~3) + ((control >> (2 * (l & 3))) & 3);                             // quad
    else if (control > 0x110 && control < 0x120) from = at >= control - 0x110 ? l - (control - 0x110) : -1;  // shift
    else if (control == 0x140) from = 16 * row + 15 - at;                                                // mirrors
    else if (control == 0x141) from = (l & ~7) + 7 - (l & 7);
    else if (control == 0x142) from = row > 0 ? 16 * row - 1 : -1;                                       // broadcasts
    else if (control == 0x143) from = row > 1 ? 31 : -1;
    else fail("dpp control");
    if (banks != 0xF) fail("dpp banks");
    return ((rows >> row) & 1) && from >= 0 ? all.at<int>(from) : old;
}

inline uint32_t perm(uint32_t a, uint32_t b, uint32_t select) {
    const uint64_t w = ((uint64_t)a << 32) | b;
    uint32_t r = 0;
    for (int i = 0; i < 4; ++i) r |= (uint32_t)((w >> (8 * ((select >> (8 * i)) & 7))) & 0xFF) << (8 * i);
    return r;
}

// The rows of 16 (32) lanes of the first operand with the second's, odd ones for even.
typedef uint32_t word2 __attribute__((ext_vector_type(2)));
inline word2 swap(uint32_t a, uint32_t b, int half) {
    struct Pair {
        uint32_t a, b;
    };
    const Values& all = exchange(Pair{a, b});
    const Pair other = all.at<Pair>(lane() ^ half);
    return lane() & half ? word2{other.b, b} : word2{a, other.a};
}

// Of 16 lanes, lane t brings elements 4 (t % 4) .. of row t / 4 and gets element t of
// the four rows.
typedef short short4 __attribute__((ext_vector_type(4)));
inline short4 read_transposed(const void* p) {
    short4 v;
    memcpy(&v, p, 8);
    const Values& all = exchange(v);
    const int t = lane() % 16, group = lane() - t;
    short4 r;
    for (int i = 0; i < 4; ++i) r[i] = all.at<short4>(group + 4 * i + t / 4)[t % 4];
    return r;
}

// D = A B + C of 16 x 16 x 32: lane 16 q + j holds K slots 8 q .. of row j of A and
// column j of B, and rows 4 q .. of column j of C and D.
typedef float float4 __attribute__((ext_vector_type(4)));
inline float as_float(uint16_t h, bool bf16) {
    return bf16 ? __builtin_bit_cast(float, (uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
}
struct Eight {
    uint16_t h[8];
};
template <bool kBf16, class V>
float4 product(const V& a, const V& b, const float4& c) {
    if (skip_products) return c;
    struct Operands {
        Eight a, b;
    };
    const Values& all = exchange(Operands{__builtin_bit_cast(Eight, a), __builtin_bit_cast(Eight, b)});
    const int q = lane() / 16, j = lane() % 16;
    float4 d = c;
    for (int i = 0; i < 4; ++i)
        for (int g = 0; g < 4; ++g) {
            const Eight x = all.at<Operands>(16 * g + 4 * q + i).a, y = all.at<Operands>(16 * g + j).b;
            for (int e = 0; e < 8; ++e) d[i] += as_float(x.h[e], kBf16) * as_float(y.h[e], kBf16);
        }
    return d;
}

// A buffer resource, and a load by it into LDS: the wave's place, 16 bytes a lane.
struct Resource {
    const unsigned char* data;
    uint32_t bytes;
};
inline void load_to_lds(const Resource& r, void* place, int size, int offset) {
    unsigned char* to = (unsigned char*)read_lane((uintptr_t)place, first());
    if (to != place) fail("LDS place differs between lanes");
    if (offset < 0 || (uint64_t)offset + size > r.bytes) fail("offset outside its buffer resource");
    memcpy(to + size * lane(), r.data + offset, size);
}

template <class T>
T unused() {
    fail("not used by these kernels");
}

}  // namespace lanes

#define threadIdx lanes::thread
#define blockIdx lanes::block
#define gridDim lanes::grid
#define hipLaunchKernelGGL(kernel, blocks, threads, lds, stream, a) \
    lanes::launch(blocks, threads, &(a), [&] { auto mine = a; (kernel)(mine); })
#define __syncthreads() lanes::block_sync()
#define __HIP_MEMORY_SCOPE_AGENT 4
#define __hip_atomic_fetch_add(...) lanes::unused<int>()
#define __amdgpu_buffer_rsrc_t lanes::Resource
#define __builtin_amdgcn_make_buffer_rsrc(p, stride, n, flags) (lanes::Resource{(const unsigned char*)(p), (uint32_t)(n)})
#define __builtin_amdgcn_raw_ptr_buffer_load_lds(r, to, n, offset, s, i, aux) lanes::load_to_lds(r, (void*)(to), n, offset)
#define __builtin_amdgcn_raw_buffer_load_b128(...) lanes::unused<u32x4>()
#define __builtin_amdgcn_raw_buffer_load_b8(...) lanes::unused<uint8_t>()
#define __builtin_amdgcn_readfirstlane(v) lanes::read_lane(v, lanes::first())
#define __builtin_amdgcn_readlane(v, l) lanes::read_lane(v, l)
#define __builtin_amdgcn_update_dpp(old, v, control, rows, banks, bound) lanes::dpp(old, v, control, rows, banks)
#define __builtin_amdgcn_perm(a, b, select) lanes::perm(a, b, select)
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __builtin_amdgcn_permlane16_swap(a, b, c, d) lanes::swap(a, b, 16)
#define __builtin_amdgcn_permlane32_swap(a, b, c, d) lanes::swap(a, b, 32)
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, x, y, z) lanes::product<true>(a, b, c)
#define __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, x, y, z) lanes::product<false>(a, b, c)
#define __builtin_amdgcn_ds_read_tr16_b64_v4i16(p) lanes::read_transposed((const void*)(p))
#define __builtin_amdgcn_s_waitcnt(x) lanes::wave_sync()
#define __builtin_amdgcn_s_barrier() lanes::block_sync()
#define __builtin_amdgcn_wave_barrier() lanes::wave_sync()
#define __builtin_amdgcn_sched_barrier(x) ((void)0)
#define __builtin_amdgcn_fence(...) ((void)0)
#define __builtin_amdgcn_kernarg_segment_ptr() lanes::arguments()

inline int __umulhi(uint32_t a, uint32_t b) { return (int)(uint32_t)(((uint64_t)a * b) >> 32); }
template <class T>
T __shfl(T v, int from) {
    return lanes::read_lane(v, from);
}
template <class T>
T __shfl_xor(T v, int mask) {
    return lanes::exchange(v).template at<T>(lanes::lane() ^ mask);
}
template <class T>
T __shfl_up(T v, int by) {
    const auto& all = lanes::exchange(v);
    return lanes::lane() >= by ? all.template at<T>(lanes::lane() - by) : v;
}
inline uint64_t __ballot(bool v) {
    const auto& all = lanes::exchange(v);
    uint64_t mask = 0;
    for (int l = 0; l < 64; ++l) mask |= (uint64_t)(((lanes::alive() >> l) & 1) && all.at<bool>(l)) << l;
    return mask;
}
inline bool __any(bool v) { return __ballot(v) != 0; }
inline bool __all(bool v) { return __ballot(!v) == 0; }
inline int __ffsll(unsigned long long v) { return __builtin_ffsll((long long)v); }
inline int __clzll(unsigned long long v) { return v ? __builtin_clzll(v) : 64; }
inline int __popcll(unsigned long long v) { return __builtin_popcountll(v); }
inline int min(int a, int b) { return a < b ? a : b; }
inline int max(int a, int b) { return a > b ? a : b; }
inline int64_t min(int64_t a, int64_t b) { return a < b ? a : b; }
inline int64_t max(int64_t a, int64_t b) { return a > b ? a : b; }
inline void sincospif(float x, float* sine, float* cosine) {
    *sine = (float)sin(M_PI * (double)x);
    *cosine = (float)cos(M_PI * (double)x);
}
