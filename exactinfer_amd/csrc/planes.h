// planes.h — what the attention kernels of prefill.hip and packed.hip share (vector types, index
// arithmetic, values kept from being hoisted), and prefill.hip's fp32 operands on bf16 matrix cores:
// the three-plane split and its product.
#pragma once

#include "common.h"

namespace ei {

typedef float floatx16 __attribute__((ext_vector_type(16)));

// n / d for small d (1..8) and n * d < 2^32 as one multiply-high: the per-pass index math
// runs on the scalar unit, which the eight waves of a CU share, so a division loop per use
// would cost thousands of cycles per pass.  m = ceil(2^32 / d); d = 1 is taken as is.
struct FastDiv {
    uint32_t m, d;
};
__device__ __forceinline__ FastDiv fast_div(uint32_t d) { return {d == 1 ? 0u : 0xFFFFFFFFu / d + 1u, d}; }
__device__ __forceinline__ int fdiv(int n, FastDiv f) {
    return f.d == 1 ? n : (int)__umulhi((uint32_t)n, f.m);
}

// A value the optimiser may not carry across loop iterations: what is derived from it is computed
// where it is used (the vector registers of the key loop are full, hoisted addresses would spill).
__device__ __forceinline__ int unhoisted(int x) {
    asm volatile("" : "+v"(x));
    return x;
}
__device__ __forceinline__ float here(float x) {  // the same of a kernel argument
    asm volatile("" : "+s"(x));
    return x;
}
__device__ __forceinline__ float uniform(float x) {  // a wave-uniform value, in a scalar register
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x)));
}

// ------------------------------------------------------------------ three-plane split
// x = h + m + l with h, m, l in bf16: h = bf16(x), m = bf16(x - h), l = x - h - m, each rounded to
// nearest.  Both differences are exact (the residual of a 24-bit value rounded to 8 bits has at
// most 16 significant bits, the second at most 8), so the three planes hold every bit of x as long
// as none of them leaves bf16's range: from kPlaneMin up, where x's last bit is a normal bf16, to
// bf16's largest value.  What lies outside is noticed and multiplied in fp32.
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int kBufferDword3 = 0x00020000;  // raw 32-bit data, gfx9-family buffer resource word 3

__device__ __forceinline__ uint32_t pk_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& h, uint32_t& m, uint32_t& l) {
#pragma clang fp contract(off)
    h = pk_bf16(a, b);
    const float ra = a - __uint_as_float(h << 16), rb = b - __uint_as_float(h & 0xFFFF0000u);
    m = pk_bf16(ra, rb);
    l = pk_bf16(ra - __uint_as_float(m << 16), rb - __uint_as_float(m & 0xFFFF0000u));
}
constexpr float kPlaneMin = 0x1p-100f;
// The planes of a small value are off by up to 2^-134, which counts for something only against a large
// partner.  From this value on an operand is taken to be one, so below it the smallest partner does
// not matter.
constexpr float kPlaneMax = 0x1p24f;
constexpr float kSmallSum = 0x1p-60f;
// |x| in the order of nonzero values, zero last
__device__ __forceinline__ uint32_t magnitude(uint32_t x) { return (x << 1) - 1u; }
__device__ __forceinline__ float of_magnitude(uint32_t m) {  // its |x|; infinite for zero
    return m == 0xFFFFFFFFu ? INFINITY : __uint_as_float((m >> 1) + 1u);
}
constexpr uint32_t kTinyMagnitude = (__builtin_bit_cast(uint32_t, kPlaneMin) << 1) - 1u;
struct Planes {  // eight values: one MFMA operand per plane
    u32x4 h, m, l;
};
__device__ __forceinline__ floatx16 mfma_bf16(u32x4 a, u32x4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}
// c += a . b without m.l, l.m and l.l (together at most 2^-24 of |a||b|).  a's planes are used up one
// after another, and next(x) refills plane x (2 l, 1 m, 0 h) with the next step's right after its last
// use: at least three matrix instructions cover each LDS read, in the registers of one step.
template <typename Next>
__device__ __forceinline__ void mfma_split(Planes& a, const Planes& b, floatx16& c, Next next) {
    constexpr int kAlu = 0x6;  // VALU and SALU work may move across, LDS reads and MFMAs stay in order
    c = mfma_bf16(a.l, b.h, c);
    __builtin_amdgcn_sched_barrier(kAlu);
    a.l = next(2);
    __builtin_amdgcn_sched_barrier(kAlu);
    c = mfma_bf16(a.m, b.m, c);
    c = mfma_bf16(a.m, b.h, c);
    __builtin_amdgcn_sched_barrier(kAlu);
    a.m = next(1);
    __builtin_amdgcn_sched_barrier(kAlu);
    c = mfma_bf16(a.h, b.l, c);
    c = mfma_bf16(a.h, b.m, c);
    c = mfma_bf16(a.h, b.h, c);
    __builtin_amdgcn_sched_barrier(kAlu);
    a.h = next(0);
    __builtin_amdgcn_sched_barrier(kAlu);
}

}  // namespace ei
