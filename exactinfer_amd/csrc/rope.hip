// rope.hip — rotary positions of packed rows on gfx950: the (cos, sin) table for plain and scaled
// frequencies, and the rotation of many heads per row, each row at a position of its own.
//
// A pair (a, b) at position p turns by p f_i: (a c - b s, a s + b c).  Both kernels move bytes: the
// table's double-precision sincos run once per context, the rotation reads and writes each head once.
#include <type_traits>

#include "common.h"
#include "launch.h"

namespace ei {

// One thread per (cos, sin), consecutive ones of a position's pairs.  Angles in double: at position 131071 an
// angle in fp32 would be off by up to 2^-8 radians.  Bound by the double sincos: 65536 positions of 64 pairs (33.5 MB)
// 22 us.
__global__ __launch_bounds__(256) void k_rope_table(float2* __restrict__ cs, long n, int half, RopeFrequencies fr) {
    for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long)gridDim.x * blockDim.x) {
        const long p = i / half;
        const double th = (double)p * fr.f[i - p * half];
        double s, c;
        sincos(th, &s, &c);
        cs[i] = make_float2((float)(c * fr.m), (float)(s * fr.m));
    }
}

// Sixteen lanes per head, eight values each, four heads per wave.  kVec: rope_dim is a multiple of 8
// (half layout) or of 4 (interleaved), so every 16-byte piece is turned whole or not at all:
//   half         lanes below rope_dim/8 hold the pieces at 4l and rope_dim/2 + 4l, partners of each
//                other; the other lanes two pieces each of the rest of the head
//   interleaved  lane l holds the pieces at 4l and 64 + 4l, two pairs each
// Otherwise lane l holds elements l + 16j and reads the partners from the row itself, all before the
// head is written.  Measured: 16384 rows of 40 heads with the norm (671 MB and the table) 131 us, 5.2 TB/s, without
// kVec 185; 1533 rows, interleaved, 64 of 128 values turned 12.6 us, 6.0 TB/s, without kVec 14.5.  48 rows take
// 3.4 us, a launch and one round trip to memory.
template <bool kHalf, bool kVec, bool kNorm>
__global__ __launch_bounds__(256) void k_rope_rows(const float* x, long x_stride, float* y, long y_stride,
                                                   int rows, int n_heads, const float* __restrict__ gamma, float eps,
                                                   const float2* __restrict__ cs, int n_pos,
                                                   const int* __restrict__ pos, int rope_dim) {
#pragma clang fp contract(off)
    const int lane = threadIdx.x & 15;
    const uint32_t unit = blockIdx.x * 16 + (threadIdx.x >> 4);  // (below 2^31 + 15)
    const uint32_t b = unit / (uint32_t)n_heads;
    if (b >= (uint32_t)rows) return;  // a whole group of sixteen; no barrier here
    const int h = (int)(unit - b * (uint32_t)n_heads);
    const int p = pos[b], half = rope_dim >> 1;
    const bool in = p >= 0 && p < n_pos;
    const float2* row = cs + (size_t)(in ? p : 0) * half;
    // the element of value j of this lane
    auto at = [&](int j) {
        if constexpr (!kVec) return lane + 16 * j;
        else if constexpr (!kHalf) return 4 * lane + 64 * (j >> 2) + (j & 3);
        else if (lane < (rope_dim >> 3)) return 4 * lane + half * (j >> 2) + (j & 3);
        else return rope_dim + 8 * (lane - (rope_dim >> 3)) + j;
    };
    float g[kNorm ? 8 : 1];
    if constexpr (kNorm) {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = gamma[at(j)];
    }
    float v[8];
    const float* src = x + (size_t)b * x_stride + (size_t)h * kHeadDim;
    if constexpr (kVec) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float4 t = *reinterpret_cast<const float4*>(src + at(4 * k));
            v[4 * k] = t.x, v[4 * k + 1] = t.y, v[4 * k + 2] = t.z, v[4 * k + 3] = t.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = src[at(j)];
    }
    // the pairs' (cos, sin): kVec half 4 of one pair per piece, interleaved 2 per piece; else one per value
    float2 t[kVec ? 4 : 8];
    if constexpr (kVec && kHalf) {
        if (lane < (rope_dim >> 3)) {
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = row[4 * lane + j];
        }
    } else if constexpr (kVec) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (at(4 * k) < rope_dim) t[2 * k] = row[at(4 * k) >> 1], t[2 * k + 1] = row[(at(4 * k) >> 1) + 1];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = at(j);
            if (e < rope_dim) t[j] = row[kHalf ? (e < half ? e : e - half) : e >> 1];
        }
    }
    float inv = 1.f;
    if constexpr (kNorm) {
        double ss = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)v[j], (double)v[j], ss);
        ss += lane_xor_f64<1>(ss);
        ss += lane_xor_f64<2>(ss);
        ss += lane_xor_f64<4>(ss);
        ss += lane_xor_f64<8>(ss);
        inv = (float)(1.0 / sqrt(ss / (double)kHeadDim + (double)eps));
    }
    auto scaled = [&](float f, int j) { return kNorm ? (f * inv) * g[j] : f; };
    float w[8];
    if (!in) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = v[j];
    } else if constexpr (kVec) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = scaled(v[j], j);
        if constexpr (kHalf) {
            if (lane < (rope_dim >> 3)) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float a = w[j], c = w[4 + j];
                    const float ac = a * t[j].x, cn = c * t[j].y, an = a * t[j].y, cc = c * t[j].x;
                    w[j] = ac - cn, w[4 + j] = an + cc;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j += 2)
                if (at(j) < rope_dim) {
                    const float a = w[j], c = w[j + 1];
                    const float2 q = t[j >> 1];
                    const float ac = a * q.x, cn = c * q.y, an = a * q.y, cc = c * q.x;
                    w[j] = ac - cn, w[j + 1] = an + cc;
                }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = at(j);
            w[j] = scaled(v[j], j);
            if (e < rope_dim) {
                const bool first = kHalf ? e < half : (e & 1) == 0;
                const int o = kHalf ? (first ? e + half : e - half) : e ^ 1;
                const float other = kNorm ? (src[o] * inv) * gamma[o] : src[o];
                const float own_c = w[j] * t[j].x, other_s = other * t[j].y;
                w[j] = first ? own_c - other_s : other_s + own_c;
            }
        }
    }
    float* dst = y + (size_t)b * y_stride + (size_t)h * kHeadDim;
    if constexpr (kVec) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            *reinterpret_cast<float4*>(dst + at(4 * k)) =
                make_float4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) dst[at(j)] = w[j];
    }
}

hipError_t launch_rope_table(hipStream_t st, float* cs, int n_pos, int rope_dim, const RopeFrequencies& fr) {
    const long n = (long)n_pos * (rope_dim >> 1);
    const long blocks = (n + 255) / 256;
    k_rope_table<<<(unsigned)(blocks < 65536 ? blocks : 65536), 256, 0, st>>>(reinterpret_cast<float2*>(cs), n,
                                                                            rope_dim >> 1, fr);
    return hipGetLastError();
}

template <bool kHalf, bool kVec, bool kNorm>
static hipError_t launch_rope_rows_as(hipStream_t st, const float* x, long x_stride, float* y, long y_stride, int rows,
                                      int n_heads, const float* gamma, float eps, const float2* cs, int n_pos,
                                      const int* pos, int rope_dim) {
    const long blocks = ((long)rows * n_heads + 15) / 16;
    k_rope_rows<kHalf, kVec, kNorm><<<(unsigned)blocks, 256, 0, st>>>(x, x_stride, y, y_stride, rows, n_heads, gamma,
                                                                    eps, cs, n_pos, pos, rope_dim);
    return hipGetLastError();
}

hipError_t launch_rope_rows(hipStream_t st, const float* x, long x_stride, float* y, long y_stride, int rows,
                            int n_heads, const float* gamma, float eps, const float* cs, int n_pos, const int* pos,
                            int rope_dim, bool half) {
    const float2* t = reinterpret_cast<const float2*>(cs);
    const bool vec = rope_dim % (half ? 8 : 4) == 0, norm = gamma != nullptr;
    auto go = [&](auto h, auto v, auto n) {
        return launch_rope_rows_as<decltype(h)::value, decltype(v)::value, decltype(n)::value>(
            st, x, x_stride, y, y_stride, rows, n_heads, gamma, eps, t, n_pos, pos, rope_dim);
    };
    using T = std::true_type;
    using F = std::false_type;
    if (half)
        return vec ? (norm ? go(T{}, T{}, T{}) : go(T{}, T{}, F{})) : (norm ? go(T{}, F{}, T{}) : go(T{}, F{}, F{}));
    return vec ? (norm ? go(F{}, T{}, T{}) : go(F{}, T{}, F{})) : (norm ? go(F{}, F{}, T{}) : go(F{}, F{}, F{}));
}

}  // namespace ei
