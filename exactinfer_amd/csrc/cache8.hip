// cache8.hip — a paged cache of 8-bit keys and values on gfx950: quantising a batch's new rows into it, reading rows
// back, attention over it (causal or over trees of drafts), and moving an accepted path's rows together.
#include <type_traits>

#include "packed.h"

namespace ei {

// ------------------------------------------------------------------ codes and their scales
// y of largest magnitude a: int8 scale a / 127, code rint(y (127 / a)); e4m3 scale a / 448, code e4m3(y (448 / a)).
// Below kNothing 127 / a and 448 / a would pass fp32's range on the way to it: such a head row is all zeros.
constexpr float kNothing = 0x1p-110f;
struct Coding {
    float scale, by;  // what a code stands for, and what a value is multiplied by
    bool bad;         // a value that is not finite: scale NaN, codes 0
};
template <bool kInt8>
__device__ __forceinline__ Coding coding(float most) {  // (infinite or NaN where a value is)
    constexpr float kTop = kInt8 ? 127.f : 448.f;
    if (!(most < INFINITY)) return {__builtin_nanf(""), 0.f, true};
    if (most < kNothing) return {0.f, 0.f, false};
    return {most / kTop, kTop / most, false};
}
// the codes of four values
template <bool kInt8>
__device__ __forceinline__ uint32_t codes_of(const float* y, const Coding& c) {
#pragma clang fp contract(off)
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = c.bad ? 0.f : y[j] * c.by;
    uint32_t u = 0;
    if constexpr (kInt8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) u |= ((uint32_t)(int)rintf(x[j]) & 0xFFu) << (8 * j);
    } else {
        u = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
        u = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], (int)u, true);
    }
    return u;
}
// two values of a code pair
template <bool kInt8, int kByte>
__device__ __forceinline__ float value_of(uint32_t codes) {
    if constexpr (kInt8) return (float)(int)(int8_t)(codes >> (8 * kByte));
    else return __builtin_amdgcn_cvt_f32_fp8((int)codes, kByte);
}
// the head row of key t in page `page`: rows of 128 codes, and scales
__device__ __forceinline__ size_t head_row(int page, int HKV, int kvh, int shift, int t) {
    return (((size_t)page * HKV + kvh) << shift) | (size_t)(t & ((1 << shift) - 1));
}

// ------------------------------------------------------------------ storing
// Sixteen lanes per head, eight values each, four heads per wave, as k_rope_rows lays them out.  kVec (rope_dim a
// multiple of 8): a lane below rope_dim / 8 holds the pieces of four at 4l and rope_dim / 2 + 4l, partners of each
// other, the others two pieces of the rest; otherwise elements l + 16j, whose partners are read from the row again.
// grid (rows, ceil((H + 2 HKV) / 16)).
//
// Bound by memory: 7644 rows of H 32 / HKV 8 (333 MB) 59 to 64 us, 5.2 to 5.6 TB/s, above a large copy's 4.7; with four
// bytes a lane instead of sixteen 83 us.  48 rows of H 16 / HKV 8 take 4 us: looking up a row's owner and its page.
template <bool kInt8, bool kVec>
__global__ __launch_bounds__(256) void k_cache8_store(const float* __restrict__ qkv, long row_stride,
                                                      float* __restrict__ q_out, Cache8Args a,
                                                      const float* __restrict__ q_gamma,
                                                      const float* __restrict__ k_gamma,
                                                      const float2* __restrict__ cs, int n_pos,
                                                      const int* __restrict__ turn_at, int rope_dim, float eps) {
#pragma clang fp contract(off)
    const int b = blockIdx.x, lane = threadIdx.x & 15, half = rope_dim >> 1;
    const int H = a.H, HKV = a.HKV, h = blockIdx.y * 16 + (threadIdx.x >> 4);
    const bool is_q = h < H, is_v = h >= H + HKV;
    auto at = [&](int j) {  // the element of value j of this lane
        if constexpr (!kVec) return lane + 16 * j;
        else if (lane < (rope_dim >> 3)) return 4 * lane + half * (j >> 2) + (j & 3);
        else return rope_dim + 8 * (lane - (rope_dim >> 3)) + j;
    };
    // (the row's values are on their way while its place is looked up; of a row that nobody owns they are not used)
    const float* src = qkv + (size_t)b * row_stride + (size_t)min(h, H + 2 * HKV - 1) * kHeadDim;
    const float* gamma = is_q ? q_gamma : k_gamma;
    float v[8], g[8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if constexpr (kVec) {
            // (plain loads: 7644 rows of H 32 / HKV 8 65 us instead of 59)
            const f32x4 t = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(src + at(4 * k)));
            v[4 * k] = t.x, v[4 * k + 1] = t.y, v[4 * k + 2] = t.z, v[4 * k + 3] = t.w;
            const float4 u = *reinterpret_cast<const float4*>(gamma + at(4 * k));
            g[4 * k] = u.x, g[4 * k + 1] = u.y, g[4 * k + 2] = u.z, g[4 * k + 3] = u.w;
        } else {
#pragma unroll
            for (int j = 4 * k; j < 4 * k + 4; ++j) v[j] = src[at(j)], g[j] = gamma[at(j)];
        }
    }
    if (!plan_fits(a.plan, a.n_seq, a.rows, H, HKV, false)) return;
    const int4* seq = reinterpret_cast<const int4*>(a.plan + kPlanSeqAt);
    const int s = row_owner(seq, a.n_seq, b, threadIdx.x & 63);  // (with the whole wave)
    if (s < 0 || h >= H + 2 * HKV || (is_q && !q_out)) return;   // sixteen lanes leave together
    const int4 e = seq[s];
    const int slot = e.z - e.y + (b - e.x);
    const int turn = turn_at ? turn_at[b] : slot;
    const bool in = slot >= 0 && slot < reinterpret_cast<const int*>(a.plan)[kHeadMaxKv] && turn >= 0 && turn < n_pos;
    const int blk = slot >> a.bshift;
    const int page = in && blk < a.max_blocks ? a.btab[(size_t)s * a.max_blocks + blk] : -1;
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = v[j];
    if (!is_v && in) {
        const float2* row = cs + (size_t)turn * half;
        double ss = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)v[j], (double)v[j], ss);
        ss += lane_xor_f64<1>(ss);
        ss += lane_xor_f64<2>(ss);
        ss += lane_xor_f64<4>(ss);
        ss += lane_xor_f64<8>(ss);
        const float inv = (float)(1.0 / sqrt(ss / (double)kHeadDim + (double)eps));
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = (v[j] * inv) * g[j];
        if constexpr (kVec) {
            if (lane < (rope_dim >> 3)) {
                const float4 t0 = *reinterpret_cast<const float4*>(row + 4 * lane);
                const float4 t1 = *reinterpret_cast<const float4*>(row + 4 * lane + 2);
                const float c[4] = {t0.x, t0.z, t1.x, t1.z}, n[4] = {t0.y, t0.w, t1.y, t1.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = w[j], y = w[4 + j];
                    const float xc = x * c[j], yn = y * n[j], xn = x * n[j], yc = y * c[j];
                    w[j] = xc - yn, w[4 + j] = xn + yc;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int i = at(j);
                if (i < rope_dim) {
                    const bool first = i < half;
                    const int o = first ? i + half : i - half;
                    const float2 t = row[first ? i : o];
                    const float other = (src[o] * inv) * gamma[o];
                    const float own_c = w[j] * t.x, other_s = other * t.y;
                    w[j] = first ? own_c - other_s : other_s + own_c;
                }
            }
        }
    }
    if (is_q) {
        float* dst = q_out + ((size_t)b * H + h) * kHeadDim;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if constexpr (kVec)
                *reinterpret_cast<float4*>(dst + at(4 * k)) =
                    make_float4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
            else
#pragma unroll
                for (int j = 4 * k; j < 4 * k + 4; ++j) dst[at(j)] = w[j];
        }
        return;
    }
    if (page < 0 || page >= a.n_blocks) return;
    // the largest magnitude, as bits: infinite and NaN ones are above the others
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(w[j]) & 0x7FFFFFFFu);
    most = max(most, __float_as_uint(lane_xor1(__uint_as_float(most))));
    most = max(most, __float_as_uint(lane_xor2(__uint_as_float(most))));
    most = max(most, __float_as_uint(lane_xor4(__uint_as_float(most))));
    most = max(most, __float_as_uint(lane_xor8(__uint_as_float(most))));
    const Coding c = coding<kInt8>(__uint_as_float(most));
    const size_t place = head_row(page, HKV, is_v ? h - H - HKV : h - H, a.bshift, slot);
    uint8_t* dst = (is_v ? a.v8 : a.k8) + place * kHeadDim;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint32_t u = codes_of<kInt8>(w + 4 * k, c);
        if constexpr (kVec) *reinterpret_cast<uint32_t*>(dst + at(4 * k)) = u;
        else
#pragma unroll
            for (int j = 0; j < 4; ++j) dst[at(4 * k + j)] = (uint8_t)(u >> (8 * j));
    }
    if (lane == 0) (is_v ? a.vs : a.ks)[place] = c.scale;
}

// ------------------------------------------------------------------ reading back
// A wave per row, a lane four codes: 32 lanes a head row, two head rows of K and V at a time.  Bound by the writes:
// 61769 rows of 8 heads (636 MB) 98 us back to back, 6.5 TB/s, and 118 over changing pools.
template <bool kInt8>
__global__ __launch_bounds__(256) void k_cache8_load(Cache8Args a, float* __restrict__ k_out,
                                                     float* __restrict__ v_out, long out_stride) {
    const int lane = threadIdx.x & 63, HKV = a.HKV;
    if (!plan_fits(a.plan, a.n_seq, a.rows, a.H, HKV, false)) return;
    const int b = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (b >= a.rows) return;
    const int4* seq = reinterpret_cast<const int4*>(a.plan + kPlanSeqAt);
    const int s = row_owner(seq, a.n_seq, b, lane);
    if (s < 0) return;
    const int4 e = seq[s];
    const int slot = e.z - e.y + (b - e.x), blk = slot >> a.bshift;
    const int page = slot >= 0 && blk < a.max_blocks ? a.btab[(size_t)s * a.max_blocks + blk] : -1;
    const bool there = page >= 0 && page < a.n_blocks;
    const int c = lane & 31;
    constexpr int kHeads = 4;  // of a lane, K and V, whose loads are in flight together
    for (int h0 = lane >> 5; h0 < HKV; h0 += 2 * kHeads) {
        uint32_t x[kHeads][2];
        float f[kHeads][2];
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const int h = h0 + 2 * i;
            const size_t at = head_row(page, HKV, min(h, HKV - 1), a.bshift, slot);
            x[i][0] = x[i][1] = 0, f[i][0] = f[i][1] = 0.f;
            if (there) {
                x[i][0] = reinterpret_cast<const uint32_t*>(a.k8 + at * kHeadDim)[c];
                x[i][1] = reinterpret_cast<const uint32_t*>(a.v8 + at * kHeadDim)[c];
                f[i][0] = a.ks[at], f[i][1] = a.vs[at];
            }
        }
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const int h = h0 + 2 * i;
            if (h >= HKV) break;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const f32x4 y = {value_of<kInt8, 0>(x[i][k]) * f[i][k], value_of<kInt8, 1>(x[i][k]) * f[i][k],
                                 value_of<kInt8, 2>(x[i][k]) * f[i][k], value_of<kInt8, 3>(x[i][k]) * f[i][k]};
                float* row = (k ? v_out : k_out) + (size_t)b * out_stride;
                f32x4* dst = reinterpret_cast<f32x4*>(row + (size_t)h * kHeadDim);
                __builtin_nontemporal_store(y, dst + c);  // (plain stores: 61769 rows 126 us instead of 100)
            }
        }
    }
}

// ------------------------------------------------------------------ the accepted path
// grid (n_seq, pieces / 256): a thread takes one piece of a sequence's rows, 16 bytes of K, then of V, then (8-bit) the
// scales.  Latency alone: the list, the lengths and the plan are read at once, a lane per entry looks its two pages
// up, then the rows are moved kKeepAtOnce at a time.  Entries rise, so kept[j] >= j: no row is read after another has
// been written over it.  Up to nine rows of 48 sequences 5 us in 8-bit pools (8.2 with a thread looking up each row).
constexpr int kKeepAtOnce = 8;
template <bool kF32>
__global__ __launch_bounds__(256) void k_cache_keep(Cache8Args a, float* __restrict__ kc, float* __restrict__ vc,
                                                    const int* __restrict__ kept, int max_kept,
                                                    const int* __restrict__ n_kept, int* __restrict__ new_len) {
    const int s = blockIdx.x, lane = threadIdx.x & 63;
    const int* list = kept + (size_t)s * max_kept;
    int row = lane < max_kept ? list[lane] : -1;
    const int want = n_kept[s];
    const int4 e = reinterpret_cast<const int4*>(a.plan + kPlanSeqAt)[s];
    if (!plan_fits(a.plan, a.n_seq, a.rows, a.H, a.HKV, false)) return;
    const int first = e.z - e.y, most = min(max(want, 0), min(max_kept, e.y));
    const int per_row = a.HKV * (kF32 ? 32 : 8);  // pieces of a row of K
    const int piece = blockIdx.y * 256 + threadIdx.x;
    const bool is_v = piece >= per_row, is_scale = !kF32 && piece >= 2 * per_row;
    const int i = is_scale ? piece - 2 * per_row : is_v ? piece - per_row : piece;  // of scales: K's, then V's
    const bool mine = piece < 2 * per_row || (is_scale && i < 2 * a.HKV);
    int before = -1, n = 0;
    for (int j0 = 0; j0 < most; j0 += 64) {
        if (j0 > 0) row = j0 + lane < max_kept ? list[j0 + lane] : -1;
        int last = __shfl_up(row, 1);
        if (lane == 0) last = before;
        const uint64_t bad = ~__builtin_amdgcn_ballot_w64(j0 + lane < most && row > last && row < e.y);
        const int count = bad ? __builtin_ctzll(bad) : 64;
        // the pages of this lane's entry: where its row is and where it goes (-1: it stays), and the rows in them
        auto page = [&](int new_row) {
            const int slot = first + new_row, blk = slot >> a.bshift;
            const int p = slot >= 0 && blk < a.max_blocks ? a.btab[(size_t)s * a.max_blocks + blk] : -1;
            return p < a.n_blocks ? p : -1;
        };
        const int in_page = (1 << a.bshift) - 1;
        int from = lane < count ? page(row) : -1;
        const int to = lane < count ? page(j0 + lane) : -1;
        if (to < 0) from = -1;
        const int from_t = (first + row) & in_page, to_t = (first + j0 + lane) & in_page;
        auto piece_at = [&](int p, int t) -> size_t {
            if constexpr (kF32) return (((size_t)p << a.bshift) | (size_t)t) * per_row + i;
            else if (is_scale) return head_row(p, a.HKV, i % a.HKV, a.bshift, t);
            else return head_row(p, a.HKV, i >> 3, a.bshift, t) * 8 + (i & 7);
        };
        for (int j = 0; j < count; j += kKeepAtOnce) {
            u32x4 x[kKeepAtOnce];
            size_t dst[kKeepAtOnce];
            bool go[kKeepAtOnce];
#pragma unroll
            for (int k = 0; k < kKeepAtOnce; ++k) {
                const int l = min(j + k, 63);
                const int p = __builtin_amdgcn_readlane(from, l);  // (-1 from `count` on)
                go[k] = mine && p >= 0 && j + k < 64;
                if (!go[k]) continue;
                const size_t src = piece_at(p, __builtin_amdgcn_readlane(from_t, l));
                dst[k] = piece_at(__builtin_amdgcn_readlane(to, l), __builtin_amdgcn_readlane(to_t, l));
                if constexpr (kF32) x[k] = reinterpret_cast<const u32x4*>(is_v ? vc : kc)[src];
                else if (is_scale) x[k].x = __float_as_uint((i < a.HKV ? a.ks : a.vs)[src]);
                else x[k] = reinterpret_cast<const u32x4*>(is_v ? a.v8 : a.k8)[src];
            }
#pragma unroll
            for (int k = 0; k < kKeepAtOnce; ++k) {
                if (!go[k]) continue;
                if constexpr (kF32) reinterpret_cast<u32x4*>(is_v ? vc : kc)[dst[k]] = x[k];
                else if (is_scale) (i < a.HKV ? a.ks : a.vs)[dst[k]] = __uint_as_float(x[k].x);
                else reinterpret_cast<u32x4*>(is_v ? a.v8 : a.k8)[dst[k]] = x[k];
            }
        }
        n += count;
        if (count < 64) break;
        before = __builtin_amdgcn_readlane(row, 63);
    }
    if (piece == 0) new_len[s] = max(first + n, 0);
}

// ------------------------------------------------------------------ attention
// Codes are exact in binary16, so a product with an fp32 operand takes two planes of it, x = h + l (22 bits of
// 24): two matrix instructions where two fp32 operands take three (packed.hip) or six (prefill.hip).
//
//   scores   q, scaled per row to a largest value of 2^14, against the codes of K; times the key's scale in fp32
//   output   weights p = 2^(s - m) F, F a power of two of the row's own, times the value's scale: the largest
//            p s_v lies between 2^14 and 2^15 at first, and F goes down where one passes that (the sums go with it), up
//            where the reference m rises (the sums stay).  So what the planes lose, 2^-39 of the row's largest
//            weight times scale, never shows, however uneven the values' scales are.  m is a whole number: every
//            factor of the sums is a power of two, exact.  The weights' sum has F too, so it stops at 2^96, and a pass
//            that ends with it there (values' scales below 2^-82) is done again with another arithmetic (pass_again).
struct Tile8 {
    u32x4 k[2][2];  // [sixteen keys][half of the lane's 32 codes]
    u32x2 v[8];
    f32x4 ks[2], vs[2];
};
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}
// Codes 2x and 2x + 1 of four as binary16: e4m3 by its conversion; int8 as 1024 + 128 + code, the code's sign bit
// flipped in the low bits of 1024, less 1152.  (`flipped`: the four codes with their sign bits flipped, for int8.)
template <bool kInt8, int x>
__device__ __forceinline__ uint32_t pair_f16(uint32_t codes) {
    if constexpr (kInt8) {
        const uint32_t biased = __builtin_amdgcn_perm(0x64646464u, codes, x ? 0x04030402u : 0x04010400u);
        const f16x2 y = __builtin_bit_cast(f16x2, biased) + f16x2{(_Float16)-1152.f, (_Float16)-1152.f};
        return __builtin_bit_cast(uint32_t, y);
    } else {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.f, x));
    }
}
// e4m3 codes that are NaN: 0x80 in the byte of each; and the codes with zeros in their place.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t codes) {
    return ((codes & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}
__device__ __forceinline__ uint32_t without_nan(uint32_t codes) {
    const uint32_t m = nan_bytes(codes);
    return codes & ~(m | (m - (m >> 7)));
}
template <bool kInt8>
__device__ __forceinline__ uint32_t flipped(uint32_t codes) { return kInt8 ? codes ^ 0x80808080u : codes; }

// Keys of the tile at t0 that a row at position qpos sees, a bit each.
__device__ __forceinline__ uint32_t causal_bits(int qpos, int t0) {
    const int n = qpos - t0 + 1;
    return n >= kKT ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
}

constexpr int kRow8 = 16;                              // rows of one matrix instruction
constexpr int kFew8ML = kWaves * kRow8 * kRowF;        // LDS: every wave's rows, then their (m, l)
constexpr int kFew8F = kFew8ML + kWaves * kRow8 * 2;
constexpr int kTopF = 96;                              // log2 F at most
constexpr float kTopW = 0x1p15f;                       // p s_v F at most
constexpr int kAgain = 64;                              // flags of passes to be done again
constexpr float kLazy8 = 8.f;                          // the reference moves when a score passes it by more
constexpr float kBigScale = 0x1p20f;                   // larger scales of values: pass_again
__device__ __forceinline__ float pow2(int e) { return __builtin_amdgcn_ldexpf(1.f, e); }

// The streaming cache policy of a buffer load, for codes that a workgroup reads once: 60000 keys of single tokens, with
// merge and host, 34.6 us, without it 37.3.  Units of 17 to 32 rows read theirs twice, by two waves, and pay 3 to 9%
// (32 drafts of 5 after 1000 keys 29.4 us, without it 26.7), 24 sequences that share all their keys 2%.
constexpr int kOnce = 2;

// ---- sixteen rows of a wave, a tile at a time: each lane its row l % 16 and quarter l / 16
//   S^T[key][row] = K . Q^T: the lane has of key 16 kb + l % 16 codes 32 quarter .. + 31, and gets the scores of the
//     keys 16 kb + 4 quarter + r (kb = 0, 1; r = 0 .. 3) for its row;
//   O^T[d][row] = V^T . P^T over the tile's 32 keys in the order of those scores: the lane has codes
//     8 (l % 16) .. + 7 of its eight keys, put together pair of keys by pair; sum y, register r is
//     d = 32 quarter + 8 r + y.
__device__ __forceinline__ Rsrc codes_rsrc(const uint8_t* codes, size_t row, int there) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(codes) + row * kHeadDim, 0, there * kHeadDim,
                                             kBufferDword3);
}
// `there` keys of the tile whose first head row is `row`
__device__ __forceinline__ void load_tile(const Cache8Args& a, size_t row, int there, Tile8& t) {
    constexpr int D = kHeadDim;
    auto scales_at = [&](const float* scales) {  // (whole tiles: pages hold them)
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(scales) + row, 0, there ? kKT * 4 : 0,
                                                 kBufferDword3);
    };
    const uint32_t ln = lane_now();
    const Rsrc rk = codes_rsrc(a.k8, row, there), rv = codes_rsrc(a.v8, row, there), sk = scales_at(a.ks),
               sv = scales_at(a.vs);
    const uint32_t ok = (ln & 15) * D + (ln >> 4) * 32, ov = (ln >> 4) * (4 * D) + (ln & 15) * 8;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
            t.k[kb][x] = __builtin_amdgcn_raw_buffer_load_b128(rk, ok + 16 * kb * D + 16 * x, 0, kOnce);
        const uint32_t os = (ln >> 4) * 16 + 64 * kb;
        t.ks[kb] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(sk, os, 0, kOnce));
        t.vs[kb] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(sv, os, 0, kOnce));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        t.v[e] = __builtin_amdgcn_raw_buffer_load_b64(rv, ov + (16 * (e >> 2) + (e & 3)) * D, 0, kOnce);
}
// The planes of a row's d = 32 quarter + 8 x + 0 .. 7, from its values and the softmax scale.
struct Query8 {
    u32x4 h[4], l[4];
    float s;  // takes the row's scaling out of its scores
    __device__ __forceinline__ void set(float4 (&q)[8], float sl2) {
        float most = 0.f;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            q[x] = make_float4(q[x].x * sl2, q[x].y * sl2, q[x].z * sl2, q[x].w * sl2);
            most = fmaxf(fmaxf(most, __builtin_fabsf(q[x].x)), __builtin_fabsf(q[x].y));
            most = fmaxf(fmaxf(most, __builtin_fabsf(q[x].z)), __builtin_fabsf(q[x].w));
        }
        most = half_max(fmaxf(most, lane_xor16(most)));
        const uint32_t f = scale_to<14>(most);
        const float fq = __uint_as_float(f);
        s = inverse(f);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const float4 v = q[2 * x + y];
                split_f16(v.x * fq, v.y * fq, hi[2 * y], lo[2 * y]);
                split_f16(v.z * fq, v.w * fq, hi[2 * y + 1], lo[2 * y + 1]);
            }
            h[x] = u32x4{hi[0], hi[1], hi[2], hi[3]};
            l[x] = u32x4{lo[0], lo[1], lo[2], lo[3]};
        }
    }
};
template <bool kInt8>
__device__ __forceinline__ void scores_of(const Tile8& t, const Query8& q, f32x4 (&s)[2]) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        s[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const uint32_t lo = flipped<kInt8>(t.k[kb][x >> 1][2 * (x & 1)]);
            const uint32_t hi = flipped<kInt8>(t.k[kb][x >> 1][2 * (x & 1) + 1]);
            const u32x4 kf = {pair_f16<kInt8, 0>(lo), pair_f16<kInt8, 1>(lo), pair_f16<kInt8, 0>(hi),
                              pair_f16<kInt8, 1>(hi)};
            s[kb] = mfma16(kf, q.l[x], s[kb]);
            s[kb] = mfma16(kf, q.h[x], s[kb]);
        }
    }
}
// (whether a code of V is NaN, and zeros in place of such ones)
__device__ __forceinline__ bool take_nans(Tile8& t) {
    uint32_t nan = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            nan |= nan_bytes(t.v[e][x]);
            t.v[e][x] = without_nan(t.v[e][x]);
        }
    return __builtin_amdgcn_ballot_w64(nan != 0) != 0;
}
struct Planes8 {  // of eight weights
    u32x4 h, l;
    __device__ __forceinline__ explicit Planes8(const float (&w)[8]) {
        uint32_t wh[4], wl[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) split_f16(w[2 * r], w[2 * r + 1], wh[r], wl[r]);
        h = u32x4{wh[0], wh[1], wh[2], wh[3]}, l = u32x4{wl[0], wl[1], wl[2], wl[3]};
    }
};
template <bool kInt8>
__device__ __forceinline__ void add_values(const Tile8& t, const Planes8& p, f32x4 (&o)[8]) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        uint32_t vf[4][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // keys 2e, 2e + 1 of the lane's eight
            const uint32_t u = t.v[2 * e][x], w = t.v[2 * e + 1][x];
            const uint32_t lo = flipped<kInt8>(__builtin_amdgcn_perm(w, u, 0x05010400u));
            const uint32_t hi = flipped<kInt8>(__builtin_amdgcn_perm(w, u, 0x07030602u));
            vf[0][e] = pair_f16<kInt8, 0>(lo), vf[1][e] = pair_f16<kInt8, 1>(lo);
            vf[2][e] = pair_f16<kInt8, 0>(hi), vf[3][e] = pair_f16<kInt8, 1>(hi);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const u32x4 v = {vf[y][0], vf[y][1], vf[y][2], vf[y][3]};
            o[4 * x + y] = mfma16(v, p.l, o[4 * x + y]);
            o[4 * x + y] = mfma16(v, p.h, o[4 * x + y]);
        }
    }
}
// NaN among the codes of a tile of V (rsrc rv) into the sums of rows that see them (`bits`).
__device__ __forceinline__ void put_nans(const Rsrc& rv, uint32_t bits, int quarter, f32x4 (&o)[8]) {
    uint32_t at = 0;  // the lane's columns d = 32 quarter + i that have one, a bit each
#pragma unroll 1
    for (int c = 0; c < kKT; ++c) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rv, c * kHeadDim + 32 * quarter + 16 * x, 0, 0);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const uint32_t nan = bits >> c & 1 ? nan_bytes(v[y]) : 0u;
                const uint32_t four = (nan >> 7 & 1) | (nan >> 14 & 2) | (nan >> 21 & 4) | (nan >> 28 & 8);
                at |= four << (16 * x + 4 * y);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (at >> i & 1) o[i & 7][i >> 3] = __builtin_nanf("");
}

// ---- units of up to 32 rows
// A workgroup's share of the few-row list.  A unit's rows are one block of sixteen or two, one per wave; waves of a
// block take its tiles in turn.
// Bound by reading the codes, two tiles of each wave in flight.  A pass is short where sequences are: the next unit
// and its pages are looked up during a pass, its queries and first tiles fetched before the waves' sums meet.
// H 32 / HKV 8, pages of 64, e4m3: 60000 keys of one sequence (127 MB) 27 us, as 24 of 2500 keys 29.6, as 96 of 625
// 32.4 (one pass after another 34.3 and 41.6); 130000 keys 49 us, 5.6 TB/s, or 6.7 past the 8 us that a call over 31
// keys takes: launch, plan, unit, page and codes one after another.
template <bool kInt8, bool kTree>
__device__ __forceinline__ void few8_walk(const Cache8Args& a, const List& list, int4 sh, int share, int kvh,
                                          FastDiv fG, float sl2, float* parts, float* smem, uint8_t* again) {
    constexpr int D = kHeadDim;
    const int tid = unhoisted(threadIdx.x), lane = tid & 63, wu = scalar(tid >> 6);
    const int j = lane & 15, quarter = lane >> 4;
    const int G = (int)fG.d;
    const int first = scalar(sh.x), first_tile = scalar(sh.y), last = scalar(sh.z), last_tile = scalar(sh.w);
    auto there = [&](int at) { return at < last || (at == last && last_tile > 0); };
    if (!there(first)) return;
    struct Unit8 : Pass {
        int nb, step, off, n_mine;  // blocks of rows; this wave's tiles: from `off` on every `step`-th, n_mine of them
    };
    auto make = [&](int at, u32x4 x, u32x4 y) {
        Unit8 p;
        const int n = (int)x.y, len = (int)x.z, cut = at == last && last_tile > 0 ? last_tile : -1;
        p.row0 = (int)x.x, p.u = (int)x.w, p.seq = (int)y.x;
        p.pos0 = len - n;
        p.nflat = n * G;
        p.T = len;  // (a few-row unit is its sequence's last: its last row sees all)
        p.kt_lo = at == first ? first_tile : 0;
        p.nrange = (cut >= 0 ? cut : (int)y.y) - p.kt_lo;
        const int place = scalar((int)part_at(true, share * a.HKV + kvh, p.kt_lo > 0 ? 0 : 1));
        p.part = p.kt_lo > 0 || cut >= 0 ? parts + place : nullptr;
        p.nb = p.nflat - kUnitRows * p.u > kRow8 ? 2 : 1;
        p.step = kWaves / p.nb, p.off = wu / p.nb;
        p.n_mine = (p.nrange - p.off + p.step - 1) / p.step;
        return p;
    };
    auto index = [&](const Unit8& p, int i) { return p.kt_lo + p.step * i + p.off; };
    auto page = [&](const Unit8& p, int i) { return page_of<true>(a, p, index(p, i) * kKT); };
    struct Place {   // of a tile
        size_t row;  // its first head row
        int there;   // keys of it
    };
    auto place = [&](const Unit8& p, int i, int pg) {
        const int t0 = index(p, i) * kKT;
        const bool ok = i < p.n_mine && pg >= 0 && pg < a.n_blocks;
        return Place{ok ? head_row(pg, a.HKV, kvh, a.bshift, t0) : 0, ok ? min(kKT, p.T - t0) : 0};
    };
    auto load = [&](Tile8& t, const Place& at) { load_tile(a, at.row, at.there, t); };
    // this lane's row of a unit (rows past the last repeat it), and its query, d = 32 quarter .. + 31
    auto row_of = [&](const Unit8& p) {
        return min(kUnitRows * p.u + kRow8 * (wu & (p.nb - 1)) + j, p.nflat - 1);
    };
    float4 q[8];
    auto load_q = [&](const Unit8& p) {
        const int row = row_of(p), tok = fdiv(row, fG);
        const float* src = a.q + ((size_t)p.row0 + tok) * a.q_stride + (size_t)(kvh * G + row - tok * G) * D;
        src += 32 * quarter;
#pragma unroll
        for (int x = 0; x < 8; ++x) q[x] = *reinterpret_cast<const float4*>(src + 4 * x);
    };

    const u32x4* unit = reinterpret_cast<const u32x4*>(&list.shares[share].start);  // a Unit's fields, in order
    Unit8 p = make(first, scalar_load(unit), scalar_load(unit + 1));
    Tile8 t0, t1;
    int pg;  // of tile 2
    auto begin = [&](const Unit8& p, int p0, int p1) {
        load_q(p);
        load(t0, place(p, 0, p0));
        load(t1, place(p, 1, p1));
    };
    begin(p, page(p, 0), page(p, 1));
    pg = page(p, 2);
    for (int at = first, turn = 0;; ++at, ++turn) {
        const bool more = there(at + 1);
        unit = reinterpret_cast<const u32x4*>(more ? list.units + at + 1 : &list.shares[share].start);
        const u32x4 nx = scalar_load(unit), ny = scalar_load(unit + 1);
        const int tok = fdiv(row_of(p), fG), qpos = p.pos0 + tok;
        const int f0 = kUnitRows * p.u, block0 = min(f0 + kRow8 * (wu & (p.nb - 1)), p.nflat - 1);
        const int nfull = max(kTree ? p.pos0 : p.pos0 + fdiv(block0, fG) + 1, 0) / kKT;
        Query8 planes;
        planes.set(q, sl2);
        const float sq = planes.s;
        f32x4 o[8];
        float m = -INFINITY, l = 0.f, limit = 0.f;  // (limit of a row without weights so far)
        int fe = 0;                                 // log2 F
#pragma unroll
        for (int y = 0; y < 8; ++y) o[y] = f32x4{0.f, 0.f, 0.f, 0.f};
        auto scale_sums = [&](float by) {
            l *= by;
#pragma unroll
            for (int y = 0; y < 8; ++y)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[y][r] *= by;
        };
        auto row_max = [&](float x) { return half_max(fmaxf(x, lane_xor16(x))); };

        int nan_tile = p.n_mine;  // the first with a NaN code that not every row sees
        auto tile = [&](Tile8& t, int i) {
            const int kt = index(p, i);
            f32x4 s[2];
            scores_of<kInt8>(t, planes, s);
            uint32_t bits = ~0u;
            if (kt >= nfull) {
                bits = kTree ? tree_bits(a, p, qpos, kt * kKT) : causal_bits(qpos, kt * kKT);
            }
            const uint32_t mine = bits >> (4 * quarter);
            auto seen = [&](int r) { return (mine >> (16 * (r >> 2) + (r & 3)) & 1) != 0; };
            float mx = -INFINITY;
#pragma unroll
            for (int r = 0; r < 8; ++r) s[r >> 2][r & 3] *= t.ks[r >> 2][r & 3];
            if (kt >= nfull) {
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (!seen(r)) s[r >> 2][r & 3] = -INFINITY;
            }
#pragma unroll
            for (int r = 0; r < 8; ++r) mx = fmaxf(mx, s[r >> 2][r & 3]);
            mx = row_max(mx) * sq;
            if (__builtin_amdgcn_ballot_w64(mx > m + kLazy8)) {  // rare after the first tile
                const float mn = fmaxf(m, ceilf(mx));
                const int up = m == -INFINITY || m == mn ? 0 : (int)fminf(mn - m, 1000.f);
                const int fn = min(fe + up, kTopF);  // the sums stay where F can go up by as much
                if (__builtin_amdgcn_ballot_w64(fn - fe != up)) scale_sums(pow2(fn - fe - up));
                fe = fn;
                m = mn;
            }
            float big = 0.f;
#pragma unroll
            for (int r = 0; r < 8; ++r) big = fmaxf(big, __builtin_fabsf(t.vs[r >> 2][r & 3]));
            if (__builtin_amdgcn_ballot_w64(big > kBigScale)) {  // (pages behind the last key may hold anything)
                big = 0.f;
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (seen(r)) big = fmaxf(big, __builtin_fabsf(t.vs[r >> 2][r & 3]));
                if (__builtin_amdgcn_ballot_w64(big > kBigScale)) again[min(turn, kAgain - 1)] = 1;
            }
            const float nb = m == -INFINITY ? 0.f : (float)fe - m;
            float sum = 0.f, wm = 0.f;
            float wt[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r >> 2][r & 3], sq, nb));
                sum += pr;
                wt[r] = pr * t.vs[r >> 2][r & 3];
            }
            l += sum;
            if (kt >= nfull) {  // (a scale that the row does not see may be anything)
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (!seen(r)) wt[r] = 0.f;
            }
#pragma unroll
            for (int r = 0; r < 8; ++r) wm = fmaxf(wm, __builtin_fabsf(wt[r]));
            wm = row_max(wm);
            if (__builtin_amdgcn_ballot_w64(wm > limit)) {  // rare after the first tile
                // the largest: 2^14 .. 2^15
                const bool over = wm > limit;
                const int fn = over ? min(fe + 127 + 14 - (int)min(__float_as_uint(wm) >> 23, 254u), kTopF) : fe;
                const float by = pow2(fn - fe);
                scale_sums(by);
#pragma unroll
                for (int r = 0; r < 8; ++r) wt[r] *= by;
                fe = fn;
                if (over) limit = kTopW;
            }
            const Planes8 w(wt);
            if constexpr (!kInt8) {
                // a NaN that not every row sees must not meet them: put in at the end
                if (kt >= nfull && take_nans(t)) nan_tile = min(nan_tile, i);
            }
            add_values<kInt8>(t, w, o);
        };
        const Unit8 next = more ? make(at + 1, nx, ny) : p;
        int n0 = -1, n1 = -1;  // the next unit's first pages
        for (int i = 0; i < p.n_mine; i += 2) {
            if (i == 0 && more) n0 = page(next, 0), n1 = page(next, 1);
            const int p3 = page(p, i + 3);
            tile(t0, i);
            __builtin_amdgcn_sched_barrier(0);
            if (i + 2 < p.n_mine) load(t0, place(p, i + 2, pg));
            __builtin_amdgcn_sched_barrier(0);
            if (i + 1 < p.n_mine) tile(t1, i + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (i + 3 < p.n_mine) load(t1, place(p, i + 3, p3));
            pg = page(p, i + 4);
            __builtin_amdgcn_sched_barrier(0);
        }
        // F stopped: scales below 2^-82 (or zeros)
        if (__builtin_amdgcn_ballot_w64(fe == kTopF)) again[min(turn, kAgain - 1)] = 1;
        if constexpr (!kInt8) {
#pragma unroll 1
            for (int i = nan_tile; i < p.n_mine; ++i) {
                const int k0 = index(p, i) * kKT;
                const Place at = place(p, i, page(p, i));
                put_nans(codes_rsrc(a.v8, at.row, at.there),
                         kTree ? tree_bits(a, p, qpos, k0) : causal_bits(qpos, k0), quarter, o);
            }
        }
        if (more) {
            if (p.n_mine <= 0) n0 = page(next, 0), n1 = page(next, 1);
            begin(next, n0, n1);
            pg = page(next, 2);
        }
        __builtin_amdgcn_sched_barrier(0);
        // every wave's rows meet, in one of two areas in turn: nobody is further than a pass ahead
        float* const area = smem + (turn & 1) * kFew8F;
        float* const own = area + wu * (kRow8 * kRowF);
        float* const ml = area + kFew8ML;
        {
            const float f = pow2(-fe);
            l *= f;
            if (m == -INFINITY) {  // (scores of -infinity beside infinite values; parts without weights are left out)
                float z = 0.f;
#pragma unroll
                for (int y = 0; y < 8; ++y)
#pragma unroll
                    for (int r = 0; r < 4; ++r) z = __builtin_fmaf(o[y][r], 0.f, z);
                l += z;
            }
            const float sum = half_sum(l + lane_xor16(l));
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int y = 0; y < 8; y += 4)
                    *reinterpret_cast<float4*>(own + j * kRowF + 32 * quarter + 8 * r + y) =
                        make_float4(o[y][r] * f, o[y + 1][r] * f, o[y + 2][r] * f, o[y + 3][r] * f);
            if (quarter == 0) *reinterpret_cast<float2*>(ml + 2 * (wu * kRow8 + j)) = make_float2(m, sum);
        }
        lds_barrier();
        const int rows = p.nflat - f0;
        auto meet = [&](auto blocks) {
            constexpr int kB = decltype(blocks)::value, kW = kWaves / kB;  // waves of a block
            const int d = 4 * (lane & 31);
            for (int i = 2 * wu + (lane >> 5); i < rows; i += 2 * kWaves) {
                const int b = kB == 1 ? 0 : i >> 4, r = i & 15;
                float2 e[kW];
                float4 v[kW];
                float M = -INFINITY, L = 0.f;
#pragma unroll
                for (int w = 0; w < kW; ++w) {
                    e[w] = *reinterpret_cast<const float2*>(ml + 2 * ((kB * w + b) * kRow8 + r));
                    v[w] = *reinterpret_cast<const float4*>(area + ((kB * w + b) * kRow8 + r) * kRowF + d);
                }
#pragma unroll
                for (int w = 0; w < kW; ++w) M = fmaxf(M, e[w].x);
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kW; ++w) {
                    // (a wave whose every score is NaN keeps m at -inf, and its NaN sum counts)
                    const float c = e[w].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(e[w].x - M);
                    L += e[w].x == -INFINITY ? e[w].y : e[w].y * c;
                    x.x = __builtin_fmaf(c, v[w].x, x.x), x.y = __builtin_fmaf(c, v[w].y, x.y);
                    x.z = __builtin_fmaf(c, v[w].z, x.z), x.w = __builtin_fmaf(c, v[w].w, x.w);
                }
                const int g = f0 + i, t = fdiv(g, fG);
                float* dst;
                if (p.part) {
                    dst = p.part + i * D;
                    if (d == 0) *reinterpret_cast<float2*>(p.part + kFewRows * D + 2 * i) = make_float2(M, L);
                } else {
                    dst = a.out + (((size_t)p.row0 + t) * a.H + kvh * G + g - t * G) * D;
                    bool none = p.pos0 + t < 0;  // a row that sees no key: zeros
                    if constexpr (kTree) none = L == 0.f && tree_sees_none(a, p.row0, p.pos0, t);
                    const float inv = none ? 0.f : 1.f / L;
                    x.x *= inv, x.y *= inv, x.z *= inv, x.w *= inv;
                }
                *reinterpret_cast<float4*>(dst + d) = x;
            }
        };
        if (p.nb == 1) meet(std::integral_constant<int, 1>{});
        else meet(std::integral_constant<int, 2>{});
        if (!more) break;
        p = next;
    }
}

// ---- a wide unit: up to 128 rows
// Groups of kS waves (four of 32 rows each, or two where the unit has no more than 64 rows) share a tile, the groups
// take the unit's tiles in turn.  Each wave turns its part of a tile's codes into binary16 in LDS, V transposed, four
// tiles of a group at a time there (or two), one barrier for half of them.  On v_mfma_f32_32x32x16_f16
// S^T[key][row] = K . Q^T gives a lane 16 of a tile's 32 keys for one row, which are the operand of
// O^T[d][row] = V^T . P^T.
//
// Matrix and vector instructions of one wave overlap where neither waits for the other: the next tile's scores are
// taken between the instructions of this one's softmax, and the next tiles' conversions and the second half of the
// weights' planes between those of P . V, by hand, since the compiler would put each kind together (and every LDS
// read right before its use).
//
// Bound by the matrix unit and its power: 1024 rows after 12000 keys (H 32 / HKV 8, int8) 407 to 465 us by box, 455 to
// 517 TFLOP/s, 0.9 to 1.0 PFLOP/s over the two plane products, 75 to 85% of what a large fp16 product reaches; the
// matrix unit is busy 48% of the cycles at 2.0 GHz of 2.4, vector instructions 54%, beside each other.  Where it takes
// 407 us: with the softmax between the products instead of among them 464, a barrier for every tile and lanes'
// addresses made anew 456.  Units of 33 to 64 rows in two groups of four waves, half of them idle: 16 trees of 48
// tokens (G 4, 192 rows: units of 128 and 64, e4m3) 188 us against 144.
constexpr int kK8RowB = 2 * kHeadDim + 16, kK8Tile = kKT * kK8RowB;  // [32 keys][128 d], rows spread over banks
constexpr int kV8RowB = 2 * kKT + 16, kV8Tile = kHeadDim * kV8RowB;  // [128 d][32 keys]
constexpr int kScales8 = 2 * kKT * 4;                                // of K, of V
constexpr int kBuf8 = kK8Tile + kV8Tile + kScales8;                  // one tile of a group
static_assert(kBuf8 % 16 == 0, "16-byte pieces");
template <int kS>
struct Wide8 {
    static constexpr int kN = kWaves / kS, kOwn = 4 / kN;  // groups, blocks of 32 d that a group finishes
    static constexpr int kRing = kS == 4 ? 4 : 2;          // tiles of a group in LDS, a barrier every kRing / 2
    // LDS, in floats: the tiles; after them the merge's exchange (m, l and the sums given away), and the rows
    static constexpr int kTilesF = kN * kRing * kBuf8 / 4;
    static constexpr int kXch = 2 + 16 * (4 - kOwn);
    static constexpr int kStage = kWaves * kXch * 64;
    static constexpr int kEnd = kStage + kS * kQB * kRowF;
    static constexpr int kF = kEnd > kTilesF ? kEnd : kTilesF;
};
constexpr int kNanAt8 = Wide8<4>::kF > Wide8<2>::kF ? Wide8<4>::kF : Wide8<2>::kF;  // a word: NaN codes were met
// Flags of passes to be done again, a byte each: 64 of the wide ones, 64 of the few-row ones (one from the 64th on).
constexpr int kAgainAt8 = kNanAt8 + 4;
constexpr int kLds8 = 4 * kAgainAt8 + 2 * kAgain;
static_assert(kLds8 <= 160 * 1024 && 2 * kFew8F <= kNanAt8, "LDS budget");
__device__ __forceinline__ floatx16 mfma32(u32x4 a, u32x4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

template <bool kInt8, bool kTree, int kS>
__device__ __forceinline__ void wide8_pass(const Cache8Args& a, const Pass& p, int kvh, FastDiv fG, float sl2,
                                           float* smem, uint8_t* again) {
    constexpr int D = kHeadDim, kN = Wide8<kS>::kN, kParts = 4 / kS;  // (of a tile, each 8 rows of K and 32 d of V)
    constexpr int kRing = Wide8<kS>::kRing, kLead = kRing / 2;
    const int tid = unhoisted(threadIdx.x), lane = tid & 63, w = tid >> 6;
    const int wu = scalar(w), hw = wu % kS, grp = wu / kS;
    const int col = lane & 31, hh = lane >> 5;
    const int G = (int)fG.d;
    char* const lds = reinterpret_cast<char*>(smem) + grp * (kRing * kBuf8);
    const int f0 = kUnitRows * p.u + kQB * hw;  // this wave's first row
    const int row = min(f0 + col, p.nflat - 1), tok = fdiv(row, fG);  // (rows past the last repeat it)
    const int qpos = p.pos0 + tok;
    const int nfull = max(kTree ? p.pos0 : p.pos0 + fdiv(min(f0, p.nflat - 1), fG) + 1, 0) / kKT;
    const int n_it = (p.nrange + kN - 1) / kN, n_mine = (p.nrange - grp + kN - 1) / kN;
    auto index = [&](int i) { return p.kt_lo + kN * i + grp; };
    auto page = [&](int i) { return page_of<true>(a, p, index(i) * kKT); };
    struct Place {   // of a tile
        size_t row;  // its first head row
        int there;   // keys of it
    };
    auto place = [&](int i, int pg) {
        const int t0 = index(i) * kKT;
        const bool ok = i < n_mine && pg >= 0 && pg < a.n_blocks;
        return Place{ok ? head_row(pg, a.HKV, kvh, a.bshift, t0) : 0, ok ? min(kKT, p.T - t0) : 0};
    };
    auto codes_at = [&](const uint8_t* codes, const Place& at) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(codes) + at.row * D, 0, at.there * D,
                                                 kBufferDword3);
    };
    // this wave's parts x of a tile, y = kParts hw + x:
    //   K: codes 16 (lane % 8) .. + 15 of row 8 y + lane / 8
    //   V: codes 32 y + 4 (lane % 8) .. + 3 of the four rows from 4 (lane / 8) on
    // and the scales, of K by the even waves, of V by the odd ones
    u32x4 tk[kParts];
    uint32_t tv[kParts][4];
    float ts;
    const uint32_t from_k = (8 * kParts * hw + (lane >> 3)) * D + 16 * (lane & 7);
    const uint32_t from_v = 4 * (lane >> 3) * D + 32 * kParts * hw + 4 * (lane & 7);
    auto load_k = [&](const Place& at) {
        const Rsrc rs = codes_at(a.k8, at);
#pragma unroll
        for (int x = 0; x < kParts; ++x)
            tk[x] = __builtin_amdgcn_raw_buffer_load_b128(rs, from_k + 8 * x * D, 0, 0);
    };
    auto load_v = [&](const Place& at) {
        const Rsrc rs = codes_at(a.v8, at);
#pragma unroll
        for (int x = 0; x < kParts; ++x)
#pragma unroll
            for (int y = 0; y < 4; ++y)
                tv[x][y] = __builtin_amdgcn_raw_buffer_load_b32(rs, from_v + 32 * x + y * D, 0, 0);
    };
    auto load_scales = [&](const Place& at) {
        const Rsrc rs = __builtin_amdgcn_make_buffer_rsrc((hw & 1 ? a.vs : a.ks) + at.row, 0, at.there * 4,
                                                          kBufferDword3);
        ts = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, 4 * (lane & 31), 0, 0));
    };
    auto buf = [&](int i) { return lds + (i & (kRing - 1)) * kBuf8; };
    // halves of 16 bytes of K's part x
    const uint32_t to_k = (8 * kParts * hw + (lane >> 3)) * kK8RowB + 32 * (lane & 7);
    auto store_k = [&](int i, int x, int half) {
        const uint32_t lo = flipped<kInt8>(tk[x][2 * half]), hi = flipped<kInt8>(tk[x][2 * half + 1]);
        *reinterpret_cast<u32x4*>(buf(i) + to_k + 8 * x * kK8RowB + 16 * half) =
            u32x4{pair_f16<kInt8, 0>(lo), pair_f16<kInt8, 1>(lo), pair_f16<kInt8, 0>(hi), pair_f16<kInt8, 1>(hi)};
    };
    // V transposed, codes 2y and 2y + 1 of part x: the keys of P . V's operand, half hh of step z, are
    // 16z + 4hh + {0 .. 3, 8 .. 11}
    const uint32_t to_v = kK8Tile + (32 * kParts * hw + 4 * (lane & 7)) * kV8RowB + 32 * (lane >> 5) +
                          16 * ((lane >> 3) & 1) + 8 * ((lane >> 4) & 1);
    auto store_v = [&](int i, int x, int y) {
        char* d = buf(i) + to_v + (32 * x + 2 * y) * kV8RowB;
        const uint32_t pick = y ? 0x07030602u : 0x05010400u;
        const uint32_t lo = flipped<kInt8>(__builtin_amdgcn_perm(tv[x][1], tv[x][0], pick));
        const uint32_t hi = flipped<kInt8>(__builtin_amdgcn_perm(tv[x][3], tv[x][2], pick));
        *reinterpret_cast<u32x2*>(d) = u32x2{pair_f16<kInt8, 0>(lo), pair_f16<kInt8, 0>(hi)};
        *reinterpret_cast<u32x2*>(d + kV8RowB) = u32x2{pair_f16<kInt8, 1>(lo), pair_f16<kInt8, 1>(hi)};
    };
    // (both halves of the wave write the same.  A big scale of V, whichever rows see it, takes the pass to pass_again:
    // F lowered for it would cost the rows that do not see it their bits)
    const uint32_t to_scales = kK8Tile + kV8Tile + 4 * kKT * (hw & 1) + 4 * col;
    auto store_scales = [&](int i) {
        if ((hw & 1) && __builtin_amdgcn_ballot_w64(__builtin_fabsf(ts) > kBigScale)) *again = 1;
        *reinterpret_cast<float*>(buf(i) + to_scales) = ts;
    };
    auto store_all_k = [&](int i) {
#pragma unroll
        for (int x = 0; x < kParts; ++x) store_k(i, x, 0), store_k(i, x, 1);
    };
    auto store_all_v = [&](int i) {
#pragma unroll
        for (int x = 0; x < kParts; ++x) store_v(i, x, 0), store_v(i, x, 1);
        store_scales(i);
    };
    {
        const Place first = place(0, page(0));
        load_k(first);
        load_v(first);
        load_scales(first);
    }
    int* const nan_met = reinterpret_cast<int*>(smem + kNanAt8);
    if constexpr (!kInt8)
        if (tid == 0) *nan_met = 0;

    // q: planes of d = 16 t + 8 hh + 0 .. 7
    u32x4 qh[8], ql[8];
    float sq;  // takes the row's scaling out of its scores
    {
        const float* src = a.q + ((size_t)p.row0 + tok) * a.q_stride + (size_t)(kvh * G + row - tok * G) * D + 8 * hh;
        float most = 0.f;
        float4 q[16];
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            const float4 v = *reinterpret_cast<const float4*>(src + 16 * (t >> 1) + 4 * (t & 1));
            q[t] = make_float4(v.x * sl2, v.y * sl2, v.z * sl2, v.w * sl2);
            most = fmaxf(fmaxf(most, __builtin_fabsf(q[t].x)), __builtin_fabsf(q[t].y));
            most = fmaxf(fmaxf(most, __builtin_fabsf(q[t].z)), __builtin_fabsf(q[t].w));
        }
        most = half_max(most);
        const uint32_t f = scale_to<14>(most);
        const float fq = __uint_as_float(f);
        sq = inverse(f);
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            uint32_t h[4], l[4];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const float4 v = q[2 * t + y];
                split_f16(v.x * fq, v.y * fq, h[2 * y], l[2 * y]);
                split_f16(v.z * fq, v.w * fq, h[2 * y + 1], l[2 * y + 1]);
            }
            qh[t] = u32x4{h[0], h[1], h[2], h[3]};
            ql[t] = u32x4{l[0], l[1], l[2], l[3]};
        }
    }
    floatx16 o[4], even, odd;  // (scores of tiles 2i, 2i + 1)
    float m = -INFINITY, l = 0.f, limit = 0.f;  // (limit of a row without weights so far)
    int fe = 0;                                 // log2 F
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
    auto scale_sums = [&](float by) {
        l *= by;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[db][r] *= by;
    };
    auto fence = [] { __builtin_amdgcn_sched_barrier(0); };

    // While tile i is worked on, V and scales of tile i + kLead and K of the one after it go to LDS, where tiles of
    // kRing before were: every wave was done with those at the last barrier, and will not need these before the next.
    store_all_k(0);
    store_all_v(0);
    Place at{};
#pragma unroll
    for (int i = 1; i <= kLead; ++i) {
        at = place(i, page(i));
        load_k(at);
        if (i < kLead) {
            load_v(at);
            load_scales(at);
            store_all_v(i);
        }
        store_all_k(i);
    }
    load_v(at);  // of kLead
    load_scales(at);
    at = place(kLead + 1, page(kLead + 1));
    load_k(at);
    int pg = page(kLead + 2);
    lds_barrier();
    u32x4 kf[3];
    auto read_k = [&](int i, int t) {
        kf[t % 3] = *reinterpret_cast<const u32x4*>(buf(i) + col * kK8RowB + 16 * hh + 32 * t);
    };
    auto score_l = [&](floatx16& next, int t) {
        if (t == 0) {
            floatx16 zero;
#pragma unroll
            for (int r = 0; r < 16; ++r) zero[r] = 0.f;
            next = mfma32(kf[t % 3], ql[t], zero);
        } else next = mfma32(kf[t % 3], ql[t], next);
    };
    auto score_h = [&](floatx16& next, int t) { next = mfma32(kf[t % 3], qh[t], next); };
    read_k(0, 0), read_k(0, 1);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        if (t + 2 < 8) read_k(0, t + 2);
        fence();
        score_l(even, t), score_h(even, t);
    }
    lds_barrier();  // (K of tile 0 has been read)
    auto tile = [&](int i, floatx16& s, floatx16& next) {
        const Place ahead = place(i + kLead + 2, pg);
        pg = page(i + kLead + 3);
        const int kt = index(i);
        const float* sc = reinterpret_cast<const float*>(buf(i) + kK8Tile + kV8Tile) + 4 * hh;
        // ---- scores times scales, while the next tile's are taken
        f32x4 f[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) f[c] = *reinterpret_cast<const f32x4*>(sc + 8 * c);
        read_k(i + 1, 0), read_k(i + 1, 1);
        fence();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[4 * c + r] *= f[c][r];
            if (c == 0) read_k(i + 1, 2);
            if (c == 1) score_l(next, 0);
            if (c == 3) score_h(next, 0);
            fence();
        }
        uint32_t bits = ~0u;
        if (kt >= nfull) {
            bits = kTree ? tree_bits(a, p, qpos, kt * kKT) : causal_bits(qpos, kt * kKT);
            const uint32_t mine = bits >> (4 * hh);
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (!(mine >> (8 * (r >> 2) + (r & 3)) & 1)) s[r] = -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        read_k(i + 1, 3);
        score_l(next, 1);
        fence();
        mx = half_max(mx) * sq;
        score_h(next, 1);
        fence();
        if (__builtin_amdgcn_ballot_w64(mx > m + kLazy8)) {  // rare after the first tile
            const float mn = fmaxf(m, ceilf(mx));
            const int up = m == -INFINITY || m == mn ? 0 : (int)fminf(mn - m, 1000.f);
            const int fn = min(fe + up, kTopF);  // the sums stay where F can go up by as much
            if (__builtin_amdgcn_ballot_w64(fn - fe != up)) scale_sums(pow2(fn - fe - up));
            fe = fn;
            m = mn;
        }
        // ---- weights times scales times F
        const float nb = m == -INFINITY ? 0.f : (float)fe - m;
        float sum = 0.f, wm = 0.f;
        f[0] = *reinterpret_cast<const f32x4*>(sc + kKT);
        fence();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (c < 3) f[(c + 1) & 3] = *reinterpret_cast<const f32x4*>(sc + kKT + 8 * (c + 1));
            read_k(i + 1, c + 4);
            score_l(next, c + 2);
#pragma unroll
            for (int r = 0; r < 4; ++r) s[4 * c + r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * c + r], sq, nb));
            fence();
            score_h(next, c + 2);
#pragma unroll
            for (int r = 0; r < 4; ++r) sum += s[4 * c + r];
#pragma unroll
            for (int r = 0; r < 4; ++r) s[4 * c + r] *= f[c][r];
            fence();
        }
        l += sum;
        if (kt >= nfull) {  // (a scale that the row does not see may be anything)
            const uint32_t mine = bits >> (4 * hh);
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (!(mine >> (8 * (r >> 2) + (r & 3)) & 1)) s[r] = 0.f;
        }
        score_l(next, 6);
#pragma unroll
        for (int r = 0; r < 16; ++r) wm = fmaxf(wm, __builtin_fabsf(s[r]));
        fence();
        score_h(next, 6);
        wm = half_max(wm);
        fence();
        score_l(next, 7);
        if (__builtin_amdgcn_ballot_w64(wm > limit)) {  // rare after the first tile
            // the largest: 2^14 .. 2^15
            const bool over = wm > limit;
            const int fn = over ? min(fe + 127 + 14 - (int)min(__float_as_uint(wm) >> 23, 254u), kTopF) : fe;
            const float by = pow2(fn - fe);
            scale_sums(by);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= by;
            fe = fn;
            if (over) limit = kTopW;
        }
        // ---- O^T += V^T . P^T
        char* const v = buf(i) + kK8Tile + col * kV8RowB + 16 * hh;
        auto place_of = [&](int y) { return reinterpret_cast<u32x4*>(v + 32 * (y & 3) * kV8RowB + 32 * (y >> 2)); };
        if constexpr (!kInt8) {
            // A NaN that not every row sees must not meet them: zero takes its place for every wave of the group, and
            // it is put in at the end.  (Of the codes' values only NaN has all exponent bits.)
            if (kt >= nfull) {
#pragma unroll
                for (int y = 0; y < 8; ++y) {
                    u32x4 x = *place_of(y);
                    uint32_t nan = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t n = ((x[j] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
                        x[j] &= ~(n | (n - (n >> 15)));
                        nan |= n;
                    }
                    if (__builtin_amdgcn_ballot_w64(nan != 0)) {
                        *place_of(y) = x;
                        *nan_met = 1;
                    }
                    fence();
                }
            }
        }
        u32x4 vf[3], ph[2], pl[2];
        auto planes = [&](int x, int j) {  // weights 8x + 2j and the next
            uint32_t hi, lo;
            split_f16(s[8 * x + 2 * j], s[8 * x + 2 * j + 1], hi, lo);
            ph[x][j] = hi, pl[x][j] = lo;
        };
        vf[0] = *place_of(0), vf[1] = *place_of(1);
        score_h(next, 7);
        fence();
#pragma unroll
        for (int j = 0; j < 4; ++j) planes(0, j);
        fence();
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            if (y + 2 < 8) vf[(y + 2) % 3] = *place_of(y + 2);
            o[y & 3] = mfma32(vf[y % 3], pl[y >> 2], o[y & 3]);
            if (y < 2) planes(1, 2 * y);
            else if (y < 4) {
#pragma unroll
                for (int x = 0; x < kParts; ++x) store_k(i + kLead + 1, x, y - 2);
            } else if (y < 6) {
#pragma unroll
                for (int x = 0; x < kParts; ++x) store_v(i + kLead, x, y - 4);
            } else if (y == 6) load_k(ahead);
            fence();
            o[y & 3] = mfma32(vf[y % 3], ph[y >> 2], o[y & 3]);
            if (y < 2) planes(1, 2 * y + 1);
            if (y == 5) store_scales(i + kLead);
            if (y == 6) load_v(at);
            if (y == 7) load_scales(at);
            fence();
        }
        at = ahead;
    };
    for (int i = 0; i < n_it; i += 2) {
        if (i < n_mine) tile(i, even, odd);
        if constexpr (kLead == 1) lds_barrier();
        if (i + 1 < n_mine) tile(i + 1, odd, even);
        lds_barrier();
    }
    if (__builtin_amdgcn_ballot_w64(fe == kTopF)) *again = 1;  // F stopped: scales below 2^-82 (or zeros)
    if constexpr (!kInt8) {
        if (scalar(*nan_met)) {
            // the group's tiles that not every row of the unit sees all of
            const int low = max(kTree ? p.pos0 : p.pos0 + fdiv(min(kUnitRows * p.u, p.nflat - 1), fG) + 1, 0) / kKT;
#pragma unroll 1
            for (int i = 0; i < n_mine; ++i) {
                const int t0 = index(i) * kKT;
                if (index(i) < low) continue;
                const uint32_t bits = kTree ? tree_bits(a, p, qpos, t0) : causal_bits(qpos, t0);
                const Rsrc rv = codes_at(a.v8, place(i, page(i)));
#pragma unroll 1
                for (int c = 0; c < kKT; ++c)
#pragma unroll
                    for (int db = 0; db < 4; ++db)
#pragma unroll
                        for (int y = 0; y < 4; ++y) {  // d = 32 db + 8y + 4hh + 0 .. 3
                            const uint32_t x =
                                __builtin_amdgcn_raw_buffer_load_b32(rv, c * D + 32 * db + 8 * y + 4 * hh, 0, 0);
                            const uint32_t nan = bits >> c & 1 ? nan_bytes(x) : 0u;
#pragma unroll
                            for (int z = 0; z < 4; ++z)
                                if (nan >> (8 * z) & 0x80) o[db][4 * y + z] = __builtin_nanf("");
                        }
            }
        }
        lds_barrier();  // (the next pass clears the word)
    }

    // ---- the groups meet through LDS: group g finishes the blocks of 32 d from kOwn g on
    scale_sums(pow2(-fe));
    if (m == -INFINITY) {  // (scores of -infinity beside infinite values; parts without weights are left out)
        float z = 0.f;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) z = __builtin_fmaf(o[db][r], 0.f, z);
        l += z;
    }
    constexpr int kOwn = Wide8<kS>::kOwn, kXch = Wide8<kS>::kXch;
    float* xw = smem + w * (kXch * 64) + lane;
    xw[0] = m;
    xw[64] = l;
    floatx16 keep[kOwn];
#pragma unroll
    for (int db = 0; db < 4; ++db) {
        if (db / kOwn != grp) {
            float* to = xw + (2 + 16 * (db < grp * kOwn ? db : db - kOwn)) * 64;
#pragma unroll
            for (int i = 0; i < 16; ++i) to[64 * i] = o[db][i];
        } else keep[db % kOwn] = o[db];
    }
    lds_barrier();
    float mt = m;
    auto of = [&](int g) { return smem + (g * kS + hw) * (kXch * 64) + lane; };
#pragma unroll
    for (int g = 0; g < kN; ++g) mt = fmaxf(mt, of(g)[0]);
    // (a group whose every score is NaN keeps m at -inf, and its NaN sum counts)
    auto factor = [&](float at) { return at == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(at - mt); };
    const float own = factor(m);
    float ls = m == -INFINITY ? l : l * own;
#pragma unroll
    for (int x = 0; x < kOwn; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) keep[x][r] *= own;
#pragma unroll
    for (int other = 1; other < kN; ++other) {
        const int g = (grp + other) % kN;
        const float* xp = of(g);
        const float mg = xp[0], lg = xp[64], c = factor(mg);
        ls += mg == -INFINITY ? lg : lg * c;
#pragma unroll
        for (int x = 0; x < kOwn; ++x) {
            const int db = grp * kOwn + x;
            const float* from = xp + (2 + 16 * (db < g * kOwn ? db : db - kOwn)) * 64;
#pragma unroll
            for (int r = 0; r < 16; ++r) keep[x][r] = __builtin_fmaf(from[64 * r], c, keep[x][r]);
        }
    }
    ls = half_sum(ls);
    float* const stage = smem + Wide8<kS>::kStage;
    {
        bool none = qpos < 0;  // a row that sees no key: zeros
        if constexpr (kTree) none = ls == 0.f && tree_sees_none(a, p.row0, p.pos0, tok);
        const float inv = p.part ? 1.f : none ? 0.f : 1.f / ls;
        float* ost = stage + (hw * kQB + col) * kRowF + 32 * kOwn * grp + 4 * hh;
#pragma unroll
        for (int x = 0; x < kOwn; ++x)
#pragma unroll
            for (int r = 0; r < 16; r += 4)  // registers r .. r + 3 of a block are d = 8 (r / 4) + 4hh + 0 .. 3 of it
                *reinterpret_cast<float4*>(ost + 32 * x + 2 * r) =
                    make_float4(keep[x][r] * inv, keep[x][r + 1] * inv, keep[x][r + 2] * inv, keep[x][r + 3] * inv);
        if (p.part && hh == 0 && grp == 0)
            *reinterpret_cast<float2*>(p.part + kUnitRows * D + 2 * (hw * kQB + col)) = make_float2(mt, ls);
    }
    lds_barrier();
    {
        const int ln = unhoisted(lane), c4 = 4 * (ln & 31);
#pragma unroll
        for (int j = 0; j < kS * kQB / (2 * kWaves); ++j) {  // two rows per instruction
            const int jj = 2 * (wu + kWaves * j) + (ln >> 5), g = kUnitRows * p.u + jj;
            const float4 v = *reinterpret_cast<const float4*>(stage + jj * kRowF + c4);
            const int t = fdiv(g, fG);
            float* dst = p.part ? p.part + jj * D : a.out + (((size_t)p.row0 + t) * a.H + kvh * G + g - t * G) * D;
            if (g < p.nflat) *reinterpret_cast<float4*>(dst + c4) = v;
        }
    }
}

// ---- sixteen rows with two references
// Where F could not serve, a pass is done again when the workgroup is through with the others: sixteen rows for each
// wave, which takes all tiles, with two references, both whole numbers: m of the weights' sum, and u of the products'
// sums, the largest log2 of a weight times its value's scale, rounded up.  The operand is (the scale's fraction)
// 2^(s + its exponent - u + 15), so that no scale overflows or underflows, whatever stands beside it; a key that the
// row does not see is in neither.  The row's largest operand lies between 2^13 and 2^15.  One tile after the other,
// nothing in flight: three to five times slower (24 tokens over 60251 keys 147 us instead of 36, 1024 rows after 12000
// keys 1436 instead of 465).
template <bool kInt8, bool kTree, bool kFew>
__device__ __forceinline__ void pass_again(const Cache8Args& a, const Pass& p, int kvh, FastDiv fG, float sl2) {
    constexpr int D = kHeadDim;
    const int tid = unhoisted(threadIdx.x), lane = tid & 63, j = lane & 15, quarter = lane >> 4, G = (int)fG.d;
    const int i0 = kRow8 * scalar(tid >> 6), f0 = kUnitRows * p.u + i0;
    if (f0 >= p.nflat) return;  // wave-uniform, no barrier here
    const int row = min(f0 + j, p.nflat - 1), tok = fdiv(row, fG), qpos = p.pos0 + tok, end = p.kt_lo + p.nrange;
    Query8 planes;
    {
        const float* src = a.q + ((size_t)p.row0 + tok) * a.q_stride + (size_t)(kvh * G + row - tok * G) * D;
        float4 q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = *reinterpret_cast<const float4*>(src + 32 * quarter + 4 * i);
        planes.set(q, sl2);
    }
    auto row_max = [&](float y) { return half_max(fmaxf(y, lane_xor16(y))); };
    f32x4 o[8];
    float m = -INFINITY, l = 0.f, u = -INFINITY;
#pragma unroll
    for (int y = 0; y < 8; ++y) o[y] = f32x4{0.f, 0.f, 0.f, 0.f};
    struct Place {
        size_t row;
        int there;
    };
    auto place = [&](int kt) {
        const int pg = page_of<true>(a, p, kt * kKT);
        const bool ok = pg >= 0 && pg < a.n_blocks;
        return Place{ok ? head_row(pg, a.HKV, kvh, a.bshift, kt * kKT) : 0, ok ? min(kKT, p.T - kt * kKT) : 0};
    };
    auto visible = [&](int kt) { return kTree ? tree_bits(a, p, qpos, kt * kKT) : causal_bits(qpos, kt * kKT); };
#pragma unroll 1
    for (int kt = p.kt_lo; kt < end; ++kt) {
        const Place at = place(kt);
        Tile8 t;
        load_tile(a, at.row, at.there, t);
        const uint32_t bits = visible(kt), mine = bits >> (4 * quarter);
        f32x4 s[2];
        scores_of<kInt8>(t, planes, s);
        float score[8], scale[8], ms = -INFINITY, us = -INFINITY;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const bool seen = (mine >> (16 * (r >> 2) + (r & 3)) & 1) != 0;
            score[r] = seen ? s[r >> 2][r & 3] * t.ks[r >> 2][r & 3] * planes.s : -INFINITY;
            scale[r] = seen ? t.vs[r >> 2][r & 3] : 0.f;
            ms = fmaxf(ms, score[r]);
            if (scale[r] != 0.f) us = fmaxf(us, score[r] + (float)__builtin_amdgcn_frexp_expf(scale[r]));
        }
        const float mn = fmaxf(m, ceilf(row_max(ms))), un = fmaxf(u, ceilf(row_max(us)));
        l *= m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        const float by = u == un ? 1.f : __builtin_amdgcn_exp2f(u - un);
#pragma unroll
        for (int y = 0; y < 8; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[y][r] *= by;
        m = mn, u = un;
        float w[8], sum = 0.f;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const float e = (float)(15 + __builtin_amdgcn_frexp_expf(scale[r]));
            sum += __builtin_amdgcn_exp2f(mn == -INFINITY ? score[r] : score[r] - mn);
            const float y = __builtin_amdgcn_frexp_mantf(scale[r]) *
                            __builtin_amdgcn_exp2f(score[r] + (un == -INFINITY ? e : e - un));
            w[r] = scale[r] == 0.f ? 0.f : y;  // (its score has not met u, and may be far above)
        }
        l += sum;
        if constexpr (kInt8) {
            add_values<kInt8>(t, Planes8(w), o);
        } else {
            const bool nans = take_nans(t);
            add_values<kInt8>(t, Planes8(w), o);
            if (nans) put_nans(codes_rsrc(a.v8, at.row, at.there), bits, quarter, o);
        }
    }
    // The weights' sum goes to 1/2 .. 1 (to 2^-17 where values may be near fp32's largest: parts are added), the sums
    // of products with it.
    const float sum = half_sum(l + lane_xor16(l)), up = fminf(fmaxf(u - m, -400.f), 400.f);
    const int down = __builtin_amdgcn_frexp_expf(sum) + (up > 64.f ? 16 : 0);
    l = __builtin_amdgcn_ldexpf(l, -down);
    m += (float)down;
#pragma unroll
    for (int y = 0; y < 8; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[y][r] = __builtin_amdgcn_ldexpf(o[y][r], (int)up - 15 - down);
    if (m == -INFINITY) {  // (scores of -infinity beside infinite values; parts without weights are left out)
        float z = 0.f;
#pragma unroll
        for (int y = 0; y < 8; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r) z = __builtin_fmaf(o[y][r], 0.f, z);
        l += z;
    }
    const float all = half_sum(l + lane_xor16(l));
    bool none = qpos < 0;  // a row that sees no key: zeros
    if constexpr (kTree) none = all == 0.f && tree_sees_none(a, p.row0, p.pos0, tok);
    const float inv = p.part ? 1.f : none ? 0.f : 1.f / all;
    float* dst = p.part ? p.part + (i0 + j) * D : a.out + (((size_t)p.row0 + tok) * a.H + kvh * G + row - tok * G) * D;
    if (f0 + j < p.nflat) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int y = 0; y < 8; y += 4)
                *reinterpret_cast<float4*>(dst + 32 * quarter + 8 * r + y) =
                    make_float4(o[y][r] * inv, o[y + 1][r] * inv, o[y + 2][r] * inv, o[y + 3][r] * inv);
        if (p.part && quarter == 0)
            *reinterpret_cast<float2*>(p.part + (kFew ? kFewRows : kUnitRows) * D + 2 * (i0 + j)) = make_float2(m, all);
    }
}

// The flagged passes of a workgroup's share.  (Not inlined: the registers of the passes before are short.)
template <bool kInt8, bool kTree>
__device__ __forceinline__ void share_again(Cache8Args a, int shares, int share, int kvh, uint64_t wides,
                                                      uint64_t fews, float* wide_parts, float* few_parts) {
    __syncthreads();  // (with the workgroup's writes done: what is written now comes after them)
    const PlanView pv = plan_view(const_cast<char*>(a.plan), a.n_seq, a.rows, a.H / a.HKV, shares);
    const FastDiv fG = fast_div((uint32_t)(a.H / a.HKV));
    const float sl2 = a.scale * 1.44269504088896340736f;
    int n = 0;
    walk_share<false>(a, pv.wide, *reinterpret_cast<const int4*>(pv.wide.shares + share),
                      scalar(reinterpret_cast<const int*>(a.plan)[kHeadRounds]), shares, share, kvh, fG, wide_parts,
                      [&](const Pass& p) {
                          if (wides >> min(n++, kAgain - 1) & 1) pass_again<kInt8, kTree, false>(a, p, kvh, fG, sl2);
                      });
    n = 0;
    walk_share<true>(a, pv.few, *reinterpret_cast<const int4*>(pv.few.shares + share), 0, shares, share, kvh, fG,
                     few_parts, [&](const Pass& p) {
                         if (fews >> min(n++, kAgain - 1) & 1) pass_again<kInt8, kTree, true>(a, p, kvh, fG, sl2);
                     });
}

// grid shares x KV heads, as k_packed_attn
template <bool kInt8, bool kTree>
__global__ __launch_bounds__(64 * kWaves) void k_cache8_attn(Cache8Args a, int shares, float* __restrict__ wide_parts,
                                                             float* __restrict__ few_parts) {
    extern __shared__ __align__(16) float smem[];
    const int kvh = blockIdx.x % a.HKV, share = blockIdx.x / a.HKV;
    const PlanView pv = plan_view(const_cast<char*>(a.plan), a.n_seq, a.rows, a.H / a.HKV, shares);
    const int rounds = scalar(reinterpret_cast<const int*>(a.plan)[kHeadRounds]);
    const int4 wide = *reinterpret_cast<const int4*>(pv.wide.shares + share);
    const int4 few = *reinterpret_cast<const int4*>(pv.few.shares + share);
    if (!plan_fits(a.plan, a.n_seq, a.rows, a.H, a.HKV, false)) return;
    const FastDiv fG = fast_div((uint32_t)(a.H / a.HKV));
    const float sl2 = a.scale * 1.44269504088896340736f;  // scores come out in log2 units
    uint8_t* const again = reinterpret_cast<uint8_t*>(smem + kAgainAt8);
    if (threadIdx.x < 2 * kAgain) again[threadIdx.x] = 0;
    int n = 0;
    walk_share<false>(a, pv.wide, wide, rounds, shares, share, kvh, fG, wide_parts, [&](const Pass& p) {
        if (n == 0) lds_barrier();  // the flags are clear before a wave sets one
        uint8_t* const flag = again + min(n++, kAgain - 1);
        if (p.nflat - kUnitRows * p.u > 2 * kQB) wide8_pass<kInt8, kTree, 4>(a, p, kvh, fG, sl2, smem, flag);
        else wide8_pass<kInt8, kTree, 2>(a, p, kvh, fG, sl2, smem, flag);
    });
    lds_barrier();  // the last wide pass's rows have been read
    few8_walk<kInt8, kTree>(a, pv.few, few, share, kvh, fG, sl2, few_parts, smem, again + kAgain);
    lds_barrier();
    const int lane = threadIdx.x & 63;
    const uint64_t wides = __builtin_amdgcn_ballot_w64(again[lane] != 0);
    const uint64_t fews = __builtin_amdgcn_ballot_w64(again[kAgain + lane] != 0);
    if (wides | fews) share_again<kInt8, kTree>(a, shares, share, kvh, wides, fews, wide_parts, few_parts);
}

// ------------------------------------------------------------------ launchers
template <typename F>
static hipError_t by_kind(const Cache8Args& a, F f) {
    return a.int8 ? f(std::true_type{}) : f(std::false_type{});
}

hipError_t launch_cache8_store(hipStream_t st, const Cache8Args& a, const float* qkv, long row_stride, float* q_out,
                               const float* q_gamma, const float* k_gamma, const float* cs, int n_pos,
                               const int* turn_at, int rope_dim, float eps) {
    const dim3 grid(a.rows, (a.H + 2 * a.HKV + 15) / 16);
    const float2* t = reinterpret_cast<const float2*>(cs);
    auto odd = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
    const bool vec = rope_dim % 8 == 0 && !odd(q_gamma) && !odd(k_gamma) && !odd(cs);  // (whole pieces of 16 bytes)
    return by_kind(a, [&](auto kind) {
        constexpr bool kInt8 = decltype(kind)::value;
        if (vec)
            k_cache8_store<kInt8, true><<<grid, 256, 0, st>>>(qkv, row_stride, q_out, a, q_gamma, k_gamma, t, n_pos,
                                                              turn_at, rope_dim, eps);
        else
            k_cache8_store<kInt8, false><<<grid, 256, 0, st>>>(qkv, row_stride, q_out, a, q_gamma, k_gamma, t, n_pos,
                                                               turn_at, rope_dim, eps);
        return hipGetLastError();
    });
}

hipError_t launch_cache8_load(hipStream_t st, const Cache8Args& a, float* k_out, float* v_out, long out_stride) {
    return by_kind(a, [&](auto kind) {
        k_cache8_load<decltype(kind)::value><<<(a.rows + 3) / 4, 256, 0, st>>>(a, k_out, v_out, out_stride);
        return hipGetLastError();
    });
}

hipError_t launch_cache_keep(hipStream_t st, const Cache8Args& a, float* kc, float* vc, const int* kept, int max_kept,
                             const int* n_kept, int* new_len) {
    const int pieces = kc ? 64 * a.HKV : 16 * a.HKV + 2 * a.HKV;
    const dim3 grid(a.n_seq, (pieces + 255) / 256);
    if (kc) k_cache_keep<true><<<grid, 256, 0, st>>>(a, kc, vc, kept, max_kept, n_kept, new_len);
    else k_cache_keep<false><<<grid, 256, 0, st>>>(a, nullptr, nullptr, kept, max_kept, n_kept, new_len);
    return hipGetLastError();
}

template <bool kInt8, bool kTree>
static hipError_t launch_cache8_attn_as(hipStream_t st, const Cache8Args& a, int shares, const PackedParts& parts) {
    static std::atomic<bool> opted;
    constexpr size_t lds = kLds8;
    if (const hipError_t e = opt_in_lds(opted, (const void*)k_cache8_attn<kInt8, kTree>, lds); e != hipSuccess)
        return e;
    k_cache8_attn<kInt8, kTree><<<shares * a.HKV, 64 * kWaves, lds, st>>>(a, shares, parts.wide, parts.few);
    return hipGetLastError();
}

hipError_t launch_cache8_attn(hipStream_t st, const Cache8Args& a, void* ws) {
    const int shares = packed_shares(a.HKV);
    const PackedParts parts = packed_parts(ws, a.rows, a.H, a.HKV);
    const hipError_t e = by_kind(a, [&](auto kind) {
        constexpr bool kInt8 = decltype(kind)::value;
        return a.mask ? launch_cache8_attn_as<kInt8, true>(st, a, shares, parts)
                      : launch_cache8_attn_as<kInt8, false>(st, a, shares, parts);
    });
    if (e != hipSuccess) return e;
    return launch_packed_combine(st, a, false, parts);
}

}  // namespace ei
