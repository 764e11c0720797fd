// packed.hip — attention of the new rows of several sequences on gfx950: the plan that lays a batch
// out over the GPU, the attention kernel over packed prompts or a paged pool, and the step's prologue.
#include <cstdlib>

#include "common.h"
#include "launch.h"
#include "planes.h"

namespace ei {

constexpr int kKT = 32;         // keys per tile
constexpr int kPassTiles = 5;   // a unit's fixed cost, in tiles

// ------------------------------------------------------------------ the plan
// The query rows of a sequence and KV head are taken flat, row f = token * G + head of the group, and
// cut into units of kUnitRows: a unit shares its K and V tiles, whatever G is and however few tokens
// there are.  Its cost is its causal key tiles and kPassTiles for everything done once per unit.
//
// `shares` workgroups serve each KV head, all heads alike.  Each takes the same cost: first whole
// units, dealt out in descending order of tiles and back and forth, round by round, so that the
// workgroups walk units of about the same keys at the same time (their tiles meet in the XCD's L2);
// then, of the last units (the smallest: one to two rounds of them, or all if there are fewer), laid
// end to end on a line, what is missing to an equal share.  The cuts on the line may fall inside a
// unit: its parts are merged by k_packed_combine.
//
// Order and cuts follow from the lengths alone (no atomics decide them), so a batch planned twice
// gives the same bits twice.
struct PlanView {
    int4* seq;    // first row, rows, keys, first unit (unit numbers run through the sequences)
    int4* units;  // in the order of the deal: sequence, unit of the sequence, tiles, 0
    int2* cuts;   // [shares + 1]: on the line, unit and first tile
};
__host__ __device__ inline size_t plan_seq_at() { return 256; }
__host__ __device__ inline size_t plan_units_at(int n_seq) { return plan_seq_at() + (size_t)n_seq * 16; }
__host__ __device__ inline long plan_max_units(int n_seq, int rows, int G) {
    return ((long)rows * G) / kUnitRows + n_seq;
}
__host__ __device__ inline size_t plan_cuts_at(int n_seq, int rows, int G) {
    return plan_units_at(n_seq) + (size_t)plan_max_units(n_seq, rows, G) * 16;
}
__device__ __forceinline__ PlanView plan_view(char* plan, int n_seq, int rows, int G) {
    return {reinterpret_cast<int4*>(plan + plan_seq_at()), reinterpret_cast<int4*>(plan + plan_units_at(n_seq)),
            reinterpret_cast<int2*>(plan + plan_cuts_at(n_seq, rows, G))};
}
int packed_shares(int HKV) { return kPackedCus / HKV > 1 ? kPackedCus / HKV : 1; }
size_t packed_plan_bytes(int n_seq, int rows, int H, int HKV) {
    const size_t b = plan_cuts_at(n_seq, rows, H / HKV) + (size_t)(packed_shares(HKV) + 1) * sizeof(int2);
    return (b + 255) & ~(size_t)255;
}

constexpr int kPlanThreads = 1024;
constexpr int kPlanSeqLds = 2048;      // sequences held in LDS (more are read from the plan)
constexpr int kMinShare = 8;           // the least cost worth a workgroup
constexpr long kMaxRankWork = 1 << 20;  // units x sequences up to which units are sorted

// Exclusive sum over the workgroup; total in every thread.
__device__ __forceinline__ long long block_scan(long long v, long long* total) {
    __shared__ long long part[kPlanThreads / 64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    long long s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const long long t = __shfl_up(s, d);
        if (lane >= d) s += t;
    }
    if (lane == 63) part[w] = s;
    __syncthreads();
    long long before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kPlanThreads / 64; ++i) {
        if (i < w) before += part[i];
        all += part[i];
    }
    __syncthreads();
    *total = all;
    return before + s - v;
}

__global__ __launch_bounds__(kPlanThreads) void k_packed_plan(const int* __restrict__ cu,
                                                              const int* __restrict__ kv_len, int n_seq, int rows,
                                                              int max_kv, int H, int HKV, int shares,
                                                              char* __restrict__ plan) {
    __shared__ int4 seq_lds[kPlanSeqLds];
    __shared__ unsigned long long load[kPackedCus];
    __shared__ long long cut_at[kPackedCus + 1];
    const int tid = threadIdx.x, G = H / HKV;
    const PlanView pv = plan_view(plan, n_seq, rows, G);

    // sequences: rows, keys, first unit
    long long units = 0;
    int bad = 0;
    for (int base = 0; base < n_seq; base += kPlanThreads) {
        const int s = base + tid;
        int lo = 0, n = 0, len = 0;
        if (s < n_seq) {
            lo = cu[s];
            const int hi = cu[s + 1];
            bad |= lo < 0 || hi < lo || hi > rows;
            n = hi - lo;
            len = kv_len ? min(max(kv_len[s], 0), max_kv) : min(n, max_kv);
        }
        bad = __syncthreads_or(bad);
        const long long nu = bad ? 0 : ((long long)n * G + kUnitRows - 1) / kUnitRows;
        long long all;
        const long long at = units + block_scan(nu, &all);
        if (s < n_seq) {
            const int4 e = make_int4(lo, n, len, (int)at);
            pv.seq[s] = e;
            if (s < kPlanSeqLds) seq_lds[s] = e;
        }
        units += all;
    }
    if (bad) units = 0;  // rows outside the batch: no call on this plan does anything
    __syncthreads();
    const bool in_lds = n_seq <= kPlanSeqLds;
    auto seq_at = [&](int s) { return in_lds ? seq_lds[s] : pv.seq[s]; };
    const int U = (int)units;
    auto units_of = [&](const int4& e) { return (int)(((long long)e.y * G + kUnitRows - 1) / kUnitRows); };
    auto unit = [&](int i) {  // sequence, unit of the sequence, tiles
        int lo = 0, hi = n_seq - 1;
        while (lo < hi) {  // the last sequence whose first unit is not past i
            const int mid = (lo + hi + 1) >> 1;
            if (seq_at(mid).w <= i) lo = mid;
            else hi = mid - 1;
        }
        const int4 e = seq_at(lo);
        const int u = i - e.w;
        const int last = min(e.y - 1, (kUnitRows * u + kUnitRows - 1) / G);
        const int keys = max(min(e.z - e.y + last + 1, e.z), 0);
        return make_int4(lo, u, (int)(((long long)keys + kKT - 1) / kKT), 0);
    };
    // units of sequence e with more than t tiles (they are its last ones)
    auto above = [&](const int4& e, int t) {
        const int nu = units_of(e);
        if (t < 0) return nu;
        const long long m = 32LL * t - (e.z - e.y);  // rows that see at most t tiles
        if (m <= 0) return nu;
        return m >= e.y ? 0 : nu - min(nu, (int)(m * G / kUnitRows));
    };

    long long mine = 0, total;
    for (int i = tid; i < U; i += kPlanThreads) mine += unit(i).z + kPassTiles;
    block_scan(mine, &total);
    const long long even = (total + shares - 1) / shares;
    const long long share = even > kMinShare ? even : kMinShare;
    // (sorting costs units x sequences: where that is much, there is enough work for the order not to matter)
    const int rounds = (long long)U * n_seq <= kMaxRankWork && U / shares > 1 ? U / shares - 1 : 0;
    const int dealt = rounds * shares, line = U - dealt;
    for (int j = tid; j < shares; j += kPlanThreads) load[j] = 0;
    __syncthreads();
    for (int i = tid; i < U; i += kPlanThreads) {
        const int4 x = unit(i);
        int at = i;
        if (rounds > 0) {
            // units before this one: more tiles, or as many in an earlier sequence, or later in its own
            at = 0;
            for (int s = 0; s < n_seq; ++s) {
                const int4 e = seq_at(s);
                at += s < x.x ? above(e, x.z - 1) : s > x.x ? above(e, x.z) : units_of(e) - 1 - x.y;
            }
        }
        pv.units[at] = x;
        if (at < dealt) {
            const int r = at / shares, j = at - r * shares;
            atomicAdd(&load[(r & 1) ? shares - 1 - j : j], (unsigned long long)(x.z + kPassTiles));
        }
    }
    __syncthreads();
    long long all;
    const long long want = tid < shares ? max(share - (long long)load[tid], 0LL) : 0;
    const long long before = block_scan(want, &all);
    if (tid <= shares) cut_at[tid] = tid == 0 ? 0 : before;  // (thread `shares` wants nothing: the sum of all)
    if (tid <= shares) pv.cuts[tid] = make_int2(tid == 0 ? 0 : line, 0);
    __syncthreads();
    // the cuts that fall on each unit of the line
    long long at = 0;
    for (int base = 0; base < line; base += kPlanThreads) {
        const int i = base + tid;
        const int tiles = i < line ? pv.units[dealt + i].z : 0;
        const long long cost = i < line ? tiles + kPassTiles : 0;
        long long sum;
        const long long a = at + block_scan(cost, &sum);
        if (i < line) {
            int lo = 1, hi = shares + 1;  // the first cut not before a
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (cut_at[mid] >= a) hi = mid;
                else lo = mid + 1;
            }
            for (; lo <= shares && cut_at[lo] < a + cost; ++lo) {
                // an even number of tiles on both sides of a cut (the key groups take turns), or none
                int t = (int)(cut_at[lo] - a) & ~1;
                if (lo == shares || t >= tiles - 1) pv.cuts[lo] = make_int2(lo == shares ? line : i + 1, 0);
                else pv.cuts[lo] = make_int2(i, t);
            }
        }
        at += sum;
    }
    if (tid == 0) {
        int* h = reinterpret_cast<int*>(plan);
        h[0] = bad ? 0 : kPlanMagic;
        h[1] = n_seq, h[2] = rows, h[3] = H, h[4] = HKV;
        h[5] = kv_len == nullptr;
        h[6] = rounds, h[7] = dealt, h[8] = line;
    }
}

// Whether the plan is one of this call's batch (and of whole prompts, where the keys are the rows).
__device__ __forceinline__ bool plan_fits(const char* plan, int n_seq, int rows, int H, int HKV, bool prompts) {
    const int* h = reinterpret_cast<const int*>(plan);
    return h[0] == kPlanMagic && h[1] == n_seq && h[2] == rows && h[3] == H && h[4] == HKV && (!prompts || h[5]);
}

// The sequence that owns row b: the last whose first row is not past it, if it has that row; else -1.
// 64 probes at a time, one per lane.
__device__ __forceinline__ int row_owner(const int4* seq, int n_seq, int b, int lane) {
    int lo = 0, n = n_seq;
    while (n > 1) {
        const int step = (n + 63) >> 6, s = lo + lane * step;
        const uint64_t le = __builtin_amdgcn_ballot_w64(lane * step < n && seq[min(s, n_seq - 1)].x <= b);
        const int k = le ? 63 - __builtin_clzll(le) : 0;
        lo += k * step;
        n = min(step, n - k * step);
    }
    const int4 e = seq[lo];
    return b >= e.x && b < e.x + e.y ? lo : -1;
}

// ------------------------------------------------------------------ attention
// Both products on v_mfma_f32_32x32x16_bf16 with fp32 operands as three bf16 planes (planes.h), six
// plane products each, as in prefill.hip, and with its wave layout: a wave holds 32 flat query rows,
// computes S^T[key][row] = K . Q^T, so that each lane owns one row and 16 of a tile's 32 keys, and
// O^T[d][row] = V^T . P^T from the same registers.
//
// Workgroup = kGroups key groups x kSlots waves: the unit's 128 rows over the waves of a group, its
// tiles over the groups in turn (tile kt to group kt % kGroups counted from the pass's first), whose
// (m, l, O) meet in LDS at the end of the pass.  A pass is a unit, or the part of it between two cuts
// of the plan's line; a part goes unnormalised to the workspace, its rows as they are numbered in the
// unit.  Waves without rows (a unit of few) take part in loading the tiles and multiply nothing.
//
// The key loop is that of prefill.hip: each wave of a group fetches a quarter of a K or V tile, 16
// floats per lane, and stores its planes (V transposed) while the group multiplies the other of the
// two; the groups run half an iteration apart, so that one has matrix work while the other is in its
// softmax.
typedef __amdgpu_buffer_rsrc_t Rsrc;
constexpr int kQB = 32;                         // flat rows per wave
constexpr int kSlots = kUnitRows / kQB;         // waves per key group
constexpr int kGroups = 2;                      // key groups per workgroup
constexpr float kLazy = 8.f;                    // lazy-rescale threshold (log2 units)
constexpr int kXchF = 34;                       // floats per lane exchanged by the merge
constexpr int kRowF = kHeadDim + 4;             // padded fp32 row of the staging area
// plane rows padded to an odd number of 16-byte pieces: the rows that an operand read takes, one per
// lane, spread over all LDS banks
constexpr int kKRowB = 2 * kHeadDim + 16, kKPlane = kKT * kKRowB;  // K plane: [32 keys][128 d] bf16
constexpr int kVRowB = 2 * kKT + 16, kVPlane = kHeadDim * kVRowB;  // V plane, transposed: [128 d][32 keys]
// LDS: the K planes of both groups, and the merge's exchange area, from 0; the V planes after it,
// and over them the staging area of the unit's rows (queries, later outputs)
constexpr int kStageF = kGroups * kSlots * kXchF * 64;
constexpr int kLdsF = kStageF + kUnitRows * kRowF;
static_assert(kGroups * 3 * kKPlane <= kStageF * 4, "K planes below the staging area");
static_assert(kStageF * 4 + kGroups * 3 * kVPlane <= kLdsF * 4, "V planes within the LDS span");
static_assert(kLdsF * 4 <= 160 * 1024, "LDS budget");

__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }

template <bool kPaged>
__global__ __launch_bounds__(64 * kSlots * kGroups) void k_packed_attn(PackedArgs a, int shares,
                                                                       float* __restrict__ parts) {
    constexpr int D = kHeadDim;
    extern __shared__ __align__(16) float smem[];
    if (!plan_fits(a.plan, a.n_seq, a.rows, a.H, a.HKV, !kPaged)) return;
    const int kvh = blockIdx.x % a.HKV, share = blockIdx.x / a.HKV;  // a KV head's workgroups share an XCD's L2
    const int H = a.H, G = a.H / a.HKV;
    const FastDiv fG = fast_div((uint32_t)G);
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int wu = scalar(w), hw = wu % kSlots, grp = wu / kSlots;
    const int col = lane & 31, hh = lane >> 5;
    const uint32_t row_bytes = (uint32_t)(a.kv_stride * 4);
    const float* const kbase = a.k + (size_t)kvh * D;
    const float* const vbase = a.v + (size_t)kvh * D;
    char* const lds = reinterpret_cast<char*>(smem);
    char* const kpl = lds + grp * 3 * kKPlane;
    char* const vpl = lds + kStageF * 4 + grp * 3 * kVPlane;
    float* const stage = smem + kStageF;
    const float sl2 = a.scale * 1.44269504088896340736f;  // goes into q: scores come out in log2 units
    const uint32_t voff_k = (uint32_t)(8 * hw + (lane >> 3)) * row_bytes + 32u * (lane & 7);
    const uint32_t voff_v =
        (uint32_t)(16 * (lane >> 5) + 4 * ((lane >> 4) & 1)) * row_bytes + 4u * (32 * hw + 2 * (lane & 15));

    const PlanView pv = plan_view(const_cast<char*>(a.plan), a.n_seq, a.rows, G);
    const int* head = reinterpret_cast<const int*>(a.plan);
    const int rounds = scalar(head[6]), dealt = scalar(head[7]);
    const int first = scalar(pv.cuts[share].x), first_tile = scalar(pv.cuts[share].y);
    const int last = scalar(pv.cuts[share + 1].x), last_tile = scalar(pv.cuts[share + 1].y);

    for (int pass = 0;; ++pass) {
        // the pass's unit, its tiles [kt_lo, kt_lo + nrange), and where its part goes (-1: whole)
        int at, kt_lo = 0, cut = -1;
        if (pass < rounds) {
            at = pass * shares + ((pass & 1) ? shares - 1 - share : share);
        } else {
            const int i = first + pass - rounds;
            if (i > last || (i == last && last_tile == 0)) break;
            at = dealt + i;
            cut = i == last ? last_tile : -1;
            kt_lo = i == first ? first_tile : 0;
        }
        const int s = scalar(pv.units[at].x), u = scalar(pv.units[at].y), tiles = scalar(pv.units[at].z);
        const int nrange = (cut >= 0 ? cut : tiles) - kt_lo;
        const bool part = kt_lo > 0 || cut >= 0;
        const int row0 = scalar(pv.seq[s].x), n = scalar(pv.seq[s].y), len = scalar(pv.seq[s].z);
        const int pos0 = len - n;                 // position of the sequence's first new row (may be negative)
        const int nflat = n * G;                  // its flat rows of this KV head
        const int f0 = kUnitRows * u + kQB * hw;  // this wave's first
        const bool live = f0 < nflat;
        const int tok = fdiv(min(f0 + col, nflat - 1), fG);
        const int qpos = pos0 + tok;              // this lane's query
        const int T = min(max(pos0 + fdiv(min(kUnitRows * u + kUnitRows, nflat) - 1, fG) + 1, 0), len);  // keys seen
        const int nfull = max(pos0 + fdiv(min(f0, nflat - 1), fG) + 1, 0) / kKT;  // tiles below the wave's diagonal
        const int n_it = (nrange + kGroups - 1) / kGroups, n_mine = (nrange - grp + kGroups - 1) / kGroups;

        // K and V of this group's i-th tile (kt_lo + kGroups * i + grp), a quarter per wave:
        //   K: row 8*hw + lane/8, d = 8c .. 8c+7 and 64 + 8c .. (c = lane%8)
        //   V: d = 32*hw + 2*(lane%16) and the next, the eight keys of chunk lane/16 (step s = chunk/2,
        //     half hh = chunk%2 of the P.V operand: keys 16s + 4hh + {0..3, 8..11})
        float rg[16];
        // the tile's visible rows as a buffer: reads past the last one give zeros
        auto tile_rsrc = [&](const float* cache, int t0) {
            size_t row = (size_t)row0 + t0;
            int there = min(kKT, T - t0);
            if constexpr (kPaged) {
                const int blk = t0 >> a.bshift;
                const int phys = blk < a.max_blocks ? a.btab[(size_t)s * a.max_blocks + blk] : -1;
                const bool ok = phys >= 0 && phys < a.n_blocks;
                row = ok ? ((size_t)phys << a.bshift) | (size_t)(t0 & ((1 << a.bshift) - 1)) : 0;
                if (!ok) there = 0;
            }
            return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(cache) + row * a.kv_stride, 0,
                                                     there ? (int)((uint32_t)(there - 1) * row_bytes + D * 4) : 0,
                                                     kBufferDword3);
        };
        auto load_k = [&](int i) {
            const Rsrc rs = tile_rsrc(kbase, (kt_lo + kGroups * i + grp) * kKT);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rs, voff_k + 256 * (j >> 1) + 16 * (j & 1), 0, 0);
                rg[4 * j] = __uint_as_float(v.x), rg[4 * j + 1] = __uint_as_float(v.y);
                rg[4 * j + 2] = __uint_as_float(v.z), rg[4 * j + 3] = __uint_as_float(v.w);
            }
        };
        auto load_v = [&](int i) {
            const Rsrc rs = tile_rsrc(vbase, (kt_lo + kGroups * i + grp) * kKT);
            const uint32_t off = unhoisted(voff_v);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const u32x2 v =
                    __builtin_amdgcn_raw_buffer_load_b64(rs, off + (8 * (j >> 2) + (j & 3)) * row_bytes, 0, 0);
                rg[2 * j] = __uint_as_float(v.x), rg[2 * j + 1] = __uint_as_float(v.y);
            }
        };
        // a value of rg past kPlaneMax turns one of them into NaN, which reaches a sum of every wave that
        // multiplies it
        auto check_planes = [&]() {
            float most = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) most = fmaxf(most, __builtin_fabsf(rg[j]));
            rg[0] = most < kPlaneMax ? rg[0] : __uint_as_float(0xFFFFFFFFu);
        };
        // half x of the conversion of rg: eight values, one 16-byte piece of each plane
        auto conv_k = [&](int x) {
            uint32_t ch[4], cm[4], cl[4];
            if (x == 0) check_planes();
#pragma unroll
            for (int j = 0; j < 4; ++j) split_pair(rg[8 * x + 2 * j], rg[8 * x + 2 * j + 1], ch[j], cm[j], cl[j]);
            char* p = kpl + (8 * hw + (lane >> 3)) * kKRowB + 16 * (lane & 7) + 128 * x;
            *reinterpret_cast<u32x4*>(p) = u32x4{ch[0], ch[1], ch[2], ch[3]};
            *reinterpret_cast<u32x4*>(p + kKPlane) = u32x4{cm[0], cm[1], cm[2], cm[3]};
            *reinterpret_cast<u32x4*>(p + 2 * kKPlane) = u32x4{cl[0], cl[1], cl[2], cl[3]};
        };
        auto conv_v = [&](int x) {  // d + x
            uint32_t ch[4], cm[4], cl[4];
            if (x == 0) check_planes();
#pragma unroll
            for (int j = 0; j < 4; ++j) split_pair(rg[4 * j + x], rg[4 * j + 2 + x], ch[j], cm[j], cl[j]);
            char* p = vpl + (32 * hw + 2 * (lane & 15) + x) * kVRowB + 16 * (lane >> 4);
            *reinterpret_cast<u32x4*>(p) = u32x4{ch[0], ch[1], ch[2], ch[3]};
            *reinterpret_cast<u32x4*>(p + kVPlane) = u32x4{cm[0], cm[1], cm[2], cm[3]};
            *reinterpret_cast<u32x4*>(p + 2 * kVPlane) = u32x4{cl[0], cl[1], cl[2], cl[3]};
        };
        auto k_frag = [&](int t, int plane) {  // K[key col][16t + 8hh ..]
            return *reinterpret_cast<const u32x4*>(kpl + col * kKRowB + 16 * hh + 32 * t + plane * kKPlane);
        };
        auto v_frag = [&](int x, int plane) {  // step s = x/4, d = 32 (x%4) + col
            return *reinterpret_cast<const u32x4*>(vpl + (32 * (x & 3) + col) * kVRowB + 32 * (x >> 2) + 16 * hh +
                                                   plane * kVPlane);
        };

        // the unit's query rows by LDS DMA, once for both groups: wave wu rows 16*wu .. of the unit
        // (rows past the sequence repeat its last), 512 contiguous bytes each
        if (pass > 0) lds_barrier();  // every wave has stored its rows from the staging area
        {
            int f = min(kUnitRows * u + (kQB / 2) * wu, nflat - 1);
            const int t0 = fdiv(f, fG);
            int g = f - t0 * G;
            uint64_t sb = (uint64_t)(uintptr_t)(a.q + ((size_t)row0 + t0) * a.q_stride + (size_t)(kvh * G + g) * D);
            const uint64_t next = (uint64_t)((a.q_stride - (long)(G - 1) * D) * 4);
            const uint32_t lb = scalar((int)lds_addr(stage + (kQB / 2) * wu * kRowF));
            if (hh == 0) {
#pragma unroll
                for (int j = 0; j < kQB / 2; ++j) {
                    dma16_s(sb, 16u * col, lb + j * (kRowF * 4));
                    if (f + 1 < nflat) {
                        ++f;
                        ++g;
                        sb += g == G ? next : (uint64_t)(D * 4);
                        if (g == G) g = 0;
                    }
                }
            }
        }
        if (n_mine > 0) load_k(0);
        wait_vmcnt<0>();
        lds_barrier();
        Planes qp[8];
        // a score on planes is off by at most 2^-134 (|q| + |k|) per element, 2^-77 with K below kPlaneMax and
        // q below 2^50; a wave with a q element past that takes its tiles in fp32 after the key loop
        uint64_t q_fp32;
        {
            const float* qs = stage + (hw * kQB + col) * kRowF + 8 * hh;
            float most = 0.f;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                float4 x = *reinterpret_cast<const float4*>(qs + 16 * t);
                float4 y = *reinterpret_cast<const float4*>(qs + 16 * t + 4);
                x.x *= sl2, x.y *= sl2, x.z *= sl2, x.w *= sl2, y.x *= sl2, y.y *= sl2, y.z *= sl2, y.w *= sl2;
#pragma unroll
                for (const float f : {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w}) most = fmaxf(most, __builtin_fabsf(f));
                uint32_t h[4], m[4], l[4];
                split_pair(x.x, x.y, h[0], m[0], l[0]);
                split_pair(x.z, x.w, h[1], m[1], l[1]);
                split_pair(y.x, y.y, h[2], m[2], l[2]);
                split_pair(y.z, y.w, h[3], m[3], l[3]);
                qp[t] = {u32x4{h[0], h[1], h[2], h[3]}, u32x4{m[0], m[1], m[2], m[3]}, u32x4{l[0], l[1], l[2], l[3]}};
            }
            q_fp32 = __builtin_amdgcn_ballot_w64(!(most < 0x1p50f));
        }
        if (n_mine > 0) {
#pragma unroll
            for (int x = 0; x < 2; ++x) conv_k(x);
            load_v(0);
        }
        floatx16 o[4];
        float m, lsum;
        auto clear = [&]() {
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
            m = -INFINITY;
            lsum = 0.f;
        };
        // scores s of tile kt -> P (in place), the running maximum and sum, O rescaled if it rose
        auto softmax = [&](int kt, floatx16& s) {
            if (kt >= nfull) {  // tile crosses the diagonal (wave-uniform)
                const int k0 = unhoisted(kt * kKT + 4 * hh);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (k0 + 8 * (r >> 2) + (r & 3) > qpos) s[r] = -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
            const float ms = half_max(mx);
            if (__builtin_amdgcn_ballot_w64(ms > m + kLazy)) {  // rare after the first tile
                const float mn = fmaxf(m, ms);
                const float corr = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
                lsum *= corr;
#pragma unroll
                for (int db = 0; db < 4; ++db)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[db][r] *= corr;
                m = mn;
            }
            const float nb_ = m == -INFINITY ? 0.f : -m;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = __builtin_amdgcn_exp2f(s[r] + nb_);
                lsum += s[r];
            }
        };
        // The two products in fp32 from the cache, for a wave that planes do not serve: see after the key
        // loop.  q comes from its row again; values 16t + 8hh .. + 7 take the registers of planes h and m.
        auto q_whole = [&]() {
            const int ln = unhoisted(lane), f = min(f0 + (ln & 31), nflat - 1), t0 = fdiv(f, fG);
            const float* row =
                a.q + ((size_t)row0 + t0) * a.q_stride + (size_t)(kvh * G + f - t0 * G) * D + 8 * (ln >> 5);
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                qp[t].h = *reinterpret_cast<const u32x4*>(row + 16 * t);
                qp[t].m = *reinterpret_cast<const u32x4*>(row + 16 * t + 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    qp[t].h[j] = __float_as_uint(__uint_as_float(qp[t].h[j]) * sl2);
                    qp[t].m[j] = __float_as_uint(__uint_as_float(qp[t].m[j]) * sl2);
                }
            }
        };
        auto qk_fp32 = [&](int i, floatx16& s) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
            const Rsrc rs = tile_rsrc(kbase, (kt_lo + kGroups * i + grp) * kKT);
            const int ln = unhoisted(lane);
            const uint32_t off = (ln & 31) * row_bytes + 32u * (ln >> 5);
#pragma unroll
            for (int t = 0; t < 8; ++t) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // d = 16t + 8hh + 2j and the next
                    const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(rs, off + 64 * t + 8 * j, 0, 0);
                    const u32x4 qv = j < 2 ? qp[t].h : qp[t].m;
                    const float q0 = __uint_as_float(qv[2 * (j & 1)]), q1 = __uint_as_float(qv[2 * (j & 1) + 1]);
                    s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(v.x), q0, s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(v.y), q1, s, 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto pv_fp32 = [&](int i, const floatx16& p) {
            const Rsrc rs = tile_rsrc(vbase, (kt_lo + kGroups * i + grp) * kKT);
            const uint32_t off = unhoisted(4 * hh) * row_bytes + 4u * col;
#pragma unroll
            for (int r = 0; r < 16; ++r) {  // lane half hh: key 8(r/4) + 4hh + r%4
#pragma unroll
                for (int db = 0; db < 4; ++db) {
                    const float v = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                        rs, off + (8 * (r >> 2) + (r & 3)) * row_bytes + 128 * db, 0, 0));
                    o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, p[r], o[db], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // The same for a tile that crosses the diagonal, key after key: a value that a row does not see
        // must not be multiplied at all (0 times infinity), and the matrix instruction takes every row
        // with every key.  P passes through the wave's own part of the exchange area, [key][row].
        auto pv_seen = [&](int i, const floatx16& p) {
            const int t0 = (kt_lo + kGroups * i + grp) * kKT;
            const Rsrc rs = tile_rsrc(vbase, t0);
            const int ln = unhoisted(lane);
            float* pw = smem + w * (kXchF * 64) + (ln & 31);
#pragma unroll
            for (int r = 0; r < 16; ++r) pw[32 * (8 * (r >> 2) + 4 * (ln >> 5) + (r & 3))] = p[r];
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (int key = 0; key < kKT; ++key) {
                const float pk = pw[32 * key];
                const uint32_t off = key * row_bytes + 16u * (ln >> 5);
                if (t0 + key <= qpos) {
#pragma unroll
                    for (int db = 0; db < 4; ++db) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) {  // d = 32 db + 8x + 4hh + 0 .. 3
                            const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rs, off + 128 * db + 32 * x, 0, 0);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                o[db][4 * x + e] = __builtin_fmaf(pk, __uint_as_float(v[e]), o[db][4 * x + e]);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
        };

        clear();
        lds_barrier();  // every wave has its q (the staging area is free for the V planes); K planes stored
        if (grp == 1) lds_barrier();
        for (int i = 0; i < n_it; ++i) {
            floatx16 s;
            if (i < n_mine) {
                // S^T = K . Q^T, while V(i) goes to its planes; then K(i+1) is fetched
                if (live) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = 0.f;
                    Planes kf;
                    kf.l = k_frag(0, 2), kf.m = k_frag(0, 1), kf.h = k_frag(0, 0);
#pragma unroll
                    for (int t = 0; t < 8; ++t) {
                        if (t == 4 || t == 6) conv_v(t == 6);
                        mfma_split(kf, qp[t], s, [&](int p) { return t < 7 ? k_frag(t + 1, p) : u32x4{}; });
                    }
                } else {
                    conv_v(0);
                    conv_v(1);
                }
                if (i + 1 < n_mine) load_k(i + 1);
            }
            lds_barrier();
            if (i < n_mine) {
                const bool more = i + 1 < n_mine;
                if (live) {
                    __builtin_amdgcn_s_setprio(1);
                    softmax(kt_lo + kGroups * i + grp, s);
                    // O^T += V^T . P^T, while K(i+1) goes to its planes; then V(i+1) is fetched
                    Planes vf, pp;
                    vf.l = v_frag(0, 2), vf.m = v_frag(0, 1), vf.h = v_frag(0, 0);
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        if ((x & 3) == 0) {
                            uint32_t ph[4], pm[4], pl[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                split_pair(s[2 * x + 2 * j], s[2 * x + 2 * j + 1], ph[j], pm[j], pl[j]);
                            pp = {u32x4{ph[0], ph[1], ph[2], ph[3]}, u32x4{pm[0], pm[1], pm[2], pm[3]},
                                  u32x4{pl[0], pl[1], pl[2], pl[3]}};
                        }
                        if (x == 4 || x == 6) conv_k(x == 6);
                        mfma_split(vf, pp, o[x & 3], [&](int p) { return x < 7 ? v_frag(x + 1, p) : u32x4{}; });
                    }
                } else {
                    conv_k(0);
                    conv_k(1);
                }
                if (more) load_v(i + 1);
                __builtin_amdgcn_s_setprio(0);
            }
            lds_barrier();
        }
        if (grp == 0) lds_barrier();

        // Which sums planes do not serve (prefill.hip has the same rule): an infinite value, or one past
        // kPlaneMax, in K or V shows as a sum that is not finite.  A V value or a weight below kPlaneMin
        // may have lost bits of its third plane, 2^-134, which shows in no sum from kSmallSum up; a smaller
        // one has the wave look through its V tiles, in the blocks of 32 columns with such a sum: it stands
        // if no V value there is below kPlaneMin and the largest one is too small for the weights' 2^-134
        // to show in it.  Otherwise, and for a q past its limit, the wave takes its tiles again in fp32.
        if (live) {
            float z = lsum * 0.f, least[4];  // per block of 32 columns
#pragma unroll
            for (int db = 0; db < 4; ++db) {
                least[db] = INFINITY;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    z = __builtin_fmaf(o[db][r], 0.f, z);
                    least[db] = fminf(least[db], __builtin_fabsf(o[db][r]));
                }
            }
            const float least_all = fminf(fminf(least[0], least[1]), fminf(least[2], least[3]));
            uint64_t redo = q_fp32 | __builtin_amdgcn_ballot_w64(z != 0.f);
            // (a lane without a visible key has no sum: m stays -inf)
            if (!redo && __builtin_amdgcn_ballot_w64(least_all < kSmallSum && m != -INFINITY)) {
                uint32_t small = 0xFFFFFFFFu, tiny = 0xFFFFFFFFu;  // the smallest nonzero sum and V value
                if (m != -INFINITY) {
#pragma unroll
                    for (int db = 0; db < 4; ++db)
#pragma unroll
                        for (int r = 0; r < 16; ++r) small = min(small, magnitude(__float_as_uint(o[db][r])));
                }
                float most = 0.f;
#pragma unroll
                for (int db = 0; db < 4; ++db) {
                    if (!__builtin_amdgcn_ballot_w64(least[db] < kSmallSum && m != -INFINITY)) continue;
                    for (int i = 0; i < n_mine; ++i) {
                        const Rsrc rs = tile_rsrc(vbase, (kt_lo + kGroups * i + grp) * kKT);
                        const int ln = unhoisted(lane);
                        const uint32_t off = (ln >> 3) * row_bytes + 16u * (ln & 7) + 128u * db;
#pragma unroll
                        for (int j = 0; j < kKT / 8; ++j) {
                            const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rs, off + 8 * j * row_bytes, 0, 0);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                tiny = min(tiny, magnitude(v[e]));
                                most = fmaxf(most, __builtin_fabsf(__uint_as_float(v[e])));
                            }
                        }
                    }
                }
                // the sums are off by up to 2^20 2^-134 most; a lane without a nonzero one has nothing to lose
                const float limit = wave_max(most) * 0x1p-84f;
                redo = __builtin_amdgcn_ballot_w64(tiny < kTinyMagnitude || limit > of_magnitude(small));
            }
            if (redo) {
                clear();
                q_whole();
                for (int i = 0; i < n_mine; ++i) {
                    floatx16 s;
                    const int kt = kt_lo + kGroups * i + grp;
                    qk_fp32(i, s);
                    softmax(kt, s);
                    if (kt >= nfull) pv_seen(i, s);
                    else pv_fp32(i, s);
                }
            }
        }

        // ---- the key groups meet through LDS (tile buffers are free after the barrier): group g finishes
        // output blocks db = 2g, 2g+1 and hands the other two to its partner
        float* xw = smem + w * (kXchF * 64) + lane;
        xw[0] = m;
        xw[64] = lsum;
        // (grp is wave-uniform: selects, not a dynamic register index)
        const floatx16 give0 = grp ? o[0] : o[2], give1 = grp ? o[1] : o[3];
        const floatx16 keep0 = grp ? o[2] : o[0], keep1 = grp ? o[3] : o[1];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            xw[(2 + i) * 64] = give0[i];
            xw[(18 + i) * 64] = give1[i];
        }
        lds_barrier();
        const float* xp = smem + ((1 - grp) * kSlots + hw) * (kXchF * 64) + lane;
        const float mp = xp[0], lp = xp[64];
        const float mt = fmaxf(m, mp);  // -inf only when the pass holds no visible key for the row
        const float c0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mt);
        const float cp = mp == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mp - mt);
        const float l = half_sum(lsum * c0 + lp * cp);
        float* dst_part = parts + (size_t)(2 * blockIdx.x + (kt_lo > 0 ? 0 : 1)) * kPartFloats;
        {
            // finished rows (normalised; a row that sees no key: zeros), or the part's, to the staging area
            const float inv = part ? 1.f : qpos < 0 ? 0.f : 1.f / l;
            float* ost = stage + (hw * kQB + col) * kRowF + 64 * grp + 4 * hh;
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                // O^T registers r .. r+3 of block db are d = 32 db + 8(r/4) + 4hh + 0 .. 3
                float v0[4], v1[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v0[j] = (keep0[r + j] * c0 + xp[(2 + r + j) * 64] * cp) * inv;
                    v1[j] = (keep1[r + j] * c0 + xp[(18 + r + j) * 64] * cp) * inv;
                }
                *reinterpret_cast<float4*>(ost + 2 * r) = make_float4(v0[0], v0[1], v0[2], v0[3]);
                *reinterpret_cast<float4*>(ost + 32 + 2 * r) = make_float4(v1[0], v1[1], v1[2], v1[3]);
            }
            if (part && hh == 0 && grp == 0)
                *reinterpret_cast<float2*>(dst_part + kUnitRows * D + 2 * (hw * kQB + col)) = make_float2(mt, l);
        }
        lds_barrier();
        {
            const int ln = unhoisted(lane), c4 = 4 * (ln & 31);
#pragma unroll
            for (int j = 0; j < kQB / 4; ++j) {  // wave wu: rows 16*wu .. of the unit, two per instruction
                const int jj = (kQB / 2) * wu + 2 * j + (ln >> 5), f = kUnitRows * u + jj;
                const float4 v = *reinterpret_cast<const float4*>(stage + jj * kRowF + c4);
                const int t0 = fdiv(f, fG);
                float* dst = part ? dst_part + jj * D
                                  : a.out + (((size_t)row0 + t0) * H + kvh * G + f - t0 * G) * D;
                if (f < nflat) *reinterpret_cast<float4*>(dst + c4) = v;
            }
        }
    }
}

// The units that the plan's cuts divide: workgroup (share, KV head; 8 rows) merges the unit that starts in
// this share and goes on in the next ones.  Part p of it is the share's own (its slot 1), then slot 0 of
// each share that it reaches.  o = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p over the parts that saw a
// key (m = -inf and l = 0 otherwise; m = -inf with a NaN l counts).
__global__ __launch_bounds__(256) void k_packed_combine(PackedArgs a, bool prompts, int shares,
                                                        const float* __restrict__ parts) {
    if (!plan_fits(a.plan, a.n_seq, a.rows, a.H, a.HKV, prompts)) return;
    const int kvh = blockIdx.x % a.HKV, share = blockIdx.x / a.HKV, G = a.H / a.HKV;
    const PlanView pv = plan_view(const_cast<char*>(a.plan), a.n_seq, a.rows, G);
    const int dealt = reinterpret_cast<const int*>(a.plan)[7];
    const int2 from = pv.cuts[share], to = pv.cuts[share + 1];
    if (to.y == 0 || (from.x == to.x && from.y > 0)) return;  // ends between units, or goes on with a unit
    const int4 x = pv.units[dealt + to.x], e = pv.seq[x.x];
    const int row = blockIdx.y * 8 + (threadIdx.x >> 5), f = kUnitRows * x.y + row, d = 4 * (threadIdx.x & 31);
    if (f >= e.y * G) return;
    const int t0 = f / G;
    int end = share + 1;  // the last share with a part
    while (pv.cuts[end + 1].x == to.x && pv.cuts[end + 1].y > 0) ++end;
    auto slot = [&](int p) {
        return parts + (size_t)(2 * (p * a.HKV + kvh) + (p == share ? 1 : 0)) * kPartFloats;
    };
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int kAtOnce = 8;  // parts whose loads are in flight together
    for (int p = share; p <= end; p += kAtOnce) {
        float2 ml[kAtOnce];
        float4 v[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const float* b = slot(min(p + i, end));
            ml[i] = *reinterpret_cast<const float2*>(b + kUnitRows * kHeadDim + 2 * row);
            v[i] = *reinterpret_cast<const float4*>(b + row * kHeadDim + d);
        }
        float mn = M;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
            if (p + i <= end) mn = fmaxf(mn, ml[i].x);
        const float c = M == mn ? 1.f : __builtin_amdgcn_exp2f(M - mn);
        M = mn;
        L *= c, o.x *= c, o.y *= c, o.z *= c, o.w *= c;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            if (p + i > end || (ml[i].x == -INFINITY && ml[i].y == 0.f)) continue;
            const float wv = __builtin_amdgcn_exp2f(ml[i].x - M);
            L = __builtin_fmaf(wv, ml[i].y, L);
            o.x = __builtin_fmaf(wv, v[i].x, o.x), o.y = __builtin_fmaf(wv, v[i].y, o.y);
            o.z = __builtin_fmaf(wv, v[i].z, o.z), o.w = __builtin_fmaf(wv, v[i].w, o.w);
        }
    }
    const float inv = e.z - e.y + t0 < 0 ? 0.f : 1.f / L;  // a row that sees no key: zeros
    *reinterpret_cast<float4*>(a.out + (((size_t)e.x + t0) * a.H + kvh * G + f - t0 * G) * kHeadDim + d) =
        make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// ------------------------------------------------------------------ the step's prologue
// grid (rows, ceil((H + HKV) / 16)), block 256: each wave four consecutive heads of the row, loads of
// all of them first.  Query heads go, normed and turned, to q_out; key heads with the V rows of the same
// KV heads to the pool.
constexpr int kPrepHeads = 4;
__global__ __launch_bounds__(256) void k_packed_prepare(const float* __restrict__ qkv, long row_stride,
                                                        float* __restrict__ q_out, PackedArgs a,
                                                        float* __restrict__ kc, float* __restrict__ vc,
                                                        const float* __restrict__ q_gamma,
                                                        const float* __restrict__ k_gamma,
                                                        const float2* __restrict__ cs, int n_pos, int rope_dim,
                                                        float eps) {
    __shared__ float scratch[4][kHeadDim];
    const int b = blockIdx.x, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int H = a.H, HKV = a.HKV, NH = H + HKV;
    const int h0 = (blockIdx.y * 4 + w) * kPrepHeads;
    if (h0 >= NH || !plan_fits(a.plan, a.n_seq, a.rows, H, HKV, false)) return;  // wave-uniform, no barrier here
    const int4* seq = reinterpret_cast<const int4*>(a.plan + plan_seq_at());
    const int s = row_owner(seq, a.n_seq, b, lane);
    if (s < 0) return;
    const int4 e = seq[s];
    const int pos = e.z - e.y + (b - e.x);
    const bool in = pos >= 0 && pos < n_pos;
    const int blk = pos >> a.bshift;
    const int phys = in && blk < a.max_blocks ? a.btab[(size_t)s * a.max_blocks + blk] : -1;
    const bool there = phys >= 0 && phys < a.n_blocks;
    const size_t crow = ((size_t)(there ? phys : 0) << a.bshift) | (size_t)(pos & ((1 << a.bshift) - 1));
    const float* row = qkv + (size_t)b * row_stride;
    const float2* cs_row = cs + (size_t)(in ? pos : 0) * (rope_dim >> 1);
    float x0[kPrepHeads], x1[kPrepHeads], v0[kPrepHeads], v1[kPrepHeads], inv[kPrepHeads];
#pragma unroll
    for (int j = 0; j < kPrepHeads; ++j) {
        const int hh = min(h0 + j, NH - 1);  // clamped: heads past NH are loaded, not used
        const float* v = row + (size_t)hh * kHeadDim;
        x0[j] = v[lane];
        x1[j] = v[lane + 64];
        const float* vs = row + (size_t)(NH + max(hh - H, 0)) * kHeadDim;  // V of a key head
        v0[j] = vs[lane];
        v1[j] = vs[lane + 64];
    }
    const float qg0 = q_gamma[lane], qg1 = q_gamma[lane + 64];
    const float kg0 = k_gamma[lane], kg1 = k_gamma[lane + 64];
    head_inv<kPrepHeads>(x0, x1, eps, inv, lane);
#pragma unroll
    for (int j = 0; j < kPrepHeads; ++j) {
        const int hh = h0 + j;
        if (hh >= NH) break;
        const bool is_k = hh >= H;
        float o0 = x0[j], o1 = x1[j];
        if (in)
            scale_rope_vals(x0[j], x1[j], inv[j], is_k ? kg0 : qg0, is_k ? kg1 : qg1, cs_row, rope_dim, scratch[w],
                            lane, &o0, &o1);
        if (!is_k) {
            float* dst = q_out + ((size_t)b * H + hh) * kHeadDim;
            dst[lane] = o0;
            dst[lane + 64] = o1;
        } else if (there) {
            const size_t at = crow * a.kv_stride + (size_t)(hh - H) * kHeadDim;
            kc[at + lane] = o0;
            kc[at + lane + 64] = o1;
            vc[at + lane] = v0[j];
            vc[at + lane + 64] = v1[j];
        }
    }
}

// ------------------------------------------------------------------ launchers
hipError_t launch_packed_plan(hipStream_t st, const int* cu, const int* kv_len, int n_seq, int rows, int max_kv, int H,
                              int HKV, void* plan) {
    k_packed_plan<<<1, kPlanThreads, 0, st>>>(cu, kv_len, n_seq, rows, max_kv, H, HKV, packed_shares(HKV),
                                              static_cast<char*>(plan));
    return hipGetLastError();
}

static size_t q_bytes(int rows, int H) { return ((size_t)rows * H * kHeadDim * 4 + 255) & ~(size_t)255; }

size_t packed_ws_bytes(int rows, int H, int HKV) {
    return q_bytes(rows, H) + (size_t)packed_shares(HKV) * HKV * 2 * kPartFloats * 4;
}

template <bool kPaged>
static hipError_t launch_packed_attn(hipStream_t st, const PackedArgs& a, int shares, float* parts) {
    static std::atomic<bool> opted;
    constexpr size_t lds = (size_t)kLdsF * sizeof(float);
    if (const hipError_t e = opt_in_lds(opted, (const void*)k_packed_attn<kPaged>, lds); e != hipSuccess) return e;
    k_packed_attn<kPaged><<<(unsigned)(shares * a.HKV), 64 * kSlots * kGroups, lds, st>>>(a, shares, parts);
    return hipGetLastError();
}

hipError_t launch_packed(hipStream_t st, const PackedArgs& a, void* ws) {
    float* parts = reinterpret_cast<float*>(static_cast<char*>(ws) + q_bytes(a.rows, a.H));
    const int shares = packed_shares(a.HKV);
    const hipError_t e = a.btab ? launch_packed_attn<true>(st, a, shares, parts)
                                : launch_packed_attn<false>(st, a, shares, parts);
    if (e != hipSuccess) return e;
    k_packed_combine<<<dim3(shares * a.HKV, kUnitRows / 8), 256, 0, st>>>(a, a.btab == nullptr, shares, parts);
    return hipGetLastError();
}

hipError_t launch_packed_step(hipStream_t st, PackedArgs a, const float* qkv, long row_stride, float* kc, float* vc,
                              const float* q_gamma, const float* k_gamma, const float* cs, int n_pos, int rope_dim,
                              float eps, void* ws) {
    float* q = static_cast<float*>(ws);
    k_packed_prepare<<<dim3(a.rows, (a.H + a.HKV + 15) / 16), 256, 0, st>>>(
        qkv, row_stride, q, a, kc, vc, q_gamma, k_gamma, reinterpret_cast<const float2*>(cs), n_pos, rope_dim, eps);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    a.q = q;
    a.q_stride = (long)a.H * kHeadDim;
    return launch_packed(st, a, ws);
}

}  // namespace ei
