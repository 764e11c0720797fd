// packed.h — what the attention kernels over batches of several sequences share (packed.hip, cache8.hip): the
// layout of the plan that k_packed_plan makes, the walk over a workgroup's share of it (cache8.hip's; packed.hip and
// the pipelined walk over few-row units, few8_walk, each read the plan by the same rules in a loop of their own), the
// parts of units that its cuts divide, masks of drafted trees, binary16 planes.
#pragma once

#include "common.h"
#include "launch.h"
#include "planes.h"

namespace ei {

constexpr int kKT = 32;         // keys per tile
constexpr int kFewRows = 32;    // a sequence's last unit of up to so many rows: few_pass

// ------------------------------------------------------------------ the plan's layout
struct Unit {
    int row0, n, len, u;    // the sequence's first row, rows and keys; the unit's number in it
    int seq, tiles, pad[2];
};
static_assert(sizeof(Unit) == 32, "two 16-byte pieces");
struct Share {
    int first, first_tile, last, last_tile;  // on the line: from tile first_tile of unit `first` to last_tile of `last`
    int merge_end;  // the last share with a part of the unit that begins here and is cut; 0: none does
    int pad[3];
    Unit start;     // what this share begins with
    Unit merge;     // the unit that merge_end speaks of
};
static_assert(sizeof(Share) == 96, "six 16-byte pieces");
struct List {
    Unit* units;    // dealt units in the order of the deal, then the line
    Share* shares;  // one per workgroup of a KV head
};
struct PlanView {
    int4* seq;     // first row, rows, keys (kv_len itself, also past max_kv), wide units before this sequence's
    List wide, few;
};
// header words past the shape: rounds of the deal, units dealt, on the wide line, few-row units, max_kv
enum { kHeadRounds = 6, kHeadDealt = 7, kHeadLine = 8, kHeadFew = 9, kHeadMaxKv = 10 };
constexpr size_t kPlanSeqAt = 256;
__host__ __device__ inline long plan_max_wide(int n_seq, int rows, int G) { return (long)rows * G / kUnitRows + n_seq; }
__host__ __device__ inline size_t plan_wide_at(int n_seq) { return kPlanSeqAt + (size_t)n_seq * sizeof(int4); }
__host__ __device__ inline size_t plan_few_at(int n_seq, int rows, int G) {
    return plan_wide_at(n_seq) + (size_t)plan_max_wide(n_seq, rows, G) * sizeof(Unit);
}
__host__ __device__ inline size_t plan_shares_at(int n_seq, int rows, int G) {
    return plan_few_at(n_seq, rows, G) + (size_t)n_seq * sizeof(Unit);
}
__device__ __forceinline__ PlanView plan_view(char* plan, int n_seq, int rows, int G, int shares) {
    Share* at = reinterpret_cast<Share*>(plan + plan_shares_at(n_seq, rows, G));
    return {reinterpret_cast<int4*>(plan + kPlanSeqAt),
            {reinterpret_cast<Unit*>(plan + plan_wide_at(n_seq)), at},
            {reinterpret_cast<Unit*>(plan + plan_few_at(n_seq, rows, G)), at + shares}};
}

// Whether the plan is one of this call's batch (and of whole prompts, where the keys are the rows).
__device__ __forceinline__ bool plan_fits(const char* plan, int n_seq, int rows, int H, int HKV, bool prompts) {
    const int* h = reinterpret_cast<const int*>(plan);
    return (h[0] == kPlanMagic) & (h[1] == n_seq) & (h[2] == rows) & (h[3] == H) & (h[4] == HKV) &
           (!prompts | (h[5] != 0));
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

// ------------------------------------------------------------------ passes
typedef __amdgpu_buffer_rsrc_t Rsrc;
constexpr int kQB = 32;                         // flat rows per wave
constexpr int kSlots = kUnitRows / kQB;         // waves per key group
constexpr int kGroups = 2;                      // key groups per workgroup
constexpr int kWaves = kSlots * kGroups;
constexpr int kRowF = kHeadDim + 4;             // padded fp32 row of the staging area

__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The lane's number, made where it is used (two instructions; kept, it would be spilled and come back by a
// load that waits for every load before it).
__device__ __forceinline__ uint32_t lane_now() {
    uint32_t zero = 0;
    asm volatile("" : "+v"(zero));
    return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, zero));
}

// A pass, all of it wave-uniform.
struct Pass {
    int seq, u;            // sequence, unit of the sequence
    int row0, pos0;        // first row of the sequence and its position (may be negative)
    int nflat;             // the sequence's flat rows of this KV head
    int T;                 // keys that the unit's last row sees
    int kt_lo, nrange;     // tiles [kt_lo, kt_lo + nrange)
    float* part;           // where its unnormalised rows go, or null: a whole unit
};

// What earlier launches wrote and this one only reads, at a wave-uniform address, by a scalar load: after the
// kernel's own stores the compiler would take a vector load, whose wait is for every load before it too.
template <typename T>
__device__ __forceinline__ T scalar_load(const T* at) {
    return *reinterpret_cast<const __attribute__((address_space(4))) T*>(reinterpret_cast<uintptr_t>(at));
}

// The pool block of the page that holds key t0 of the pass's sequence, -1 past the table's end.
template <bool kPaged>
__device__ __forceinline__ int page_of(const PackedArgs& a, const Pass& p, int t0) {
    if constexpr (!kPaged) return 0;
    const int blk = t0 >> a.bshift;
    const int e = scalar_load(a.btab + (size_t)p.seq * a.max_blocks + min(blk, a.max_blocks - 1));
    return blk < a.max_blocks ? e : -1;
}

// A workgroup's parts in its kernel's share of the workspace: slot 0 of the unit that it goes on with, slot 1
// of the one that it begins; O rows, then (m, l) of each.
constexpr size_t kWidePart = kUnitRows * (kHeadDim + 2), kFewPart = kFewRows * (kHeadDim + 2);
__device__ __forceinline__ size_t part_at(bool few, int block, int slot) {
    return (size_t)(2 * block + slot) * (few ? kFewPart : kWidePart);
}

// A workgroup's part of a list: `sh` its share of the line (first unit, first tile, last unit, last tile), before
// it `rounds` whole units.  run(pass) does one of them.
template <bool kFew, typename Run>
__device__ __forceinline__ void walk_share(const PackedArgs& a, const List& list, int4 sh, int rounds, int shares,
                                           int share, int kvh, FastDiv fG, float* parts, Run run) {
    const int dealt = rounds * shares;
    const int first = scalar(sh.x), first_tile = scalar(sh.y), last = scalar(sh.z), last_tile = scalar(sh.w);
    for (int pass = 0;; ++pass) {
        int at, cut = -1;
        Pass p;
        p.kt_lo = 0;
        if (pass < rounds) {
            at = pass * shares + ((pass & 1) ? shares - 1 - share : share);
        } else {
            const int i = first + pass - rounds;
            if (i > last || (i == last && last_tile == 0)) break;
            at = dealt + i;
            cut = i == last ? last_tile : -1;
            p.kt_lo = i == first ? first_tile : 0;
        }
        // (the share's own copy comes with the line just read: no wait for a list entry)
        const u32x4* unit = reinterpret_cast<const u32x4*>(pass == 0 ? &list.shares[share].start : list.units + at);
        const u32x4 x = scalar_load(unit), y = scalar_load(unit + 1);  // a Unit's fields, in order
        const int n = (int)x.y, len = (int)x.z;
        p.row0 = (int)x.x, p.u = (int)x.w, p.seq = (int)y.x;
        p.pos0 = len - n;
        p.nflat = n * (int)fG.d;
        p.T = min(max(p.pos0 + fdiv(min(kUnitRows * p.u + kUnitRows, p.nflat) - 1, fG) + 1, 0), len);
        p.nrange = (cut >= 0 ? cut : (int)y.y) - p.kt_lo;
        // (its place in scalar registers: kept in vector ones it would be spilled)
        const int place = scalar((int)part_at(kFew, share * a.HKV + kvh, p.kt_lo > 0 ? 0 : 1));
        p.part = p.kt_lo > 0 || cut >= 0 ? parts + place : nullptr;
        if (pass > 0) lds_barrier();  // the last pass's rows have been read
        run(p);
    }
}

// ------------------------------------------------------------------ trees of drafts
// Keys of the tile at t0 that a row sees, a bit each: those before its sequence's new rows, and of the new ones,
// row for row, those whose bit is set in its mask, up to itself.  (Two 32-bit words of the mask, shifted.)
__device__ __forceinline__ uint32_t tree_bits(const PackedArgs& a, const Pass& p, int qpos, int t0) {
    const uint32_t* row = a.mask + (size_t)(p.row0 + qpos - p.pos0) * a.mask_words;
    const int j0 = t0 - p.pos0, at = j0 >> 5;  // (rounded down)
    auto word = [&](int i) { return i < 0 ? ~0u : i < a.mask_words ? row[i] : 0u; };
    const uint64_t both = (uint64_t)word(at + 1) << 32 | word(at);
    const uint32_t bits = (uint32_t)(both >> (j0 & 31));
    const int n = qpos - t0 + 1;  // causal: not past itself
    return n >= 32 ? bits : n <= 0 ? 0u : bits & ((1u << n) - 1u);
}

// Whether new row `tok` of a sequence, its first new key at pos0, sees no key at all.  (Asked where a row's weights sum
// to zero; scores of -infinity do that too, and give NaN.)
__device__ __forceinline__ bool tree_sees_none(const PackedArgs& a, int row0, int pos0, int tok) {
    if (pos0 > 0) return false;
    const uint32_t* row = a.mask + (size_t)(row0 + tok) * a.mask_words;
    uint32_t any = 0;
    for (int w = max(-pos0, 0) >> 5; w <= tok >> 5 && w < a.mask_words; ++w) {
        uint32_t bits = row[w];
        if (w == -pos0 >> 5) bits &= ~0u << (-pos0 & 31);
        if (w == tok >> 5) bits &= ~0u >> (31 - (tok & 31));
        any |= bits;
    }
    return any == 0;
}

// ------------------------------------------------------------------ two binary16 planes
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& h, uint32_t& l) {
    h = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
    float ra, rb;  // a - h's low half, b - its high half, in one instruction each
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(h), "v"(a));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(h), "v"(b));
    l = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{ra, rb}, f16x2));
}
// The power of two that brings `most` to 2^kTop .. 2^(kTop+1), and its inverse: `most`'s exponent (biased) is kept
// where both are normal numbers, and up to `limit`: planes of what passes that by two overflow to infinities, their
// products to NaN, and the waves that meet them take their keys again in fp32.
template <int kTop>
__device__ __forceinline__ uint32_t scale_to(float most, uint32_t limit = 254) {
    const uint32_t e = min(max(__float_as_uint(most) >> 23, kTop + 2u), limit);
    return (254u + kTop - e) << 23;
}
__device__ __forceinline__ float inverse(uint32_t scale) { return __uint_as_float(0x7F000000u - scale); }

}  // namespace ei
