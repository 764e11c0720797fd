// packed.hip — attention of the new rows of several sequences on gfx950: the plan that lays a batch
// out over the GPU, the attention kernel over packed prompts or a paged pool, and the step's prologue.
#include <type_traits>

#include "packed.h"

namespace ei {

// ------------------------------------------------------------------ the plan
// The query rows of a sequence and KV head are taken flat, row f = token * G + head of the group, and
// cut into units of kUnitRows: a unit shares its K and V tiles, whatever G is and however few tokens
// there are.  A sequence's last unit, if it has at most kFewRows rows (single tokens, drafts, tails of
// prompts), goes to the list of few-row units, the others to the wide list.
//
// `shares` workgroups serve each KV head, all heads alike.  A unit costs its causal key tiles, and something for what
// is done once per unit.  Of the wide list each workgroup first takes whole units, dealt out in descending order of
// tiles and back and forth, round by round, so that the workgroups walk units of about the same keys at the same
// time (their tiles meet in the XCD's L2); the rest (less than a round, or the last full one too, if some workgroup
// would have more than an equal share of everything and 1/32 with it) is laid end to end on a line, of which each gets
// what is missing to an equal share.  The few-row units lie on a line of their own, of which each workgroup gets
// what its wide work leaves of an equal share of everything.  A cut may fall inside a unit: its parts are merged by
// k_packed_combine.
//
// So the workgroups' shares are equal where the units are, and where there is less than a round of them (to within
// what cuts are moved by); a unit of an earlier round is dealt whole, whatever it costs.  One chunk of 64 rows after
// 30000 keys among 64 prompts of 32 rows (H 32 / HKV 8, 66 units for 32 workgroups) is 945 tiles for one workgroup of
// each head, against an equal share of 72, and 1333 us; in a batch of its own, where it is cut, it takes 130, the
// prompts 34.
//
// Dealing the last full round, against leaving it on the line in any case (H 32, HKV 8): 8 prompts of 250
// rows 42 us against 52, one of 2048 132 against 145, 1500 rows after 8000 keys 729 against 770, 1024 after
// 30000 with a prompt of 400 1747 against 1810; at worst (H 40, prompts of 900 and 700) 97 against 89.
//
// Order and cuts follow from the lengths alone (no atomics decide them), so a batch planned twice
// gives the same bits twice.
//
// One workgroup, a thread per sequence, unit or cut, everything in LDS as long as it fits: its time is the
// latency of a dozen steps that need each other, 8 us for 5 sequences, 10 for 6 of up to 8192 rows (490 wide
// units), 6 to 8 in a graph; once per forward pass, not per layer.  With many sequences it is the sorting, which looks
// at every sequence for every unit (in a graph): 256 single tokens 6.5 us, 64 prompts of 32 rows 18, 256 of 64 rows
// 48, 512 of 64 rows 169, the most there is (kMaxRankWork); beyond, unsorted, 1000 of 64 rows 17, 16000 tokens 85.
int packed_shares(int HKV) { return kPackedCus / HKV > 1 ? kPackedCus / HKV : 1; }
size_t packed_plan_bytes(int n_seq, int rows, int H, int HKV) {
    const size_t b = plan_shares_at(n_seq, rows, H / HKV) + 2 * (size_t)packed_shares(HKV) * sizeof(Share);
    return (b + 255) & ~(size_t)255;
}

constexpr int kPlanThreads = 512;
constexpr int kPlanSeqLds = 1024;       // sequences held in LDS (more are read from the plan)
constexpr int kPlanLineLds = 512;       // units of a line held in LDS (likewise)
constexpr long kMaxRankWork = 1 << 20;  // wide units x sequences up to which units are sorted
constexpr int kDealSlack = 32;          // whole units may pass an equal share by 1/32 (by 1/128: 1024 rows after
                                        // 30000 keys take 1770 us instead of 1715; by all of it: H 64, prompts of
                                        // 600 rows after 9000 keys, 300 and 200, 928 instead of 644)

// What a list's work costs, in tiles: `pass` for everything done once per unit or part of one; a cut leaves
// whole turns (the tiles that a workgroup's waves take at a time, a power of two; less where all the work there is
// would not give each one) on both sides, and keeps off a unit's ends by what a pass costs, so that a share does not
// run one for a few tiles.  Without the smaller turns one token at 2000 keys takes 20.3 us instead of 13.7, at 255
// 14.3 instead of 11.0, a draft of 5 of H 32 after 1000 keys 21.4 instead of 15.5.
struct ListCost {
    int pass, turn;
};
// Measured (H / HKV, single tokens): a few-row pass at 5 instead of 8, 24 sequences of 2001 keys 77 us against 85
// (16/8), 50 of up to 4000 117 against 122 (16/8), 6 of 4 tokens after 3000 keys 38 against 41 (32/8); 16 of 5
// tokens after 1024 to 1579 keys 57 against 55.  A wide pass at 7 instead of 5: one prompt of 1024 rows 66 us
// against 61.
constexpr ListCost kWideCost = {5, 2}, kFewCost = {5, 8};

// Sum over the lanes up to this one, by DPP: within rows of 16, then the last lane of each row (15), of
// the two upper rows (31) onwards.
template <int kCtrl, int kRows>
__device__ __forceinline__ long long dpp_add(long long v) {
    const int lo = __builtin_amdgcn_update_dpp(0, (int)v, kCtrl, kRows, 0xF, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), kCtrl, kRows, 0xF, false);
    return v + (long long)(((unsigned long long)(unsigned)hi << 32) | (unsigned)lo);
}
__device__ __forceinline__ long long wave_scan(long long v) {
    v = dpp_add<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);  // row_bcast:15
    return dpp_add<0x143, 0xC>(v);  // row_bcast:31
}
// Exclusive sum over the workgroup; total in every thread.
__device__ __forceinline__ long long block_scan(long long v, long long* total) {
    constexpr int kN = kPlanThreads / 64;
    __shared__ long long part[kN];
    const int w = threadIdx.x >> 6;
    const long long s = wave_scan(v);
    __syncthreads();  // the last call's sums have been read
    if ((threadIdx.x & 63) == 63) part[w] = s;
    __syncthreads();
    long long before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        if (i < w) before += part[i];
        all += part[i];
    }
    *total = all;
    return before + s - v;
}

__global__ __launch_bounds__(kPlanThreads) void k_packed_plan(const int* __restrict__ cu,
                                                              const int* __restrict__ kv_len, int n_seq, int rows,
                                                              int max_kv, int H, int HKV, int shares, FastDiv by_g,
                                                              FastDiv by_shares, double one_share,
                                                              char* __restrict__ plan) {
    __shared__ int4 seq_lds[kPlanSeqLds];
    __shared__ Unit wide_lds[kPlanLineLds], few_lds[kPlanLineLds];  // the lines' units
    __shared__ unsigned long long load[kPackedCus], few_cost, wide_cost;
    __shared__ int last_round[kPackedCus];  // the cost of the units of the last full round, share by share
    __shared__ int2 cuts[kPackedCus + 1];
    __shared__ long long cut_cost[kPackedCus + 1];  // the line's cost before each cut
    __shared__ long long line_at[kPlanThreads];     // units of the line: cost before, tiles
    __shared__ int line_tiles[kPlanThreads];
    const int tid = threadIdx.x, G = H / HKV;
    const PlanView pv = plan_view(plan, n_seq, rows, G, shares);
    // keys that rows up to `row` of a sequence of n rows and len keys see, in tiles
    auto tiles_of = [](int n, int len, int row) { return (max(min(len - n + row + 1, len), 0) + kKT - 1) / kKT; };
    auto wide_of = [&](int n) { return (int)((unsigned)(n * G + kUnitRows - 1 - kFewRows) / kUnitRows); };
    // a share of a cost, rounded up (one_share = 1 / shares; what its rounding adds is below the 2^-20)
    auto share_of = [&](unsigned long long cost) {
        return (long long)ceil((double)(long long)cost * one_share - 0x1p-20);
    };

    if (tid == 0) few_cost = wide_cost = 0;
    for (int j = tid; j < shares; j += kPlanThreads) load[j] = 0;
    // sequences: rows, keys, first wide unit; the few-row units
    long long units = 0, few = 0;
    int bad = 0;
    for (int base = 0; base < n_seq; base += kPlanThreads) {
        const int s = base + tid;
        int lo = 0, n = 0, len = 0, all_keys = 0;
        if (s < n_seq) {
            lo = cu[s];
            const int hi = cu[s + 1];
            bad |= lo < 0 || hi < lo || hi > rows;
            n = hi - lo;
            all_keys = kv_len ? max(kv_len[s], 0) : n;
            len = min(all_keys, max_kv);
        }
        bad = __syncthreads_or(bad);
        if (bad) n = 0;  // rows outside the batch: no call on this plan does anything
        const int nw = wide_of(n), is_few = n * G > nw * kUnitRows;
        const int tiles = is_few ? tiles_of(n, len, n - 1) : 0;
        long long all;
        const long long at = block_scan((long long)nw << 32 | is_few, &all);  // (both sums stay below 2^31)
        if (s < n_seq) {
            const int first = (int)(units + (at >> 32));
            pv.seq[s] = make_int4(lo, n, all_keys, first);
            if (s < kPlanSeqLds) seq_lds[s] = make_int4(lo, n, len, first);
        }
        if (is_few) {
            const int i = (int)(few + (at & 0xFFFFFFFF));
            const Unit x{lo, n, len, nw, s, tiles, {0, 0}};
            pv.few.units[i] = x;
            if (i < kPlanLineLds) few_lds[i] = x;
        }
        const long long cost = wave_scan(is_few ? tiles + kFewCost.pass : 0);
        if ((tid & 63) == 63 && cost > 0) atomicAdd(&few_cost, (unsigned long long)cost);
        units += all >> 32;
        few += all & 0xFFFFFFFF;
    }
    if (bad) units = few = 0;
    const int U = (int)units;
    __syncthreads();
    const bool in_lds = n_seq <= kPlanSeqLds;
    auto seq_at = [&](int s) {
        if (in_lds) return seq_lds[s];
        int4 e = pv.seq[s];
        e.z = min(e.z, max_kv);
        return e;
    };
    auto unit = [&](int i) {
        int lo = 0, hi = n_seq - 1;
        while (lo < hi) {  // the last sequence whose first unit is not past i
            const int mid = (lo + hi + 1) >> 1;
            if (seq_at(mid).w <= i) lo = mid;
            else hi = mid - 1;
        }
        const int4 e = seq_at(lo);
        const int u = i - e.w;
        const int row = min(e.y - 1, fdiv(kUnitRows * u + kUnitRows - 1, by_g));
        return Unit{e.x, e.y, e.z, u, lo, tiles_of(e.y, e.z, row), {0, 0}};
    };
    // wide units of sequence e with more than t tiles (they are its last ones)
    auto above = [&](const int4& e, int t) {
        const int nw = wide_of(e.y);
        if (t < 0) return nw;
        const long long m = 32LL * t - (e.z - e.y);  // rows that see at most t tiles
        if (m <= 0) return nw;
        return m >= e.y ? 0 : nw - min(nw, (int)((unsigned)((int)m * G) / kUnitRows));
    };
    // (sorting costs units x sequences: where that is much, there is enough work for the order not to matter)
    const int full = (long long)U * n_seq <= kMaxRankWork ? fdiv(U, by_shares) : 0, sure = max(full - 1, 0) * shares;
    long long mine = 0;
    for (int i = tid; i < U; i += kPlanThreads) {
        const Unit x = unit(i);
        const int cost = x.tiles + kWideCost.pass;
        mine += cost;
        int at = i;
        if (full > 0) {
            // units before this one: more tiles, or as many in an earlier sequence, or later in its own
            at = 0;
#pragma unroll 4
            for (int s = 0; s < n_seq; ++s) {
                const int4 e = seq_at(s);
                at += s < x.seq ? above(e, x.tiles - 1) : s > x.seq ? above(e, x.tiles) : wide_of(e.y) - 1 - x.u;
            }
        }
        pv.wide.units[at] = x;
        const int r = fdiv(at, by_shares), j = at - r * shares;
        if (at < sure) atomicAdd(&load[(r & 1) ? shares - 1 - j : j], (unsigned long long)cost);
        else if (r < full) last_round[(r & 1) ? shares - 1 - j : j] = cost;
        if (at >= sure && at - sure < kPlanLineLds) wide_lds[at - sure] = x;
    }
    mine = wave_scan(mine);
    if ((tid & 63) == 63 && mine > 0) atomicAdd(&wide_cost, (unsigned long long)mine);
    __syncthreads();
    // all rounds, or all but one
    const long long both = share_of(wide_cost + few_cost);
    const bool over = full > 0 && tid < shares && (long long)load[tid] + last_round[tid] > both + both / kDealSlack;
    const int rounds = __syncthreads_or(over) ? full - 1 : full;
    const int dealt = rounds * shares;
    if (rounds > 0 && rounds == full && tid < shares) load[tid] += last_round[tid];
    // The wide line's shares, then the few-row line's.  Share j's end lies where the sum of what shares 0 .. j want
    // falls on the line's running cost.  (One code for both: a single workgroup waits for each instruction once.)
    long long taken = tid < shares ? (long long)load[tid] : 0;  // the share's work so far
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
        const List& list = which ? pv.few : pv.wide;
        const int line = which ? (int)few : U - dealt, first = which ? 0 : dealt;
        const int pass = which ? kFewCost.pass : kWideCost.pass;
        const long long share = share_of(which ? few_cost : wide_cost);
        // the line's units in LDS, where it fits
        const bool fits = (which ? line : U - sure) <= kPlanLineLds;
        const Unit* lds = which ? few_lds : wide_lds + (dealt - sure);
        auto unit_at = [&](int i) { return fits ? lds[i] : list.units[first + i]; };
        int turn = which ? kFewCost.turn : kWideCost.turn;
        while (both < kFewCost.turn && turn > 1 && turn > share) turn >>= 1;  // (idle waves cost nothing then)
        const int keep = max(turn, (int)min(share / 2, (long long)pass));
        long long total;
        long long mine = block_scan(tid < shares ? max((which ? both : share) - taken, 0LL) : 0, &total);
        int2 cut = make_int2(tid == 0 ? 0 : line, 0);  // thread j: the end of share j - 1
        long long cost_at = tid == 0 ? 0 : -1;
        if (tid == 0 || tid >= shares) mine = -1;
        long long at = 0;
        for (int base = 0; base < line; base += kPlanThreads) {
            const int i = base + tid;
            const int tiles = i >= line ? 0 : fits ? lds[i].tiles : list.units[first + i].tiles;
            long long sum;
            const long long a = at + block_scan(i < line ? tiles + pass : 0, &sum);
            line_at[tid] = a, line_tiles[tid] = tiles;
            __syncthreads();
            if (mine >= at && mine < at + sum) {
                int lo = 0, hi = min(line - base, kPlanThreads) - 1;
                while (lo < hi) {  // the last unit that begins at or before the cut
                    const int mid = (lo + hi + 1) >> 1;
                    if (line_at[mid] <= mine) lo = mid;
                    else hi = mid - 1;
                }
                const long long in = mine - line_at[lo];
                const int n = line_tiles[lo], t = (int)min(in, (long long)n) & ~(turn - 1);
                // inside the unit, or at the end of it whose `keep` tiles it falls in (the nearer one, if it is
                // too short to be cut at all): later cuts never come before earlier ones
                const bool inside = t >= keep && t + keep <= n;
                const bool after = !inside && (n >= 2 * keep ? t >= keep : 2 * in >= n + pass);
                cut = make_int2(base + lo + after, inside ? t : 0);
                cost_at = line_at[lo] + (inside ? t : after ? n + pass : 0);
            }
            at += sum;
        }
        if (tid <= shares) cuts[tid] = cut, cut_cost[tid] = cost_at < 0 ? at : cost_at;  // (past the end: all of it)
        __syncthreads();
        if (tid < shares) {
            const int2 from = cuts[tid], to = cuts[tid + 1];
            taken += cut_cost[tid + 1] - cut_cost[tid];
            Share& x = list.shares[tid];
            x.first = from.x, x.first_tile = from.y, x.last = to.x, x.last_tile = to.y;
            if (first > 0) x.start = list.units[tid];
            else if (from.x < line) x.start = unit_at(from.x);
            int end = 0;
            if (to.y > 0 && !(from.x == to.x && from.y > 0)) {  // a unit begins here and goes on
                end = tid + 1;
                for (int hi = shares - 1; end < hi;) {  // to the last cut that is not past it
                    const int mid = (end + hi + 1) >> 1;
                    if (cuts[mid].x == to.x) end = mid;
                    else hi = mid - 1;
                }
                x.merge = unit_at(to.x);
            }
            x.merge_end = end;
        }
    }
    if (tid == 0) {
        int* h = reinterpret_cast<int*>(plan);
        h[0] = bad ? 0 : kPlanMagic;
        h[1] = n_seq, h[2] = rows, h[3] = H, h[4] = HKV;
        h[5] = kv_len == nullptr;
        h[kHeadRounds] = rounds, h[kHeadDealt] = dealt, h[kHeadLine] = U - dealt, h[kHeadFew] = (int)few;
        h[kHeadMaxKv] = max_kv;
    }
}

// ------------------------------------------------------------------ attention
// Wide units multiply on v_mfma_f32_32x32x16_f16 with every fp32 operand in two binary16 planes, x = h + l:
// h = f16(x) and l = f16(x - h), after a scaling by a power of two that brings the largest of its fellows
// to 2^14 .. 2^16: the residual is exact, and l keeps it to 2^-22 of x (2^-24.6 in the root mean square)
// or to 2^-25, 2^-39 of the largest, whichever is more.  Three of the four plane products are taken; l.l
// is at most 2^-22 of |a||b|, 2^-23.6 in the root mean square.  Together that is about what fp32 loses in
// adding 128 products, for half the matrix instructions of three bf16 planes (prefill.hip), which keep
// every bit.  The scalings:
//   q, with the softmax scale in it: per row, taken back in the exponent's FMA
//   K: per key, taken back in the scores (16 products per tile and lane), before q's
//   V: per 32 columns, the running largest value of the tiles so far; sums are rescaled when it grows
//   P: 2^14 against the row's reference, so that weights of up to 2^kLazy fit; the weights' sum has it too.  The
//     reference is the running maximum until a tile's largest score lies more than kWindow below it; then it
//     goes down after the tile.  (Behind a key that takes nearly all of the weight, 2^-39 of it, the planes' end, would
//     be 2^-13 of an ordinary weight.)  What its planes may still be off by is counted, 32 times 2^-25 a tile.
// What the planes of q and K lose at their lower end, 2^-39 of a row's largest value, is at most 2^-31 of the product
// of the two largest in a score, which shows where that product is large and the score is not (a channel of q far
// above the others that meets zeros, and one of K).  So a key's planes go up to the exponent at which its largest
// value times the unit's largest q is 2^13 (2^-18 of a log2 unit is left), and what is larger overflows, which is
// noticed; and up to kMostK, where the sum of 128 products of up to 2^32 is finite with K's scaling taken out: one that
// went to -infinity on the way would leave no trace.
// What the scalings of V and P cannot hold is noticed at the end of a pass (planes_failed) and multiplied in fp32.
//
// What bounds it: matrix and vector instructions follow one another.  8192, 4096, 2048, 1024, 300 and 17 rows (H 32 /
// HKV 8) take 2271 to 2334 us by box, 313 to 322 TFLOP/s, with the matrix unit busy 45% of the cycles and the other
// vector instructions (splits, softmax, scalings; four cycles each) another 37%, at 1.87 GHz of 2.4 under this load.
// With two products of three taken out 1530 us, with the loop's loads out 11% less, with the LDS reads out 3%; more
// fragments in flight, other interleavings of the splits and no priorities all came within 3%.  Three bf16 planes:
// 3370 us.
//
// A wave holds 32 flat query rows and computes S^T[key][row] = K . Q^T, so that each lane owns one row and
// 16 of a tile's 32 keys, and O^T[d][row] = V^T . P^T from the same registers.
//
// A workgroup of eight waves walks its share of a list pass by pass: a pass is a unit, or the part of it
// between two cuts of the list's line.  A part goes unnormalised to the workspace.
//
// Wide units (wide_pass): two key groups of four waves; a group's waves hold 32 rows
// each and share its tiles, which take turns (tile kt to group (kt - first) % 2).  The key loop is that
// of prefill.hip: each wave of a group fetches a quarter of a K or V tile, 16 floats per lane, and
// stores its planes in LDS (V transposed) while the group multiplies the other of the two; the groups
// run half an iteration apart, so that one has matrix work while the other is in its softmax.  Waves
// without rows repeat the sequence's last one and write nothing (a branch round their products costs the
// other waves registers).
//
// Few-row units (few_pass), single tokens and short drafts, read much and multiply little: every wave holds
// the same rows and a tile of its own, loaded straight into the operands' registers, and multiplies in
// fp32, which needs no planes.  (Both kinds of pass in one loop leave the compiler short of registers in
// both: a workgroup walks its wide units first, then its few-row ones.)
// lazy-rescale thresholds (log2 units): sums are rescaled when the running maximum has risen by more (for
// wide units, what a weight may pass 1 by comes off the range of its planes)
constexpr float kLazy = 1.f, kFewLazy = 8.f;
// Wide units' reference goes down where a tile's scores are all more than kWindow below it, to kWindow / 2 above them,
// as long as the sums stay below 2^kTopSum.  So a tile's largest weight is 2^2 or more, with its 2^14, and what its
// weights may be off by, 2^-20, shows only where their values are small too.  8192 rows (H 32 / HKV 8), scores of
// standard deviation 4: 1793 us (at 8 1843, never going down 1686); of 1: 1703 (1702, 1690).
constexpr float kWindow = 12.f;
constexpr int kTopSum = 64;
// the largest (biased) exponents of a query's planes, of a key's, and of both together
constexpr uint32_t kMostQ = 127 + 121, kMostK = 127 + 100, kMostQK = 2 * 127 + 10;
constexpr float kPBits = 14.f;                  // wide units' weights and sums are times 2^kPBits
constexpr int kXchF = 34;                       // floats per lane exchanged by the merge
// plane rows padded to an odd number of 16-byte pieces: the rows that an operand read takes, one per
// lane, spread over all LDS banks
constexpr int kKRowB = 2 * kHeadDim + 16, kKPlane = kKT * kKRowB;  // K plane: [32 keys][128 d] binary16
constexpr int kVRowB = 2 * kKT + 16, kVPlane = kHeadDim * kVRowB;  // V plane, transposed: [128 d][32 keys]
// LDS of a wide pass: the K planes of both groups, and the merge's exchange area, from 0; the V planes
// after it, and over them the staging area of the unit's rows (queries, later outputs); then the scalings,
// of K [group][tile parity][key] and of V [group][32 columns], each wave's largest q, each lane's Before.  Of a
// few-rows pass: every wave's rows, and their (m, l).
constexpr int kStageF = kWaves * kXchF * 64;
constexpr int kScaleK = kStageF + kUnitRows * kRowF, kScaleV = kScaleK + kGroups * 2 * kKT;
constexpr int kMaxQ = kScaleV + kGroups * 4, kBefore = kMaxQ + kWaves, kWideF = kBefore + 3 * kWaves * 64;
constexpr int kFewBlock = 16;                   // rows of one matrix instruction of few_pass
constexpr int kFewML = kWaves * kFewRows * kRowF;
constexpr int kFewF = kFewML + kWaves * kFewRows * 2;
static_assert(kWaves * 64 == kFewRows * 16, "sixteen threads stage a row");
static_assert(kSlots == 4, "a float4 of the largest q");
static_assert(kGroups * 2 * kKPlane <= kStageF * 4, "K planes below the staging area");
static_assert(kStageF * 4 + kGroups * 2 * kVPlane <= kScaleK * 4, "V planes within the LDS span");
static_assert(kWideF * 4 <= 160 * 1024 && kFewF * 4 <= 160 * 1024, "LDS budget");

// The visible rows of a tile as a buffer: reads past the last one, and of a missing page, give zeros (all
// reads, if the tile is not `wanted`).
template <bool kPaged>
__device__ __forceinline__ Rsrc tile_rsrc(const PackedArgs& a, const Pass& p, const float* cache, int t0, int page,
                                          bool wanted = true) {
    size_t row = (size_t)p.row0 + t0;
    int there = wanted ? min(kKT, p.T - t0) : 0;
    if constexpr (kPaged) {
        const bool ok = page >= 0 && page < a.n_blocks;
        row = ok ? ((size_t)page << a.bshift) | (size_t)(t0 & ((1 << a.bshift) - 1)) : 0;
        if (!ok) there = 0;
    }
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<float*>(cache) + row * a.kv_stride, 0,
        there ? (int)((uint32_t)(there - 1) * (uint32_t)(a.kv_stride * 4) + kHeadDim * 4) : 0, kBufferDword3);
}

struct Sums {  // of 32 rows, one per lane and its lane ^ 32: O^T, their reference (log2 units), sum of weights
    floatx16 o[4];
    float m, l;
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
        m = -INFINITY;
        l = 0.f;
    }
};

// What a row's sums leave behind where its reference goes down, kept in LDS, a float per lane of each: the weights' sum
// (small weights added to a sum that one key has nearly all of would be lost), the tiles summed so far, each counted as
// one of the reference it was summed against (or of a higher one), and the reference that both are in.
struct Before {
    float* at;
    int from;    // the tile at which a reference of the wave went down last
    float rest;  // of sums in fp32 alone, whose reference never does: what rounding has kept from the weights' sum
};
constexpr int kTiles = kWaves * 64, kRef = 2 * kWaves * 64;
__device__ __forceinline__ float moved(float from, float to) {  // a sum's factor for another reference
    return from == to ? 1.f : __builtin_amdgcn_exp2f(from - to);
}

// Scores s of tile kt (times sq: log2 units) -> P (in place; with planes times 2^kPBits) and its sum; O rescaled if the
// reference moves: to the tile's maximum, if that is higher by more than kLazy, and with planes down towards it
// (kWindow).  Tiles from nfull on cross the diagonal of the wave's rows.  The wave's i-th tile.
template <bool kPlanes, bool kTree>
__device__ __forceinline__ void softmax_tile(const PackedArgs& a, const Pass& p, Sums& x, floatx16& s, float sq, int kt,
                                             int nfull, int qpos, int hh, Before& before, int i) {
    if (kt >= nfull) {
        if constexpr (kTree) {
            const uint32_t bits = tree_bits(a, p, qpos, kt * kKT) >> (4 * hh);
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (!(bits >> (8 * (r >> 2) + (r & 3)) & 1)) s[r] = -INFINITY;
        } else {
            const int k0 = unhoisted(kt * kKT + 4 * hh);
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (k0 + 8 * (r >> 2) + (r & 3) > qpos) s[r] = -INFINITY;
        }
    }
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    const float ms = half_max(mx) * sq;
    const bool out = kPlanes ? __builtin_fabsf(ms - x.m + 0.5f * (kWindow - kLazy)) > 0.5f * (kWindow + kLazy)
                             : ms > x.m + kLazy;
    if (__builtin_amdgcn_ballot_w64(out)) {  // rare after the first tile
        float mn = fmaxf(x.m, ms);
        const bool down = kPlanes && ms < x.m - kWindow && ms > -INFINITY;
        if (kPlanes && __builtin_amdgcn_ballot_w64(down)) {
            const float by = moved(before.at[kRef], x.m);
            const float sum = __builtin_fmaf(before.at[0], by, x.l);
            const float tiles = __builtin_fmaf(before.at[kTiles], by, (float)(i - before.from));
            const int room = max(127 + kTopSum - (int)(__float_as_uint(half_max(sum)) >> 23), 0);
            if (down) mn = fmaxf(ms + 0.5f * kWindow, x.m - (float)room);
            const float now = moved(x.m, mn);
            before.at[0] = sum * now, before.at[kTiles] = tiles * now, before.at[kRef] = mn;
            before.from = i;
            x.l = 0.f;
        }
        if (!kPlanes || __builtin_amdgcn_ballot_w64(x.m != mn)) {  // (not for rows that see nothing of the tile)
            const float corr = moved(x.m, mn);
            x.l *= corr;
            if constexpr (!kPlanes) before.rest *= corr;
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) x.o[db][r] *= corr;
            x.m = mn;
        }
    }
    const float nb = x.m == -INFINITY ? 0.f : (kPlanes ? kPBits : 0.f) - x.m;
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], sq, nb));
        sum += s[r];
    }
    if constexpr (kPlanes) {
        x.l += sum;
    } else {
        const float l = x.l + sum;
        before.rest += sum > x.l ? x.l - (l - sum) : sum - (l - x.l);
        x.l = l;
    }
}

// ---- two binary16 planes
struct Halves {  // eight values: one MFMA operand per plane
    u32x4 h, l;
};
__device__ __forceinline__ floatx16 mfma_f16(u32x4 a, u32x4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}
__device__ __forceinline__ void mfma_halves(const Halves& a, const Halves& b, floatx16& c) {
    c = mfma_f16(a.l, b.h, c);
    c = mfma_f16(a.h, b.l, c);
    c = mfma_f16(a.h, b.h, c);
}
constexpr uint32_t kNoScale = 253u << 23;  // of columns that have been zero so far

// The planes of P's half x (registers 8x .. 8x + 7): the B operand of two steps' worth of keys.
__device__ __forceinline__ Halves split_p(const floatx16& s, int x) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) split_f16(s[8 * x + 2 * j], s[8 * x + 2 * j + 1], h[j], l[j]);
    return {u32x4{h[0], h[1], h[2], h[3]}, u32x4{l[0], l[1], l[2], l[3]}};
}

// Takes V's scalings and P's 2^kPBits out of the sums, and says whether the planes did not serve them:
//   - a sum is not finite (an infinite value or NaN in K or V, seen by the row or not, or q and K out of range);
//   - a row's sums are so small, against V's largest values on the way and the sum of weights, that the 2^-25 which
//     planes keep of scaled values of V may show (2^-22 of the row's largest sum);
//   - or so small that the 2^-25 which they keep of scaled weights may: 32 weights a tile, times values of up to 2^16
//     as scaled, together 2^-17 of the row's largest sum (`tiles`: see Before).
__device__ __forceinline__ bool planes_failed(Sums& x, const uint32_t (&scale)[4], float tiles) {
    constexpr float kOne = 0x1p-14f;
    static_assert(kPBits == 14.f, "kOne is its inverse");
    x.l *= kOne, tiles *= kOne;
    float l = half_sum(x.l);
    if (__builtin_amdgcn_ballot_w64(l > 0x1p26f)) {  // the reference went far down: up again, by a power of two
        const uint32_t e = l > 0x1p26f ? min(__float_as_uint(l) >> 23, 253u) : 127u;
        const float by = __uint_as_float((127u + 127u - e) << 23);
        l *= by, x.l *= by, tiles *= by;
        x.m += (float)((int)e - 127);
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) x.o[db][r] *= by;
    }
    float z = x.l * 0.f, most = 0.f, step = 0.f;
#pragma unroll
    for (int db = 0; db < 4; ++db) {
        const float inv = scale[db] == kNoScale ? 0.f : inverse(scale[db]);
        step = fmaxf(step, inv);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            z = __builtin_fmaf(x.o[db][r], 0.f, z);
            x.o[db][r] *= inv * kOne;
            most = fmaxf(most, __builtin_fabsf(x.o[db][r]));
        }
    }
    most = half_max(most);
    const bool small = l * step * 0x1p-25f > most * 0x1p-22f || (l > 0.f && tiles * step * 0x1p-4f > most * 0x1p-17f);
    return __builtin_amdgcn_ballot_w64(z != 0.f || small) != 0;
}

// A wave's tiles again, both products in fp32 from the cache.  In a tile that crosses the diagonal a
// value that a row does not see must not be multiplied at all (0 times infinity), and the matrix
// instruction takes every row with every key: P . V goes key by key there, P through p_lds, 32 x 32
// floats of the wave's own.
template <bool kTree, typename KTile, typename VTile, typename Index>
__device__ __forceinline__ void redo_fp32(Sums& x, const PackedArgs& a, const Pass& p, const float* q_row, float sl2,
                                          int n_mine, KTile k_tile, VTile v_tile, Index index, int nfull, int qpos,
                                          uint32_t row_bytes, float* p_lds, int lane) {
    const int col = lane & 31, hh = lane >> 5;
    // values 16t + 8hh .. + 7 of the row
    float q[64];
#pragma unroll
    for (int t = 0; t < 16; ++t) {
        const float4 v = *reinterpret_cast<const float4*>(q_row + 16 * (t >> 1) + 4 * (t & 1) + 8 * hh);
        q[4 * t] = v.x * sl2, q[4 * t + 1] = v.y * sl2, q[4 * t + 2] = v.z * sl2, q[4 * t + 3] = v.w * sl2;
    }
    x.clear();
    Before before{};
    for (int i = 0; i < n_mine; ++i) {
        const int kt = index(i);
        floatx16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
        {
            const Rsrc rs = k_tile(i);
            const uint32_t off = unhoisted(col) * row_bytes + 32u * hh;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // d = 16t + 8hh + 2j and the next
                    const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(rs, off + 64 * t + 8 * j, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(v.x), q[8 * t + 2 * j], s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(v.y), q[8 * t + 2 * j + 1], s, 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        softmax_tile<false, kTree>(a, p, x, s, 1.f, kt, nfull, qpos, hh, before, i);
        const Rsrc rs = v_tile(i);
        if (kt < nfull) {
            const uint32_t off = unhoisted(4 * hh) * row_bytes + 4u * col;
#pragma unroll
            for (int r = 0; r < 16; ++r) {  // lane half hh: key 8(r/4) + 4hh + r%4
#pragma unroll
                for (int db = 0; db < 4; ++db) {
                    const float v = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                        rs, off + (8 * (r >> 2) + (r & 3)) * row_bytes + 128 * db, 0, 0));
                    x.o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, s[r], x.o[db], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            continue;
        }
        const int ln = unhoisted(lane);
        float* pw = p_lds + (ln & 31);
#pragma unroll
        for (int r = 0; r < 16; ++r) pw[32 * (8 * (r >> 2) + 4 * (ln >> 5) + (r & 3))] = s[r];
        __builtin_amdgcn_wave_barrier();
        uint32_t bits = 0;
        if constexpr (kTree) bits = tree_bits(a, p, qpos, kt * kKT);
#pragma unroll 1
        for (int key = 0; key < kKT; ++key) {
            const float pk = pw[32 * key];
            const uint32_t off = key * row_bytes + 16u * (ln >> 5);
            if (kTree ? (bits >> key & 1) != 0 : kt * kKT + key <= qpos) {
#pragma unroll
                for (int db = 0; db < 4; ++db) {
#pragma unroll
                    for (int y = 0; y < 4; ++y) {  // d = 32 db + 8y + 4hh + 0 .. 3
                        const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rs, off + 128 * db + 32 * y, 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            x.o[db][4 * y + e] = __builtin_fmaf(pk, __uint_as_float(v[e]), x.o[db][4 * y + e]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    x.l += before.rest;
}

// ---- a wide unit
template <bool kPaged, bool kTree>
__device__ __forceinline__ void wide_pass(const PackedArgs& a, const Pass& p, int kvh, FastDiv fG, float sl2,
                                          float* smem) {
    constexpr int D = kHeadDim;
    // (what follows from the thread's number is computed in each pass: kept over passes it would spill)
    const int tid = unhoisted(threadIdx.x), lane = tid & 63, w = tid >> 6;
    const int wu = scalar(w), hw = wu % kSlots, grp = wu / kSlots;
    const int col = lane & 31, hh = lane >> 5;
    const int G = (int)fG.d;
    const uint32_t row_bytes = (uint32_t)(a.kv_stride * 4);
    char* const lds = reinterpret_cast<char*>(smem);
    char* const kpl = lds + grp * 2 * kKPlane;
    char* const vpl = lds + kStageF * 4 + grp * 2 * kVPlane;
    float* const stage = smem + kStageF;
    float* const k_scale = smem + kScaleK + grp * 2 * kKT;
    uint32_t* const v_scale = reinterpret_cast<uint32_t*>(smem + kScaleV) + grp * 4;
    const uint32_t voff_k = (uint32_t)(8 * hw + (lane >> 3)) * row_bytes + 32u * (lane & 7);
    const uint32_t voff_v =
        (uint32_t)(16 * (lane >> 5) + 4 * ((lane >> 4) & 1)) * row_bytes + 4u * (32 * hw + 2 * (lane & 15));
    const int f0 = kUnitRows * p.u + kQB * hw;  // this wave's first row
    const bool live = f0 < p.nflat;
    const int qpos = p.pos0 + fdiv(min(f0 + col, p.nflat - 1), fG);  // this lane's query
    // tiles below the wave's diagonal (before a tree)
    const int nfull = max(kTree ? p.pos0 : p.pos0 + fdiv(min(f0, p.nflat - 1), fG) + 1, 0) / kKT;
    const int n_it = (p.nrange + kGroups - 1) / kGroups, n_mine = (p.nrange - grp + kGroups - 1) / kGroups;
    auto index = [&](int i) { return p.kt_lo + kGroups * i + grp; };
    auto page = [&](int i) { return page_of<kPaged>(a, p, index(i) * kKT); };
    auto k_tile = [&](int i, int pg) { return tile_rsrc<kPaged>(a, p, a.k + (size_t)kvh * D, index(i) * kKT, pg); };
    auto v_tile = [&](int i, int pg) { return tile_rsrc<kPaged>(a, p, a.v + (size_t)kvh * D, index(i) * kKT, pg); };

    // K and V of this group's i-th tile, a quarter per wave:
    //   K: row 8*hw + lane/8, d = 8c .. 8c+7 and 64 + 8c .. (c = lane%8)
    //   V: d = 32*hw + 2*(lane%16) and the next, the eight keys of chunk lane/16 (step s = chunk/2,
    //     half hh = chunk%2 of the P.V operand: keys 16s + 4hh + {0..3, 8..11})
    float rg[16];
    auto load_k = [&](int i, int pg) {
        const Rsrc rs = k_tile(i, pg);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rs, voff_k + 256 * (j >> 1) + 16 * (j & 1), 0, 0);
            rg[4 * j] = __uint_as_float(v.x), rg[4 * j + 1] = __uint_as_float(v.y);
            rg[4 * j + 2] = __uint_as_float(v.z), rg[4 * j + 3] = __uint_as_float(v.w);
        }
    };
    auto load_v = [&](int i, int pg) {
        const Rsrc rs = v_tile(i, pg);
        const uint32_t off = unhoisted(voff_v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(rs, off + (8 * (j >> 2) + (j & 3)) * row_bytes, 0, 0);
            rg[2 * j] = __uint_as_float(v.x), rg[2 * j + 1] = __uint_as_float(v.y);
        }
    };
    auto largest = [&]() {
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) most = fmaxf(most, __builtin_fabsf(rg[j]));
        return most;
    };
    // half x of the conversion of rg, eight values, one 16-byte piece of each plane; the first half finds the
    // scaling: of K the row's, of V the running one of the wave's 32 columns (twice its largest value
    // fits, so it changes rarely)
    float fk;
    uint32_t k_limit;
    auto conv_k = [&](int x, int parity) {
        uint32_t ch[4], cl[4];
        if (x == 0) {
            float most = largest();
            most = fmaxf(most, lane_xor1(most));
            most = fmaxf(most, lane_xor2(most));
            most = fmaxf(most, lane_xor4(most));
            const uint32_t f = scale_to<14>(most, k_limit);
            fk = __uint_as_float(f);
            if ((lane & 7) == 0) k_scale[kKT * parity + 8 * hw + (lane >> 3)] = inverse(f);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) split_f16(rg[8 * x + 2 * j] * fk, rg[8 * x + 2 * j + 1] * fk, ch[j], cl[j]);
        char* d = kpl + (8 * hw + (lane >> 3)) * kKRowB + 16 * (lane & 7) + 128 * x;
        *reinterpret_cast<u32x4*>(d) = u32x4{ch[0], ch[1], ch[2], ch[3]};
        *reinterpret_cast<u32x4*>(d + kKPlane) = u32x4{cl[0], cl[1], cl[2], cl[3]};
    };
    uint32_t fv = kNoScale;
    float limit = 0.f;
    auto conv_v = [&](int x) {  // d + x
        uint32_t ch[4], cl[4];
        if (x == 0) {
            const float most = largest();
            if (__builtin_amdgcn_ballot_w64(most > limit)) {
                fv = scalar(scale_to<14>(wave_max(most)));
                limit = uniform(65000.f * inverse(fv));
            }
            if (lane == 0) v_scale[hw] = fv;
        }
        const float f = __uint_as_float(fv);
#pragma unroll
        for (int j = 0; j < 4; ++j) split_f16(rg[4 * j + x] * f, rg[4 * j + 2 + x] * f, ch[j], cl[j]);
        char* d = vpl + (32 * hw + 2 * (lane & 15) + x) * kVRowB + 16 * (lane >> 4);
        *reinterpret_cast<u32x4*>(d) = u32x4{ch[0], ch[1], ch[2], ch[3]};
        *reinterpret_cast<u32x4*>(d + kVPlane) = u32x4{cl[0], cl[1], cl[2], cl[3]};
    };
    auto k_frag = [&](int t) {  // K[key col][16t + 8hh ..]
        const char* k = kpl + col * kKRowB + 16 * hh + 32 * t;
        return Halves{*reinterpret_cast<const u32x4*>(k), *reinterpret_cast<const u32x4*>(k + kKPlane)};
    };
    auto v_frag = [&](int x) {  // step s = x/4, d = 32 (x%4) + col
        const char* v = vpl + (32 * (x & 3) + col) * kVRowB + 32 * (x >> 2) + 16 * hh;
        return Halves{*reinterpret_cast<const u32x4*>(v), *reinterpret_cast<const u32x4*>(v + kVPlane)};
    };

    // the unit's query rows by LDS DMA, once for both groups: wave wu rows 16*wu .. of the unit
    // (rows past the sequence repeat its last), 512 contiguous bytes each
    {
        int f = min(kUnitRows * p.u + (kQB / 2) * wu, p.nflat - 1);
        const int t0 = fdiv(f, fG);
        int g = f - t0 * G;
        uint64_t sb = (uint64_t)(uintptr_t)(a.q + ((size_t)p.row0 + t0) * a.q_stride + (size_t)(kvh * G + g) * D);
        const uint64_t next = (uint64_t)((a.q_stride - (long)(G - 1) * D) * 4);
        const uint32_t lb = scalar((int)lds_addr(stage + (kQB / 2) * wu * kRowF));
        if (hh == 0) {
#pragma unroll
            for (int j = 0; j < kQB / 2; ++j) {
                dma16_s(sb, 16u * col, lb + j * (kRowF * 4));
                if (f + 1 < p.nflat) {
                    ++f;
                    ++g;
                    sb += g == G ? next : (uint64_t)(D * 4);
                    if (g == G) g = 0;
                }
            }
        }
    }
    int pg = page(0);  // of the tile that is loaded next
    if (n_mine > 0) load_k(0, pg);
    wait_vmcnt<0>();
    lds_barrier();
    Halves qp[8];
    float sq;  // takes the row's scaling out of its scores
    {
        const float* qs = stage + (hw * kQB + col) * kRowF + 8 * hh;
        float most = 0.f;
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            const float4 v = *reinterpret_cast<const float4*>(qs + 16 * (t >> 1) + 4 * (t & 1));
            most = fmaxf(fmaxf(most, __builtin_fabsf(v.x * sl2)), __builtin_fabsf(v.y * sl2));
            most = fmaxf(fmaxf(most, __builtin_fabsf(v.z * sl2)), __builtin_fabsf(v.w * sl2));
        }
        most = half_max(most);
        const uint32_t f = scale_to<14>(most, kMostQ);
        const float fq = __uint_as_float(f);
        sq = inverse(f);
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const float4 u = *reinterpret_cast<const float4*>(qs + 16 * t);
            const float4 v = *reinterpret_cast<const float4*>(qs + 16 * t + 4);
            uint32_t h[4], l[4];
            split_f16(u.x * sl2 * fq, u.y * sl2 * fq, h[0], l[0]);
            split_f16(u.z * sl2 * fq, u.w * sl2 * fq, h[1], l[1]);
            split_f16(v.x * sl2 * fq, v.y * sl2 * fq, h[2], l[2]);
            split_f16(v.z * sl2 * fq, v.w * sl2 * fq, h[3], l[3]);
            qp[t] = {u32x4{h[0], h[1], h[2], h[3]}, u32x4{l[0], l[1], l[2], l[3]}};
        }
        // the unit's largest q, from the group's four waves, sets how large a key's planes may be
        most = wave_max(most);
        if (lane == 0) smem[kMaxQ + wu] = most;
        lds_barrier();
        const float4 m = *reinterpret_cast<const float4*>(smem + kMaxQ + kSlots * grp);
        const float unit = fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w));
        k_limit = scalar(min(kMostQK - min(max(__float_as_uint(unit) >> 23, 16u), kMostQ), kMostK));
    }
    if (n_mine > 0) {
#pragma unroll
        for (int x = 0; x < 2; ++x) conv_k(x, 0);
        load_v(0, pg);
        pg = page(1);
    }
    Sums x;
    x.clear();
    uint32_t scale[4] = {kNoScale, kNoScale, kNoScale, kNoScale};  // V's, as the sums have it
    Before before{smem + kBefore + tid, 0, 0.f};
    before.at[0] = before.at[kTiles] = 0.f;
    before.at[kRef] = -INFINITY;
    lds_barrier();  // every wave has its q (the staging area is free for the V planes); K planes stored
    if (grp == 1) lds_barrier();
    for (int i = 0; i < n_it; ++i) {
        floatx16 s;
        if (i < n_mine) {
            // S^T = K . Q^T, while V(i) goes to its planes; then K(i+1) is fetched
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
            Halves kf[2];
            kf[0] = k_frag(0);
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                if (t < 7) kf[(t + 1) & 1] = k_frag(t + 1);
                if (t == 2 || t == 4) conv_v(t == 4);
                mfma_halves(kf[t & 1], qp[t], s);
            }
            if (i + 1 < n_mine) load_k(i + 1, pg);
            const float* ks = k_scale + kKT * (i & 1) + 4 * hh;
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const float4 f = *reinterpret_cast<const float4*>(ks + 2 * r);
                s[r] *= f.x, s[r + 1] *= f.y, s[r + 2] *= f.z, s[r + 3] *= f.w;
            }
        }
        lds_barrier();
        if (i < n_mine) {
            __builtin_amdgcn_s_setprio(1);
            const u32x4 f = *reinterpret_cast<const u32x4*>(v_scale);
#pragma unroll
            for (int db = 0; db < 4; ++db) {
                const uint32_t now = scalar(f[db]);
                if (now != scale[db]) {  // rare after the first tile
                    const float by = __uint_as_float(now) * inverse(scale[db]);
#pragma unroll
                    for (int r = 0; r < 16; ++r) x.o[db][r] *= by;
                    scale[db] = now;
                }
            }
            softmax_tile<true, kTree>(a, p, x, s, sq, index(i), nfull, qpos, hh, before, i);
            // O^T += V^T . P^T, while K(i+1) goes to its planes; then V(i+1) is fetched
            const bool more = i + 1 < n_mine;
            Halves vf[2], pp;
            vf[0] = v_frag(0);
#pragma unroll
            for (int y = 0; y < 8; ++y) {
                if ((y & 3) == 0) pp = split_p(s, y >> 2);
                if (y < 7) vf[(y + 1) & 1] = v_frag(y + 1);
                if (y == 4 || y == 6) conv_k(y == 6, (i + 1) & 1);
                mfma_halves(vf[y & 1], pp, x.o[y & 3]);
            }
            if (more) load_v(i + 1, pg);
            pg = page(i + 2);  // (looked up here, its wait is the barrier's)
            __builtin_amdgcn_s_setprio(0);
        }
        lds_barrier();
    }
    if (grp == 0) lds_barrier();

    const float by = moved(before.at[kRef], x.m);
    x.l = __builtin_fmaf(before.at[0], by, x.l);
    if (planes_failed(x, scale, __builtin_fmaf(before.at[kTiles], by, (float)(n_mine - before.from))) && live) {
        const int f = min(f0 + col, p.nflat - 1), t0 = fdiv(f, fG);
        const float* q_row = a.q + ((size_t)p.row0 + t0) * a.q_stride + (size_t)(kvh * G + f - t0 * G) * D;
        redo_fp32<kTree>(
            x, a, p, q_row, sl2, n_mine, [&](int i) { return k_tile(i, page(i)); },
            [&](int i) { return v_tile(i, page(i)); }, index, nfull, qpos, row_bytes,
                  smem + w * (kXchF * 64), lane);
    }

    // ---- the key groups meet through LDS (tile buffers are free after the barrier): group g finishes
    // output blocks db = 2g, 2g+1 and hands the other two to its partner
    float* xw = smem + w * (kXchF * 64) + lane;
    xw[0] = x.m;
    xw[64] = x.l;
    // (grp is wave-uniform: selects, not a dynamic register index)
    const floatx16 give0 = grp ? x.o[0] : x.o[2], give1 = grp ? x.o[1] : x.o[3];
    const floatx16 keep0 = grp ? x.o[2] : x.o[0], keep1 = grp ? x.o[3] : x.o[1];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        xw[(2 + i) * 64] = give0[i];
        xw[(18 + i) * 64] = give1[i];
    }
    lds_barrier();
    const float* xp = smem + ((1 - grp) * kSlots + hw) * (kXchF * 64) + lane;
    const float mp = xp[0], lp = xp[64];
    const float mt = fmaxf(x.m, mp);  // (references) -inf only when the pass holds no visible key for the row
    const float c0 = x.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.m - mt);
    const float cp = mp == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mp - mt);
    const float l = half_sum(x.l * c0 + lp * cp);
    {
        // finished rows (normalised; a row that sees no key: zeros), or the part's, to the staging area
        bool none = qpos < 0;
        if constexpr (kTree) none = l == 0.f && tree_sees_none(a, p.row0, p.pos0, qpos - p.pos0);
        const float inv = p.part ? 1.f : none ? 0.f : 1.f / l;
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
        if (p.part && hh == 0 && grp == 0)
            *reinterpret_cast<float2*>(p.part + kUnitRows * D + 2 * (hw * kQB + col)) = make_float2(mt, l);
    }
    lds_barrier();
    {
        const int ln = unhoisted(lane), c4 = 4 * (ln & 31);
#pragma unroll
        for (int j = 0; j < kQB / 4; ++j) {  // wave wu: rows 16*wu .. of the unit, two per instruction
            const int jj = (kQB / 2) * wu + 2 * j + (ln >> 5), f = kUnitRows * p.u + jj;
            const float4 v = *reinterpret_cast<const float4*>(stage + jj * kRowF + c4);
            const int t0 = fdiv(f, fG);
            float* dst = p.part ? p.part + jj * D : a.out + (((size_t)p.row0 + t0) * a.H + kvh * G + f - t0 * G) * D;
            if (f < p.nflat) *reinterpret_cast<float4*>(dst + c4) = v;
        }
    }
}

// ---- a unit of few rows
// On v_mfma_f32_16x16x4_f32: S^T[key][row] = K . Q^T and O^T[d][row] = V^T . P^T for kBlocks sixteens of
// rows; lane = row l % 16 of each, quarter l / 16.  Of a tile's half kb a lane holds the scores of the keys
// 16 kb + 4 quarter + r (r = 0 .. 3), which are the operand of P . V for the steps (kb, r): step by step a
// quarter of the lanes takes each of four keys.  K: step (x, e) takes d = 16x + 4 quarter + e, so that a
// lane's row comes in 16-byte pieces; V: a lane's pieces hold d = 64y + 4 (l % 16) + e, sum 4y + e takes
// element e.  Pieces of the next tile are fetched as this one's are used up.
//
// kQuad: four more rows (or the only ones), row l % 4 of them, on v_mfma_f32_4x4x1_16b_f32 from the same K and V
// registers, at a quarter of the time: its block l / 4 holds keys 4 (l/4 % 4) .. + 3 of the half for the scores,
// the same of d for O, and the quarters' products (of d, of keys) are summed afterwards.
//
// Single tokens are bound by reading K and V: 24 sequences of 57000 keys in all (H 16 / HKV 8, pages of 64),
// 494 MB in 87 to 91 us, 5.4 to 5.7 TB/s.  Where sequences share their keys and have more rows it is the matrix
// instructions and what a pass does once: 16 drafts of 5 tokens after 1024 shared keys and up to 555 more (H 32 / HKV 8)
// 41 us.
// By rows (H 32 / HKV 8, 32 sequences of 480 keys, with the merge): four 26.2 us (27.1 as sixteen), sixteen 27
// (37 as 32), twenty 32.3 (35.5 as 32), 32 rows 36 (44 as a wide unit; of 4067 keys 192 against 297; single
// tokens as wide units 44, and of 4059 keys 290 against 179).
template <bool kPaged, bool kTree, int kBlocks, bool kQuad>
__device__ __forceinline__ void few_pass(const PackedArgs& a, const Pass& p, int kvh, FastDiv fG, float sl2,
                                         float* smem) {
    constexpr int D = kHeadDim, kSets = kBlocks + kQuad, kRows = kFewBlock * kBlocks + 4 * kQuad;
    const int tid = unhoisted(threadIdx.x), lane = tid & 63, wu = scalar(tid >> 6);
    const int j = lane & 15, quarter = lane >> 4;
    const int G = (int)fG.d;
    const uint32_t row_bytes = (uint32_t)(a.kv_stride * 4);
    const int f0 = kUnitRows * p.u, last = p.nflat - 1, rows = p.nflat - f0;
    const int nfull = max(kTree ? p.pos0 : p.pos0 + fdiv(f0, fG) + 1, 0) / kKT;
    const int n_mine = (p.nrange - wu + kWaves - 1) / kWaves;
    auto index = [&](int i) { return p.kt_lo + kWaves * i + wu; };
    auto page = [&](int i) { return page_of<kPaged>(a, p, index(i) * kKT); };
    auto k_tile = [&](int i, int pg, bool wanted = true) {
        return tile_rsrc<kPaged>(a, p, a.k + (size_t)kvh * D, index(i) * kKT, pg, wanted);
    };
    auto v_tile = [&](int i, int pg, bool wanted = true) {
        return tile_rsrc<kPaged>(a, p, a.v + (size_t)kvh * D, index(i) * kKT, pg, wanted);
    };
    u32x4 kr[2][8], vr[8][2];
    auto load_k = [&](const Rsrc& rs, int x, uint32_t off) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
            kr[kb][x] = __builtin_amdgcn_raw_buffer_load_b128(rs, off + 16 * kb * row_bytes + 64 * x, 0, 0);
    };
    auto k_offset = [&]() {
        const uint32_t ln = lane_now();
        return (ln & 15) * row_bytes + (ln & 48);
    };
    auto load_v = [&](const Rsrc& rs, int t, uint32_t off) {
        const uint32_t at = off + (uint32_t)(16 * (t >> 2) + (t & 3)) * row_bytes;
        vr[t][0] = __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, 0);
        vr[t][1] = __builtin_amdgcn_raw_buffer_load_b128(rs, at + 256, 0, 0);
    };
    auto v_offset = [&]() {
        const uint32_t ln = lane_now();
        return (ln >> 4) * 4 * row_bytes + 16 * (ln & 15);
    };
    int pg = page(0);  // of the tile that is loaded next
    // q first (a wait for it is not one for the tiles), by the first rows' lanes; more than sixteen rows' goes
    // through LDS (registers), [row][d]
    auto quad = [](int rb) { return rb == kBlocks; };  // the set of four
    auto row_of = [&](int rb) { return kFewBlock * rb + (quad(rb) ? j & 3 : j); };
    int qpos[kSets];  // (rows past the last repeat it)
#pragma unroll
    for (int rb = 0; rb < kSets; ++rb) qpos[rb] = p.pos0 + fdiv(min(f0 + row_of(rb), last), fG);
    auto q_row = [&](int f) {
        const int tok = fdiv(f, fG);
        return a.q + ((size_t)p.row0 + tok) * a.q_stride + (size_t)(kvh * G + f - tok * G) * D;
    };
    float4 q_raw[kSets == 1 ? 8 : 2];
    if constexpr (kSets == 1) {
        const float* src = q_row(min(f0 + row_of(0), last)) + 4 * quarter;
#pragma unroll
        for (int x = 0; x < 8; ++x) q_raw[x] = *reinterpret_cast<const float4*>(src + 16 * x);
    } else {
        const float* src = q_row(min(f0 + (tid >> 4), last)) + 8 * (tid & 15);
        q_raw[0] = *reinterpret_cast<const float4*>(src);
        q_raw[1] = *reinterpret_cast<const float4*>(src + 4);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (n_mine > 0) {
        const Rsrc rk = k_tile(0, pg), rv = v_tile(0, pg);
#pragma unroll
        for (int x = 0; x < 8; ++x) load_k(rk, x, k_offset());
#pragma unroll
        for (int t = 0; t < 8; ++t) load_v(rv, t, v_offset());
        pg = page(1);
    }
    auto scaled = [&](const float4& v) { return f32x4{v.x * sl2, v.y * sl2, v.z * sl2, v.w * sl2}; };
    f32x4 q[kSets == 1 ? 8 : 1];
    if constexpr (kSets == 1) {
#pragma unroll
        for (int x = 0; x < 8; ++x) q[x] = scaled(q_raw[x]);
    } else {
        float* dst = smem + (tid >> 4) * kRowF + 8 * (tid & 15);
        *reinterpret_cast<f32x4*>(dst) = scaled(q_raw[0]);
        *reinterpret_cast<f32x4*>(dst + 4) = scaled(q_raw[1]);
        lds_barrier();
    }
    auto q_at = [&](int rb, int x) -> f32x4 {
        if constexpr (kSets == 1) return q[x];
        else return *reinterpret_cast<const f32x4*>(smem + row_of(rb) * kRowF + 16 * x + 4 * quarter);
    };
    f32x4 o[kSets][8];
    float m[kSets], l[kSets];
#pragma unroll
    for (int rb = 0; rb < kSets; ++rb) {
#pragma unroll
        for (int y = 0; y < 8; ++y) o[rb][y] = f32x4{0.f, 0.f, 0.f, 0.f};
        m[rb] = -INFINITY;
        l[rb] = 0.f;
    }
    auto mma = [&](int rb, uint32_t x, float y, f32x4 c) {
        return quad(rb) ? __builtin_amdgcn_mfma_f32_4x4x1f32(__uint_as_float(x), y, c, 0, 0, 0)
                        : __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x), y, c, 0, 0, 0);
    };
    for (int i = 0; i < n_mine; ++i) {
        const bool more = i + 1 < n_mine;
        const int kt = index(i);
        const Rsrc rk = k_tile(more ? i + 1 : i, pg, more), rv = v_tile(more ? i + 1 : i, pg, more);
        f32x4 s[kSets][2];
#pragma unroll
        for (int rb = 0; rb < kSets; ++rb) s[rb][0] = s[rb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
        const uint32_t off_k = k_offset();
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            f32x4 qx[kSets];
#pragma unroll
            for (int rb = 0; rb < kSets; ++rb) qx[rb] = q_at(rb, x);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int rb = 0; rb < kSets; ++rb)
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
                        s[rb][kb] = mma(rb, kr[kb][x][e], qx[rb][e], s[rb][kb]);
            __builtin_amdgcn_sched_barrier(0);
            load_k(rk, x, off_k);
        }
#pragma unroll
        for (int rb = 0; rb < kSets; ++rb) {
            if (quad(rb)) {  // the quarters' sums, then each quarter its four keys of every sixteen
                const int from = 4 * (20 * quarter + (lane & 3));
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    float v = s[rb][r >> 2][r & 3];
                    v += lane_xor16(v);
                    v += lane_xor32(v);
                    s[rb][r >> 2][r & 3] =
                        __uint_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_uint(v)));
                }
            }
            if (kt >= nfull) {
                if constexpr (kTree) {
                    const uint32_t bits = tree_bits(a, p, qpos[rb], kt * kKT) >> (4 * quarter);
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (!(bits >> (16 * (r >> 2) + (r & 3)) & 1)) s[rb][r >> 2][r & 3] = -INFINITY;
                } else {
                    const int k0 = unhoisted(kt * kKT + 4 * quarter);
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (k0 + 16 * (r >> 2) + (r & 3) > qpos[rb]) s[rb][r >> 2][r & 3] = -INFINITY;
                }
            }
            float mx = s[rb][0][0];
#pragma unroll
            for (int r = 1; r < 8; ++r) mx = fmaxf(mx, s[rb][r >> 2][r & 3]);
            mx = half_max(fmaxf(mx, lane_xor16(mx)));
            if (__builtin_amdgcn_ballot_w64(mx > m[rb] + kFewLazy)) {  // rare after the first tile
                const float mn = fmaxf(m[rb], mx);
                const float corr = m[rb] == mn ? 1.f : __builtin_amdgcn_exp2f(m[rb] - mn);
                l[rb] *= corr;
#pragma unroll
                for (int y = 0; y < 8; ++y)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[rb][y][r] *= corr;
                m[rb] = mn;
            }
            const float nb = m[rb] == -INFINITY ? 0.f : -m[rb];
            float sum = 0.f;  // (the tile's first: small weights would be lost one by one beside a large one)
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                s[rb][r >> 2][r & 3] = __builtin_amdgcn_exp2f(s[rb][r >> 2][r & 3] + nb);
                sum += s[rb][r >> 2][r & 3];
            }
            l[rb] += sum;
        }
        const uint32_t off_v = v_offset();
        pg = page(i + 2);
#pragma unroll
        for (int t = 0; t < 8; ++t) {
#pragma unroll
            for (int rb = 0; rb < kSets; ++rb)
#pragma unroll
                for (int y = 0; y < 8; ++y)
                    o[rb][y] = mma(rb, vr[t][y >> 2][y & 3], s[rb][t >> 2][t & 3], o[rb][y]);
            __builtin_amdgcn_sched_barrier(0);
            load_v(rv, t, off_v);
        }
    }
    // A sum that is not finite: an infinite value or NaN among the keys, seen by the row or not (the matrix
    // instruction multiplies every row with every key, and 0 times infinity is NaN).  The wave then takes
    // its tiles again, key by key: a lane has 32 products of its row's score and 32 columns of its sums.
    {
        float z = 0.f;
#pragma unroll
        for (int rb = 0; rb < kSets; ++rb) {
            z = __builtin_fmaf(l[rb], 0.f, z);
#pragma unroll
            for (int y = 0; y < 8; ++y)
#pragma unroll
                for (int r = 0; r < 4; ++r) z = __builtin_fmaf(o[rb][y][r], 0.f, z);
        }
        if (__builtin_amdgcn_ballot_w64(z != 0.f)) {
#pragma unroll
            for (int rb = 0; rb < kSets; ++rb) {
#pragma unroll
                for (int y = 0; y < 8; ++y) o[rb][y] = f32x4{0.f, 0.f, 0.f, 0.f};
                m[rb] = -INFINITY;
                l[rb] = 0.f;
#pragma unroll 1
                for (int c = 0; c < n_mine * kKT; ++c) {
                    const int at = page(c / kKT);
                    const Rsrc rk = k_tile(c / kKT, at), rv = v_tile(c / kKT, at);
                    const uint32_t row = (uint32_t)(c % kKT) * row_bytes;
                    if constexpr (kTree) {
                        if (!(tree_bits(a, p, qpos[rb], index(c / kKT) * kKT) >> (c % kKT) & 1)) continue;
                    } else if (index(c / kKT) * kKT + c % kKT > qpos[rb]) continue;
                    float dot = 0.f;
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const u32x4 k = __builtin_amdgcn_raw_buffer_load_b128(rk, row + 16 * quarter + 64 * x, 0, 0);
                        const f32x4 qx = q_at(rb, x);
#pragma unroll
                        for (int e = 0; e < 4; ++e) dot = __builtin_fmaf(__uint_as_float(k[e]), qx[e], dot);
                    }
                    // (the four lanes of a row see the same keys: the exchange stays among active lanes)
                    dot += lane_xor16(dot);
                    dot += lane_xor32(dot);
                    const float mn = fmaxf(m[rb], dot);
                    const float corr = m[rb] == mn ? 1.f : __builtin_amdgcn_exp2f(m[rb] - mn);
                    const float w = __builtin_amdgcn_exp2f(dot - (mn == -INFINITY ? 0.f : mn));
                    m[rb] = mn;
                    l[rb] = quarter == 0 ? l[rb] * corr + w : 0.f;  // (summed over the quarters below)
                    if (quad(rb) && quarter > 0) continue;          // (the sums too)
                    const int part = quad(rb) ? j >> 2 : quarter;
#pragma unroll
                    for (int x = 0; x < 8; ++x) {  // d = 64 (x/4) + 16 part + 4 (x%4) + e
                        const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(
                            rv, row + 64 * part + 256 * (x >> 2) + 16 * (x & 3), 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            f32x4& sum = o[rb][4 * (x >> 2) + e];
                            sum[x & 3] = __builtin_fmaf(w, __uint_as_float(v[e]), sum[x & 3] * corr);
                        }
                    }
                }
            }
        }
    }
    // every wave's rows meet: register r of sum 4y + e is d = 64y + 16 quarter + 4r + e
    if constexpr (kSets > 1) lds_barrier();  // q has been read
    float* const mine = smem + wu * (kRows * kRowF);
    float* const ml_at = smem + kFewML;
#pragma unroll
    for (int rb = 0; rb < kSets; ++rb) {
        const float sum = half_sum(l[rb] + lane_xor16(l[rb]));
        const int row = row_of(rb);
        if (quad(rb)) {
            // register r of sum 4y + e is d = 64y + 16 (j / 4) + 4r + e there, over a quarter's keys: quarter r of
            // the lanes sums and writes it, handing on the others
            float sums[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) {
                float half[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float lo = o[rb][y][2 * i], hi = o[rb][y][2 * i + 1];
                    half[i] = (quarter & 1 ? hi : lo) + lane_xor16(quarter & 1 ? lo : hi);
                }
                sums[y] = (quarter & 2 ? half[1] : half[0]) + lane_xor32(quarter & 2 ? half[0] : half[1]);
            }
#pragma unroll
            for (int y = 0; y < 2; ++y)
                *reinterpret_cast<float4*>(mine + row * kRowF + 64 * y + 16 * (j >> 2) + 4 * quarter) =
                    make_float4(sums[4 * y], sums[4 * y + 1], sums[4 * y + 2], sums[4 * y + 3]);
        } else {
#pragma unroll
            for (int x = 0; x < 8; ++x)
                *reinterpret_cast<float4*>(mine + row * kRowF + 64 * (x >> 2) + 16 * quarter + 4 * (x & 3)) =
                    make_float4(o[rb][4 * (x >> 2)][x & 3], o[rb][4 * (x >> 2) + 1][x & 3],
                                o[rb][4 * (x >> 2) + 2][x & 3], o[rb][4 * (x >> 2) + 3][x & 3]);
        }
        if (quarter == 0 && (!quad(rb) || j < 4))
            *reinterpret_cast<float2*>(ml_at + 2 * (wu * kRows + row)) = make_float2(m[rb], sum);
    }
    lds_barrier();
    // two rows per wave and round, a lane four columns
    const int d = 4 * (lane & 31);
    for (int row = 2 * wu + (lane >> 5); row < rows; row += 2 * kWaves) {
        float M = -INFINITY, L = 0.f;
        float2 ml[kWaves];
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            ml[i] = *reinterpret_cast<const float2*>(ml_at + 2 * (i * kRows + row));
            M = fmaxf(M, ml[i].x);
        }
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            const float c = ml[i].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[i].x - M);
            // (a wave whose every score is NaN keeps m at -inf, and its NaN sum counts)
            L += ml[i].x == -INFINITY ? ml[i].y : ml[i].y * c;
            const float4 v = *reinterpret_cast<const float4*>(smem + (i * kRows + row) * kRowF + d);
            x.x = __builtin_fmaf(c, v.x, x.x), x.y = __builtin_fmaf(c, v.y, x.y);
            x.z = __builtin_fmaf(c, v.z, x.z), x.w = __builtin_fmaf(c, v.w, x.w);
        }
        const int g = f0 + row, t0 = fdiv(g, fG);
        float* dst;
        if (p.part) {
            dst = p.part + row * D;
            if (d == 0) *reinterpret_cast<float2*>(p.part + kFewRows * D + 2 * row) = make_float2(M, L);
        } else {
            dst = a.out + (((size_t)p.row0 + t0) * a.H + kvh * G + g - t0 * G) * D;
            bool none = p.pos0 + t0 < 0;  // a row that sees no key: zeros
            if constexpr (kTree) none = L == 0.f && tree_sees_none(a, p.row0, p.pos0, t0);
            const float inv = none ? 0.f : 1.f / L;
            x.x *= inv, x.y *= inv, x.z *= inv, x.w *= inv;
        }
        *reinterpret_cast<float4*>(dst + d) = x;
    }
}

// A workgroup's part of a list: `sh` its share of the line (first unit, first tile, last unit, last tile), before
// it `rounds` whole units.
// (walk_share of packed.h, spelt out: through it the passes are compiled otherwise, and prompts of 17 to 8192 rows take
// 0.7% longer.)
template <bool kPaged, bool kTree, bool kFew>
__device__ __forceinline__ void walk_list(const PackedArgs& a, const List& list, int4 sh, int rounds, int shares,
                                          int share, int kvh, float* parts, float* smem) {
    const FastDiv fG = fast_div((uint32_t)(a.H / a.HKV));
    const float sl2 = a.scale * 1.44269504088896340736f;  // scores come out in log2 units
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
        p.part = p.kt_lo > 0 || cut >= 0 ? parts + part_at(kFew, share * a.HKV + kvh, p.kt_lo > 0 ? 0 : 1) : nullptr;
        if (pass > 0) lds_barrier();  // the last pass's rows have been read
        if constexpr (kFew) {
            const int rows = p.nflat - kUnitRows * p.u;
            // (up to so many rows: the fewest matrix instructions that hold them)
            if (rows <= 4) few_pass<kPaged, kTree, 0, true>(a, p, kvh, fG, sl2, smem);
            else if (rows <= kFewBlock) few_pass<kPaged, kTree, 1, false>(a, p, kvh, fG, sl2, smem);
            else if (rows <= kFewBlock + 4) few_pass<kPaged, kTree, 1, true>(a, p, kvh, fG, sl2, smem);
            else few_pass<kPaged, kTree, kFewRows / kFewBlock, false>(a, p, kvh, fG, sl2, smem);
        } else wide_pass<kPaged, kTree>(a, p, kvh, fG, sl2, smem);
    }
}

// grid shares x KV heads (a KV head's workgroups share an XCD's L2): each workgroup's part of the wide list, then of
// the few-row list.  The plan's header and both shares are read before anything waits for them.
template <bool kPaged, bool kTree>
__global__ __launch_bounds__(64 * kWaves) void k_packed_attn(PackedArgs a, int shares, float* __restrict__ wide_parts,
                                                             float* __restrict__ few_parts) {
    extern __shared__ __align__(16) float smem[];
    const int kvh = blockIdx.x % a.HKV, share = blockIdx.x / a.HKV;
    const PlanView pv = plan_view(const_cast<char*>(a.plan), a.n_seq, a.rows, a.H / a.HKV, shares);
    const int rounds = scalar(reinterpret_cast<const int*>(a.plan)[kHeadRounds]);
    const int4 wide = *reinterpret_cast<const int4*>(pv.wide.shares + share);
    const int4 few = *reinterpret_cast<const int4*>(pv.few.shares + share);
    if (!plan_fits(a.plan, a.n_seq, a.rows, a.H, a.HKV, !kPaged)) return;
    walk_list<kPaged, kTree, false>(a, pv.wide, wide, rounds, shares, share, kvh, wide_parts, smem);
    lds_barrier();  // the last wide pass's rows have been read
    walk_list<kPaged, kTree, true>(a, pv.few, few, 0, shares, share, kvh, few_parts, smem);
}

// The units that the cuts divide.  Part p of a unit is slot 1 of the share that it begins in, then slot 0 of each share
// that it reaches: o = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p over the parts that saw a key (m = -inf and
// l = 0 otherwise; m = -inf with a NaN l counts).
//
// Every workgroup of a KV head collects the head's cut units from the shares, and they take eight rows at a time in
// turn, a thread four columns of one.  A round trip to memory for the shares, one for the parts: those of one
// unit on many CUs, since one CU draws some 20 KB/us.
// 64 rows after 448 keys (8 parts each) 5 us, against 17 with four workgroups per unit.  1024 workgroups instead of 512
// cost 0.5 us where there is nothing to merge.
constexpr int kCombineRows = 8, kCombineWgs = 512;
struct Merge {
    Unit x;
    int share, end;
};
__global__ __launch_bounds__(32 * kCombineRows) void k_packed_combine(PackedArgs a, bool prompts, int shares, int wgs,
                                                                      const float* __restrict__ wide_parts,
                                                                      const float* __restrict__ few_parts) {
    __shared__ Merge merges[2 * kPackedCus];  // by share, few-row ones after the wide ones
    __shared__ uint64_t cut[2 * kPackedCus / 64];
    __shared__ int order[2 * kPackedCus];     // the shares with one, in order
    const int tid = threadIdx.x, kvh = blockIdx.x % a.HKV, G = a.H / a.HKV;
    const PlanView pv = plan_view(const_cast<char*>(a.plan), a.n_seq, a.rows, G, shares);
    if (!plan_fits(a.plan, a.n_seq, a.rows, a.H, a.HKV, prompts)) return;
    for (int t = tid; t < 2 * kPackedCus; t += 32 * kCombineRows) {
        int end = 0;
        if (t < 2 * shares) {
            const Share* at = pv.wide.shares + t;  // (the few-row list's follow)
            end = at->merge_end;
            merges[t] = {at->merge, t < shares ? t : t - shares, end};
        }
        const uint64_t cuts = __builtin_amdgcn_ballot_w64(end > 0);
        if ((t & 63) == 0) cut[t >> 6] = cuts;
    }
    __syncthreads();
    auto before = [&](int t) {  // shares below t with a cut unit
        int n = 0;
#pragma unroll
        for (int i = 0; i < 2 * kPackedCus / 64; ++i) {
            const int in = min(max(t - 64 * i, 0), 64);
            n += __builtin_popcountll(in == 64 ? cut[i] : cut[i] & ((1ull << in) - 1));
        }
        return n;
    };
    for (int t = tid; t < 2 * shares; t += 32 * kCombineRows)
        if (cut[t >> 6] >> (t & 63) & 1) order[before(t)] = t;
    const int wide = before(shares), few_rows = before(2 * shares) - wide;
    __syncthreads();
    const int n_wide = wide * (kUnitRows / kCombineRows), n_few = few_rows * (kFewRows / kCombineRows);
    const int d = 4 * (tid & 31);
    for (int i = blockIdx.x / a.HKV; i < n_wide + n_few; i += wgs) {
        const bool few = i >= n_wide;
        const int j = few ? i - n_wide : i, n = few ? few_rows : wide;
        const Merge& m = merges[order[few ? wide + j % n : j % n]];
        const int row = j / n * kCombineRows + (tid >> 5), f = kUnitRows * m.x.u + row;
        if (f >= m.x.n * G) continue;
        const float* parts = few ? few_parts : wide_parts;
        float M = -INFINITY, L = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        constexpr int kAtOnce = 8;  // parts whose loads are in flight together
        for (int p = m.share; p <= m.end; p += kAtOnce) {
            float2 ml[kAtOnce];
            float4 v[kAtOnce];
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const int q = min(p + k, m.end);
                const float* b = parts + part_at(few, q * a.HKV + kvh, q == m.share ? 1 : 0);
                ml[k] = *reinterpret_cast<const float2*>(b + (few ? kFewRows : kUnitRows) * kHeadDim + 2 * row);
                v[k] = *reinterpret_cast<const float4*>(b + row * kHeadDim + d);
            }
            float mn = M;
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) mn = fmaxf(mn, ml[k].x);
            const float c = M == mn ? 1.f : __builtin_amdgcn_exp2f(M - mn);
            M = mn;
            // (these parts' sum first: fewer roundings of a long unit's)
            float l = 0.f;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                // (past the end the last part was read again: no row then, since zero times an infinite one is NaN)
                const bool none = (p + k > m.end) | ((ml[k].x == -INFINITY) & (ml[k].y == 0.f));
                const float wv = none ? 0.f : __builtin_amdgcn_exp2f(ml[k].x - M);
                const float4 x = none ? make_float4(0.f, 0.f, 0.f, 0.f) : v[k];
                l = __builtin_fmaf(wv, ml[k].y, l);
                sum.x = __builtin_fmaf(wv, x.x, sum.x), sum.y = __builtin_fmaf(wv, x.y, sum.y);
                sum.z = __builtin_fmaf(wv, x.z, sum.z), sum.w = __builtin_fmaf(wv, x.w, sum.w);
            }
            L = __builtin_fmaf(L, c, l);
            o.x = __builtin_fmaf(o.x, c, sum.x), o.y = __builtin_fmaf(o.y, c, sum.y);
            o.z = __builtin_fmaf(o.z, c, sum.z), o.w = __builtin_fmaf(o.w, c, sum.w);
        }
        const int t0 = f / G;
        const int pos0 = m.x.len - m.x.n;  // a row that sees no key: zeros
        const bool none = a.mask ? L == 0.f && tree_sees_none(a, m.x.row0, pos0, t0) : pos0 + t0 < 0;
        const float inv = none ? 0.f : 1.f / L;
        *reinterpret_cast<float4*>(a.out + (((size_t)m.x.row0 + t0) * a.H + kvh * G + f - t0 * G) * kHeadDim + d) =
            make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
}

// ------------------------------------------------------------------ the step's prologue
// Bound by memory, after the latency of two lookups (the row's owner, its page): 824 rows of H 16 / HKV 8 9.2 us
// (27 MB), 1424 of H 32 / HKV 8 18.6 us (70 MB, 3.8 TB/s).
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
                                                        float eps, const int* __restrict__ turn_at) {
    __shared__ float scratch[4][kHeadDim];
    const int b = blockIdx.x, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int H = a.H, HKV = a.HKV, NH = H + HKV;
    const int h0 = (blockIdx.y * 4 + w) * kPrepHeads;
    if (h0 >= NH) return;  // wave-uniform, no barrier here
    // (the row's values are on their way while its place is looked up; of a row that nobody owns they are not used)
    const float* row = qkv + (size_t)b * row_stride;
    float x0[kPrepHeads], x1[kPrepHeads], v0[kPrepHeads], v1[kPrepHeads], inv[kPrepHeads];
#pragma unroll
    for (int j = 0; j < kPrepHeads; ++j) {
        const int hh = min(h0 + j, NH - 1);  // clamped: heads past NH are loaded, not used
        const float* v = row + (size_t)hh * kHeadDim;
        x0[j] = v[lane];
        x1[j] = v[lane + 64];
        v0[j] = v1[j] = 0.f;
        if (hh >= H) {
            const float* vs = row + (size_t)(NH + hh - H) * kHeadDim;  // V of a key head
            v0[j] = vs[lane];
            v1[j] = vs[lane + 64];
        }
    }
    if (!plan_fits(a.plan, a.n_seq, a.rows, H, HKV, false)) return;
    const int4* seq = reinterpret_cast<const int4*>(a.plan + kPlanSeqAt);
    const int s = row_owner(seq, a.n_seq, b, lane);
    if (s < 0) return;
    const int4 e = seq[s];
    const int pos = e.z - e.y + (b - e.x);
    const int turn = turn_at ? turn_at[b] : pos;
    const bool in = pos >= 0 && pos < reinterpret_cast<const int*>(a.plan)[kHeadMaxKv] && turn >= 0 && turn < n_pos;
    const int blk = pos >> a.bshift;
    const int phys = in && blk < a.max_blocks ? a.btab[(size_t)s * a.max_blocks + blk] : -1;
    const bool there = phys >= 0 && phys < a.n_blocks;
    const size_t crow = ((size_t)(there ? phys : 0) << a.bshift) | (size_t)(pos & ((1 << a.bshift) - 1));
    const float2* cs_row = cs + (size_t)(in ? turn : 0) * (rope_dim >> 1);
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
    const int shares = packed_shares(HKV);
    auto by = [](uint32_t d) { return FastDiv{d == 1 ? 0u : 0xFFFFFFFFu / d + 1u, d}; };
    k_packed_plan<<<1, kPlanThreads, 0, st>>>(cu, kv_len, n_seq, rows, max_kv, H, HKV, shares, by((uint32_t)(H / HKV)),
                                              by((uint32_t)shares), 1.0 / shares, static_cast<char*>(plan));
    return hipGetLastError();
}

static size_t q_bytes(int rows, int H) { return ((size_t)rows * H * kHeadDim * 4 + 255) & ~(size_t)255; }

size_t packed_ws_bytes(int rows, int H, int HKV) {
    return q_bytes(rows, H) + (size_t)packed_shares(HKV) * HKV * 2 * (kWidePart + kFewPart) * sizeof(float);
}

PackedParts packed_parts(void* ws, int rows, int H, int HKV) {
    float* wide = reinterpret_cast<float*>(static_cast<char*>(ws) + q_bytes(rows, H));
    return {static_cast<float*>(ws), wide, wide + (size_t)packed_shares(HKV) * HKV * 2 * kWidePart};
}

template <bool kPaged, bool kTree>
static hipError_t launch_packed_attn(hipStream_t st, const PackedArgs& a, int shares, const PackedParts& parts) {
    static std::atomic<bool> opted;
    constexpr size_t lds = (size_t)(kWideF > kFewF ? kWideF : kFewF) * sizeof(float);
    if (const hipError_t e = opt_in_lds(opted, (const void*)k_packed_attn<kPaged, kTree>, lds); e != hipSuccess)
        return e;
    k_packed_attn<kPaged, kTree><<<shares * a.HKV, 64 * kWaves, lds, st>>>(a, shares, parts.wide, parts.few);
    return hipGetLastError();
}

hipError_t launch_packed_combine(hipStream_t st, const PackedArgs& a, bool prompts, const PackedParts& parts) {
    const int wgs = kCombineWgs / a.HKV > 1 ? kCombineWgs / a.HKV : 1;
    k_packed_combine<<<wgs * a.HKV, 32 * kCombineRows, 0, st>>>(a, prompts, packed_shares(a.HKV), wgs, parts.wide,
                                                               parts.few);
    return hipGetLastError();
}

hipError_t launch_packed(hipStream_t st, const PackedArgs& a, void* ws) {
    const int shares = packed_shares(a.HKV);
    const PackedParts parts = packed_parts(ws, a.rows, a.H, a.HKV);
    const hipError_t e = !a.btab ? launch_packed_attn<false, false>(st, a, shares, parts)
                         : a.mask ? launch_packed_attn<true, true>(st, a, shares, parts)
                                  : launch_packed_attn<true, false>(st, a, shares, parts);
    if (e != hipSuccess) return e;
    return launch_packed_combine(st, a, a.btab == nullptr, parts);
}

hipError_t launch_packed_step(hipStream_t st, PackedArgs a, const float* qkv, long row_stride, float* kc, float* vc,
                              const float* q_gamma, const float* k_gamma, const float* cs, int n_pos, int rope_dim,
                              float eps, void* ws, const int* turn_at) {
    float* q = static_cast<float*>(ws);
    k_packed_prepare<<<dim3(a.rows, (a.H + a.HKV + 15) / 16), 256, 0, st>>>(
        qkv, row_stride, q, a, kc, vc, q_gamma, k_gamma, reinterpret_cast<const float2*>(cs), n_pos, rope_dim, eps,
        turn_at);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    a.q = q;
    a.q_stride = (long)a.H * kHeadDim;
    return launch_packed(st, a, ws);
}

}  // namespace ei
