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
// One wave per row and head, lane l on values 2l and 2l + 1: running maximum and sum over the keys.
__global__ __launch_bounds__(256) void k_packed_rows(PackedArgs a) {
    const int lane = threadIdx.x & 63;
    if (!plan_fits(a.plan, a.n_seq, a.rows, a.H, a.HKV, !a.btab)) return;
    const long id = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int b = (int)(id / a.H), h = (int)(id - (long)b * a.H);
    if (b >= a.rows) return;
    const int4* seq = reinterpret_cast<const int4*>(a.plan + plan_seq_at());
    const int s = row_owner(seq, a.n_seq, b, lane);
    if (s < 0) return;
    const int4 e = seq[s];
    const int keys = min(e.z - e.y + (b - e.x) + 1, e.z);
    const float2 q = *reinterpret_cast<const float2*>(a.q + (size_t)b * a.q_stride + (size_t)h * kHeadDim + 2 * lane);
    const int kvh = h / (a.H / a.HKV);
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int t = 0; t < keys; ++t) {
        size_t row = (size_t)e.x + t;
        bool there = true;
        if (a.btab) {
            const int blk = t >> a.bshift;
            const int phys = blk < a.max_blocks ? a.btab[(size_t)s * a.max_blocks + blk] : -1;
            there = phys >= 0 && phys < a.n_blocks;
            row = ((size_t)phys << a.bshift) | (size_t)(t & ((1 << a.bshift) - 1));
        }
        float2 k = make_float2(0.f, 0.f), v = k;
        if (there) {
            k = *reinterpret_cast<const float2*>(a.k + row * a.kv_stride + (size_t)kvh * kHeadDim + 2 * lane);
            v = *reinterpret_cast<const float2*>(a.v + row * a.kv_stride + (size_t)kvh * kHeadDim + 2 * lane);
        }
        const float x = wave_sum(q.x * k.x + q.y * k.y) * a.scale * 1.44269504088896340736f;
        const float mn = fmaxf(m, x);
        const float c = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        const float p = __builtin_amdgcn_exp2f(x - (mn == -INFINITY ? 0.f : mn));
        l = l * c + p;
        o0 = o0 * c + p * v.x;
        o1 = o1 * c + p * v.y;
        m = mn;
    }
    const float inv = keys <= 0 ? 0.f : 1.f / l;  // a row that sees no key: zeros
    *reinterpret_cast<float2*>(a.out + ((size_t)b * a.H + h) * kHeadDim + 2 * lane) = make_float2(o0 * inv, o1 * inv);
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

hipError_t launch_packed(hipStream_t st, const PackedArgs& a, void* ws) {
    (void)ws;
    const long waves = (long)a.rows * a.H;
    k_packed_rows<<<(unsigned)((waves + 3) / 4), 256, 0, st>>>(a);
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
