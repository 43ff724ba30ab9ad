// How attention over cached or packed keys is dealt out to workgroups, and the merge of what several of them leave of a unit:
// shared by the kernels over 16-bit keys (attn.hip) and over the 8-bit cache (attn_fp8.hip).
#pragma once
#include "attn.h"

#define ATTN_XCD_GROUP 8     // row groups of a (sequence, KV head) that go to one XCD together, at most

// ---- how the work is dealt out -----------------------------------------------------------------------
// A sequence is KVH * rg units, each of `steps` list steps of g keys (a sequence without keys still owns
// output rows, which are written as zeros: one step).  A sequence takes no more of the list than the host sized
// the launch for: a context longer than its table is walked by the last step of its units, and row groups
// past the bound on the query lengths are left out, so that the others' shares stay where they are.
struct SeqCost {
    int L, ql, rg, steps, cost;
};
__device__ __forceinline__ void seq_steps(const AttnParams &p, SeqCost &c, const int g) {
    c.steps = max(1, (min(c.L, p.max_keys) + g - 1) / g);
    c.cost = c.rg * p.KVH * c.steps;
}
__device__ __forceinline__ SeqCost seq_cost(const AttnParams &p, const int s, const int rows_per_unit, const int g) {
    SeqCost c{0, 0, 0, 0, 0};
    if (s < p.n_seqs) {
        if (p.cu_k) {
            c.L = p.cu_k[s + 1] - p.cu_k[s];
            c.ql = p.cu_q[s + 1] - p.cu_q[s];
        } else {
            c.L = p.context_lens[s];
            c.ql = p.q_lens ? p.q_lens[s] : 1;
        }
        c.ql = min(max(c.ql, 0), p.n_tokens);
        c.rg = min((c.ql * p.Gq + rows_per_unit - 1) / rows_per_unit, p.max_rg);
        seq_steps(p, c, g);
    }
    return c;
}
// inclusive prefix sum over the wavefront
__device__ __forceinline__ int wave_scan(int v) {
#define ATTN_SCAN(CTRL, ROWMASK) v += __builtin_amdgcn_update_dpp(0, v, CTRL, ROWMASK, 0xF, false)
    ATTN_SCAN(0x111, 0xF);   // row_shr:1, 2, 4, 8
    ATTN_SCAN(0x112, 0xF);
    ATTN_SCAN(0x114, 0xF);
    ATTN_SCAN(0x118, 0xF);
    ATTN_SCAN(0x142, 0xA);   // row_bcast:15 into rows 1 and 3
    ATTN_SCAN(0x143, 0xC);   // row_bcast:31 into rows 2 and 3
#undef ATTN_SCAN
    return v;
}
__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// Where a sequence stands in the list: found either by a position in the list or by its number.
struct SeqAt {
    int seq, L, ql, rg, steps;
    int first;       // list position of its first step
    int q0;          // its first query token (packed form: cu_q[seq], wherever the offsets begin)
};
struct ListPlan {
    int g;                   // keys per list step
    int total, share;        // steps in all, steps per workgroup
    SeqAt at;
    int me;                  // the share (unit) that is this workgroup's
    bool found;
};
// Workgroups go round the 8 XCDs, each with an L2 of its own, and the row groups of a (sequence, KV head) read the same
// keys.  Unsplit units: `group` neighbours of the list go to workgroups that are 8 apart, in whole periods of 8 groups
// (what is left at the end stays as it is), so that the groups still go round.  (32 / 4 heads of 128, 8 queries a row group, us,
// workgroup = unit or share / so: unsplit, 64 sequences of 1024 keys x 16 queries 40.2 / 35.9, 100 of 900 x 12 55.7 / 45.0; split, 8
// of 3000 x 16 29.3 / 27.9, x 40 43.9 / 40.8, 30 of 1777 x 9 39.2 / 38.4; one row group each: no difference.)
__device__ __forceinline__ int unit_of_workgroup(const int wg, const int n, const int group) {
    if (group <= 1) return wg;
    const int period = 8 * group, o = wg % period;
    return wg - o + period > n ? wg : wg - o + (o & 7) * group + (o >> 3);
}
// Shares, which cost the same: a contiguous eighth of the `used` ones to each XCD, so that the pieces of a unit and the units of
// a sequence are neighbours there.  Not below `used`: a workgroup without a share.  Shares of one step stay as they are (9 sequences
// of 1225 keys x 24 24.3 / 25.0; others no difference).  With more, as above; two of 15 such lose (2 of 1939 x 160, 16 / 2 heads, 26.2 / 27.0,
// 7 of 1294 x 24, 64 / 4 heads of 64, 22.9 / 23.7).
__device__ __forceinline__ int share_of_workgroup(const int wg, const int used) {
    if (wg >= used) return wg;
    const int q = used >> 3, r = used & 7, x = wg & 7;
    return x * q + min(x, r) + (wg >> 3);
}
// fine, coarse: the two granularities.  The list is cut at multiples of `fine` keys when every workgroup gets at
// least `coarse` keys that way; otherwise at multiples of `coarse`, so that short units stay whole.
// SPLIT, UNSPLIT: the launches that the caller is compiled for (p.whole: its direct way to the unit).  BY_XCD: `who` is a
// workgroup, and its share or unit is chosen by the two functions above.
template <bool BY_SEQ, bool SPLIT, bool UNSPLIT, bool BY_XCD = false>
__device__ __forceinline__ ListPlan list_plan(const AttnParams &p, const int rows_per_unit, const int fine,
                                              const int coarse, int who) {
    const int lane = lane_id();
    ListPlan pl;
    if (BY_XCD && !SPLIT) who = unit_of_workgroup(who, p.n_wg, min(p.max_rg, ATTN_XCD_GROUP));
    pl.me = who;
    if (UNSPLIT && p.whole) {
        // A workgroup per (sequence, KV head, row group that a sequence can have), found without the list: with
        // 512 sequences its scan cost every workgroup two rounds of 8 dependent loads (MANY, below).
        pl.g = 1 << 30;                       // (longer than any sequence: one step per unit, whatever its length)
        pl.total = 0x7fffffff;
        pl.share = 1;
        const int per_seq = p.KVH * p.whole, s = who / per_seq, l = who - s * per_seq;
        // (the query lengths before s in front of everything that waits for the sequence's own)
        int tok = 0;
        if (!p.cu_k && p.q_lens)
            for (int i = lane; i < s; i += 64) tok += max(p.q_lens[i], 0);
        const SeqCost c = seq_cost(p, s, rows_per_unit, pl.g);
        pl.found = l < __builtin_amdgcn_readfirstlane(c.cost);
        if (p.cu_k) tok = p.cu_q[s];
        else tok = p.q_lens ? lane_value(wave_scan(tok), 63) : s;
        pl.at = SeqAt{s, __builtin_amdgcn_readfirstlane(c.L), __builtin_amdgcn_readfirstlane(c.ql),
                      __builtin_amdgcn_readfirstlane(c.rg), 1, who - l, __builtin_amdgcn_readfirstlane(tok)};
        return pl;
    }
    pl.g = SPLIT ? fine : 1 << 30;                        // (unsplit: each unit is one step)
    SeqCost c0 = seq_cost(p, lane, rows_per_unit, pl.g);
    int s0, total;
    for (;;) {
        s0 = wave_scan(c0.cost);
        total = lane_value(s0, 63);
        for (int b = 64; b < p.n_seqs; b += 64)
            total += lane_value(wave_scan(seq_cost(p, b + lane, rows_per_unit, pl.g).cost), 63);
        if (!SPLIT || pl.g == coarse || total >= (coarse / fine) * p.n_wg) break;
        pl.g = coarse;
        seq_steps(p, c0, coarse);
    }
    pl.total = total;
    pl.share = max(1, (total + p.n_wg - 1) / p.n_wg);
    pl.found = false;
    if (BY_XCD && SPLIT && pl.share > 1) pl.me = who = share_of_workgroup(who, (total + pl.share - 1) / pl.share);
    const int target = BY_SEQ ? 0 : who * pl.share;
    if (!BY_SEQ && target >= total) return pl;
    int before = 0, tok = 0;
    SeqCost c = c0;
    int sc = s0;
    for (int b = 0; b < p.n_seqs; b += 64) {
        if (b > 0) {
            c = seq_cost(p, b + lane, rows_per_unit, pl.g);
            sc = wave_scan(c.cost);
        }
        const int tc = wave_scan(c.ql);
        const int sum = lane_value(sc, 63);
        if (BY_SEQ ? who < b + 64 : target < before + sum) {
            const int l = BY_SEQ ? who - b : __builtin_ctzll(__ballot(before + sc > target));
            pl.at = SeqAt{b + l, lane_value(c.L, l), lane_value(c.ql, l), lane_value(c.rg, l), lane_value(c.steps, l),
                          before + lane_value(sc, l) - lane_value(c.cost, l),
                          p.cu_k ? __builtin_amdgcn_readfirstlane(p.cu_q[b + l]) : tok + lane_value(tc, l) - lane_value(c.ql, l)};
            pl.found = true;
            return pl;
        }
        before += sum;
        tok += lane_value(tc, 63);
    }
    return pl;
}

// the unit after this one: of the same sequence, or of the next one that has any
__device__ __forceinline__ void next_unit(const AttnParams &p, SeqAt &sq, int &unit, int &step, const int rows_per_unit,
                                          const int g) {
    step = 0;
    if (++unit < p.KVH * sq.rg) return;
    unit = 0;
    sq.first += p.KVH * sq.rg * sq.steps;
    do {                                                   // (a sequence without queries has no units)
        ++sq.seq;
        sq.q0 = p.cu_k ? __builtin_amdgcn_readfirstlane(p.cu_q[sq.seq]) : sq.q0 + sq.ql;
        const SeqCost nx = seq_cost(p, sq.seq, rows_per_unit, g);
        sq.L = __builtin_amdgcn_readfirstlane(nx.L);
        sq.ql = __builtin_amdgcn_readfirstlane(nx.ql);
        sq.rg = __builtin_amdgcn_readfirstlane(nx.rg);
        sq.steps = __builtin_amdgcn_readfirstlane(nx.steps);
    } while (sq.rg == 0);
}

// Merge of the pieces of a unit: out[row] = sum_s exp2(m_s - m) O_s / sum_s exp2(m_s - m) l_s, pieces in
// order.  One workgroup per (sequence, KV head, unit, 1024 / HD rows): a thread owns 4 neighbouring output
// elements of a row and walks the pieces, 4 at a time.  Units that were finished in place are left alone.
// BY_SHARE: one workgroup per bound between two shares instead, and 1024 / HD rows; the first bound inside a unit
// does the work.  (For launches that allow for many row groups, which need not be there: 64 sequences of 8
// queries with the query lengths bounded by the 512 tokens of the call only, 900 keys: 131072 workgroups
// otherwise, 96 us the call.)
// G: threads that share the walk over a row's pieces, and join what they have through LDS (1024 / HD / G rows to a workgroup then)
template <typename T, int HD, int ROWS, int FINE, int COARSE, bool BY_SHARE = false, int G = 1>
__global__ __launch_bounds__(256) void attn_merge_kernel(const AttnParams p) {
    constexpr int XROW = HD + 4;
    constexpr int TPR = HD / 4, RPW = 256 / TPR / G;
    int kvh, rg, a;                                                // a: list position of the unit's first step
    const ListPlan pl = list_plan<!BY_SHARE, true, false>(p, ROWS, FINE, COARSE, BY_SHARE ? blockIdx.x + 1 : blockIdx.x / p.KVH);
    const SeqAt &sq = pl.at;
    if (BY_SHARE) {
        if (!pl.found) return;
        const int at = ((int)blockIdx.x + 1) * pl.share - sq.first, unit = at / sq.steps;
        kvh = unit / sq.rg;
        rg = sq.rg - 1 - (unit - kvh * sq.rg);
        a = sq.first + unit * sq.steps;
    } else {
        kvh = blockIdx.x % p.KVH;
        rg = blockIdx.y;
        if (rg >= sq.rg) return;
        a = sq.first + (kvh * sq.rg + sq.rg - 1 - rg) * sq.steps;
    }
    const int wa = a / pl.share, wb = (a + sq.steps - 1) / pl.share;
    if (wa == wb || (BY_SHARE && wa != (int)blockIdx.x)) return;
    const int row = (int)blockIdx.z * RPW + (int)threadIdx.x / TPR % RPW, d = 4 * ((int)threadIdx.x % TPR), g = (int)threadIdx.x / (TPR * RPW);
    const int r = rg * ROWS + row;
    const bool there = row < ROWS && r < sq.ql * p.Gq;
    // (G > 1: all threads of a workgroup that has a row come to the barrier below)
    if (G == 1 ? !there : rg * ROWS + (int)blockIdx.z * RPW >= sq.ql * p.Gq) return;
    const float *base = p.part + row * XROW;
    const size_t slot = (size_t)ROWS * XROW;
    auto piece = [&](const int w) { return base + (size_t)(2 * w + (w == wa && a > wa * pl.share ? 1 : 0)) * slot; };
    float m = -INFINITY, l = 0.0f;
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
    constexpr int SB = 4;
    for (int w0 = wa + SB * g; there && w0 <= wb; w0 += SB * G) {
        float ms[SB], ls[SB];
        float4_t os[SB];
#pragma unroll
        for (int u = 0; u < SB; ++u) {
            // (every load unconditional, on a clamped piece: loads under a branch serialise)
            const float *rp = piece(min(w0 + u, wb));
            const float2_t ml = *(const float2_t *)(rp + HD);
            ms[u] = ml.x;
            ls[u] = ml.y;
            os[u] = *(const float4_t *)(rp + d);
        }
#pragma unroll
        for (int u = 0; u < SB; ++u) {
            if (w0 + u > wb) {
                ms[u] = -INFINITY;
                ls[u] = 0.0f;
                os[u] = float4_t{0.f, 0.f, 0.f, 0.f};
            }
        }
        float mb = m;
#pragma unroll
        for (int u = 0; u < SB; ++u) mb = fmaxf(mb, ms[u]);
        const float ref = mb == -INFINITY ? 0.0f : mb;
        const float keep = __builtin_amdgcn_exp2f(m - ref);            // m = -inf -> 0
        l *= keep;
        acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
#pragma unroll
        for (int u = 0; u < SB; ++u) {
            const float f = __builtin_amdgcn_exp2f(ms[u] - ref);
            l += f * ls[u];
            acc.x += f * os[u].x; acc.y += f * os[u].y; acc.z += f * os[u].z; acc.w += f * os[u].w;
        }
        m = mb;
    }
    if constexpr (G > 1) {
        __shared__ float2_t ml[G][RPW * TPR];
        __shared__ float4_t os[G][RPW * TPR];
        const int at = (int)threadIdx.x % (RPW * TPR);
        ml[g][at] = float2_t{m, l};
        os[g][at] = acc;
        __syncthreads();
        if (g > 0 || !there) return;
#pragma unroll
        for (int u = 1; u < G; ++u) m = fmaxf(m, ml[u][at].x);
        const float ref = m == -INFINITY ? 0.0f : m;
        l = 0.0f;
        acc = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < G; ++u) {
            const float f = __builtin_amdgcn_exp2f(ml[u][at].x - ref);
            const float4_t o = os[u][at];
            l += f * ml[u][at].y;
            acc.x += f * o.x; acc.y += f * o.y; acc.z += f * o.z; acc.w += f * o.w;
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const int tok = r / p.Gq, hq = r - tok * p.Gq;
    if ((uint32_t)(sq.q0 + tok) >= (uint32_t)p.n_tokens) return;
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    *(u32x2 *)((uint16_t *)p.out + ((size_t)(sq.q0 + tok) * p.H + kvh * p.Gq + hq) * HD + d) =
        u32x2{AttnT<T>::pack2(acc.x * inv, acc.y * inv), AttnT<T>::pack2(acc.z * inv, acc.w * inv)};
}
