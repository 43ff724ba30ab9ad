// Causal attention over the 8-bit paged cache: decode, verify, and a chunk of a prompt.
//
// With query row i, key j of block b(j), codes kc, vc and the block's scales sk, sv of the KV head:
//   s_ij = scale * sk(b(j)) * sum_d q_id kc_jd                       (j <= L - ql + token of i)
//   o_i  = sum_j exp(s_ij) sv(b(j)) vc_j / sum_j exp(s_ij)
// The scale of V joins the exponent: w_ij = 2^(s_ij log2 e + log2 sv - m_i) is what the matrix product takes, m_i the running
// maximum of that exponent, and l_i sums w_ij / sv in fp32.  A w below 2^-126 vanishes; beside the row's largest, 1 or more, it is less than
// 2^-46 of l_i while the scales of V that the row meets are within 2^80 of each other.  (Blocks of zeros have the smallest scale, 2^-64: V up to
// 2^24 may stand beside them, and with it all that fp16 holds.)  Codes become 16-bit operands of q's type in registers (exact); products
// and sums are fp32; w, 2^8 at most, is rounded to q's type once (half a step, as in the kernels over 16-bit keys; fp16 has steps of 2^-24 below
// 2^-14), the result once.
//
// A unit -- up to 16, 32, 64 or 128 query rows of a (sequence, KV head) -- and the way units are cut into shares of keys are those of
// attn_list.h.  V is stored transposed, so 16 bytes are 16 keys of one dimension, and the rows of S^T = K Q^T are dealt so that a lane
// (c, kq) gets the scores of keys 16 kq .. 16 kq + 15 of query row c: those of its own V bytes, as the B operand of O^T = V^T P^T, and all in
// one block, whose scales are lane values.  A lane's 16 bytes of a K row are the k indices of two products; the query's fragments have the
// same order.  The cache holds what the matrix instructions want as it lies.
//
// Up to 16 rows (a token of each sequence) bytes bound it: no barrier and no LDS in the loop, the next tile's bytes requested into the registers
// that the present one has just left.  More rows would read each key once per wavefront that has it, and widening it once per 16 rows is what
// they wait for: the keys go through LDS, a step is copied while the one before is worked on, and a wavefront has 32 rows for every code
// it widens.  (32 / 4 heads of 128, 8 tokens of 32 sequences of up to 2000 keys: 42 us with keys straight to registers, 30 through LDS; a
// chunk of 2048 tokens at 4096 keys 397 and 226.)
//
// Measured, 32 / 4 heads of 128, bf16, in a graph: a token each of 64 sequences of 750 to 3000 keys 29 us, 4.2 TB/s of codes; 4 tokens each of 64
// sequences of 8000 to 8192 keys 114 us, 4.7 TB/s; a chunk of 512 tokens each of 8 sequences of 8192 keys 497 us, 1020 TFLOP/s.  A short call is a
// list, a lookup, a tile and a merge, each waiting for the one before: one sequence of 777 keys 8.0 us.
#include "attn_list.h"
#include "fp8.h"
#include "w4_gemm.h"

#define FP8_WG 512           // workgroups that share the keys: two per CU
#define FP8_JOIN 8           // threads that share the merge of a row's pieces where units are few
#define FP8_STEP 256         // keys of a list step, 64 per wavefront
#define FP8_WHOLE 512        // no sequence longer: nothing is split

struct AttnFp8Params : AttnParams {
    const float *scales;     // [n_blocks, KVH, 2]
    int n_blocks;
    uint32_t gq_inverse;     // ceil(2^32 / Gq), 0 for 1
};
// query token of a row: row / Gq (exact: rows * Gq stays below 2^32)
__device__ __forceinline__ int fp8_token(const AttnFp8Params &p, const int row) {
    return p.gq_inverse ? (int)__umulhi((uint32_t)row, p.gq_inverse) : row;
}

// ---- 64 keys of 16 RB query rows ------------------------------------------------------------------------
// Lane (c, kq) has the raw scores st[rb][t] of keys k0 + 16 kq + 4 t + i of query row 16 rb + c.  Returns the weights as the B operands of
// O^T = V^T P^T and keeps the rows' reference points, this lane's part of their sums, and O^T.  sc, ev, iv: of the block of the lane's
// keys, scale * sk * log2 e, log2 sv and 1 / sv.
template <typename T, int RB, int NDB>
__device__ __forceinline__ void fp8_weights(const float4_t (&st)[RB][4], const float sc, const float ev, const float iv, const bool masked,
                                            const int k, const int (&kmax)[RB], float (&m_run)[RB], float (&l_run)[RB],
                                            float4_t (&o)[RB][NDB], typename AttnT<T>::V8 (&pf)[RB][2]) {
    typedef typename AttnT<T>::V8 V8;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        float a[16];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            a[4 * t] = st[rb][t].x; a[4 * t + 1] = st[rb][t].y; a[4 * t + 2] = st[rb][t].z; a[4 * t + 3] = st[rb][t].w;
        }
        if (masked) {
#pragma unroll
            for (int e = 0; e < 16; ++e) a[e] = k + e <= kmax[rb] ? a[e] : -INFINITY;
        }
        float mx = a[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = fmaxf(mx, a[e]);
        mx = fmaf(mx, sc, ev);
        // The reference point moves only when a weight of the wavefront would pass 2^8 (weights up to 256 are as exact in fp16 / bf16 as
        // those below 1, and the sums are fp32): most tiles need no exchange between lanes
        if (__any(mx > m_run[rb] + 8.0f)) {
            mx = fmaxf(mx, __shfl_xor(mx, 16, ODSD_WAVE));
            mx = fmaxf(mx, __shfl_xor(mx, 32, ODSD_WAVE));
            const float m_new = fmaxf(m_run[rb], mx);
            // a row with nothing to attend yet keeps m = -inf: use 0 as the reference point then
            const float alpha = __builtin_amdgcn_exp2f(m_run[rb] - (m_new == -INFINITY ? 0.0f : m_new));
            l_run[rb] *= alpha;
            m_run[rb] = m_new;
#pragma unroll
            for (int db = 0; db < NDB; ++db) {
                o[rb][db].x *= alpha; o[rb][db].y *= alpha; o[rb][db].z *= alpha; o[rb][db].w *= alpha;
            }
        }
        const float ref = m_run[rb] == -INFINITY ? ev : ev - m_run[rb];
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) a[e] = __builtin_amdgcn_exp2f(fmaf(a[e], sc, ref));      // masked -> 0
#pragma unroll
        for (int e = 0; e < 16; e += 4) sum += (a[e] + a[e + 1]) + (a[e + 2] + a[e + 3]);
        l_run[rb] = fmaf(sum, iv, l_run[rb]);
#pragma unroll
        for (int u = 0; u < 2; ++u)
            pf[rb][u] = __builtin_bit_cast(V8, uint4_t{AttnT<T>::pack2(a[8 * u], a[8 * u + 1]), AttnT<T>::pack2(a[8 * u + 2], a[8 * u + 3]),
                                                       AttnT<T>::pack2(a[8 * u + 4], a[8 * u + 5]), AttnT<T>::pack2(a[8 * u + 6], a[8 * u + 7])});
    }
}
// Codes of V, 16 keys of one dimension from key k on, of a tile in which some row does not see some key.  Bytes past the last key are what a
// block held before: they count as zeros.  A NaN of a key that some rows see and others do not must not reach the others as 0 * NaN: before
// the tile's weights are there fp8_nan_rows counts such codes for the rows that see them, by a product of its own, and makes their sums
// NaN; in the product itself they are zeros.
__device__ __forceinline__ uint4_t fp8_keep(const int k, const int L) {
    uint4_t keep;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int left = L - k - 4 * w;
        keep[w] = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
    }
    return keep;
}
__device__ __forceinline__ uint32_t fp8_nan_bits(const uint32_t v) { return ((v & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint4_t fp8_clean(uint4_t v, const uint4_t keep) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const uint32_t f = fp8_nan_bits(v[w]);
        v[w] &= keep[w] & ~((f << 1) - (f >> 7));
    }
    return v;
}
template <typename T, int RB, int NDB, typename PIECE>
__device__ __forceinline__ void fp8_nan_rows(const PIECE &piece, const uint4_t keep, const int k, const int (&kmax)[RB], float4_t (&o)[RB][NDB]) {
    typedef typename AttnT<T>::V8 V8;
    uint32_t any = 0u;
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
        const uint4_t v = piece(db);
#pragma unroll
        for (int w = 0; w < 4; ++w) any |= fp8_nan_bits(v[w] & keep[w]);
    }
    if (!__any(any != 0u)) return;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        V8 sees[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float s[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = k + 8 * u + e <= kmax[rb] ? 1.0f : 0.0f;
            sees[u] = __builtin_bit_cast(V8, uint4_t{AttnT<T>::pack2(s[0], s[1]), AttnT<T>::pack2(s[2], s[3]),
                                                     AttnT<T>::pack2(s[4], s[5]), AttnT<T>::pack2(s[6], s[7])});
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
            uint4_t ones = piece(db);                      // 1.0 where the code is no number
#pragma unroll
            for (int w = 0; w < 4; ++w) ones[w] = (fp8_nan_bits(ones[w] & keep[w]) >> 7) * 0x38u;
            float4_t cnt = AttnT<T>::mfma(fp8_widen8<T>(ones[0], ones[1]), sees[0], float4_t{0.f, 0.f, 0.f, 0.f});
            cnt = AttnT<T>::mfma(fp8_widen8<T>(ones[2], ones[3]), sees[1], cnt);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (cnt[i] > 0.0f) o[rb][db][i] = __builtin_nanf("");
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}
// fragments of the unit's query rows from row0 on, and the last position that each attends
template <typename T, int HD, int RB>
__device__ __forceinline__ void fp8_queries(const AttnFp8Params &p, const SeqAt &sq, const int kvh, const int row0, int lane,
                                            typename AttnT<T>::V8 (&qf)[RB][HD / 32], int (&kmax)[RB]) {
    asm volatile("" : "+v"(lane));                         // (computed here, not kept from piece to piece)
    const int c = lane & 15, kq = lane >> 4, rows_total = sq.ql * p.Gq;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int row = row0 + 16 * rb + c;
        int tok = fp8_token(p, row);
        const bool ok = row < rows_total && (uint32_t)(sq.q0 + tok) < (uint32_t)p.n_tokens;
        tok = ok ? tok : 0;
        const int hq = ok ? row - tok * p.Gq : 0;
        kmax[rb] = ok ? min(sq.L - sq.ql + tok, p.max_keys - 1) : -1;
        const uint16_t *qp = (const uint16_t *)p.q + ((size_t)(sq.q0 + tok) * p.H + kvh * p.Gq + hq) * HD + 16 * kq;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {                // dims 64 (j / 2) + 16 kq + 8 (j % 2) ..
            uint4_t raw = {0u, 0u, 0u, 0u};
            if (ok) raw = *(const uint4_t *)(qp + 64 * (j >> 1) + 8 * (j & 1));
            qf[rb][j] = __builtin_bit_cast(typename AttnT<T>::V8, raw);
        }
    }
}
// block of the KV head (block * KVH + kvh) and token of it of position kp; an entry that is negative or beyond the cache reads block 0
__device__ __forceinline__ void fp8_locate(const AttnFp8Params &p, const int32_t *bt, const int kvh, const int kp, uint32_t &gk, uint32_t &off) {
    const int blk = kp / p.block_size;
    const int32_t b = bt[min(blk, p.max_blocks - 1)];
    gk = (b >= 0 && b < p.n_blocks && blk < p.max_blocks ? (uint32_t)b : 0u) * (uint32_t)p.KVH + (uint32_t)kvh;
    off = (uint32_t)(kp - blk * p.block_size);
}
// its scales as the scores want them: scale * sk * log2 e, log2 sv, 1 / sv.  A product that fp32 does not hold counts as the smallest or the largest
// normal number: -inf stands for a key that is not seen, and -inf * 0 would be no number (nor 0 * inf, of a score of 0).
__device__ __forceinline__ void fp8_scales(const AttnFp8Params &p, const uint32_t gk, float &sc, float &ev, float &iv) {
    const float2_t s2 = *(const float2_t *)(p.scales + 2 * (size_t)gk);
    const float sv = fmaxf(s2.y, FP8_MIN_SCALE);
    sc = __builtin_amdgcn_fmed3f(p.scale_log2e * fmaxf(s2.x, FP8_MIN_SCALE), 1.17549435e-38f, 3.40282347e38f);
    ev = __builtin_amdgcn_logf(sv);
    iv = __builtin_amdgcn_rcpf(sv);
}
// The sums of WK wavefronts that had other keys of the same rows (and of WR groups of them, with other rows), 16 rows of each group at
// a time through LDS; `whole`: the unit is done, otherwise the results go to `part`.
template <typename T, int HD, int RB, int WR>
__device__ __forceinline__ void fp8_finish(const AttnFp8Params &p, const SeqAt &sq, const int kvh, const int row0, int tid, const bool whole,
                                           float *part, const float (&m_run)[RB], const float (&l_run)[RB], const float4_t (&o)[RB][HD / 16],
                                           float *xch) {
    constexpr int WK = 4 / WR, XROW = HD + 4, TPR = 16 / WR, PIECES = HD / 4 / TPR;      // threads of a row, float4 each
    asm volatile("" : "+v"(tid));                          // (what follows from it is computed here, not kept through the loop over the keys)
    const int lane = tid & 63, wave = tid >> 6, c = lane & 15, kq = lane >> 4;
    const int rows_here = min(16 * RB * WR, sq.ql * p.Gq - row0);
    const int x = tid / TPR;                               // this thread's row of the 16 WR
    const float *xs = xch + ((x >> 4) * WK * 16 + (x & 15)) * XROW;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        __syncthreads();                                   // the area is free
        float *xr = xch + (wave * 16 + c) * XROW;          // wavefront: group wave / WK, keys wave % WK
        float l = l_run[rb];
        l += __shfl_xor(l, 16, ODSD_WAVE);
        l += __shfl_xor(l, 32, ODSD_WAVE);
#pragma unroll
        for (int db = 0; db < HD / 16; ++db) *(float4_t *)(xr + 16 * db + 4 * kq) = o[rb][db];
        if (kq == 0) {
            xr[HD] = m_run[rb];
            xr[HD + 1] = l;
        }
        __syncthreads();
        const int r = 16 * RB * (x >> 4) + 16 * rb + (x & 15);
        const int tok = fp8_token(p, row0 + r), hq = row0 + r - tok * p.Gq;
        if (r >= rows_here || (uint32_t)(sq.q0 + tok) >= (uint32_t)p.n_tokens) continue;
        float m = -INFINITY, f[WK], ls = 0.0f;
#pragma unroll
        for (int w = 0; w < WK; ++w) m = fmaxf(m, xs[w * 16 * XROW + HD]);
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < WK; ++w) {
            f[w] = __builtin_amdgcn_exp2f(xs[w * 16 * XROW + HD] - ref);      // -inf -> 0
            ls += f[w] * xs[w * 16 * XROW + HD + 1];
        }
        if (whole) {
            const float inv = ls > 0.0f ? 1.0f / ls : 0.0f;
#pragma unroll
            for (int w = 0; w < WK; ++w) f[w] *= inv;
        }
        uint16_t *to = (uint16_t *)p.out + ((size_t)(sq.q0 + tok) * p.H + kvh * p.Gq + hq) * HD;
        float *pr = part + r * XROW;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int d = 4 * (tid % TPR + TPR * i);
            float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < WK; ++w) {
                const float4_t v = *(const float4_t *)(xs + w * 16 * XROW + d);
                acc.x += f[w] * v.x; acc.y += f[w] * v.y; acc.z += f[w] * v.z; acc.w += f[w] * v.w;
            }
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            if (whole) *(u32x2 *)(to + d) = u32x2{AttnT<T>::pack2(acc.x, acc.y), AttnT<T>::pack2(acc.z, acc.w)};
            else *(float4_t *)(pr + d) = acc;
        }
        if (!whole && tid % TPR == 0) {
            pr[HD] = m;
            pr[HD + 1] = ls;
        }
    }
}

// ---- up to 16 rows: the keys straight to registers --------------------------------------------------------
template <typename T, int HD, bool ALIGNED>
__global__ __launch_bounds__(256, 2) void attn_fp8_kernel(const AttnFp8Params p) {
    typedef typename AttnT<T>::V8 V8;
    constexpr int NC = HD / 64;          // 16-byte pieces of a K row per lane
    constexpr int NDB = HD / 16;         // 16-dim blocks of the output
    constexpr int ROWS = 16, XROW = HD + 4;
    constexpr int MOST = ALIGNED ? 64 : 16;              // tiles whose blocks are looked up at a time
    __shared__ __attribute__((aligned(16))) float xch[4 * 16 * XROW];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, kq = lane >> 4;

    const ListPlan pl = list_plan<false, true, true>(p, ROWS, FP8_STEP, FP8_STEP, blockIdx.x);
    if (!pl.found) return;
    const int first_pos = pl.me * pl.share;
    int pos = first_pos;                                   // list position of the next step
    const int end = min(pl.total, pos + pl.share);
    SeqAt sq = pl.at;
    int unit = sq.steps == 1 ? pos - sq.first : (pos - sq.first) / sq.steps;      // unit of the sequence, step inside the unit
    int step = (pos - sq.first) - unit * sq.steps;

    const int bs = p.block_size;
    const uint32_t block_bytes = (uint32_t)(bs * HD);
    const char *kc = (const char *)p.k_cache, *vc = (const char *)p.v_cache;
    // K: the rows of product t are keys 16 (m / 4) + 4 t + m % 4; V: 16 keys of dimension 16 db + c
    const uint32_t k_lane = (uint32_t)((ALIGNED ? 16 * (c >> 2) + (c & 3) : (c & 3)) * HD + 16 * kq);
    const uint32_t v_lane = (uint32_t)(c * bs + (ALIGNED ? 16 * kq : 0));

    while (pos < end) {
        // ---- one piece: steps step .. step + n - 1 of one unit ----------------------------------------
        const int n = min(end - pos, sq.steps - step);
        const int kvh = sq.rg == 1 ? unit : unit / sq.rg, rg = sq.rg - 1 - (unit - kvh * sq.rg);
        const int L = min(sq.L, p.max_keys), row0 = rg * ROWS;       // (what is past the table is not attended)
        const int32_t *bt = p.block_tables + (size_t)sq.seq * p.max_blocks;
        V8 qf[1][HD / 32];
        int kmax[1];
        fp8_queries<T, HD, 1>(p, sq, kvh, row0, lane, qf, kmax);
        const int kmin = min(sq.L - sq.ql + fp8_token(p, row0), p.max_keys - 1);       // of the unit's first row: tiles that end at or before it need no mask
        float m_run[1] = {-INFINITY}, l_run[1] = {0.0f};
        float4_t o[1][NDB];
#pragma unroll
        for (int db = 0; db < NDB; ++db) o[0][db] = float4_t{0.f, 0.f, 0.f, 0.f};
        const int key_end = step + n == sq.steps ? L : pl.g * (step + n);
        for (int key0 = pl.g * step + 64 * wave; key0 < key_end; key0 += MOST * FP8_STEP) {
            const int nt = min(MOST, (key_end - key0 + FP8_STEP - 1) / FP8_STEP);
            // the blocks of this wavefront's next tiles, one tile (ALIGNED: it lies in one block) or one group of 16 keys per lane;
            // keys past the last one are its group's
            uint32_t gk_l, off_l;
            float sc_l, ev_l, iv_l;
            fp8_locate(p, bt, kvh, min(ALIGNED ? key0 + FP8_STEP * lane : key0 + FP8_STEP * (lane >> 2) + 16 * (lane & 3),
                                       ALIGNED ? (L - 1) & ~63 : (L - 1) & ~15), gk_l, off_l);
            fp8_scales(p, gk_l, sc_l, ev_l, iv_l);

            uint4_t kreg[4][NC], vreg[NDB];
            auto k_from = [&](const int i) {
                const char *at;
                if constexpr (ALIGNED)
                    at = kc + (uint64_t)(uint32_t)lane_value((int)gk_l, i) * block_bytes + (uint32_t)lane_value((int)off_l, i) * (uint32_t)HD + k_lane;
                else
                    at = kc + (uint64_t)(uint32_t)__shfl((int)gk_l, 4 * i + (c >> 2), ODSD_WAVE) * block_bytes +
                         (uint32_t)__shfl((int)off_l, 4 * i + (c >> 2), ODSD_WAVE) * (uint32_t)HD + k_lane;
                return at;
            };
            auto v_from = [&](const int i) {
                const char *at;
                if constexpr (ALIGNED)
                    at = vc + (uint64_t)(uint32_t)lane_value((int)gk_l, i) * block_bytes + (uint32_t)lane_value((int)off_l, i) + v_lane;
                else
                    at = vc + (uint64_t)(uint32_t)__shfl((int)gk_l, 4 * i + kq, ODSD_WAVE) * block_bytes +
                         (uint32_t)__shfl((int)off_l, 4 * i + kq, ODSD_WAVE) + v_lane;
                return at;
            };
            auto fetch_k = [&](const char *at, const int t) {
#pragma unroll
                for (int h = 0; h < NC; ++h) kreg[t][h] = __builtin_nontemporal_load((const uint4_t *)(at + 4 * t * HD + 64 * h));
            };
            auto fetch_v = [&](const char *at, const int db) {
                vreg[db] = *(const uint4_t *)(at + (uint32_t)(16 * db * bs));
            };
            // one tile.  FETCH: there is a next one, whose bytes are requested as registers come free (the scheduling barriers keep
            // the compiler from widening all of a tile first, which costs 64 registers)
            auto tile = [&](auto fetch_c, const int i) {
                const int k0 = key0 + FP8_STEP * i;
                float sc, ev, iv;
                if constexpr (ALIGNED) {
                    sc = __uint_as_float((uint32_t)lane_value((int)__float_as_uint(sc_l), i));
                    ev = __uint_as_float((uint32_t)lane_value((int)__float_as_uint(ev_l), i));
                    iv = __uint_as_float((uint32_t)lane_value((int)__float_as_uint(iv_l), i));
                } else {
                    sc = __shfl(sc_l, 4 * i + kq, ODSD_WAVE);
                    ev = __shfl(ev_l, 4 * i + kq, ODSD_WAVE);
                    iv = __shfl(iv_l, 4 * i + kq, ODSD_WAVE);
                }
                const bool masked = k0 + 63 > kmin;
                if (masked) {
                    const uint4_t keep = fp8_keep(k0 + 16 * kq, L);
                    fp8_nan_rows<T, 1, NDB>([&](const int db) { return vreg[db]; }, keep, k0 + 16 * kq, kmax, o);
#pragma unroll
                    for (int db = 0; db < NDB; ++db) vreg[db] = fp8_clean(vreg[db], keep);
                    __builtin_amdgcn_sched_barrier(0);
                }
                float4_t st[1][4];
                const char *next = nullptr;
                if constexpr (decltype(fetch_c)::value) next = k_from(i + 1);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    st[0][t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int h = 0; h < NC; ++h) {
                        const V8 lo = fp8_widen8<T>(kreg[t][h].x, kreg[t][h].y), hi = fp8_widen8<T>(kreg[t][h].z, kreg[t][h].w);
                        st[0][t] = AttnT<T>::mfma(lo, qf[0][2 * h], st[0][t]);
                        st[0][t] = AttnT<T>::mfma(hi, qf[0][2 * h + 1], st[0][t]);
                    }
                    if constexpr (decltype(fetch_c)::value) fetch_k(next, t);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if constexpr (decltype(fetch_c)::value) next = v_from(i + 1);
                V8 pf[1][2];
                fp8_weights<T, 1, NDB>(st, sc, ev, iv, masked, k0 + 16 * kq, kmax, m_run, l_run, o, pf);
#pragma unroll
                for (int db = 0; db < NDB; ++db) {
                    const V8 lo = fp8_widen8<T>(vreg[db].x, vreg[db].y), hi = fp8_widen8<T>(vreg[db].z, vreg[db].w);
                    o[0][db] = AttnT<T>::mfma(lo, pf[0][0], o[0][db]);
                    o[0][db] = AttnT<T>::mfma(hi, pf[0][1], o[0][db]);
                    if constexpr (decltype(fetch_c)::value) fetch_v(next, db);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            {
                const char *ka = k_from(0), *va = v_from(0);
#pragma unroll
                for (int t = 0; t < 4; ++t) fetch_k(ka, t);
#pragma unroll
                for (int db = 0; db < NDB; ++db) fetch_v(va, db);
            }
            int i = 0;
            for (; i + 1 < nt; ++i) tile(std::true_type{}, i);
            tile(std::false_type{}, i);
        }

        // (a piece that begins where its workgroup's share begins goes to the workgroup's first slot)
        fp8_finish<T, HD, 1, 1>(p, sq, kvh, row0, tid, n == sq.steps, p.part + (size_t)(2 * pl.me + (pos > first_pos ? 1 : 0)) * (ROWS * XROW),
                                 m_run, l_run, o, xch);
        pos += n;
        if (pos < end) next_unit(p, sq, unit, step, ROWS, pl.g);
    }
}

// ---- more rows: the keys through LDS -----------------------------------------------------------------------
// Steps of 128 keys, copied to LDS as they are (asynchronously, the next step's while this one is worked on) for all four wavefronts.  A
// wavefront has 32 rows; WR of them next to each other, the others have other keys of a step (two of 64; with WR = 4 every one both).
// 16-byte pieces are stored XORed with bits of their row, so that the 16 rows that are read together lie in all banks: K rows (keys
// 16 a + 4 t + b, a and b from the lane) by a and the upper bit of b, V rows (dimensions) by their number / 2.
#define FP8_TILE 128         // keys of a step
#define FP8_TILES 32         // steps whose blocks are looked up at a time

template <typename T, int HD, int RB, int WR, bool ALIGNED, bool SPLIT>
__global__ __launch_bounds__(256, 2) void attn_fp8_tile_kernel(const AttnFp8Params p) {
    typedef typename AttnT<T>::V8 V8;
    constexpr int WK = 4 / WR, ROWS = 16 * RB * WR, XROW = HD + 4;
    constexpr int NC = HD / 64, NDB = HD / 16, NP = HD / 16;       // NP: pieces of a K row
    constexpr int TILEB = FP8_TILE * HD;                  // bytes of K (and of V) of a step
    constexpr int COPIES = TILEB / 1024 / 4;              // copies of K (and of V) per wavefront
    __shared__ __attribute__((aligned(16))) char lds[2 * 2 * TILEB];
    __shared__ uint32_t at_block[FP8_TILES * 8], at_token[FP8_TILES * 8];      // of every 16 keys
    __shared__ float4_t at_scale[FP8_TILES * 8];
    static_assert(2 * 2 * TILEB >= 4 * 16 * XROW * 4, "the exchange area is in the tiles");
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, kq = lane >> 4, wr = wave / WK, wk = wave % WK;

    const ListPlan pl = list_plan<false, SPLIT, !SPLIT, true>(p, ROWS, FP8_TILE, FP8_TILE, blockIdx.x);
    if (!pl.found) return;
    const int first_pos = pl.me * pl.share;
    int pos = first_pos;
    const int end = min(pl.total, pos + pl.share);
    SeqAt sq = pl.at;
    int unit = sq.steps == 1 ? pos - sq.first : (pos - sq.first) / sq.steps;
    int step = (pos - sq.first) - unit * sq.steps;
    const int bs = p.block_size;
    const uint32_t block_bytes = (uint32_t)(bs * HD);

    // copies: K rows RPC i + lane / NP of the tile, V rows 8 i + lane / 8 (dimensions); where a lane's pieces begin, in the tile's block
    // (ALIGNED: the whole tile lies in one) or in the block of the lane's 16 keys
    constexpr int RPC = 64 / NP;
    const int k_row = lane / NP, k_slot = lane % NP, v_row = lane >> 3, v_slot = lane & 7;
    uint32_t k_from[COPIES], v_from[COPIES], v_group[COPIES];
#pragma unroll
    for (int u = 0; u < COPIES; ++u) {
        const int r = RPC * (COPIES * wave + u) + k_row, a = (r >> 4) & 3, f = HD == 128 ? ((r >> 1) & 1) + 2 * a : a;
        const int d = 8 * (COPIES * wave + u) + v_row;
        v_group[u] = (uint32_t)(v_slot ^ ((d >> 1) & 7));
        k_from[u] = (uint32_t)((ALIGNED ? r : r & 15) * HD + (k_slot ^ f) * 16);
        v_from[u] = (uint32_t)(d * bs) + (ALIGNED ? 16u * v_group[u] : 0u);
    }
    // fragments
    const int ka = c >> 2, kb = c & 3;
    uint32_t k_at[NC];
#pragma unroll
    for (int h = 0; h < NC; ++h) {
        const int f = HD == 128 ? (kb >> 1) + 2 * ka : ka;
        k_at[h] = (uint32_t)((16 * ka + kb) * HD + ((kq + 4 * h) ^ f) * 16);
    }

    while (pos < end) {
        const int n = min(end - pos, sq.steps - step);
        const int kvh = sq.rg == 1 ? unit : unit / sq.rg, rg = sq.rg - 1 - (unit - kvh * sq.rg);      // row groups with the most keys first
        const int L = min(sq.L, p.max_keys), row0 = rg * ROWS;       // (what is past the table is not attended)
        const int32_t *bt = p.block_tables + (size_t)sq.seq * p.max_blocks;
        V8 qf[RB][HD / 32];
        int kmax[RB];
        fp8_queries<T, HD, RB>(p, sq, kvh, row0 + 16 * RB * wr, lane, qf, kmax);
        const int kmin = min(sq.L - sq.ql + fp8_token(p, row0 + 16 * RB * wr), p.max_keys - 1);     // of the wavefront's first row
        const bool active = row0 + 16 * RB * wr < sq.ql * p.Gq;
        float m_run[RB], l_run[RB];
        float4_t o[RB][NDB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            m_run[rb] = -INFINITY;
            l_run[rb] = 0.0f;
#pragma unroll
            for (int db = 0; db < NDB; ++db) o[rb][db] = float4_t{0.f, 0.f, 0.f, 0.f};
        }
        int key_end = step + n == sq.steps ? L : pl.g * (step + n);
        if (sq.rg > 1)                                     // (no further than the unit's last row sees)
            key_end = min(key_end, sq.L - sq.ql + min(sq.ql, fp8_token(p, row0 + ROWS - 1) + 1));
        for (int key0 = pl.g * step; key0 < key_end; key0 += FP8_TILES * FP8_TILE) {
            const int nt = min(FP8_TILES, (key_end - key0 + FP8_TILE - 1) / FP8_TILE);
            __syncthreads();                               // tables and tiles are free
            uint32_t gk = 0u, off;
            if (tid < 8 * nt) {
                fp8_locate(p, bt, kvh, min(key0 + 16 * tid, (L - 1) & ~15), gk, off);
                at_block[tid] = gk;
                at_token[tid] = off;
            }
            __syncthreads();
            // (Q has come in before the table entries; without this the compiler would wait for it, and with it for every copy, at
            // its first use)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) asm volatile("" : "+v"(qf[rb][j]));
            auto copy = [&](const int i) {
                char *dst = lds + (i & 1) * (2 * TILEB) + 1024 * COPIES * wave;
                if constexpr (ALIGNED) {
                    const uint32_t gk1 = __builtin_amdgcn_readfirstlane(at_block[8 * i]), off1 = __builtin_amdgcn_readfirstlane(at_token[8 * i]);
                    const global_char *kb1 = scalar_base((const global_char *)p.k_cache + (uint64_t)gk1 * block_bytes + off1 * (uint32_t)HD);
                    const global_char *vb1 = scalar_base((const global_char *)p.v_cache + (uint64_t)gk1 * block_bytes + off1);
#pragma unroll
                    for (int u = 0; u < COPIES; ++u) dma16_to_lds(kb1, k_from[u], (lds_void *)(dst + 1024 * u));
#pragma unroll
                    for (int u = 0; u < COPIES; ++u) dma16_to_lds(vb1, v_from[u], (lds_void *)(dst + TILEB + 1024 * u));
                } else {
#pragma unroll
                    for (int u = 0; u < COPIES; ++u) {
                        const int g = 8 * i + (RPC * (COPIES * wave + u) + k_row) / 16;
                        dma16_from_to_lds((const char *)p.k_cache + (uint64_t)at_block[g] * block_bytes + (at_token[g] * (uint32_t)HD + k_from[u]),
                                          (lds_void *)(dst + 1024 * u));
                    }
#pragma unroll
                    for (int u = 0; u < COPIES; ++u) {
                        const int g = 8 * i + (int)v_group[u];
                        dma16_from_to_lds((const char *)p.v_cache + (uint64_t)at_block[g] * block_bytes + (at_token[g] + v_from[u]),
                                          (lds_void *)(dst + TILEB + 1024 * u));
                    }
                }
            };
            copy(0);
            if (tid < 8 * nt) {                            // (the scales are wanted behind the first barrier only)
                float sc, ev, iv;
                fp8_scales(p, gk, sc, ev, iv);
                at_scale[tid] = float4_t{sc, ev, iv, 0.f};
            }
            for (int i = 0; i < nt; ++i) {
                // (128 rows: a wavefront that has got as far as a step's first product with V goes in front of the SIMD's other one until the step
                // ends; the two then want the matrix pipe and the vector unit at different times: a chunk 236 / 226 us, 2048 tokens of one
                // sequence 140 / 129.  In front during every product 227, during those with K 232, with V 231.)
                if constexpr (WR == 4) __builtin_amdgcn_s_setprio(0);
                ODSD_WAIT_VMCNT_LGKM0(0);                  // this wavefront's copies of step i have landed
                __builtin_amdgcn_s_barrier();              // ... everybody's, and all are done with step i - 1
                if (i + 1 < nt) copy(i + 1);
                if (!active) continue;
                const char *kt = lds + (i & 1) * (2 * TILEB), *vt = kt + TILEB;
                // 64 keys.  While a fragment is multiplied the next one is widened and the one behind it read; the scheduling barriers keep
                // the compiler from doing that for all of them first, whose registers would push others out to memory.  masked: some row
                // does not see some key.
                auto keys64 = [&](const auto masked, const int half, const int k0) {
                    const float4_t sc = at_scale[8 * i + 4 * half + kq];
                    const char *v_at = vt + c * FP8_TILE + ((4 * half + kq) ^ (c >> 1)) * 16;
                    auto k_piece = [&](const int x) { return *(const uint4_t *)(kt + k_at[x % NC] + (64 * half + 4 * (x / NC)) * HD); };
                    auto v_piece = [&](const int db) { return *(const uint4_t *)(v_at + 16 * db * FP8_TILE); };
                    uint4_t keep = {0u, 0u, 0u, 0u};
                    if (masked) {
                        keep = fp8_keep(k0 + 16 * kq, L);
                        fp8_nan_rows<T, RB, NDB>(v_piece, keep, k0 + 16 * kq, kmax, o);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    float4_t st[RB][4];
                    uint4_t w = k_piece(0);
                    V8 lo = fp8_widen8<T>(w.x, w.y), hi = fp8_widen8<T>(w.z, w.w);
                    w = k_piece(1);
#pragma unroll
                    for (int x = 0; x < 4 * NC; ++x) {
                        const int t = x / NC, h = x % NC;
                        const uint4_t next = x + 2 < 4 * NC ? k_piece(x + 2) : v_piece(x + 2 - 4 * NC);
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) st[rb][t] = AttnT<T>::mfma(lo, qf[rb][2 * h], h == 0 ? float4_t{0.f, 0.f, 0.f, 0.f} : st[rb][t]);
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) st[rb][t] = AttnT<T>::mfma(hi, qf[rb][2 * h + 1], st[rb][t]);
                        if (x + 1 < 4 * NC) {
                            lo = fp8_widen8<T>(w.x, w.y);
                            hi = fp8_widen8<T>(w.z, w.w);
                            w = next;
                        }
                        __builtin_amdgcn_sched_barrier(0);
                        if (x + 1 == 4 * NC) {
                            V8 pf[RB][2];
                            fp8_weights<T, RB, NDB>(st, sc.x, sc.y, sc.z, masked, k0 + 16 * kq, kmax, m_run, l_run, o, pf);
                            __builtin_amdgcn_sched_barrier(0);
                            if constexpr (WR == 4) __builtin_amdgcn_s_setprio(1);
                            // (w is V's first piece, next its second)
                            uint4_t wn = next;
                            auto widen = [&]() {
                                if (masked) w = fp8_clean(w, keep);
                                lo = fp8_widen8<T>(w.x, w.y);
                                hi = fp8_widen8<T>(w.z, w.w);
                                w = wn;
                            };
                            widen();
#pragma unroll
                            for (int db = 0; db < NDB; ++db) {
                                if (db + 2 < NDB) wn = v_piece(db + 2);
#pragma unroll
                                for (int rb = 0; rb < RB; ++rb) o[rb][db] = AttnT<T>::mfma(lo, pf[rb][0], o[rb][db]);
#pragma unroll
                                for (int rb = 0; rb < RB; ++rb) o[rb][db] = AttnT<T>::mfma(hi, pf[rb][1], o[rb][db]);
                                if (db + 1 < NDB) widen();
                                __builtin_amdgcn_sched_barrier(0);
                            }
                        }
                    }
                };
#pragma unroll
                for (int sub = 0; sub < (WK == 1 ? 2 : 1); ++sub) {
                    const int half = WK == 1 ? sub : wk, k0 = key0 + FP8_TILE * i + 64 * half;
                    // (One body for both costs a branch here and there, two copy the accumulators where they meet and put some registers in
                    // memory: 128 rows, whose tiles are nearly all full, a chunk 228 / 220 us; 64 rows, verify of 32 x 8 28.7 / 29.6.)
                    if constexpr (WR < 4) keys64(k0 + 63 > kmin, half, k0);
                    else if (k0 + 63 > kmin) keys64(std::true_type{}, half, k0);
                    else keys64(std::false_type{}, half, k0);
                }
            }
        }
        fp8_finish<T, HD, RB, WR>(p, sq, kvh, row0, tid, n == sq.steps, p.part + (size_t)(2 * pl.me + (pos > first_pos ? 1 : 0)) * (ROWS * XROW),
                                  m_run, l_run, o, (float *)lds);
        pos += n;
        if (pos < end) next_unit(p, sq, unit, step, ROWS, pl.g);
    }
}

// ---- host side -----------------------------------------------------------------------------------------
// What a call does, from its shape alone; the size function and the launch both ask here.
struct AttnFp8Plan {
    int rows;                     // per unit
    int64_t rg, units;            // row groups per (sequence, KV head), units
    int n_wg, shares;             // workgroups that share the list, those that can get a share
    bool split;                   // units may be split: partial results and a merge
    int join;                     // threads that share the merge of a row's pieces
    size_t bytes;                 // workspace that splitting takes
};
static AttnFp8Plan attn_fp8_plan(int64_t n_seqs, int64_t max_q, int gq, int64_t max_keys, int kvh, int head_dim) {
    AttnFp8Plan pl;
    const int64_t rows = max_q * gq;
    pl.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    pl.rg = (rows + pl.rows - 1) / pl.rows;
    pl.units = n_seqs * kvh * pl.rg;
    const int step = pl.rows <= 16 ? FP8_STEP : FP8_TILE;
    const int64_t steps = (max_keys + step - 1) / step;
    pl.n_wg = FP8_WG;
    // Whole units need no merge (4 to 6 us) and leave no pieces; split ones level mixed lengths out and fill the chip.  (32 / 4 heads of 128, whole /
    // split, us.  16 rows: 64 sequences of 512 keys 9.9 / 13.9, 1024 15.1 / 18.8, 2048 25.1 / 28.6, 750 to 3001 31.6 / 29.4; 128 of 1024 25.4 /
    // 29.1; 16 of 1024 12.0 / 10.0; one of 777 10.0 / 8.0: what a CU reads a microsecond bounds a unit, so heads of 64 stay whole for twice the keys, 14 /
    // 2 heads, one of 1024 5.3 / 6.7, 2048 7.6 / 7.3; 64 of 2048 9.7 / 12.3; 128 of 4096 23.1 / 28.0.  64 rows: 32 sequences of 512 keys 14.6 / 21.2, 1024 20.4 / 23.8, 2048 31.9 / 28.9;
    // 64 of 2048 41.7 / 45.1, 512 to 2048 33.9 / 39.3; 8 of 2048 30.6 / 22.0.  32 rows: 64 of 2048 33.2 / 37.2, 8 of 4096 37.9 / 18.6.  128 rows: 4
    // sequences of 8192 keys 279 / 286, one 160 / 86.)  List positions are 32 bits wide.  What this costs: from 2048 units on nothing is split however
    // long one of them is (16 rows, 512 sequences of 500 keys 49, with one of 131072 among them 1059; 510 and one, which are split, 89).
    const int64_t whole = pl.rows <= 16 ? (pl.units >= 256 ? 2048 : pl.units >= 128 ? 1024 : FP8_WHOLE) * 128 / head_dim : max((int64_t)FP8_WHOLE, 12 * pl.units);
    pl.split = !(max_keys <= whole || pl.units >= 4 * pl.n_wg || pl.units * steps > (1LL << 30));
    // Few units are many pieces each, which are long to walk for one thread (one / eight, us: 4 units of 16 rows and 32768 keys 31.2 / 16.2, 16 of
    // 16384 22.9 / 19.2, 64 of 4096 19.6 / 19.9; 4 of 64 rows and 32768 keys 39.8 / 24.9, 32 of 16384 45.9 / 46.5, 128 of 4096 46.1 / 52.2; one
    // sequence of 777 keys, four pieces a unit, 8.0 / 8.3).
    pl.join = pl.units <= 32 && steps > FP8_JOIN ? FP8_JOIN : 1;
    pl.shares = (int)min(pl.units * steps, (int64_t)pl.n_wg);
    pl.bytes = pl.split ? odsd_round_up((size_t)2 * pl.shares * pl.rows * (head_dim + 4) * sizeof(float), 256) : 0;
    return pl;
}
static bool attn_fp8_shape_ok(int64_t n_seqs, int64_t max_q_len, int num_heads, int num_kv_heads, int head_dim, int block_size, int max_blocks) {
    return n_seqs > 0 && max_q_len > 0 && num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0 &&
           (head_dim == 64 || head_dim == 128) && block_size > 0 && block_size % 16 == 0 && block_size <= FP8_MAX_BLOCK && max_blocks > 0 &&
           (int64_t)max_blocks * block_size <= (1LL << 30) &&                     // (a position and a list step behind it are 31 bits)
           (max_q_len * (num_heads / num_kv_heads) + 63) / 64 <= 65535 &&
           ((max_q_len + 128) * (num_heads / num_kv_heads) + 128) * (num_heads / num_kv_heads) < (1LL << 32) && n_seqs * num_kv_heads <= 0x7fffffffLL &&
           n_seqs * num_kv_heads * ((max_q_len * (num_heads / num_kv_heads) + 63) / 64) <= (1LL << 24) - 1;
}

extern "C" size_t odsd_paged_attention_fp8_workspace_bytes(int32_t n_seqs, int32_t max_q_len, int32_t num_heads,
                                                           int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                                           int32_t max_blocks) {
    if (!attn_fp8_shape_ok(n_seqs, max_q_len, num_heads, num_kv_heads, head_dim, block_size, max_blocks)) return 0;
    const AttnFp8Plan pl = attn_fp8_plan(n_seqs, max_q_len, num_heads / num_kv_heads, (int64_t)max_blocks * block_size, num_kv_heads, head_dim);
    return pl.split ? pl.bytes : 256;
}

extern "C" int odsd_paged_attention_fp8(const void *q, const void *k_cache, const void *v_cache, const float *scales,
                                        const int32_t *block_tables, const int32_t *context_lens, const int32_t *q_lens,
                                        int32_t n_tokens, int32_t n_seqs, int32_t max_q_len, int32_t num_heads, int32_t num_kv_heads,
                                        int32_t head_dim, int32_t block_size, int32_t max_blocks, int32_t n_blocks,
                                        float softmax_scale, int32_t dtype, void *out, void *workspace,
                                        size_t workspace_bytes, void *stream) {
    if (n_tokens < 0 || n_seqs < 0 || max_q_len <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || block_size <= 0 ||
        block_size % 16 || max_blocks <= 0 || n_blocks <= 0 || !(softmax_scale > 0.0f) || !(softmax_scale < INFINITY))
        return ODSD_ERR_SHAPE;
    if (dtype != ODSD_DT_BF16 && dtype != ODSD_DT_F16) return ODSD_ERR_DTYPE;
    if (n_seqs == 0 || n_tokens == 0) return (head_dim == 64 || head_dim == 128) && block_size <= FP8_MAX_BLOCK ? ODSD_OK : ODSD_ERR_UNSUPPORTED;
    if (!attn_fp8_shape_ok(n_seqs, max_q_len, num_heads, num_kv_heads, head_dim, block_size, max_blocks) ||
        (int64_t)n_blocks * num_kv_heads > 0x7fffffffLL)
        return ODSD_ERR_UNSUPPORTED;
    if (!q || !k_cache || !v_cache || !scales || !block_tables || !context_lens || !out) return ODSD_ERR_NULL;
    if (!odsd_aligned16(q) || !odsd_aligned16(k_cache) || !odsd_aligned16(v_cache) || ((uintptr_t)scales & 7u) || ((uintptr_t)out & 7u))
        return ODSD_ERR_ALIGN;
    const int64_t max_keys = (int64_t)max_blocks * block_size;
    const AttnFp8Plan pl = attn_fp8_plan(n_seqs, max_q_len, num_heads / num_kv_heads, max_keys, num_kv_heads, head_dim);
    AttnFp8Params p{};
    p.q = q; p.k_cache = k_cache; p.v_cache = v_cache; p.out = out;
    p.q_lens = q_lens; p.context_lens = context_lens; p.block_tables = block_tables;
    p.n_seqs = n_seqs; p.n_tokens = n_tokens; p.H = num_heads; p.KVH = num_kv_heads; p.Gq = num_heads / num_kv_heads;
    p.max_blocks = max_blocks; p.block_size = block_size;
    p.scale_log2e = softmax_scale * 1.4426950408889634f;
    p.scales = scales; p.n_blocks = n_blocks;
    p.gq_inverse = p.Gq > 1 ? (uint32_t)(((1ULL << 32) + (uint64_t)p.Gq - 1) / (uint64_t)p.Gq) : 0u;
    p.max_keys = (int)max_keys;
    p.max_rg = (int)pl.rg;
    if (pl.split) {
        if (!workspace) return ODSD_ERR_NULL;
        if (!odsd_aligned16(workspace)) return ODSD_ERR_ALIGN;
        if (workspace_bytes < pl.bytes) return ODSD_ERR_WORKSPACE;
        p.part = (float *)workspace;
        p.n_wg = pl.n_wg;
    } else {
        p.n_wg = (int)pl.units;
        p.whole = (int)pl.rg;
    }
    const unsigned grid = (unsigned)(pl.split ? pl.shares : p.n_wg);
    const dim3 mgrid((unsigned)(n_seqs * num_kv_heads), (unsigned)pl.rg, (unsigned)((pl.rows * head_dim * pl.join + 1023) / 1024));
    hipStream_t st = (hipStream_t)stream;
    const bool aligned = block_size % (pl.rows <= 16 ? 64 : FP8_TILE) == 0;       // a tile lies in one block
#define FP8_MERGE(T, HDV, ROWSV, STEPV)                                                                   \
    do {                                                                                                  \
        if (!pl.split) break;                                                                             \
        if (pl.join > 1) attn_merge_kernel<T, HDV, ROWSV, STEPV, STEPV, false, FP8_JOIN><<<mgrid, 256, 0, st>>>(p); \
        else attn_merge_kernel<T, HDV, ROWSV, STEPV, STEPV><<<mgrid, 256, 0, st>>>(p);                    \
    } while (0)
#define FP8_GO(T, HDV)                                                                                    \
    do {                                                                                                  \
        if (aligned) attn_fp8_kernel<T, HDV, true><<<grid, 256, 0, st>>>(p);                              \
        else attn_fp8_kernel<T, HDV, false><<<grid, 256, 0, st>>>(p);                                     \
        FP8_MERGE(T, HDV, 16, FP8_STEP);                                                                  \
    } while (0)
#define FP8_GO_TILE(T, HDV, RBV, WRV)                                                                          \
    do {                                                                                                  \
        if (pl.split) {                                                                                   \
            if (aligned) attn_fp8_tile_kernel<T, HDV, RBV, WRV, true, true><<<grid, 256, 0, st>>>(p);       \
            else attn_fp8_tile_kernel<T, HDV, RBV, WRV, false, true><<<grid, 256, 0, st>>>(p);              \
        } else if (aligned) attn_fp8_tile_kernel<T, HDV, RBV, WRV, true, false><<<grid, 256, 0, st>>>(p);   \
        else attn_fp8_tile_kernel<T, HDV, RBV, WRV, false, false><<<grid, 256, 0, st>>>(p);                 \
        FP8_MERGE(T, HDV, 16 * RBV * WRV, FP8_TILE);                                                      \
    } while (0)
#define FP8_GO_RB(T, HDV)                                                                                 \
    do {                                                                                                  \
        if (pl.rows == 16) FP8_GO(T, HDV);                                                                \
        else if (pl.rows == 32) FP8_GO_TILE(T, HDV, 1, 2);                                                \
        else if (pl.rows == 64) FP8_GO_TILE(T, HDV, 2, 2);                                                \
        else FP8_GO_TILE(T, HDV, 2, 4);                                                                      \
    } while (0)
    if (dtype == ODSD_DT_F16) {
        if (head_dim == 128) FP8_GO_RB(half_t, 128);
        else FP8_GO_RB(half_t, 64);
    } else {
        if (head_dim == 128) FP8_GO_RB(__bf16, 128);
        else FP8_GO_RB(__bf16, 64);
    }
#undef FP8_GO_RB
#undef FP8_GO_TILE
#undef FP8_GO
#undef FP8_MERGE
    ODSD_CHECK_LAUNCH();
    return ODSD_OK;
}
