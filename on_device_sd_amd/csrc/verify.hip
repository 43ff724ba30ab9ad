// Verification of drafted tokens against the target's probabilities from given random numbers (speculative sampling); with
// no drafts, the sampling of a decode step.
//
// Sequence s has n rows of target logits (n - 1 drafted tokens and the row behind the last).  p_j = softmax(row j / T), q_j
// likewise from the draft model's logits (one-hot at the drafted token without them).  Draft j is kept while u_j <
// min(1, p_j(d_j) / q_j(d_j)); at the first that is not, the next token is drawn from max(p_j - q_j, 0), behind the last from
// p.  Drawn means: the lowest token whose inclusive cumulative weight exceeds r times the total.  T = 0: p is one-hot at the
// largest logit (the lowest index of equals).
//
// All probabilities and sums are fp64.  A cumulative sum over 100 000 tokens in fp32 has borders that are off by more than
// many tokens' probability, and p - q of two good models is a small difference; in fp64 a token does not depend on the
// order of the sums or the accuracy of exp but with a probability of about 1e-11 a draw.  On this chip an fp64 FMA issues at
// the rate of an unpacked fp32 one, so the 20 instructions of exp stay near the time that the logits take to arrive.
#include "common.h"

#define VER_THREADS 256
#define VER_CHUNK 8192          // logits of one row that a workgroup takes: 32 a thread, kept in registers
#define VER_SUB 512             // granularity of the sums that the draw walks over: 8 consecutive logits a lane

struct VerifyParams {
    const void *logits, *draft_logits;
    int64_t ld_t, ld_d;
    const int64_t *drafts;
    const int32_t *query_lens;      // or null: one row each
    const float *temperature;       // [S] or null
    float temperature_all;
    const float *accept_u, *sample_u;
    int S, max_q, n_q, n_d, V;
    int splits, subs;               // chunks of a row, VER_SUB blocks of a row
    int64_t *tokens;
    int32_t *num_accepted;
    float *accept_probs;
    struct Stat *stats;             // [n_q + n_d][splits]
    double *sums;                   // [S][subs]
    struct Choice *choice;          // [S]
};
// of a chunk of a row: its largest logit, the lowest index that has it, and sum exp((l - max) / T)
struct Stat {
    float top;
    int at;
    double z;
};
// which distribution the next token of a sequence is drawn from
struct Choice {
    int row, draft;                 // row of the target, of the draft (-1: none); row -1: no row is left
    int count;                      // accepted drafts
    int greedy;                     // or token of the one-hot target, -1: not greedy
    int one_hot;                    // draft without logits: the drafted token, else -1
    float top_p, top_q;
    int pad;
    double z_p, z_q, k;             // k: log2(e) / T
};

// e^(ln2 t) = 2^t for t <= 0 (anything below -1100, and NaN, gives 0): 2^n by the exponent, 2^f, |f| <= 1/2, as the Taylor
// polynomial of degree 10 in f ln 2 (remainder 0.347^11 / 11! = 2e-13 relative)
__device__ __forceinline__ double exp2_neg(double t) {
    t = fmax(t, -1100.0);
    const double n = rint(t);
    const double f = (t - n) * 0.69314718055994530942;
    double e = 2.7557319223985891e-7;
    e = fma(e, f, 2.7557319223985893e-6);
    e = fma(e, f, 2.4801587301587302e-5);
    e = fma(e, f, 1.9841269841269841e-4);
    e = fma(e, f, 1.3888888888888889e-3);
    e = fma(e, f, 8.3333333333333333e-3);
    e = fma(e, f, 4.1666666666666667e-2);
    e = fma(e, f, 1.6666666666666667e-1);
    e = fma(e, f, 0.5);
    e = fma(e, f, 1.0);
    e = fma(e, f, 1.0);
    return ldexp(e, (int)n);
}
// exp((l - top) / T).  A row whose largest logit is +inf has its weight on the +inf entries; one without any number has none.
__device__ __forceinline__ double weight_of(float l, float top, double k) {
    if (top == INFINITY) return l == INFINITY ? 1.0 : 0.0;
    if (top == -INFINITY) return 0.0;
    return exp2_neg(((double)l - (double)top) * k);
}

__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ float up(__bf16 v) { return (float)v; }
__device__ __forceinline__ float up(half_t v) { return (float)v; }

// eight consecutive logits of a row, at the elements' own alignment; NaN and what is behind the row's end count as -inf
template <typename T> __device__ __forceinline__ void load8(const T *row, int i, int V, float *l) {
    T e[8];
    if (i + 8 <= V) {
        __builtin_memcpy(e, row + i, sizeof e);
#pragma unroll
        for (int j = 0; j < 8; ++j) l[j] = up(e[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) l[j] = i + j < V ? up(row[i + j]) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) l[j] = l[j] == l[j] ? l[j] : -INFINITY;
}

// the larger logit, the lower index of equals
__device__ __forceinline__ void better(float &top, int &at, float t2, int a2) {
    if (t2 > top || (t2 == top && a2 < at)) {
        top = t2;
        at = a2;
    }
}

__device__ __forceinline__ float temperature_of(const VerifyParams &p, int s) { return p.temperature ? p.temperature[s] : p.temperature_all; }
__device__ __forceinline__ int len_of(const VerifyParams &p, int s) { return p.query_lens ? max(p.query_lens[s], 0) : 1; }
// log2(e) / T; 0 says greedy
__device__ __forceinline__ double factor_of(float t) { return t > 0.0f ? 1.4426950408889634074 / (double)t : 0.0; }

// the sequence that row `r` of the target (or of the drafts) belongs to: by the whole wavefront
__device__ __forceinline__ int sequence_of(const VerifyParams &p, int r, bool draft) {
    int before = 0;
    for (int s0 = 0; s0 < p.S; s0 += 64) {
        const int s = s0 + lane_id();
        int n = s < p.S ? len_of(p, s) : 0;
        if (draft) n = max(n - 1, 0);
        int sum = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(sum, o, ODSD_WAVE);
            if (lane_id() >= o) sum += v;
        }
        const uint64_t past = __ballot(before + sum > r);
        if (past) return s0 + __builtin_ctzll(past);
        before += __shfl(sum, 63, ODSD_WAVE);
    }
    return -1;
}

// ---- statistics of every row ---------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(VER_THREADS) void verify_stats_kernel(VerifyParams p) {
    __shared__ float s_top[4];
    __shared__ int s_at[4];
    __shared__ double s_z[4];
    const int row = blockIdx.x / p.splits, c = blockIdx.x - row * p.splits;
    const bool draft = row >= p.n_q;
    const int r = draft ? row - p.n_q : row;
    const T *src = draft ? (const T *)p.draft_logits + (int64_t)r * p.ld_d : (const T *)p.logits + (int64_t)r * p.ld_t;
    float l[32];
#pragma unroll
    for (int i = 0; i < 4; ++i) load8(src, c * VER_CHUNK + i * (VER_THREADS * 8) + (int)threadIdx.x * 8, p.V, l + 8 * i);
    float t = p.temperature_all;
    if (p.temperature) {
        const int s = sequence_of(p, r, draft);
        t = s < 0 ? 0.0f : p.temperature[s];
    }
    const double k = factor_of(t);
    float top = -INFINITY;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < 32; ++i) better(top, at, l[i], c * VER_CHUNK + (i >> 3) * (VER_THREADS * 8) + (int)threadIdx.x * 8 + (i & 7));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) better(top, at, __shfl_xor(top, o, ODSD_WAVE), __shfl_xor(at, o, ODSD_WAVE));
    const int wave = threadIdx.x >> 6;
    if (lane_id() == 0) {
        s_top[wave] = top;
        s_at[wave] = at;
    }
    __syncthreads();
    top = s_top[0];
    at = s_at[0];
    for (int w = 1; w < 4; ++w) better(top, at, s_top[w], s_at[w]);
    double z = 0.0;
    if (k > 0.0) {
#pragma unroll
        for (int i = 0; i < 32; ++i) z += weight_of(l[i], top, k);
        z = wave_sum(z);
        if (lane_id() == 0) s_z[wave] = z;
        __syncthreads();
        z = (s_z[0] + s_z[1]) + (s_z[2] + s_z[3]);
    }
    if (threadIdx.x == 0) p.stats[(int64_t)row * p.splits + c] = Stat{top, at, z};
}

// the whole row's, by one wavefront
__device__ __forceinline__ Stat row_stat(const VerifyParams &p, int row, double k) {
    Stat all{-INFINITY, 0x7fffffff, 0.0};
    const Stat *st = p.stats + (int64_t)row * p.splits;
    for (int c = lane_id(); c < p.splits; c += 64) better(all.top, all.at, st[c].top, st[c].at);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) better(all.top, all.at, __shfl_xor(all.top, o, ODSD_WAVE), __shfl_xor(all.at, o, ODSD_WAVE));
    for (int c = lane_id(); c < p.splits; c += 64) all.z += st[c].z * weight_of(st[c].top, all.top, k);
    all.z = wave_sum(all.z);
    return all;
}

// ---- which drafts stay -----------------------------------------------------------------------------
// One workgroup per sequence, a wavefront per draft.
template <typename T>
__global__ __launch_bounds__(VER_THREADS) void verify_accept_kernel(VerifyParams p) {
    __shared__ int s_start[4], s_dstart[4], s_first;
    const int s = blockIdx.x, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) s_first = 0x7fffffff;
    int start = 0, dstart = 0;
    for (int i = threadIdx.x; i < s; i += VER_THREADS) {
        const int n = len_of(p, i);
        start += n;
        dstart += max(n - 1, 0);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        start += __shfl_xor(start, o, ODSD_WAVE);
        dstart += __shfl_xor(dstart, o, ODSD_WAVE);
    }
    if (lane_id() == 0) {
        s_start[wave] = start;
        s_dstart[wave] = dstart;
    }
    __syncthreads();
    start = s_start[0] + s_start[1] + s_start[2] + s_start[3];
    dstart = s_dstart[0] + s_dstart[1] + s_dstart[2] + s_dstart[3];
    // rows and drafts that are really there; drafts that no row verifies are not accepted
    int n = min(min(len_of(p, s), p.max_q), p.n_q - start);
    n = min(n, p.n_d - dstart + 1);
    const int d_end = s == p.S - 1 ? p.n_d : min(dstart + max(len_of(p, s) - 1, 0), p.n_d);
    for (int j = dstart + max(n - 1, 0) + (int)threadIdx.x; j < d_end; j += VER_THREADS) p.accept_probs[j] = 0.0f;
    const float t = temperature_of(p, s);
    const double k = factor_of(t);
    for (int j = wave; j < n - 1; j += 4) {
        const int64_t d = p.drafts[dstart + j];
        double a = 0.0;
        if (d >= 0 && d < p.V) {
            const Stat sp = row_stat(p, start + j, k);
            const float lp = up(((const T *)p.logits)[(int64_t)(start + j) * p.ld_t + d]);
            double pd, qd = 1.0;
            if (k > 0.0) {
                pd = sp.z > 0.0 ? weight_of(lp, sp.top, k) / sp.z : 0.0;
                if (p.draft_logits) {
                    const Stat sq = row_stat(p, p.n_q + dstart + j, k);
                    const float lq = up(((const T *)p.draft_logits)[(int64_t)(dstart + j) * p.ld_d + d]);
                    qd = sq.z > 0.0 ? weight_of(lq, sq.top, k) / sq.z : 0.0;
                }
            } else {
                pd = sp.top > -INFINITY && sp.at == (int)d ? 1.0 : 0.0;
            }
            a = pd >= qd ? (pd > 0.0 ? 1.0 : 0.0) : pd / qd;
        }
        if (lane_id() == 0) {
            p.accept_probs[dstart + j] = (float)a;
            if (!((double)p.accept_u[dstart + j] < a)) atomicMin(&s_first, j);
        }
    }
    __syncthreads();
    const int count = max(min(s_first, n - 1), 0);
    int64_t *out = p.tokens + (int64_t)s * p.max_q;
    for (int j = threadIdx.x; j < p.max_q; j += VER_THREADS)
        if (j != count) out[j] = j < count ? p.drafts[dstart + j] : -1;
    if (wave != 0) return;
    Choice c;
    c.row = n > 0 ? start + count : -1;
    c.draft = n > 0 && count < n - 1 && p.draft_logits && k > 0.0 ? dstart + count : -1;
    c.one_hot = n > 0 && count < n - 1 && !p.draft_logits ? (int)min(max(p.drafts[dstart + count], (int64_t)-1), (int64_t)0x7fffffff) : -1;
    c.count = count;
    c.greedy = -1;
    c.k = k;
    c.pad = 0;
    c.top_p = c.top_q = 0.0f;
    c.z_p = c.z_q = 1.0;
    if (n > 0) {
        const Stat sp = row_stat(p, c.row, k);
        c.top_p = sp.top;
        c.z_p = sp.z;
        if (!(sp.top > -INFINITY)) c.row = -1;                     // a row without a number: nothing to draw from
        else if (!(k > 0.0)) c.greedy = sp.at;
        if (c.draft >= 0) {
            const Stat sq = row_stat(p, p.n_q + c.draft, k);
            c.top_q = sq.top;
            c.z_q = sq.z;
            if (!(sq.z > 0.0)) c.draft = -1;                       // q is nowhere: p - q is p
        }
    }
    if (lane_id() == 0) {
        p.choice[s] = c;
        p.num_accepted[s] = count;
        if (c.row < 0 || c.greedy >= 0) {
            if (count < p.max_q) out[count] = c.row < 0 ? -1 : c.greedy;
        }
    }
}

// weights of eight consecutive tokens: p, and max(p - q, 0)
template <typename T>
__device__ __forceinline__ void weights8(const VerifyParams &p, const Choice &c, int i, bool rest, double *w) {
    float l[8];
    load8((const T *)p.logits + (int64_t)c.row * p.ld_t, i, p.V, l);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = weight_of(l[j], c.top_p, c.k) / c.z_p;
    if (!rest) return;
    if (c.draft >= 0) {
        load8((const T *)p.draft_logits + (int64_t)c.draft * p.ld_d, i, p.V, l);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = fmax(w[j] - weight_of(l[j], c.top_q, c.k) / c.z_q, 0.0);
    } else if (c.one_hot >= 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = i + j == c.one_hot ? 0.0 : w[j];
    }
}

// ---- sums of the weights that the next token is drawn from -------------------------------------------
template <typename T>
__global__ __launch_bounds__(VER_THREADS) void verify_sums_kernel(VerifyParams p) {
    const int s = blockIdx.y;
    const Choice c = p.choice[s];
    if (c.row < 0 || c.greedy >= 0) return;
    const int wave = threadIdx.x >> 6;
    for (int i = 0; i < 4; ++i) {
        const int sub = blockIdx.x * (VER_CHUNK / VER_SUB) + i * 4 + wave;
        if (sub >= p.subs) return;
        double w[8], v[8];
        weights8<T>(p, c, sub * VER_SUB + lane_id() * 8, true, w);
        weights8<T>(p, c, sub * VER_SUB + lane_id() * 8, false, v);
        double a = 0.0, b = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            a += w[j];
            b += v[j];
        }
        a = wave_sum(a);
        b = wave_sum(b);
        if (lane_id() == 0) {
            p.sums[(int64_t)s * 2 * p.subs + sub] = a;
            p.sums[((int64_t)s * 2 + 1) * p.subs + sub] = b;
        }
    }
}

__device__ __forceinline__ double wave_scan(double v) {       // inclusive
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(v, o, ODSD_WAVE);
        if (lane_id() >= o) v += u;
    }
    return v;
}

// ---- the draw: one wavefront per sequence --------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(64) void verify_draw_kernel(VerifyParams p) {
    const int s = blockIdx.x;
    const Choice c = p.choice[s];
    if (c.row < 0 || c.greedy >= 0) return;
    bool rest = c.draft >= 0 || c.one_hot >= 0;
    const double *sums = p.sums + (int64_t)s * 2 * p.subs;
    double total = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
        if (pass == 1 || !rest) {                              // nothing of p exceeds q: p itself
            rest = false;
            sums = p.sums + ((int64_t)s * 2 + 1) * p.subs;
        }
        total = 0.0;
        for (int b = 0; b < p.subs; b += 64) total += __shfl(wave_scan(b + lane_id() < p.subs ? sums[b + lane_id()] : 0.0), 63, ODSD_WAVE);
        if (total > 0.0 || !rest) break;
    }
    const double aim = (double)p.sample_u[s] * total;
    // the first block of VER_SUB tokens whose inclusive sum exceeds the aim (else the last one that has any weight)
    double before = 0.0, at_before = 0.0;
    int sub = -1;
    for (int b = 0; b < p.subs && sub < 0; b += 64) {
        const double own = b + lane_id() < p.subs ? sums[b + lane_id()] : 0.0;
        const double run = wave_scan(own);
        const uint64_t past = __ballot(before + run > aim && own > 0.0);
        if (past) {
            const int l = __builtin_ctzll(past);
            sub = b + l;
            at_before = before + __shfl(run - own, l, ODSD_WAVE);
        }
        before += __shfl(run, 63, ODSD_WAVE);
    }
    if (sub < 0) {
        for (int b = (p.subs - 1) / 64 * 64; b >= 0 && sub < 0; b -= 64) {
            const uint64_t any = __ballot(b + lane_id() < p.subs && sums[b + lane_id()] > 0.0);
            if (any) sub = b + 63 - __builtin_clzll(any);
        }
        at_before = -INFINITY;                                 // no sum exceeds the aim: the last token with a weight is taken
        if (sub < 0) {
            if (lane_id() == 0) p.tokens[(int64_t)s * p.max_q + c.count] = -1;
            return;
        }
    }
    double w[8], own = 0.0;
    const int i0 = sub * VER_SUB + lane_id() * 8;
    weights8<T>(p, c, i0, rest, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) own += w[j];
    const double run = at_before + (wave_scan(own) - own);
    // the first token of this lane whose cumulative weight exceeds the aim, and the last that has any weight
    int hit = 0x7fffffff, last = -1;
    double cum = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        cum += w[j];
        if (w[j] > 0.0) {
            if (hit == 0x7fffffff && run + cum > aim) hit = i0 + j;
            last = i0 + j;
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        hit = min(hit, __shfl_xor(hit, o, ODSD_WAVE));
        last = max(last, __shfl_xor(last, o, ODSD_WAVE));
    }
    if (lane_id() == 0) p.tokens[(int64_t)s * p.max_q + c.count] = hit != 0x7fffffff ? hit : last;
}

// ---- entry points ------------------------------------------------------------------------------------
struct VerifyLayout {
    size_t stats, sums, choice, total;
    int splits, subs;
};
static bool verify_layout(int64_t S, int64_t n_q, int64_t n_d, int64_t V, bool draft_logits, VerifyLayout &l) {
    l.splits = (int)((V + VER_CHUNK - 1) / VER_CHUNK);
    l.subs = (int)((V + VER_SUB - 1) / VER_SUB);
    size_t o = 0;
    auto take = [&](size_t bytes) { const size_t at = o; o += odsd_round_up(bytes, 256); return at; };
    l.stats = take((size_t)(n_q + (draft_logits ? n_d : 0)) * l.splits * sizeof(Stat));
    l.sums = take((size_t)S * 2 * l.subs * 8);
    l.choice = take((size_t)S * sizeof(Choice));
    l.total = o;
    return (n_q + n_d) * l.splits <= 0x7fffffffLL && S <= 65535;
}
static bool verify_sizes_ok(int32_t S, int32_t max_q, int32_t n_q, int32_t n_d, int32_t V) {
    return S >= 0 && max_q >= 0 && n_q >= 0 && n_d >= 0 && V > 0;
}

extern "C" size_t odsd_verify_workspace_bytes(int32_t n_seqs, int32_t max_q_len, int32_t n_rows, int32_t n_drafts,
                                              int32_t vocab, int32_t has_draft_logits) {
    VerifyLayout l;
    if (!verify_sizes_ok(n_seqs, max_q_len, n_rows, n_drafts, vocab) || vocab > 0x7fffffff - VER_CHUNK ||
        !verify_layout(n_seqs, n_rows, n_drafts, vocab, has_draft_logits != 0, l)) return 0;
    return l.total > 256 ? l.total : 256;
}

template <typename T> static int launch_verify(const VerifyParams &p, hipStream_t st) {
    const int rows = p.n_q + (p.draft_logits ? p.n_d : 0);
    if (rows > 0) verify_stats_kernel<T><<<(unsigned)(rows * p.splits), VER_THREADS, 0, st>>>(p);
    verify_accept_kernel<T><<<(unsigned)p.S, VER_THREADS, 0, st>>>(p);
    verify_sums_kernel<T><<<dim3((unsigned)p.splits, (unsigned)p.S), VER_THREADS, 0, st>>>(p);
    verify_draw_kernel<T><<<(unsigned)p.S, 64, 0, st>>>(p);
    ODSD_CHECK_LAUNCH();
    return ODSD_OK;
}

extern "C" int odsd_verify_drafts(const void *logits, int64_t logits_stride, const void *draft_logits,
                                  int64_t draft_stride, int32_t dtype, const int64_t *draft_tokens,
                                  const int32_t *query_lens, const float *temperature, float temperature_all,
                                  const float *accept_u, const float *sample_u, int32_t n_seqs, int32_t max_q_len,
                                  int32_t n_rows, int32_t n_drafts, int32_t vocab, int64_t *tokens,
                                  int32_t *num_accepted, float *accept_probs, void *workspace, size_t workspace_bytes,
                                  void *stream) {
    if (!verify_sizes_ok(n_seqs, max_q_len, n_rows, n_drafts, vocab) || logits_stride < vocab ||
        (draft_logits && draft_stride < vocab)) return ODSD_ERR_SHAPE;
    if (dtype != ODSD_DT_F32 && dtype != ODSD_DT_BF16 && dtype != ODSD_DT_F16) return ODSD_ERR_DTYPE;
    if (!temperature && !(temperature_all >= 0.0f)) return ODSD_ERR_SHAPE;
    const size_t need = odsd_verify_workspace_bytes(n_seqs, max_q_len, n_rows, n_drafts, vocab, draft_logits != nullptr);
    if (need == 0) return ODSD_ERR_UNSUPPORTED;
    if (n_seqs == 0 || max_q_len == 0) return ODSD_OK;
    if (!tokens || !num_accepted || !sample_u || !workspace || (n_rows && !logits)) return ODSD_ERR_NULL;
    if (n_drafts && (!draft_tokens || !accept_u || !accept_probs || !query_lens)) return ODSD_ERR_NULL;
    const uintptr_t mask = dtype == ODSD_DT_F32 ? 3 : 1;
    if ((((uintptr_t)logits | (uintptr_t)draft_logits) & mask) || !odsd_aligned16(workspace)) return ODSD_ERR_ALIGN;
    if (workspace_bytes < need) return ODSD_ERR_WORKSPACE;
    VerifyLayout l;
    verify_layout(n_seqs, n_rows, n_drafts, vocab, draft_logits != nullptr, l);
    char *ws = (char *)workspace;
    VerifyParams p{logits, draft_logits, logits_stride, draft_stride, draft_tokens, query_lens, temperature,
                   temperature_all, accept_u, sample_u, n_seqs, max_q_len, n_rows, n_drafts, vocab, l.splits, l.subs,
                   tokens, num_accepted, accept_probs, (Stat *)(ws + l.stats), (double *)(ws + l.sums),
                   (Choice *)(ws + l.choice)};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ODSD_DT_F32) return launch_verify<float>(p, st);
    if (dtype == ODSD_DT_BF16) return launch_verify<__bf16>(p, st);
    return launch_verify<half_t>(p, st);
}
