// Verification of drafted tokens against the target's probabilities from given random numbers (speculative sampling); with
// no drafts, the sampling of a decode step.
//
// Sequence s has n rows of target logits (n - 1 drafted tokens and the row behind the last).  p_j = softmax(row j / T), q_j
// likewise from the draft model's logits (one-hot at the drafted token without them).  Draft j is kept while u_j <
// min(1, p_j(d_j) / q_j(d_j)); at the first that is not, the next token is drawn from max(p_j - q_j, 0), behind the last from
// p.  Drawn means: the lowest token whose inclusive cumulative weight exceeds r times the total.  T = 0: p is one-hot at the
// largest logit (the lowest index of equals).
//
// What a token is drawn from is fp64: a cumulative sum over 100 000 tokens in fp32 has borders that are off by more than many
// tokens' probability, and p - q of two good models is a small difference; in fp64 a token depends on the order of the sums
// and the accuracy of exp (4e-14) with a probability of about 1e-11 a draw.  Only the row that a sequence draws from needs
// that; whether a draft is kept takes the statistics of every row, and those are one pass in fp32: exp2 by the hardware (1 ulp)
// of an argument to 48 bits, sums in fp32 over 4 logits and by a tree over 32, in fp64 above that.  A sum is off by less than
// 2^-23 + 6 2^-24 relative, plus 17 ln 2 2^-24 where l - top is not exact (16-bit logits 2^16 times below the largest).
//
// Launches: statistics of all rows (with drafts); which drafts stay, and the exact sums of p and q of the rows at hand (with
// draft logits); sums of the weights, 512 tokens each; the draw.
#include "common.h"
#include <type_traits>

#define VER_THREADS 256
#define VER_CHUNK 8192          // logits of one row that a workgroup takes: 32 a thread, kept in registers
#define VER_SUB 512             // granularity of the sums that the draw walks over: 8 consecutive logits a lane

// of a chunk of a row: its largest logit, the lowest index that has it (greedy), else sum exp((l - top) / T)
struct Stat {
    float top;
    int at;
    double z;
};
// which distribution the next token of a sequence is drawn from
struct Choice {
    int row, draft;                 // row of the target, of the draft (-1: none); row -1: nothing to draw from
    int count;                      // kept drafts
    int greedy;                     // the token of the one-hot target, -1: not greedy
    int one_hot;                    // refused draft without logits: its token, else -1
    float top_p, top_q;             // the rows' largest logits (only with draft >= 0)
    int pad;
    double k;                       // log2(e) / T
};
// of VER_SUB tokens: the sum of their weights relative to exp((top - row's top) / T)
struct Block {
    double sum;
    float top;
    int pad;
};
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
    Stat *stats;                    // [n_q + n_d][splits]
    double *z;                      // [S][splits][2]: exact sums of the chunks of p and q of the chosen rows
    Block *blocks;                  // [S][subs]
    Choice *choice;                 // [S]
};

// 2^t for t <= 0, not far below -1100: 2^n by the exponent, 2^f, |f| <= 1/2, as 1 + f P(f), P the interpolation of
// (2^f - 1) / f at the nine Chebyshev points of the interval (3.7e-14 relative).  2^0 is exactly 1, and every t here is a
// difference of logits times k, so a row's largest logits weigh exactly 1: sums over a row of equals are whole numbers, and a
// token at a border of theirs is the definition's.
#define EXP2_1 0.6931471805599453
#define EXP2_2 0.2402265069581299
#define EXP2_3 0.055504108664760424
#define EXP2_4 0.009618129159402558
#define EXP2_5 0.0013333558179043112
#define EXP2_6 0.00015403455852453838
#define EXP2_7 1.525268684626772e-05
#define EXP2_8 1.3255224878668817e-06
#define EXP2_9 1.0203121063391729e-07
__device__ __forceinline__ double exp2_neg(double t) {
    const double n = rint(t), f = t - n;
    double e = EXP2_9;
    e = fma(e, f, EXP2_8);
    e = fma(e, f, EXP2_7);
    e = fma(e, f, EXP2_6);
    e = fma(e, f, EXP2_5);
    e = fma(e, f, EXP2_4);
    e = fma(e, f, EXP2_3);
    e = fma(e, f, EXP2_2);
    e = fma(e, f, EXP2_1);
    e = fma(e, f, 1.0);
    return ldexp(e, (int)n);
}
__device__ __forceinline__ float max3(float a, float b, float c) {      // a NaN in front of numbers counts as nothing
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float max3_or_nan(float a, float b, float c) {
    float r;
    asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// exp((l - top) / T).  A row whose largest logit is +inf has its weight on the +inf entries; one without any number has none.
__device__ __forceinline__ double weight_of(float l, float top, double k) {
    if (top == INFINITY) return l == INFINITY ? 1.0 : 0.0;
    if (!(l > -INFINITY) || top == -INFINITY) return 0.0;
    const double t = ((double)l - (double)top) * k;
    return t > -1100.0 ? exp2_neg(t) : 0.0;
}
// The same for many logits of a row: where nothing is out of the ordinary, a clamp in fp32 stands for all cases (NaN, -inf and
// what weighs nothing become 2^-1200, which is 0).  (l k - top k as one FMA saves an instruction, but leaves the rounding of
// top k in the weight of the largest logit.)  Eight at a time, so that the chains of FMAs hide each other's latency, with the
// coefficients in scalar registers (as literals they cost two moves an FMA): 18 instructions a logit, 39 one by one.
struct Weigh {
    double k;
    float low, top;
    bool plain;
    __device__ __forceinline__ Weigh(float top_, double k_) : k(k_), top(top_) {
        low = (float)((double)top - 1200.0 / k);
        const double least = ((double)top - (double)low) * k;
        plain = fabsf(top) < 1e30f && k > 1e-20 && k < 1e20 && least > 1100.0 && least < 1e6;
        plain = __builtin_amdgcn_readfirstlane(plain);
    }
    template <typename R> __device__ __forceinline__ void operator()(const R &r, double *w) const {
        const double c[10] = {1.0, EXP2_1, EXP2_2, EXP2_3, EXP2_4, EXP2_5, EXP2_6, EXP2_7, EXP2_8, EXP2_9};
        double f[8], n[8];
        if (plain) {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = ((double)max3(r.get(j), low, low) - (double)top) * k;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float l = r.get(j);
                const double t = top == INFINITY ? (l == INFINITY ? 0.0 : -1200.0) : ((double)l - (double)top) * k;
                f[j] = t > -1200.0 ? t : -1200.0;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            n[j] = rint(f[j]);
            f[j] -= n[j];
            w[j] = c[9];
        }
#pragma unroll
        for (int i = 8; i >= 0; --i) {
            double ci = c[i];
            asm("" : "+s"(ci));
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = fma(w[j], f[j], ci);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = ldexp(w[j], (int)n[j]);
    }
};

// Eight consecutive logits as they lie in memory, at the elements' own alignment.  A row's last eight are loaded where it
// ends: `base` is where, and what is in front of the eight asked for (or all, behind the end) becomes -inf by clip().  No lane
// branches before its loads, so those of a thread are on their way together.  (Rows have 8 logits at least: pad_kernel.)
template <typename T> struct Raw8 {
    uint32_t w[sizeof(T) * 2];
    int base, skip;
    __device__ __forceinline__ void load(const T *row, int i, int V) {
        base = min(i, V - 8);
        skip = i - base;
        __builtin_memcpy(w, row + base, sizeof w);
    }
    __device__ __forceinline__ void clip() {
        if (!__any(skip > 0)) return;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = j < skip ? 0xff800000u : w[j];
        } else {
            constexpr uint32_t low = std::is_same<T, __bf16>::value ? 0xff80u : 0xfc00u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (2 * j < skip) w[j] = (w[j] & 0xffff0000u) | low;
                if (2 * j + 1 < skip) w[j] = (w[j] & 0xffffu) | (low << 16);
            }
        }
    }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[j]);
        } else {
            const uint32_t two = w[j >> 1];
            if constexpr (std::is_same<T, __bf16>::value) return __uint_as_float(j & 1 ? two & 0xffff0000u : two << 16);
            else return (float)__builtin_bit_cast(half_t, (uint16_t)(j & 1 ? two >> 16 : two));
        }
    }
};
// The largest of eight, NaN none of them.  (Told by the bits: a signalling NaN as an operand of the hardware's ordinary maximum
// makes the result NaN, and the other operand is lost.)
template <typename T> __device__ __forceinline__ float largest8(const Raw8<T> &r) {
    const float t = max3_or_nan(max3_or_nan(r.get(0), r.get(1), r.get(2)), max3_or_nan(r.get(3), r.get(4), r.get(5)), max3_or_nan(r.get(6), r.get(7), -INFINITY));
    if (t == t) return t;
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t bits = __float_as_uint(r.get(j));
        m = fmaxf(m, __uint_as_float((bits & 0x7fffffffu) > 0x7f800000u ? 0xff800000u : bits));
    }
    return m;
}

// Reductions by DPP: a step is one or two vector instructions, where a shuffle through the LDS hardware waits for it; these
// kernels are chains of them.  Within a row of 16 lanes (every lane has the result): rotations.  Over the wavefront (the result
// is uniform): shifts within the rows, then the rows' last lanes.
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ int dpp(int old, int v) {
    return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ float dpp(float old, float v) {
    return __int_as_float(dpp<CTRL, ROWS>(__float_as_int(old), __float_as_int(v)));
}
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ double dpp(double old, double v) {
    return __hiloint2double(dpp<CTRL, ROWS>(__double2hiint(old), __double2hiint(v)), dpp<CTRL, ROWS>(__double2loint(old), __double2loint(v)));
}
enum { ROW_SHR = 0x110, ROW_ROR = 0x120, ROW_BCAST15 = 0x142, ROW_BCAST31 = 0x143 };
template <typename V, typename F> __device__ __forceinline__ V row_all(V v, F f) {
    v = f(v, dpp<ROW_ROR + 8>(v, v));
    v = f(v, dpp<ROW_ROR + 4>(v, v));
    v = f(v, dpp<ROW_ROR + 2>(v, v));
    return f(v, dpp<ROW_ROR + 1>(v, v));
}
// inclusive, over the lanes; `zero` leaves f's other argument as it is
template <typename V, typename F> __device__ __forceinline__ V scan_all(V v, V zero, F f) {
    v = f(dpp<ROW_SHR + 1>(zero, v), v);
    v = f(dpp<ROW_SHR + 2>(zero, v), v);
    v = f(dpp<ROW_SHR + 4>(zero, v), v);
    v = f(dpp<ROW_SHR + 8>(zero, v), v);
    v = f(dpp<ROW_BCAST15, 0xa>(zero, v), v);
    return f(dpp<ROW_BCAST31, 0xc>(zero, v), v);
}
__device__ __forceinline__ int last_lane(int v) { return __builtin_amdgcn_readlane(v, 63); }
__device__ __forceinline__ float last_lane(float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63)); }
__device__ __forceinline__ double last_lane(double v) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), 63), __builtin_amdgcn_readlane(__double2loint(v), 63));
}
template <typename V> __device__ __forceinline__ V plus(V a, V b) { return a + b; }
__device__ __forceinline__ double all_sum(double v) { return last_lane(scan_all(v, 0.0, plus<double>)); }
// (modulo 2^32: lengths are the caller's)
__device__ __forceinline__ int wrapping_plus(int a, int b) { return (int)((uint32_t)a + (uint32_t)b); }
__device__ __forceinline__ int all_sum(int v) { return last_lane(scan_all(v, 0, wrapping_plus)); }
__device__ __forceinline__ float all_max(float v) { return last_lane(scan_all(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); })); }
__device__ __forceinline__ int all_min(int v) { return last_lane(scan_all(v, 0x7fffffff, [](int a, int b) { return min(a, b); })); }
__device__ __forceinline__ int all_max(int v) { return last_lane(scan_all(v, -0x7fffffff - 1, [](int a, int b) { return max(a, b); })); }

// the larger logit, the lower index of equals
__device__ __forceinline__ void better(float &top, int &at, float t2, int a2) {
    if (t2 > top || (t2 == top && a2 < at)) {
        top = t2;
        at = a2;
    }
}

__device__ __forceinline__ float temperature_of(const VerifyParams &p, int s) { return p.temperature ? p.temperature[s] : p.temperature_all; }
__device__ __forceinline__ int len_of(const VerifyParams &p, int s) { return p.query_lens ? max(p.query_lens[s], 0) : 1; }
// log2(e) / T; 0 says greedy (an infinite T: all finite logits alike)
__device__ __forceinline__ double factor_of(float t) { return t > 0.0f ? fmax(1.4426950408889634074 / (double)t, 1e-300) : 0.0; }

// rows of fewer than 8 logits, as rows of 8
template <typename T>
__global__ __launch_bounds__(VER_THREADS) void verify_pad_kernel(const T *src, int64_t ld, T *dst, int rows, int V) {
    const int64_t i = (int64_t)blockIdx.x * VER_THREADS + threadIdx.x;
    const int64_t row = i >> 3;
    const int j = (int)(i & 7);
    if (row < rows) dst[i] = j < V ? src[row * ld + j] : (T)-INFINITY;
}

// the sequence that row `r` of the target (or of the drafts) belongs to: by the whole wavefront
__device__ __forceinline__ int sequence_of(const VerifyParams &p, int r, bool draft) {
    int before = 0;
    for (int s0 = 0; s0 < p.S; s0 += 64) {
        const int s = s0 + lane_id();
        int n = s < p.S ? len_of(p, s) : 0;
        if (draft) n = max(n - 1, 0);
        const int sum = scan_all(n, 0, wrapping_plus);
        const uint64_t past = __ballot(wrapping_plus(before, sum) > r);
        if (past) return s0 + __builtin_ctzll(past);
        before = wrapping_plus(before, last_lane(sum));
    }
    return -1;
}

// ---- statistics of every row ---------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(VER_THREADS) void verify_stats_kernel(VerifyParams p) {
    __shared__ float s_top[4];
    __shared__ int s_at[4];
    __shared__ double s_z[4];
    const int row = blockIdx.x / p.splits, c = blockIdx.x - row * p.splits, wave = threadIdx.x >> 6;
    const bool draft = row >= p.n_q;
    const int r = draft ? row - p.n_q : row;
    const T *src = draft ? (const T *)p.draft_logits + (int64_t)r * p.ld_d : (const T *)p.logits + (int64_t)r * p.ld_t;
    const int first = c * VER_CHUNK + (int)threadIdx.x * 8;
    Raw8<T> raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i].load(src, first + i * (VER_THREADS * 8), p.V);
    float t = p.temperature_all;
    if (p.temperature) {
        const int s = sequence_of(p, r, draft);
        t = s < 0 ? 0.0f : p.temperature[s];
    }
    const double k = factor_of(t);
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i].clip();
    float top = max3(largest8(raw[0]), largest8(raw[1]), fmaxf(largest8(raw[2]), largest8(raw[3])));
    const float own = top;
    top = all_max(top);
    if (lane_id() == 0) s_top[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
    int at = 0x7fffffff;
    double z = 0.0;
    if (!(k > 0.0)) {                                  // greedy: where it is, nothing else
        if (own == top) {
#pragma unroll
            for (int i = 3; i >= 0; --i)
#pragma unroll
                for (int j = 7; j >= 0; --j)
                    if (raw[i].get(j) == top && j >= raw[i].skip) at = raw[i].base + j;
        }
        at = all_min(at);
        if (lane_id() == 0) s_at[wave] = at;
    } else {
        if (fabsf(top) < INFINITY && k > 1e-30 && k < 1e30) {
            // x = (l - top) k to 48 bits: a part that exp2 takes as it is, and its rest times the derivative
            const float kh = (float)k, kl = (float)(k - (double)kh), low = -160.0f / kh;
            // sum e (1 + ln 2 lo) as sum e + ln 2 sum e lo
            float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f}, more[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float l = raw[i].get(j), d0 = l - top;
                    const float d = max3(d0, low, low);                          // (NaN and -inf: 2^-160)
                    const float hi = d * kh;
                    float lo = fmaf(d, kl, fmaf(d, kh, -hi));
                    if (sizeof(T) == 4) {                                        // what l - top lost (16-bit logits: as good as nothing)
                        const float b = l - d0;
                        const float lost = (l - (d0 + b)) + (b - top);
                        lo = d > low ? fmaf(lost, kh, lo) : lo;
                    }
                    const float e = __builtin_amdgcn_exp2f(hi);
                    sum[j] += e;
                    more[j & 1] = fmaf(e, lo, more[j & 1]);
                }
            z = (double)(((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]))) +
                0.69314718055994530942 * (double)(more[0] + more[1]);
        } else {
            // (any temperature, any logits; read again, one by one)
#pragma unroll 1
            for (int i = 0; i < 32; ++i) {
                const int at = first + (i >> 3) * (VER_THREADS * 8) + (i & 7);
                if (at < p.V) z += weight_of((float)src[at], top, k);
            }
        }
        z = all_sum(z);
        if (lane_id() == 0) s_z[wave] = z;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        Stat st{top, 0x7fffffff, 0.0};
        if (k > 0.0) st.z = (s_z[0] + s_z[1]) + (s_z[2] + s_z[3]);
        else st.at = min(min(s_at[0], s_at[1]), min(s_at[2], s_at[3]));
        p.stats[(int64_t)row * p.splits + c] = st;
    }
}

// the whole row's, by 16 neighbouring lanes
__device__ __forceinline__ Stat row_stat(const VerifyParams &p, int row, double k) {
    const Stat *st = p.stats + (int64_t)row * p.splits;
    const int l = lane_id() & 15;
    Stat own{-INFINITY, 0x7fffffff, 0.0};
    if (l < p.splits) own = st[l];
    float top = own.top;
    int at = own.at;
    double z = 0.0;
    if (k > 0.0) {
        for (int c = l + 16; c < p.splits; c += 16) top = fmaxf(top, st[c].top);
        top = row_all(top, [](float a, float b) { return fmaxf(a, b); });
        z = own.z * weight_of(own.top, top, k);
        for (int c = l + 16; c < p.splits; c += 16) z += st[c].z * weight_of(st[c].top, top, k);
        z = row_all(z, plus<double>);
    } else {
        for (int c = l + 16; c < p.splits; c += 16) better(top, at, st[c].top, st[c].at);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) better(top, at, __shfl_xor(top, o, ODSD_WAVE), __shfl_xor(at, o, ODSD_WAVE));
    }
    return Stat{top, at, z};
}

// ---- which drafts stay -----------------------------------------------------------------------------
// By a whole workgroup; every workgroup of a sequence comes to the same answer, one (`writes`) leaves it.  Rows in batches of
// 32: their statistics by 16 lanes each, then a lane per draft.  Without drafts in the call (DRAFTS: there may be some) there are
// no statistics and nothing to decide but the row.
template <typename T, bool DRAFTS>
__device__ Choice choose(const VerifyParams &p, const int s, const bool writes) {
    __shared__ int s_start[4], s_dstart[4];
    __shared__ Stat s_p[32], s_q[32];
    __shared__ Choice s_choice;
    __shared__ bool s_done;
    const int wave = threadIdx.x >> 6;
    int start = 0, dstart = 0;
    const float t = temperature_of(p, s);
    const int len = len_of(p, s);
    if (p.query_lens) {
        for (int i = threadIdx.x; i < s; i += VER_THREADS) {
            const int n = len_of(p, i);
            start = wrapping_plus(start, n);
            if (DRAFTS) dstart = wrapping_plus(dstart, max(n - 1, 0));
        }
        start = all_sum(start);
        if (DRAFTS) dstart = all_sum(dstart);
        if (lane_id() == 0) {
            s_start[wave] = start;
            s_dstart[wave] = dstart;
        }
        __syncthreads();
        start = wrapping_plus(wrapping_plus(s_start[0], s_start[1]), wrapping_plus(s_start[2], s_start[3]));
        dstart = wrapping_plus(wrapping_plus(s_dstart[0], s_dstart[1]), wrapping_plus(s_dstart[2], s_dstart[3]));
        // behind the last row, however far (lengths that do not belong to these rows): the sequence has none
        if ((uint32_t)start > (uint32_t)p.n_q) start = p.n_q;
        if ((uint32_t)dstart > (uint32_t)p.n_d) dstart = p.n_d;
    } else {
        start = s;
    }
    // rows and drafts that are really there; drafts that no row verifies are not kept
    const int n = max(min(min(min(len, p.max_q), p.n_q - start), p.n_d - dstart + 1), 0);
    if (writes) {
        const int d_end = s == p.S - 1 ? p.n_d : dstart + min(max(len - 1, 0), p.n_d - dstart);
        for (int j = dstart + max(n - 1, 0) + (int)threadIdx.x; j < d_end; j += VER_THREADS) p.accept_probs[j] = 0.0f;
    }
    const double k = factor_of(t);
    Choice c{n > 0 ? start : -1, -1, 0, -1, -1, 0.0f, 0.0f, 0, k};
    if (DRAFTS && p.n_d > 0) {
        if (threadIdx.x == 0) {
            s_choice = c;
            s_done = false;
        }
        __syncthreads();
        const bool with_q = p.draft_logits && k > 0.0;
        for (int j0 = 0; j0 < n; j0 += 32) {
            const int rows = min(32, n - j0), drafts = min(32, n - 1 - j0);
            // the drafts' own logits, on their way meanwhile: by the wavefront that has rows last
            const int j = lane_id();
            int64_t d = -1;
            float u = 0.0f, lp = -INFINITY, lq = -INFINITY;
            if (wave == 3 && j < drafts) {
                d = p.drafts[dstart + j0 + j];
                u = p.accept_u[dstart + j0 + j];
                if (d >= 0 && d < p.V) {
                    lp = (float)((const T *)p.logits)[(int64_t)(start + j0 + j) * p.ld_t + d];
                    if (with_q) lq = (float)((const T *)p.draft_logits)[(int64_t)(dstart + j0 + j) * p.ld_d + d];
                }
            }
            for (int g = threadIdx.x >> 4; g < (with_q ? 64 : 32); g += VER_THREADS / 16) {
                const int j = g & 31;
                if (g < 32 ? j >= rows : j >= drafts) continue;
                const Stat st = row_stat(p, g < 32 ? start + j0 + j : p.n_q + dstart + j0 + j, k);
                if ((lane_id() & 15) == 0) (g < 32 ? s_p : s_q)[j] = st;
            }
            __syncthreads();
            if (wave == 3) {
                double a = 0.0;
                if (j < drafts && d >= 0 && d < p.V) {
                    const Stat sp = s_p[j];
                    double pd, qd = 1.0;
                    if (k > 0.0) {
                        pd = sp.z > 0.0 ? weight_of(lp, sp.top, k) / sp.z : 0.0;
                        if (with_q) qd = s_q[j].z > 0.0 ? weight_of(lq, s_q[j].top, k) / s_q[j].z : 0.0;
                    } else {
                        pd = sp.top > -INFINITY && sp.at == (int)d ? 1.0 : 0.0;
                    }
                    a = pd >= qd ? (pd > 0.0 ? 1.0 : 0.0) : pd / qd;
                }
                if (writes && j < drafts) p.accept_probs[dstart + j0 + j] = (float)a;
                const uint64_t refused = __ballot(j < drafts && !((double)u < a));
                const bool ends = refused != 0 || j0 + rows == n;
                if (!s_done && ends) {
                    const int at = refused ? __builtin_ctzll(refused) : rows - 1;      // of the batch: the row that is drawn from
                    const int64_t d_at = __shfl(d, at, ODSD_WAVE);
                    if (j == 0) {
                        Choice c = s_choice;
                        c.row = start + j0 + at;
                        c.count = j0 + at;
                        c.top_p = s_p[at].top;
                        if (!(c.top_p > -INFINITY)) c.row = -1;                        // a row without a number: nothing to draw from
                        else if (!(k > 0.0)) c.greedy = s_p[at].at;
                        if (refused && with_q) {
                            c.top_q = s_q[at].top;
                            if (s_q[at].z > 0.0) c.draft = dstart + j0 + at;           // (q is nowhere: p - q is p)
                        }
                        if (refused && !p.draft_logits && d_at >= 0 && d_at < p.V) c.one_hot = (int)d_at;
                        s_choice = c;
                        s_done = true;
                    }
                }
            }
            __syncthreads();
            if (s_done && !writes) break;
        }
        c = s_choice;
    }
    if (writes) {
        int64_t *out = p.tokens + (int64_t)s * p.max_q;
        // (the token behind the kept ones is the draw's, unless it is known here)
        const bool drawn = c.row >= 0 && c.greedy < 0;
        for (int j = threadIdx.x; j < p.max_q; j += VER_THREADS)
            if (j != c.count || !drawn) out[j] = j < c.count ? p.drafts[dstart + j] : j == c.count && c.row >= 0 ? c.greedy : -1;
        if (threadIdx.x == 0) {
            p.choice[s] = c;
            p.num_accepted[s] = c.count;
        }
    }
    return c;
}

// The exact sums of a chunk of p and of q of the rows that a refused draft leaves (with draft logits).
template <typename T>
__global__ __launch_bounds__(VER_THREADS) void verify_choose_kernel(VerifyParams p) {
    __shared__ double s_z[2][4];
    const int s = blockIdx.y;
    const Choice c = choose<T, true>(p, s, blockIdx.x == 0);
    if (c.row < 0 || c.greedy >= 0 || c.draft < 0) return;
    Raw8<T> rp[4], rq[4];
    const T *lp = (const T *)p.logits + (int64_t)c.row * p.ld_t, *lq = (const T *)p.draft_logits + (int64_t)c.draft * p.ld_d;
    const int first = blockIdx.x * VER_CHUNK + (int)threadIdx.x * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        rp[i].load(lp, first + i * (VER_THREADS * 8), p.V);
        rq[i].load(lq, first + i * (VER_THREADS * 8), p.V);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        rp[i].clip();
        rq[i].clip();
    }
    double zp = 0.0, zq = 0.0;
    const Weigh wp(c.top_p, c.k), wq(c.top_q, c.k);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        double w[8], v[8];
        wp(rp[i], w);
        wq(rq[i], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            zp += w[j];
            zq += v[j];
        }
    }
    zp = all_sum(zp);
    zq = all_sum(zq);
    if (lane_id() == 0) {
        s_z[0][threadIdx.x >> 6] = zp;
        s_z[1][threadIdx.x >> 6] = zq;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        const double *z = s_z[threadIdx.x];
        p.z[((int64_t)s * p.splits + blockIdx.x) * 2 + threadIdx.x] = (z[0] + z[1]) + (z[2] + z[3]);
    }
}

// the row's sums from its chunks', in their order: by a whole wavefront
__device__ __forceinline__ void exact_sums(const VerifyParams &p, int s, double &zp, double &zq) {
    zp = zq = 0.0;
    for (int c = lane_id(); c < p.splits; c += 64) {
        zp += p.z[((int64_t)s * p.splits + c) * 2];
        zq += p.z[((int64_t)s * p.splits + c) * 2 + 1];
    }
    zp = all_sum(zp);
    zq = all_sum(zq);
}

// The weights of eight consecutive tokens that one is drawn from, relative to exp((top - row's top) / T): max(p - q, 0) with
// top = 0 by agreement (`rest`, with draft logits), else the exponentials, the refused draft's taken out; by a whole wavefront.
// (`r` and `q`: loaded, q only with draft logits)
template <typename T>
__device__ __forceinline__ float weights8(const Choice &c, Raw8<T> &r, Raw8<T> &q, bool rest, double ip, double iq, double *w) {
    r.clip();
    if (rest && c.draft >= 0) {
        q.clip();
        const Weigh wp(c.top_p, c.k), wq(c.top_q, c.k);
        double v[8];
        wp(r, w);
        wq(q, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double d = w[j] * ip - v[j] * iq;
            w[j] = d > 0.0 ? d : 0.0;
        }
        return 0.0f;
    }
    const float top = all_max(largest8(r));
    if (c.k > 0.0) {
        const Weigh wp(top, c.k);
        wp(r, w);
    } else {                                                            // greedy, in a call without statistics
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = top > -INFINITY && r.get(j) == top && j >= r.skip ? 1.0 : 0.0;
    }
    if (rest && c.one_hot >= 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = r.base + j == c.one_hot ? 0.0 : w[j];
    }
    return top;
}
template <typename T>
__device__ __forceinline__ void load_pair(const VerifyParams &p, const Choice &c, int i, Raw8<T> &r, Raw8<T> &q) {
    r.load((const T *)p.logits + (int64_t)c.row * p.ld_t, i, p.V);
    if (c.draft >= 0) q.load((const T *)p.draft_logits + (int64_t)c.draft * p.ld_d, i, p.V);
}

// ---- sums of the weights that the next token is drawn from -------------------------------------------
// Which row: chosen by the launch before (draft logits), by this one (drafts without), or no drafts in the call.  (The last as
// an instance of its own: without the drafts' registers a CU holds five workgroups of fp32 logits instead of three.)
enum { VER_CHOSEN, VER_CHOOSE, VER_SAMPLE };
template <typename T, int ROW>
__global__ __launch_bounds__(VER_THREADS) void verify_sums_kernel(VerifyParams p) {
    const int s = blockIdx.y;
    Choice c;
    if (ROW == VER_CHOSEN) c = p.choice[s];
    else c = choose<T, ROW == VER_CHOOSE>(p, s, blockIdx.x == 0);
    if (c.row < 0 || c.greedy >= 0) return;
    Raw8<T> r[4], q[4];
    const int sub0 = blockIdx.x * (VER_CHUNK / VER_SUB) + (int)(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < 4; ++i) load_pair(p, c, (sub0 + i * 4) * VER_SUB + lane_id() * 8, r[i], q[i]);
    double ip = 0.0, iq = 0.0;
    if (c.draft >= 0) {
        exact_sums(p, s, ip, iq);
        ip = 1.0 / ip;
        iq = 1.0 / iq;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int sub = sub0 + i * 4;
        double w[8];
        const float top = weights8<T>(c, r[i], q[i], true, ip, iq, w);
        const double a = all_sum(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
        if (sub < p.subs && lane_id() == 0) p.blocks[(int64_t)s * p.subs + sub] = Block{a, top, 0};
    }
}

// ---- the draw: one wavefront per sequence --------------------------------------------------------------
// A lane has `per` neighbouring blocks; one scan over the lanes finds whose, that lane its block, the wavefront the token in it.
template <typename T>
__global__ __launch_bounds__(64) void verify_draw_kernel(VerifyParams p) {
    const int s = blockIdx.x, per = (p.subs + 63) / 64, b0 = min((int)lane_id() * per, p.subs), b1 = min(b0 + per, p.subs);
    Block *blocks = p.blocks + (int64_t)s * p.subs;
    const Choice c = p.choice[s];
    const float u = p.sample_u[s];
    if (c.row < 0 || c.greedy >= 0) return;
    double ip = 0.0, iq = 0.0;
    if (c.draft >= 0) {
        exact_sums(p, s, ip, iq);
        ip = 1.0 / ip;
        iq = 1.0 / iq;
    }
    bool rest = true;
    double lane_sum, total;
    float top;
    constexpr int KEEP = 4;                                   // blocks of a lane that stay in registers (131 072 tokens)
    Block v[KEEP];
    auto block_weight = [&](const Block &v) {                 // relative to the largest block's top
        return c.k > 0.0 ? v.sum * weight_of(v.top, top, c.k) : v.top == top ? v.sum : 0.0;
    };
    for (;;) {
#pragma unroll
        for (int i = 0; i < KEEP; ++i) v[i] = b0 + i < b1 ? blocks[b0 + i] : Block{0.0, -INFINITY, 0};
        if (rest && c.draft >= 0) {
            top = 0.0f;                                       // (by agreement: these sums are absolute)
        } else {
            top = -INFINITY;
#pragma unroll
            for (int i = 0; i < KEEP; ++i) top = fmaxf(top, v[i].sum > 0.0 ? v[i].top : -INFINITY);
            for (int b = b0 + KEEP; b < b1; ++b) top = fmaxf(top, blocks[b].sum > 0.0 ? blocks[b].top : -INFINITY);
            top = all_max(top);
        }
        lane_sum = 0.0;
#pragma unroll
        for (int i = 0; i < KEEP; ++i) lane_sum += v[i].sum = block_weight(v[i]);
        for (int b = b0 + KEEP; b < b1; ++b) lane_sum += block_weight(blocks[b]);
        total = all_sum(lane_sum);
        if (total > 0.0 || !rest) break;
        // nothing of p exceeds q: p itself.  (Two equal distributions keep every draft, so this is rare: the sums are made here.)
        rest = false;
        for (int b = 0; b < p.subs; ++b) {
            double w[8];
            Raw8<T> r1, q1;
            load_pair(p, c, b * VER_SUB + lane_id() * 8, r1, q1);
            const float t = weights8<T>(c, r1, q1, false, ip, iq, w);
            const double a = all_sum(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
            if (lane_id() == 0) blocks[b] = Block{a, t, 0};
        }
        __threadfence();
    }
    int64_t *out = p.tokens + (int64_t)s * p.max_q + c.count;
    if (!(total > 0.0)) {
        if (lane_id() == 0) *out = -1;
        return;
    }
    const double aim = c.k > 0.0 ? (double)u * total : 0.0;    // (greedy: the first of the largest)
    // the first lane whose inclusive sum exceeds the aim (else the last that has any weight), and of its blocks likewise
    const double run = scan_all(lane_sum, 0.0, plus<double>);
    const uint64_t past = __ballot(run > aim && lane_sum > 0.0), any = __ballot(lane_sum > 0.0);
    const int owner = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(any);
    int sub = -1;
    double before = run - lane_sum;
    if ((int)lane_id() == owner) {
        int last = -1;
        double last_before = 0.0, sum = before;
        auto step = [&](int b, double w) {
            if (sub >= 0) return;
            if (w > 0.0) {
                last = b;
                last_before = sum;
                if (past && sum + w > aim) sub = b;
            }
            sum += w;
        };
#pragma unroll
        for (int i = 0; i < KEEP; ++i) step(b0 + i, v[i].sum);
        for (int b = b0 + KEEP; b < b1; ++b) step(b, block_weight(blocks[b]));
        // (rounding between the scan and this sum, or no block past the aim: the last token with a weight is taken)
        before = sub >= 0 ? last_before : -INFINITY;
        if (sub < 0) sub = last;
    }
    sub = __builtin_amdgcn_readlane(sub, owner);
    before = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(before), owner), __builtin_amdgcn_readlane(__double2loint(before), owner));
    double w[8], own = 0.0;
    Raw8<T> r1, q1;
    load_pair(p, c, sub * VER_SUB + lane_id() * 8, r1, q1);
    const float block_top = weights8<T>(c, r1, q1, rest, ip, iq, w);
    const double scale = c.k > 0.0 ? weight_of(block_top, top, c.k) : 1.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        w[j] *= scale;
        own += w[j];
    }
    // the first token of this lane whose cumulative weight exceeds the aim, and the last that has any weight
    const double up_to = before + (scan_all(own, 0.0, plus<double>) - own);
    int hit = 0x7fffffff, last = -1;
    double cum = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        cum += w[j];
        if (w[j] > 0.0) {
            if (hit == 0x7fffffff && up_to + cum > aim) hit = r1.base + j;
            last = r1.base + j;
        }
    }
    hit = all_min(hit);
    last = all_max(last);
    if (lane_id() == 0) *out = hit != 0x7fffffff ? hit : last;
}

// ---- entry points ------------------------------------------------------------------------------------
struct VerifyLayout {
    size_t stats, z, blocks, choice, padded, total;
    int splits, subs;
};
static bool verify_layout(int64_t S, int64_t n_q, int64_t n_d, int64_t V, bool draft_logits, VerifyLayout &l) {
    l.splits = (int)((V + VER_CHUNK - 1) / VER_CHUNK);
    l.subs = (int)((V + VER_SUB - 1) / VER_SUB);
    size_t o = 0;
    auto take = [&](size_t bytes) { const size_t at = o; o += odsd_round_up(bytes, 256); return at; };
    l.stats = take(n_d ? (size_t)(n_q + (draft_logits ? n_d : 0)) * l.splits * sizeof(Stat) : 0);
    l.z = take(draft_logits ? (size_t)S * l.splits * 16 : 0);
    l.blocks = take((size_t)S * l.subs * sizeof(Block));
    l.choice = take((size_t)S * sizeof(Choice));
    l.padded = take(V < 8 ? (size_t)(n_q + n_d) * 8 * 4 : 0);
    l.total = o;
    return (n_q + n_d) * l.splits < (1LL << 32) / VER_THREADS && S <= 65535;      // a launch has fewer than 2^32 threads
}
static bool verify_sizes_ok(int32_t S, int32_t max_q, int32_t n_q, int32_t n_d, int32_t V) {
    return S >= 0 && max_q >= 0 && n_q >= 0 && n_d >= 0 && V > 0;
}

extern "C" size_t odsd_verify_workspace_bytes(int32_t n_seqs, int32_t max_q_len, int32_t n_rows, int32_t n_drafts,
                                              int32_t vocab, int32_t has_draft_logits) {
    VerifyLayout l;
    // a row of logits and one of tokens are stepped over in 31 bits, by chunks and by a workgroup's threads
    if (!verify_sizes_ok(n_seqs, max_q_len, n_rows, n_drafts, vocab) || vocab > 0x7fffffff - VER_CHUNK ||
        max_q_len > 0x7fffffff - VER_THREADS || !verify_layout(n_seqs, n_rows, n_drafts, vocab, has_draft_logits != 0, l)) return 0;
    return l.total > 256 ? l.total : 256;
}

template <typename T> static int launch_verify(VerifyParams &p, void *padded, hipStream_t st) {
    if (p.V < 8) {
        T *rows = (T *)padded, *draft_rows = rows + (int64_t)p.n_q * 8;
        auto pad = [&](const void *src, int64_t ld, T *dst, int n) {
            if (n > 0) verify_pad_kernel<T><<<(unsigned)(((int64_t)n * 8 + VER_THREADS - 1) / VER_THREADS), VER_THREADS, 0, st>>>((const T *)src, ld, dst, n, p.V);
        };
        pad(p.logits, p.ld_t, rows, p.n_q);
        if (p.draft_logits) {
            pad(p.draft_logits, p.ld_d, draft_rows, p.n_d);
            p.draft_logits = draft_rows;
        }
        p.logits = rows;
        p.ld_t = p.ld_d = p.V = 8;
    }
    const dim3 chunks((unsigned)p.splits, (unsigned)p.S);
    if (p.n_d > 0 && p.n_q > 0) verify_stats_kernel<T><<<(unsigned)((p.n_q + (p.draft_logits ? p.n_d : 0)) * p.splits), VER_THREADS, 0, st>>>(p);
    if (p.draft_logits) {
        verify_choose_kernel<T><<<chunks, VER_THREADS, 0, st>>>(p);
        verify_sums_kernel<T, VER_CHOSEN><<<chunks, VER_THREADS, 0, st>>>(p);
    } else if (p.n_d > 0) {
        verify_sums_kernel<T, VER_CHOOSE><<<chunks, VER_THREADS, 0, st>>>(p);
    } else {
        verify_sums_kernel<T, VER_SAMPLE><<<chunks, VER_THREADS, 0, st>>>(p);
    }
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
                   tokens, num_accepted, accept_probs, (Stat *)(ws + l.stats), (double *)(ws + l.z),
                   (Block *)(ws + l.blocks), (Choice *)(ws + l.choice)};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ODSD_DT_F32) return launch_verify<float>(p, ws + l.padded, st);
    if (dtype == ODSD_DT_BF16) return launch_verify<__bf16>(p, ws + l.padded, st);
    return launch_verify<half_t>(p, ws + l.padded, st);
}
