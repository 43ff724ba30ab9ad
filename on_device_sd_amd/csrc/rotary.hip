// Rotary positions of the queries and keys of a step, with one or several position axes, the per-head RMSNorm in front
// of them (optional), and the KV-cache store behind them (optional).
//
// Frequency i in [0, R/2) turns the pair (x[i], x[i + R/2]) of a head (pairs side by side: x[2i], x[2i + 1]) by the angle
// pos[axis(i)] * inv_freq[i]; columns from R on pass.  Angles in fp64, in whole turns: a position of a million times a
// frequency of 1 has 20 bits before the point, which leaves fp32 none of the digits that an fp32 result needs behind it.  (Three
// roundings: less than 3 2^-53 of the number of turns, below the fraction's 2^-26 in fp32 up to positions of 2^28.)
// Everything else in fp32, one rounding at the end.
#include "common.h"

#define ROT_THREADS 256

struct RotaryParams {
    const void *q, *k, *v;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;   // elements between two tokens / two heads
    const void *positions;          // [n_axes][pos_ld], int32 or int64
    int64_t pos_ld;
    const double *inv_freq;         // [R / 2]
    int sec_end[4];                 // frequencies [sec_end[a-1], sec_end[a]) belong to axis a
    const void *q_weight, *k_weight;
    float eps;
    void *q_out;                    // [n, Hq, D]
    void *k_out;                    // [n, Hk, D] or null
    void *k_cache, *v_cache;        // [num_slots, Hk * D] or null
    const int32_t *slots, *src;
    int64_t num_slots;
    int n, n_store;                 // tokens; rows that are stored
    int Hq, Hk, D, R;
    int q_tokens, kv_tokens, q_wgs; // tokens of a workgroup, workgroups that have queries
};

// sin and cos of t turns, |t| <= 1/2: reduced to an eighth of a turn and the quarter it lies in, Taylor polynomials there
// (|x| <= pi/4: the next term is below 2^-27)
__device__ __forceinline__ void sincos_turns(float t, float &s, float &c) {
    const float q = rintf(t * 4.0f);
    const float x = (t - q * 0.25f) * 6.28318530717958648f;        // t - q/4 is exact
    const float x2 = x * x;
    const float sn = x + x * x2 * (-1.6666666666666667e-1f + x2 * (8.3333333333333333e-3f + x2 * (-1.9841269841269841e-4f + x2 * 2.7557319223985893e-6f)));
    const float cs = 1.0f + x2 * (-0.5f + x2 * (4.1666666666666667e-2f + x2 * (-1.3888888888888889e-3f + x2 * (2.4801587301587302e-5f - x2 * 2.7557319223985888e-7f))));
    const int iq = (int)q & 3;
    const float a = iq & 1 ? cs : sn, b = iq & 1 ? sn : cs;
    s = iq & 2 ? -a : a;
    c = (iq + 1) & 2 ? -b : b;
}

// What a workgroup has: the heads of `rows` tokens of q, or of rows that go to k_out and the cache with the values beside them.
struct RotaryPart {
    bool is_q;
    int row0, rows, H;
    const void *src, *weight;
    int64_t token_ld, head_ld;
};
__device__ __forceinline__ RotaryPart rotary_part(const RotaryParams &p) {
    RotaryPart w;
    w.is_q = (int)blockIdx.x < p.q_wgs;
    const int per = w.is_q ? p.q_tokens : p.kv_tokens;
    w.row0 = (w.is_q ? blockIdx.x : blockIdx.x - p.q_wgs) * per;
    w.rows = min(per, (w.is_q ? p.n : p.n_store) - w.row0);
    w.H = w.is_q ? p.Hq : p.Hk;
    w.src = w.is_q ? p.q : p.k;
    w.weight = w.is_q ? p.q_weight : p.k_weight;
    w.token_ld = w.is_q ? p.q_token : p.k_token;
    w.head_ld = w.is_q ? p.q_head : p.k_head;
    return w;
}
__device__ __forceinline__ int rotary_token(const RotaryParams &p, const RotaryPart &w, int r) {
    const int t = w.is_q || !p.src ? w.row0 + r : p.src[w.row0 + r];
    return t >= 0 && t < p.n ? t : -1;
}
__device__ __forceinline__ int64_t rotary_slot(const RotaryParams &p, const RotaryPart &w, int r) {
    const int64_t slot = p.slots[w.row0 + r];
    return slot >= 0 && slot < p.num_slots ? slot : -1;
}
// (cos, sin) of every frequency of the workgroup's tokens
template <typename POS>
__device__ __forceinline__ void rotary_angles(const RotaryParams &p, const RotaryPart &w, float2 *trig) {
    const int half = p.R / 2;
    for (int i = threadIdx.x; i < w.rows * half; i += ROT_THREADS) {
        const int r = i / half, f = i - r * half;
        const int t = rotary_token(p, w, r);
        float s = 0.0f, c = 1.0f;
        if (t >= 0) {
            const int axis = (f >= p.sec_end[0]) + (f >= p.sec_end[1]) + (f >= p.sec_end[2]);
            const double turns = (double)((const POS *)p.positions)[axis * p.pos_ld + t] * (p.inv_freq[f] * 0.15915494309189533577);
            sincos_turns((float)(turns - rint(turns)), s, c);
        }
        trig[i] = make_float2(c, s);
    }
}
// Where a head of a token goes: its place in q_out or k_out, and in the cache, if its row has one.
template <typename T>
__device__ __forceinline__ void rotary_targets(const RotaryParams &p, const RotaryPart &w, int r, int t, int h, T *&dst, T *&dst2) {
    dst = w.is_q ? (T *)p.q_out + ((int64_t)t * p.Hq + h) * p.D : p.k_out ? (T *)p.k_out + ((int64_t)t * p.Hk + h) * p.D : nullptr;
    dst2 = nullptr;
    if (!w.is_q && p.k_cache) {
        const int64_t slot = rotary_slot(p, w, r);
        if (slot >= 0) dst2 = (T *)p.k_cache + (slot * p.Hk + h) * p.D;
    }
}
// The first columns of the two halves of unit u: V frequencies with both members of their pairs, or 2 V columns that pass.
template <int V, bool SIDE>
__device__ __forceinline__ void rotary_columns(const RotaryParams &p, int u, int &c0, int &c1) {
    const int half = p.R / 2;
    if (u < half / V) {
        c0 = SIDE ? 2 * V * u : V * u;
        c1 = SIDE ? c0 + V : c0 + half;
    } else {
        c0 = p.R + (u - half / V) * 2 * V;
        c1 = c0 + V;
    }
}
template <int V, bool SIDE>
__device__ __forceinline__ void rotary_turn(float *x, const float2 *cs) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int lo = SIDE ? 2 * i : i, hi = SIDE ? 2 * i + 1 : V + i;
        const float c = cs[i].x, s = cs[i].y, x1 = x[lo], x2 = x[hi];
        x[lo] = x1 * c - x2 * s;
        x[hi] = x2 * c + x1 * s;
    }
}

// Everything in pieces of eight 16-bit values, 16-byte aligned.  A head's units (two pieces each) lie on LG neighbouring lanes,
// which add up its squares; a thread's first unit is requested before the angles are made, so that its way from memory and
// the sines hide each other.  Bytes bound it: 16384 tokens of 32 + 4 heads of 128 on three axes in 57 to 61 us, 4.9 to
// 5.3 TB/s; two units a thread 60, four 69 (fewer workgroups at once); one token a workgroup for the keys, too, 73 to 84.
template <typename T, bool SIDE, typename POS>
__global__ __launch_bounds__(ROT_THREADS) void rotary_wide_kernel(RotaryParams p, int LG) {
    typedef T T8 __attribute__((ext_vector_type(8)));
    extern __shared__ float2 trig[];                      // [rows][R / 2]: (cos, sin)
    const RotaryPart w = rotary_part(p);
    const int half = p.R / 2, units = p.D / 16, per_pass = ROT_THREADS / LG, total = w.rows * w.H;
    const int sub = threadIdx.x % LG, first = threadIdx.x / LG;
    int c0, c1;
    rotary_columns<8, SIDE>(p, min(sub, units - 1), c0, c1);
    T8 a, b, wa, wb;
    int token;
    auto fetch = [&](int hr) {
        const int r = min(hr, total - 1) / w.H, h = min(hr, total - 1) - r * w.H;
        token = rotary_token(p, w, r);
        const T *row = (const T *)w.src + max(token, 0) * w.token_ld + h * w.head_ld;
        a = *(const T8 *)(row + c0);
        b = *(const T8 *)(row + c1);
    };
    fetch(first);
    if (w.weight) {
        wa = *(const T8 *)((const T *)w.weight + c0);
        wb = *(const T8 *)((const T *)w.weight + c1);
    }
    if (!w.is_q && p.v_cache) {
        const int chunks = p.Hk * (p.D / 8);
        for (int i = threadIdx.x; i < w.rows * chunks; i += ROT_THREADS) {
            const int r = i / chunks, c = i - r * chunks, h = c / (p.D / 8), at = (c - h * (p.D / 8)) * 8;
            const int t = rotary_token(p, w, r);
            const int64_t slot = rotary_slot(p, w, r);
            if (t >= 0 && slot >= 0)
                *(T8 *)((T *)p.v_cache + (slot * p.Hk + h) * p.D + at) = *(const T8 *)((const T *)p.v + t * p.v_token + h * p.v_head + at);
        }
    }
    rotary_angles<POS>(p, w, trig);
    __syncthreads();
    for (int hr = first; hr < total; hr += per_pass) {
        if (hr != first) fetch(hr);
        const int r = hr / w.H, h = hr - r * w.H;
        float x[16];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = (float)a[e];
            x[8 + e] = (float)b[e];
        }
        if (w.weight) {
            float ss = 0.0f;
            if (sub < units) {
#pragma unroll
                for (int e = 0; e < 16; ++e) ss += x[e] * x[e];
            }
            for (int o = LG / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, ODSD_WAVE);   // (all LG lanes of a head are here)
            const float scale = rsqrtf(ss / (float)p.D + p.eps);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] *= scale * (float)wa[e];
                x[8 + e] *= scale * (float)wb[e];
            }
        }
        if (sub >= units || token < 0) continue;
        if (sub < half / 8) rotary_turn<8, SIDE>(x, trig + r * half + sub * 8);
        T8 ya, yb;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            ya[e] = (T)x[e];
            yb[e] = (T)x[8 + e];
        }
        T *dst, *dst2;
        rotary_targets(p, w, r, token, h, dst, dst2);
        if (dst) {
            *(T8 *)(dst + c0) = ya;
            *(T8 *)(dst + c1) = yb;
        }
        if (dst2) {
            *(T8 *)(dst2 + c0) = ya;
            *(T8 *)(dst2 + c1) = yb;
        }
    }
}

// Any head size, strides and alignment: value by value, a unit is one pair; a head's units lie on LG lanes in turns.  16384 tokens
// of 32 + 4 heads of 128 without norms, 2 bytes off alignment: 142 us, 2.1 TB/s (aligned, by the kernel above: 60).
template <typename T, bool SIDE, typename POS>
__global__ __launch_bounds__(ROT_THREADS) void rotary_any_kernel(RotaryParams p, int LG) {
    extern __shared__ float2 trig[];
    const RotaryPart w = rotary_part(p);
    rotary_angles<POS>(p, w, trig);
    __syncthreads();
    const int half = p.R / 2, units = p.D / 2, sub = threadIdx.x % LG;
    for (int hr = threadIdx.x / LG; hr < w.rows * w.H; hr += ROT_THREADS / LG) {
        const int r = hr / w.H, h = hr - r * w.H;
        const int t = rotary_token(p, w, r);
        if (t < 0) continue;                              // (all LG lanes of the head agree)
        T *dst, *dst2;
        rotary_targets(p, w, r, t, h, dst, dst2);
        const T *row = (const T *)w.src + t * w.token_ld + h * w.head_ld, *weight = (const T *)w.weight;
        float scale = 1.0f;
        int c0, c1;
        if (weight) {
            float ss = 0.0f;
            for (int u = sub; u < units; u += LG) {
                rotary_columns<1, SIDE>(p, u, c0, c1);
                ss += (float)row[c0] * (float)row[c0] + (float)row[c1] * (float)row[c1];
            }
            for (int o = LG / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, ODSD_WAVE);
            scale = rsqrtf(ss / (float)p.D + p.eps);
        }
        for (int u = sub; u < units; u += LG) {
            rotary_columns<1, SIDE>(p, u, c0, c1);
            float x[2] = {(float)row[c0], (float)row[c1]};
            if (weight) {
                x[0] *= scale * (float)weight[c0];
                x[1] *= scale * (float)weight[c1];
            }
            if (u < half) rotary_turn<1, SIDE>(x, trig + r * half + u);
            if (dst) {
                dst[c0] = (T)x[0];
                dst[c1] = (T)x[1];
            }
            if (dst2) {
                dst2[c0] = (T)x[0];
                dst2[c1] = (T)x[1];
            }
        }
    }
    if (w.is_q || !p.v_cache) return;
    for (int i = threadIdx.x; i < w.rows * p.Hk * p.D; i += ROT_THREADS) {
        const int r = i / (p.Hk * p.D), c = i - r * (p.Hk * p.D), h = c / p.D, at = c - h * p.D;
        const int t = rotary_token(p, w, r);
        const int64_t slot = rotary_slot(p, w, r);
        if (t >= 0 && slot >= 0) ((T *)p.v_cache)[(slot * p.Hk + h) * p.D + at] = ((const T *)p.v)[t * p.v_token + h * p.v_head + at];
    }
}

template <typename T, bool SIDE, typename POS>
static int launch_rotary(RotaryParams &p, bool wide, hipStream_t st) {
    const int units = wide ? p.D / 16 : p.D / 2;
    int LG = 1;
    while (LG < units && LG < 64) LG *= 2;
    // Tokens of a workgroup: one while there are few workgroups, else as many as give each thread a unit (at most 32: their
    // angles, 4 KB a token for 1024 columns, stay within the LDS)
    const bool many = wide && (int64_t)p.n + p.n_store >= 2048;
    auto tokens = [&](int H) { return many ? max(1, min(ROT_THREADS / (LG * H), 32)) : 1; };
    p.q_tokens = tokens(p.Hq);
    p.kv_tokens = tokens(p.Hk);
    p.q_wgs = (p.n + p.q_tokens - 1) / p.q_tokens;
    const unsigned grid = (unsigned)(p.q_wgs + (p.n_store + p.kv_tokens - 1) / p.kv_tokens);
    if (grid >= (1u << 24)) return ODSD_ERR_UNSUPPORTED;       // 2^32 threads
    const size_t lds = (size_t)max(p.q_tokens, p.kv_tokens) * (p.R / 2) * sizeof(float2);
    if (wide) rotary_wide_kernel<T, SIDE, POS><<<grid, ROT_THREADS, lds, st>>>(p, LG);
    else rotary_any_kernel<T, SIDE, POS><<<grid, ROT_THREADS, lds, st>>>(p, LG);
    ODSD_CHECK_LAUNCH();
    return ODSD_OK;
}

extern "C" int odsd_rotary(const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k,
                           int64_t k_token_stride, int64_t k_head_stride, const void *v, int64_t v_token_stride,
                           int64_t v_head_stride, int32_t n, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                           int32_t rotary_dim, int32_t interleaved, int32_t dtype, const void *positions,
                           int32_t position_bytes, int32_t n_axes, int64_t position_stride, const int32_t *sections,
                           const double *inv_freq, const void *q_weight, const void *k_weight, float eps, void *q_out,
                           void *k_out, void *k_cache, void *v_cache, const int32_t *slot_mapping,
                           const int32_t *src_index, int32_t n_store, int64_t num_slots, void *stream) {
    if (n < 0 || n_store < 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || rotary_dim <= 0 || (rotary_dim & 1) ||
        (head_dim & 1) || rotary_dim > head_dim || n_axes < 1 || num_slots < 0) return ODSD_ERR_SHAPE;
    // a token's columns and the rows of a call are counted in 31 bits, the columns in steps of a workgroup's threads
    if (head_dim > 1024 || n_axes > 4 || (int64_t)n + n_store > 0x7fffffffLL ||
        (int64_t)max(num_heads, num_kv_heads) * head_dim > 0x7fffffffLL - ROT_THREADS) return ODSD_ERR_UNSUPPORTED;
    if (dtype != ODSD_DT_BF16 && dtype != ODSD_DT_F16) return ODSD_ERR_DTYPE;
    if (position_bytes != 4 && position_bytes != 8) return ODSD_ERR_DTYPE;
    RotaryParams p;
    int end = 0;
    for (int a = 0; a < 4; ++a) {
        if (a < n_axes) {
            const int count = n_axes == 1 && !sections ? rotary_dim / 2 : sections ? sections[a] : -1;
            if (count < 0) return ODSD_ERR_SHAPE;
            end += count;
            if (end > rotary_dim / 2) return ODSD_ERR_SHAPE;
        }
        p.sec_end[a] = a < n_axes - 1 ? end : rotary_dim / 2;
    }
    if (end != rotary_dim / 2) return ODSD_ERR_SHAPE;
    const bool store = k_cache || v_cache;
    if (n == 0) return ODSD_OK;
    if (!q || !k || !q_out || !positions || !inv_freq) return ODSD_ERR_NULL;
    if (!k_out && !store) return ODSD_ERR_NULL;
    if (store && (!k_cache || !v_cache || !v || (n_store && !slot_mapping))) return ODSD_ERR_NULL;
    if (store && !src_index && n_store != n && (n_store != 0 || k_out)) return ODSD_ERR_SHAPE;
    if (store && src_index && k_out) return ODSD_ERR_UNSUPPORTED;      // keys that are not stored would not be computed
    if (!store && n_store != 0) return ODSD_ERR_SHAPE;
    p.q = q; p.k = k; p.v = v;
    p.q_token = q_token_stride; p.q_head = q_head_stride;
    p.k_token = k_token_stride; p.k_head = k_head_stride;
    p.v_token = v_token_stride; p.v_head = v_head_stride;
    p.positions = positions; p.pos_ld = position_stride;
    p.inv_freq = inv_freq;
    p.q_weight = q_weight; p.k_weight = k_weight; p.eps = eps;
    p.q_out = q_out; p.k_out = k_out; p.k_cache = k_cache; p.v_cache = v_cache;
    p.slots = slot_mapping; p.src = src_index; p.num_slots = num_slots;
    p.n = n; p.n_store = store ? n_store : n;
    p.Hq = num_heads; p.Hk = num_kv_heads; p.D = head_dim; p.R = rotary_dim;
    const uintptr_t bytes = (uintptr_t)q | (uintptr_t)k | (uintptr_t)(store ? v : nullptr) | (uintptr_t)q_weight |
                            (uintptr_t)k_weight | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)k_cache | (uintptr_t)v_cache;
    uint64_t elems = (uint64_t)q_token_stride | (uint64_t)q_head_stride | (uint64_t)k_token_stride | (uint64_t)k_head_stride;
    if (store) elems |= (uint64_t)v_token_stride | (uint64_t)v_head_stride;
    if (bytes & 1) return ODSD_ERR_ALIGN;
    if (((uintptr_t)positions & (position_bytes - 1)) || ((uintptr_t)inv_freq & 7)) return ODSD_ERR_ALIGN;
    const bool wide = (bytes & 15) == 0 && (elems & 7) == 0 && rotary_dim % 16 == 0 && head_dim % 16 == 0;
    hipStream_t st = (hipStream_t)stream;
#define ROT_GO(T, POS) (interleaved ? launch_rotary<T, true, POS>(p, wide, st) : launch_rotary<T, false, POS>(p, wide, st))
    if (dtype == ODSD_DT_BF16) return position_bytes == 8 ? ROT_GO(__bf16, int64_t) : ROT_GO(__bf16, int32_t);
    return position_bytes == 8 ? ROT_GO(half_t, int64_t) : ROT_GO(half_t, int32_t);
#undef ROT_GO
}
