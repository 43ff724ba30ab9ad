// Rotary positions of the queries and keys of a step, with one or several position axes, the per-head RMSNorm in front
// of them (optional), and the KV-cache store behind them (optional).
//
// Frequency i in [0, R/2) turns the pair (x[i], x[i + R/2]) of a head (pairs side by side: x[2i], x[2i + 1]) by the angle
// pos[axis(i)] * inv_freq[i]; columns from R on pass.  Angles in fp64, in whole turns: a position of a million times a
// frequency of 1 has 20 bits before the point, which leaves fp32 none of the digits that an fp32 result needs behind it.
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
    int tokens_per_wg, q_wgs;
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

// V: values per access (8: 16-bit elements, everything 16-byte aligned, R and D - R multiples of 16; else 1).
// A unit is 2 V columns of a head: V frequencies with both members of their pairs, or 2 V columns that pass.  The units of a
// head lie on LG neighbouring lanes (a power of two), which add up its squares.
template <typename T, int V, bool SIDE, typename POS>
__global__ __launch_bounds__(ROT_THREADS) void rotary_kernel(RotaryParams p, int LG) {
    typedef T TV __attribute__((ext_vector_type(V)));
    extern __shared__ float2 trig[];                      // [tokens_per_wg][R / 2]: (cos, sin)
    const int half = p.R / 2;
    const bool is_q = (int)blockIdx.x < p.q_wgs;
    const int row0 = (is_q ? blockIdx.x : blockIdx.x - p.q_wgs) * p.tokens_per_wg;
    const int rows = min(p.tokens_per_wg, (is_q ? p.n : p.n_store) - row0);
    auto token_of = [&](int r) { return is_q || !p.src ? row0 + r : p.src[row0 + r]; };
    for (int i = threadIdx.x; i < rows * half; i += ROT_THREADS) {
        const int r = i / half, f = i - r * half;
        const int t = token_of(r);
        float s = 0.0f, c = 1.0f;
        if (t >= 0 && t < p.n) {
            const int axis = (f >= p.sec_end[0]) + (f >= p.sec_end[1]) + (f >= p.sec_end[2]);
            const double turns = (double)((const POS *)p.positions)[axis * p.pos_ld + t] * (p.inv_freq[f] * 0.15915494309189533577);
            sincos_turns((float)(turns - rint(turns)), s, c);
        }
        trig[i] = make_float2(c, s);
    }
    __syncthreads();

    const int units = half / V + (p.D - p.R) / (2 * V);
    const int H = is_q ? p.Hq : p.Hk;
    const int per_pass = ROT_THREADS / LG;
    const int sub = threadIdx.x % LG;
    const T *src = (const T *)(is_q ? p.q : p.k), *weight = (const T *)(is_q ? p.q_weight : p.k_weight);
    const int64_t token_ld = is_q ? p.q_token : p.k_token, head_ld = is_q ? p.q_head : p.k_head;
    for (int hr = threadIdx.x / LG; hr < rows * H; hr += per_pass) {
        const int r = hr / H, h = hr - r * H;
        const int t = token_of(r);
        if (t < 0 || t >= p.n) continue;                  // (all LG lanes of the head agree)
        T *dst = is_q ? (T *)p.q_out + ((int64_t)t * p.Hq + h) * p.D
                      : p.k_out ? (T *)p.k_out + ((int64_t)t * p.Hk + h) * p.D : nullptr;
        T *dst2 = nullptr;                                // the head's place in the cache, if its row has one
        if (!is_q && p.k_cache) {
            const int64_t slot = p.slots[row0 + r];
            if (slot >= 0 && slot < p.num_slots) dst2 = (T *)p.k_cache + (slot * p.Hk + h) * p.D;
        }
        if (!dst && !dst2) continue;
        const T *row = src + t * token_ld + h * head_ld;
        float scale = 1.0f;
        auto columns = [&](int u, int &c0, int &c1) {     // the first columns of a unit's two halves
            if (u < half / V) {
                c0 = SIDE ? 2 * V * u : V * u;
                c1 = SIDE ? c0 + V : c0 + half;
            } else {
                c0 = p.R + (u - half / V) * 2 * V;
                c1 = c0 + V;
            }
        };
        if (weight) {
            float ss = 0.0f;
            for (int u = sub; u < units; u += LG) {
                int c0, c1;
                columns(u, c0, c1);
                const TV a = *(const TV *)(row + c0), b = *(const TV *)(row + c1);
#pragma unroll
                for (int i = 0; i < V; ++i) ss += (float)a[i] * (float)a[i] + (float)b[i] * (float)b[i];
            }
            for (int o = LG / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, ODSD_WAVE);
            scale = rsqrtf(ss / (float)p.D + p.eps);
        }
        for (int u = sub; u < units; u += LG) {
            int c0, c1;
            columns(u, c0, c1);
            const TV a = *(const TV *)(row + c0), b = *(const TV *)(row + c1);
            float x[2 * V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                x[i] = (float)a[i];
                x[V + i] = (float)b[i];
            }
            if (weight) {
                const TV wa = *(const TV *)(weight + c0), wb = *(const TV *)(weight + c1);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    x[i] *= scale * (float)wa[i];
                    x[V + i] *= scale * (float)wb[i];
                }
            }
            if (u < half / V) {
                const float2 *cs = trig + r * half + u * V;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int lo = SIDE ? 2 * i : i, hi = SIDE ? 2 * i + 1 : V + i;
                    const float c = cs[i].x, s = cs[i].y, x1 = x[lo], x2 = x[hi];
                    x[lo] = x1 * c - x2 * s;
                    x[hi] = x2 * c + x1 * s;
                }
            }
            TV ya, yb;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                ya[i] = (T)x[i];
                yb[i] = (T)x[V + i];
            }
            if (dst) {
                *(TV *)(dst + c0) = ya;
                *(TV *)(dst + c1) = yb;
            }
            if (dst2) {
                *(TV *)(dst2 + c0) = ya;
                *(TV *)(dst2 + c1) = yb;
            }
        }
    }
    if (is_q || !p.v_cache) return;
    const int chunks = p.D / V;
    for (int i = threadIdx.x; i < rows * p.Hk * chunks; i += ROT_THREADS) {
        const int r = i / (p.Hk * chunks), c = i - r * (p.Hk * chunks);
        const int t = token_of(r);
        const int64_t slot = p.slots[row0 + r];
        if (t < 0 || t >= p.n || slot < 0 || slot >= p.num_slots) continue;
        const int h = c / chunks, at = (c - h * chunks) * V;
        *(TV *)((T *)p.v_cache + (slot * p.Hk + h) * p.D + at) = *(const TV *)((const T *)p.v + t * p.v_token + h * p.v_head + at);
    }
}

template <typename T, int V, bool SIDE>
static void launch_rotary(RotaryParams &p, int pos_bytes, hipStream_t st) {
    const int units = p.R / 2 / V + (p.D - p.R) / (2 * V);
    int LG = 1;
    while (LG < units && LG < 64) LG *= 2;
    p.tokens_per_wg = 1;
    p.q_wgs = p.n;
    const int kv_wgs = p.n_store;
    const size_t lds = (size_t)p.tokens_per_wg * (p.R / 2) * sizeof(float2);
    if (pos_bytes == 8) rotary_kernel<T, V, SIDE, int64_t><<<p.q_wgs + kv_wgs, ROT_THREADS, lds, st>>>(p, LG);
    else rotary_kernel<T, V, SIDE, int32_t><<<p.q_wgs + kv_wgs, ROT_THREADS, lds, st>>>(p, LG);
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
    if (head_dim > 1024 || n_axes > 4 || (int64_t)n + n_store > 0x7fffffffLL) return ODSD_ERR_UNSUPPORTED;
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
#define ROT_GO(T)                                                                        \
    do {                                                                                 \
        if (wide) {                                                                      \
            if (interleaved) launch_rotary<T, 8, true>(p, position_bytes, st);           \
            else launch_rotary<T, 8, false>(p, position_bytes, st);                      \
        } else {                                                                         \
            if (interleaved) launch_rotary<T, 1, true>(p, position_bytes, st);           \
            else launch_rotary<T, 1, false>(p, position_bytes, st);                      \
        }                                                                                \
    } while (0)
    if (dtype == ODSD_DT_BF16) ROT_GO(__bf16);
    else ROT_GO(half_t);
#undef ROT_GO
    ODSD_CHECK_LAUNCH();
    return ODSD_OK;
}
