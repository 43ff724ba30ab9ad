// Store of a step's keys and values to the 8-bit paged cache, with one power-of-two scale per block and KV head for K and for V:
//   code = nearest e4m3 of x / s,   s >= amax / 448 over the rows of the block,   K [block][head][token][dim], V [block][head][dim][token]
// Powers of two, so that a row stored earlier keeps its value when a later one raises the scale: the codes are divided by a power of
// two, which only those lose bits by that fall below e4m3's normal numbers.
//
// A (block, head) is written by one workgroup, K and V each by one wavefront or workgroup, so scale and codes need no atomics and the same
// call gives the same bits.  The rows of a block may stand anywhere in slot_mapping: the workgroup of the first of them (the leader) looks through
// the list and notes which row goes to which token of the block (of two with one slot the last).  Rows that follow one of the same block,
// which is what a prompt's are, end at once.  In a long list the leader looks only into those chunks of 256 entries whose bitmap, made by a
// launch of its own, has the block's bit.
// Many rows of a block (a prompt) are read once and stay in registers between their maximum and their codes; V's codes are turned
// through LDS, four rows of four dimensions at a time, and leave as 16 bytes of a dimension.  A few rows write V's bytes one by one.
// Traffic bounds a prompt, 3 bytes a value: 32767 tokens of 8 heads of 128, 201 MB, 58 us (and 5 for the bitmaps), 3.5 TB/s.  The 16
// loads of a thread have no branch between them (rows that are not there load the leader's and count as zeros): with one each 76 us.
// Three workgroups to a CU; with four the registers do not suffice (87).
// A decode step is a chain of four trips to memory, 64 rows of 8 heads 5.1 us, and then a number of workgroups: where the leader's sixteenth neighbour
// behind is no row of its block, a workgroup looks through the list once for several heads, and its wavefronts take one K or V after the other, the
// next one's rows on their way meanwhile.  (A workgroup for each K and V / so: 128 rows 14.7 / 6.4, 512 44 / 18, 1024 of 4 heads 48 / 15.  Without
// asking ahead 1024 take 20, and 64 rows 5.0 instead of 5.3.)  Those are steps in which no scale rises.  Where one does, its wavefront goes through all codes
// of the block, a load after the other: 64 rows of 4 heads of 128, every scale rising, blocks of 256 20 us for 4.8, of 1024 73 for 5.1, of 16 (8 heads) 5.2 for 4.2.
#include "fp8.h"
#include <type_traits>

#define KV8_THREADS 256
#define KV8_CHUNK 256          // list entries with one bitmap
#define KV8_BITS 256           // bits of a bitmap
#define KV8_LONG 4096          // a longer list has bitmaps
#define KV8_WINDOW 256         // tokens of a block that are turned at a time
#define KV8_FEW 16             // rows of a block that are not turned
#define KV8_WGS 512            // workgroups that a list of few rows a block goes to (1024: 256 rows of 8 heads 13.1 us for 11.0)

struct KvFp8Params {
    const uint16_t *key, *value;
    int64_t key_token, key_head, value_token, value_head;      // strides in elements
    uint8_t *k_cache, *v_cache;
    float *scales;                                             // [n_blocks, KVH, 2]
    const int32_t *slots, *src;
    uint32_t *bitmaps;                                         // [KV8_BITS / 32][n_chunks], or null
    int N, n_src, KVH, bs, n_blocks, n_chunks;
    int per_wg;                                                // list entries of a workgroup
    int run_wgs;                                               // workgroups that have a head's K or V each; behind them those for few rows of a block,
    int few_groups, few_heads, few_entries;                    // which have a range of entries and some heads
};

__device__ __forceinline__ uint32_t kv_bit(const int block) { return ((uint32_t)block * 0x9e3779b1u) >> 24; }      // of KV8_BITS
// whether list entry i names a slot and a row that exist; its slot
__device__ __forceinline__ bool kv_entry(const KvFp8Params &p, const int i, int &slot) {
    slot = p.slots[i];
    const bool row = !p.src || (p.src[i] >= 0 && p.src[i] < p.n_src);
    return slot >= 0 && slot / p.bs < p.n_blocks && row;
}

// Whether a block whose first entry is e has a run of rows: its leader is looked for by the workgroups of a head's K or V, otherwise by
// those for few rows.
__device__ __forceinline__ bool kv_run(const KvFp8Params &p, const int e, const int block) {
    int slot;
    return p.run_wgs > 0 && e + KV8_FEW < p.N && kv_entry(p, e + KV8_FEW, slot) && slot / p.bs == block;
}

__global__ __launch_bounds__(KV8_CHUNK) void kv_bitmap_kernel(const KvFp8Params p) {
    __shared__ uint32_t bits[KV8_BITS / 32];
    const int i = blockIdx.x * KV8_CHUNK + threadIdx.x;
    if (threadIdx.x < KV8_BITS / 32) bits[threadIdx.x] = 0u;
    __syncthreads();
    int slot;
    if (i < p.N && kv_entry(p, i, slot)) {
        const uint32_t b = kv_bit(slot / p.bs);
        atomicOr(&bits[b >> 5], 1u << (b & 31));
    }
    __syncthreads();
    if (threadIdx.x < KV8_BITS / 32) p.bitmaps[(size_t)threadIdx.x * p.n_chunks + blockIdx.x] = bits[threadIdx.x];
}

// what the codes under one scale are multiplied by for the next; 0: the block held nothing.  A quotient that fp32 does not hold as a
// normal number leaves of every number zero, and so does the smallest one that it does hold: with a 0 a NaN would go too.
__device__ __forceinline__ float kv_ratio(const float old, const float scale) { return old > 0.0f ? fmaxf(old / scale, 1.17549435e-38f) : 0.0f; }
// n times 16 codes of a block times `ratio`, a power of two (0: the block held nothing, whatever its bytes are)
__device__ __forceinline__ void kv_rescale(uint8_t *codes, const int n, const float ratio, const int first, const int step) {
#pragma unroll 1
    for (int i = first; i < n; i += step) {
        uint4_t w = *(const uint4_t *)(codes + 16 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = ratio > 0.0f ? fp8_rescale4(w[j], ratio) : 0u;
        *(uint4_t *)(codes + 16 * i) = w;
    }
}

template <typename T> __device__ __forceinline__ float kv_value(uint16_t b);
template <> __device__ __forceinline__ float kv_value<__bf16>(uint16_t b) { return bf16_to_f32(b); }
template <> __device__ __forceinline__ float kv_value<half_t>(uint16_t b) { return (float)__builtin_bit_cast(half_t, b); }

template <bool VEC>
__device__ __forceinline__ uint4_t kv_load8(const uint16_t *p) {
    if constexpr (VEC) return __builtin_nontemporal_load((const uint4_t *)p);
    uint4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
    return w;
}
// Magnitudes are compared as the integers that they are without their sign; from KvBits<T>::INF on they are infinities and NaN.
template <typename T> struct KvBits { static constexpr uint32_t INF = std::is_same<T, half_t>::value ? 0x7c00u : 0x7f80u; };
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
// the larger of m and the magnitudes of eight values, in two halves; FINITE: infinities and NaN do not count
template <typename T, bool FINITE>
__device__ __forceinline__ uint32_t kv_top8(const uint4_t w, uint32_t m) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t a = w[i] & 0x7fff7fffu;
        if constexpr (FINITE) a = ((a & 0xffffu) < KvBits<T>::INF ? a & 0xffffu : 0u) | ((a >> 16) < KvBits<T>::INF ? a & 0xffff0000u : 0u);
        m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, a)));
    }
    return m;
}
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// Codes of eight values over the scale.  FINITE: all are numbers, and 448 scales at most: the conversion that divides by a power of two on its way does
// two at a time (nearest, ties to even: the same codes as below for every value of both types).
template <typename T, bool FINITE>
__device__ __forceinline__ u32x2 kv_codes8(const uint4_t w, const float scale) {
    if constexpr (FINITE) {
        typedef short s16x2 __attribute__((ext_vector_type(2)));
        u32x2 out;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            s16x2 c = {0, 0};
            if constexpr (std::is_same<T, half_t>::value) {
                c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, __builtin_bit_cast(half2_t, (uint32_t)w[2 * i]), scale, false);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, __builtin_bit_cast(half2_t, (uint32_t)w[2 * i + 1]), scale, true);
            } else {
                typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
                c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2, (uint32_t)w[2 * i]), scale, false);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2, (uint32_t)w[2 * i + 1]), scale, true);
            }
            out[i] = __builtin_bit_cast(uint32_t, c);
        }
        return out;
    }
    const float inv = 1.0f / scale;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = kv_value<T>((uint16_t)(w[i >> 1] >> (16 * (i & 1)))) * inv;
    return u32x2{fp8_pack4(x[0], x[1], x[2], x[3]), fp8_pack4(x[4], x[5], x[6], x[7])};
}
// codes of eight dimensions of a token to their place
template <int HD>
__device__ __forceinline__ void kv_put(uint8_t *codes, const int bs, const bool is_v, const int r, const int d, const u32x2 c) {
    if (!is_v) {
        *(u32x2 *)(codes + r * HD + d) = c;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) codes[(d + j) * bs + r] = (uint8_t)(c[j >> 2] >> (8 * (j & 3)));
    }
}
__device__ __forceinline__ uint32_t kv_wave_top(uint32_t m) {
    m = max(m & 0xffffu, m >> 16);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, ODSD_WAVE));
    return m;
}

// Blocks without a run of rows, in short lists: the leader's workgroup has several heads, and a wavefront takes one of their Ks and Vs after
// the other, with nothing to wait for between them.
template <typename T, int HD, bool VEC>
__device__ __forceinline__ void kv_store_few(const KvFp8Params &p, const int wg, int *row_of, int *first, int *count, uint16_t *present) {
    constexpr int NP = HD / 8, HELD = KV8_FEW * NP / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), bs = p.bs;
    const int range = wg / p.few_groups, h0 = (wg - range * p.few_groups) * p.few_heads, heads = min(p.few_heads, p.KVH - h0);
    const int begin = range * p.few_entries, stop = min(p.N, begin + p.few_entries);
    for (int e0 = begin; e0 < stop; e0 += 64) {
        const int le = e0 + lane;
        int slot_l = -1, before;
        bool may = false;
        if (le < stop && kv_entry(p, le, slot_l)) {
            const int block = slot_l / bs;
            may = (le == 0 || !kv_entry(p, le - 1, before) || before / bs != block) && !kv_run(p, le, block);
        }
        for (uint64_t leaders = __ballot(may); leaders; leaders &= leaders - 1) {
            const int l = __builtin_ctzll(leaders), e = e0 + l;
            const int block = __builtin_amdgcn_readlane(slot_l, l) / bs, base = block * bs;
            __syncthreads();                    // the arrays are free
            for (int i = tid; i < bs; i += KV8_THREADS) row_of[i] = -1;
            if (tid == 0) {
                *first = 0x7fffffff;
                *count = 0;
            }
            __syncthreads();
            for (int i = tid; i < p.N; i += KV8_THREADS) {
                const int slot = p.slots[i], at = slot - base;
                if (slot >= base && at < bs && (!p.src || (p.src[i] >= 0 && p.src[i] < p.n_src))) {
                    atomicMax(&row_of[at], i);
                    atomicMin(first, i);
                }
            }
            __syncthreads();
            if (*first != e) continue;          // (another entry's)
            for (int i = tid; i < bs; i += KV8_THREADS)
                if (row_of[i] >= 0) present[atomicAdd(count, 1)] = (uint16_t)i;
            __syncthreads();
            const int rows = *count, pieces = rows * NP;
            const bool anew = row_of[0] >= 0, held = rows <= KV8_FEW;
            auto source = [&](const int i) {        // the row of piece i
                const int from = row_of[present[i / NP]];
                return p.src ? p.src[from] : from;
            };
            int64_t rows_at[HELD];              // of this lane's pieces, where they can be held
#pragma unroll
            for (int u = 0; u < HELD; ++u) rows_at[u] = held && lane + 64 * u < pieces ? source(lane + 64 * u) : 0;
            // a K or V: what is asked for (`ask`) while the one before is worked on (`put`)
            struct Task {
                uint4_t hold[HELD];
                float was;
            };
            auto ask = [&](Task &k, const int t) {
                const int h = h0 + (t >> 1);
                const bool is_v = t & 1;
                const uint16_t *x = (is_v ? p.value : p.key) + (int64_t)h * (is_v ? p.value_head : p.key_head);
                const int64_t token = is_v ? p.value_token : p.key_token;
                k.was = p.scales[2 * ((int64_t)block * p.KVH + h) + (is_v ? 1 : 0)];
#pragma unroll
                for (int u = 0; u < HELD; ++u) {
                    k.hold[u] = uint4_t{0u, 0u, 0u, 0u};
                    if (held && lane + 64 * u < pieces) k.hold[u] = kv_load8<VEC>(x + rows_at[u] * token + 8 * ((lane + 64 * u) % NP));
                }
            };
            auto put = [&](const Task &k, const int t) {
                const int h = h0 + (t >> 1);
                const bool is_v = t & 1;
                const uint16_t *x = (is_v ? p.value : p.key) + (int64_t)h * (is_v ? p.value_head : p.key_head);
                const int64_t token = is_v ? p.value_token : p.key_token, bh = (int64_t)block * p.KVH + h;
                auto load = [&](const int i) { return kv_load8<VEC>(x + source(i) * token + 8 * (i % NP)); };
                auto top_of = [&](auto finite_c) {
                    constexpr bool FINITE = decltype(finite_c)::value;
                    uint32_t m = 0u;
                    if (held) {
#pragma unroll
                        for (int u = 0; u < HELD; ++u) m = kv_top8<T, FINITE>(k.hold[u], m);
                    } else {
#pragma unroll 1
                        for (int i = lane; i < pieces; i += 64) m = kv_top8<T, FINITE>(load(i), m);
                    }
                    return kv_wave_top(m);
                };
                uint32_t top = top_of(std::false_type{});
                const bool finite = top < KvBits<T>::INF;
                if (!finite) top = top_of(std::true_type{});
                const float old = anew ? 0.0f : k.was, scale = fmaxf(old, fp8_scale_of(kv_value<T>((uint16_t)top)));
                uint8_t *codes = (is_v ? p.v_cache : p.k_cache) + bh * bs * HD;
                if (!anew && old < scale) {
                    kv_rescale(codes, bs * HD / 16, kv_ratio(old, scale), lane, 64);
                    __threadfence_block();      // (the codes are there before the new ones come)
                }
                if (lane == 0) p.scales[2 * bh + (is_v ? 1 : 0)] = scale;
                auto store = [&](const int i, const uint4_t w) {
                    kv_put<HD>(codes, bs, is_v, present[i / NP], 8 * (i % NP), finite ? kv_codes8<T, true>(w, scale) : kv_codes8<T, false>(w, scale));
                };
                if (held) {
#pragma unroll
                    for (int u = 0; u < HELD; ++u)
                        if (lane + 64 * u < pieces) store(lane + 64 * u, k.hold[u]);
                } else {
#pragma unroll 1
                    for (int i = lane; i < pieces; i += 64) store(i, load(i));
                }
            };
            constexpr int W = KV8_THREADS / 64;
            Task k[2];
            if (wave < 2 * heads) ask(k[0], wave);
            for (int t = wave; t < 2 * heads; t += 2 * W) {
                if (t + W < 2 * heads) ask(k[1], t + W);
                put(k[0], t);
                if (t + 2 * W < 2 * heads) ask(k[0], t + 2 * W);
                if (t + W < 2 * heads) put(k[1], t + W);
            }
        }
    }
}

// LONG: the list has bitmaps, and no workgroups for few rows
template <typename T, int HD, bool VEC, bool LONG>
__global__ __launch_bounds__(KV8_THREADS, 3) void kv_store_fp8_kernel(const KvFp8Params p) {
    constexpr int NP = HD / 8;                           // pieces of 8 values of a row
    constexpr int HELD = KV8_WINDOW * NP / KV8_THREADS;          // pieces of a window per thread
    constexpr int RPT = KV8_THREADS / NP;                // rows that a workgroup's pieces are at a time
    constexpr int ROW = HD + 8;                          // bytes of a row in LDS: 16 rows on, other banks
    __shared__ int row_of[FP8_MAX_BLOCK];      // list entry that goes to a token of the block, -1: none
    __shared__ int first, count;
    __shared__ uint32_t red[2][KV8_THREADS / 64];
    __shared__ __attribute__((aligned(16))) uint8_t turn[KV8_WINDOW * ROW];
    uint16_t *present = (uint16_t *)turn;      // tokens that get a row, in no order; where V is turned only until then
    const int tid = threadIdx.x, lane = tid & 63, row0 = tid / NP, piece = tid % NP;
    if constexpr (!LONG) {
        if ((int)blockIdx.x >= p.run_wgs) return kv_store_few<T, HD, VEC>(p, (int)blockIdx.x - p.run_wgs, row_of, &first, &count, present);
    }
    const int which = blockIdx.x / 2, h = which % p.KVH;
    const bool is_v = blockIdx.x & 1;
    const uint16_t *x = (is_v ? p.value : p.key) + (int64_t)h * (is_v ? p.value_head : p.key_head);
    const int64_t token = is_v ? p.value_token : p.key_token;
    const int bs = p.bs;
    const int begin = which / p.KVH * p.per_wg;
    const int stop = min(p.N, begin + p.per_wg);
    for (int e0 = begin; e0 < stop; e0 += 64) {
    // entries that may be leaders: those whose neighbour in front is of another block
    uint64_t leaders;
    int slot_l = -1;
    {
        const int e = e0 + lane;
        bool may = false;
        if (e < stop && kv_entry(p, e, slot_l)) {
            int before;
            const int block = slot_l / bs;
            may = (e == 0 || !kv_entry(p, e - 1, before) || before / bs != block) && (LONG || kv_run(p, e, block));
        }
        leaders = __ballot(may);
    }
    for (; leaders; leaders &= leaders - 1) {
        const int l = __builtin_ctzll(leaders), e = e0 + l;
        const int block = __builtin_amdgcn_readlane(slot_l, l) / bs, base = block * bs;
        const int64_t bh = (int64_t)block * p.KVH + h;
        float *scale_at = p.scales + 2 * bh + (is_v ? 1 : 0);
        const float was = *scale_at;            // (nobody else writes it, unless this workgroup turns out not to be the leader)
        // ---- the block's rows ------------------------------------------------------------------------
        __syncthreads();                        // the arrays are free
        for (int i = tid; i < (bs + KV8_WINDOW - 1) / KV8_WINDOW * KV8_WINDOW; i += KV8_THREADS) row_of[i] = -1;
        if (tid == 0) {
            first = 0x7fffffff;
            count = 0;
        }
        __syncthreads();
        auto look = [&](const int i) {          // (block is a block of the cache, so its slots need no check)
            const int slot = p.slots[i], at = slot - base;
            if (slot >= base && at < bs && (!p.src || (p.src[i] >= 0 && p.src[i] < p.n_src))) {
                atomicMax(&row_of[at], i);
                atomicMin(&first, i);
            }
        };
        if constexpr (LONG) {
            const uint32_t bit = kv_bit(block);
            const uint32_t *maps = p.bitmaps + (size_t)(bit >> 5) * p.n_chunks;
            for (int c0 = 0; c0 < p.n_chunks; c0 += 64) {
                const bool has = c0 + lane < p.n_chunks && (maps[c0 + lane] >> (bit & 31)) & 1;
                for (uint64_t todo = __ballot(has); todo; todo &= todo - 1) {
                    const int i = (c0 + __builtin_ctzll(todo)) * KV8_CHUNK + tid;
                    if (i < p.N) look(i);
                }
            }
        } else {
            for (int i = tid; i < p.N; i += KV8_THREADS) look(i);
        }
        __syncthreads();
        if (first != e) continue;               // (another workgroup's)
        for (int i = tid; i < bs; i += KV8_THREADS)
            if (row_of[i] >= 0) present[atomicAdd(&count, 1)] = (uint16_t)i;
        __syncthreads();
        const int rows = count;
        const bool turned = rows > KV8_FEW, held = turned && bs <= KV8_WINDOW;
        auto source = [&](const int i) { return x + (int64_t)(p.src ? p.src[i] : i) * token; };
        // the pieces of a window: piece `piece` of rows row0 + RPT u; bit u of `have`: there is one (the others are zeros)
        uint4_t hold[HELD];
        uint32_t have = 0u;
        auto load_window = [&](const int w0) {
            const int *rows_at = row_of + w0 + row0;
            int from[HELD];
            have = 0u;
#pragma unroll
            for (int u = 0; u < HELD; ++u) {
                from[u] = rows_at[RPT * u];
                have |= from[u] >= 0 ? 1u << u : 0u;
                from[u] = from[u] >= 0 ? from[u] : e;
            }
            if (p.src) {
#pragma unroll
                for (int u = 0; u < HELD; ++u) from[u] = p.src[from[u]];
            }
            const uint16_t *at = x + 8 * piece;
#pragma unroll
            for (int u = 0; u < HELD; ++u) hold[u] = kv_load8<VEC>(at + from[u] * token);
#pragma unroll
            for (int u = 0; u < HELD; ++u)
                if (!(have >> u & 1)) hold[u] = uint4_t{0u, 0u, 0u, 0u};
        };
        // ---- the scale -------------------------------------------------------------------------------
        auto top_of = [&](auto finite_c, uint32_t *part) {       // the largest magnitude of the workgroup's rows
            constexpr bool FINITE = decltype(finite_c)::value;
            uint32_t m = 0u;
            if (held) {
#pragma unroll
                for (int u = 0; u < HELD; ++u) m = kv_top8<T, FINITE>(hold[u], m);
            } else {
#pragma unroll 1
                for (int i = tid; i < rows * NP; i += KV8_THREADS) m = kv_top8<T, FINITE>(kv_load8<VEC>(source(row_of[present[i / NP]]) + 8 * (i % NP)), m);
            }
            m = kv_wave_top(m);
            if (lane == 0) part[tid >> 6] = m;
            __syncthreads();
            return max(max(part[0], part[1]), max(part[2], part[3]));
        };
        if (held) load_window(0);
        uint32_t top = top_of(std::false_type{}, red[0]);
        const bool finite = top < KvBits<T>::INF;
        if (!finite) top = top_of(std::true_type{}, red[1]);
        const float amax = kv_value<T>((uint16_t)top);
        const bool anew = row_of[0] >= 0;       // the block starts: what it held before is given up
        const float old = anew ? 0.0f : was;
        const float scale = fmaxf(old, fp8_scale_of(amax));
        uint8_t *codes = (is_v ? p.v_cache : p.k_cache) + bh * bs * HD;
        if (!anew && old < scale) {
            kv_rescale(codes, bs * HD / 16, kv_ratio(old, scale), tid, KV8_THREADS);
        }
        __syncthreads();                        // (the codes are there before the new ones come)
        if (tid == 0) *scale_at = scale;
        // ---- the codes -------------------------------------------------------------------------------
        if (!turned) {
#pragma unroll 1
            for (int i = tid; i < rows * NP; i += KV8_THREADS) {
                const int r = present[i / NP], d = 8 * (i % NP);
                const uint4_t w = kv_load8<VEC>(source(row_of[r]) + d);
                kv_put<HD>(codes, bs, is_v, r, d, finite ? kv_codes8<T, true>(w, scale) : kv_codes8<T, false>(w, scale));
            }
            continue;
        }
        for (int w0 = 0; w0 < bs; w0 += KV8_WINDOW) {
            if (!held) load_window(w0);
            if (is_v) __syncthreads();          // the last window has left LDS
            auto coded = [&](auto finite_c) {
#pragma unroll
                for (int u = 0; u < HELD; ++u) {
                    const u32x2 c = kv_codes8<T, decltype(finite_c)::value>(hold[u], scale);
                    hold[u].x = c.x;
                    hold[u].y = c.y;
                    if (!decltype(finite_c)::value) __builtin_amdgcn_sched_barrier(0);      // (one at a time: registers)
                }
            };
            if (finite) coded(std::true_type{});
            else coded(std::false_type{});
#pragma unroll
            for (int u = 0; u < HELD; ++u) {
                const u32x2 c = {hold[u].x, hold[u].y};
                if (is_v) *(u32x2 *)(turn + row0 * ROW + 8 * piece + RPT * ROW * u) = c;
                else if (have >> u & 1) *(u32x2 *)(codes + (w0 + row0) * HD + 8 * piece + RPT * HD * u) = c;
            }
            if (!is_v) continue;
            __syncthreads();
            // 16 tokens of 4 dimensions a turn
            const int here = min(KV8_WINDOW, bs - w0);
#pragma unroll 1
            for (int i = tid; i < here / 16 * (HD / 4); i += KV8_THREADS) {
                const int r0 = 16 * (i / (HD / 4)), d = 4 * (i % (HD / 4));
                uint32_t there = 0u;
#pragma unroll
                for (int r = 0; r < 16; ++r) there |= row_of[w0 + r0 + r] >= 0 ? 1u << r : 0u;
                if (!there) continue;
                uint4_t out[4];                 // [dimension], four tokens a word
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t w[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) w[r] = *(const uint32_t *)(turn + (r0 + 4 * q + r) * ROW + d);
                    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
                    const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), e4 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
                    out[0][q] = __builtin_amdgcn_perm(b, a, 0x05040100u);
                    out[1][q] = __builtin_amdgcn_perm(b, a, 0x07060302u);
                    out[2][q] = __builtin_amdgcn_perm(e4, c, 0x05040100u);
                    out[3][q] = __builtin_amdgcn_perm(e4, c, 0x07060302u);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint8_t *to = codes + (d + j) * bs + w0 + r0;
                    if (there == 0xffffu) {
                        *(uint4_t *)to = out[j];
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (there >> r & 1) to[r] = (uint8_t)(out[j][r >> 2] >> (8 * (r & 3)));
                    }
                }
            }
        }
    }
    }
}

extern "C" size_t odsd_kv_store_fp8_workspace_bytes(int32_t N) {
    if (N < 0 || N > (1 << 28)) return 0;
    return N <= KV8_LONG ? 256 : odsd_round_up((size_t)((N + KV8_CHUNK - 1) / KV8_CHUNK) * (KV8_BITS / 8), 256);
}

extern "C" int odsd_kv_store_fp8(const void *key, int64_t key_token_stride, int64_t key_head_stride, const void *value,
                                 int64_t value_token_stride, int64_t value_head_stride, void *k_cache, void *v_cache,
                                 float *scales, const int32_t *slot_mapping, const int32_t *src_index, int32_t N,
                                 int32_t n_src, int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int32_t n_blocks,
                                 int32_t dtype, void *workspace, size_t workspace_bytes, void *stream) {
    if (N < 0 || n_src < 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || block_size % 16 || n_blocks < 0 ||
        (!src_index && N != n_src))
        return ODSD_ERR_SHAPE;
    if (dtype != ODSD_DT_BF16 && dtype != ODSD_DT_F16) return ODSD_ERR_DTYPE;
    // (slots are 31 bits, and so is a block's number times the heads)
    if ((head_dim != 64 && head_dim != 128) || block_size > FP8_MAX_BLOCK || (int64_t)n_blocks * block_size > 0x7fffffffLL ||
        (int64_t)n_blocks * num_kv_heads > 0x7fffffffLL || num_kv_heads > 65535 || N > (1 << 28))
        return ODSD_ERR_UNSUPPORTED;
    if (N == 0 || n_blocks == 0) return ODSD_OK;
    if (!key || !value || !k_cache || !v_cache || !scales || !slot_mapping) return ODSD_ERR_NULL;
    if (!odsd_aligned16(k_cache) || !odsd_aligned16(v_cache) || ((uintptr_t)scales & 7u) || (((uintptr_t)key | (uintptr_t)value) & 1u))
        return ODSD_ERR_ALIGN;
    KvFp8Params p{};
    hipStream_t st = (hipStream_t)stream;
    p.key = (const uint16_t *)key; p.value = (const uint16_t *)value;
    p.key_token = key_token_stride; p.key_head = key_head_stride; p.value_token = value_token_stride; p.value_head = value_head_stride;
    p.k_cache = (uint8_t *)k_cache; p.v_cache = (uint8_t *)v_cache; p.scales = scales;
    p.slots = slot_mapping; p.src = src_index;
    p.N = N; p.n_src = n_src; p.KVH = num_kv_heads; p.bs = block_size; p.n_blocks = n_blocks;
    // Enough workgroups for the chip; no more entries each than a block of a prompt takes, so that every one has about one leader (a workgroup
    // that has none holds its place for two trips to memory: with 64 entries each and blocks of 256 three of four, 94 us where this took 76).
    p.per_wg = (int)max((int64_t)1, min((int64_t)min(256, block_size), (int64_t)N * num_kv_heads / 1024));
    int64_t few = 0;
    if (N <= KV8_LONG) {
        p.per_wg = 64;                                        // (leaders of runs stand further apart than others)
        const int64_t heads = ((int64_t)N * num_kv_heads + KV8_WGS - 1) / KV8_WGS;
        p.few_heads = (int)min((int64_t)num_kv_heads, max((int64_t)2, heads));
        p.few_groups = (num_kv_heads + p.few_heads - 1) / p.few_heads;
        p.few_entries = (int)max((int64_t)1, (int64_t)N * p.few_groups / KV8_WGS);
        few = ((int64_t)N + p.few_entries - 1) / p.few_entries * p.few_groups;
    }
    // (a block of few tokens has no run)
    const int64_t wgs = few && block_size <= KV8_FEW ? 0 : ((int64_t)N + p.per_wg - 1) / p.per_wg * num_kv_heads * 2;
    if (wgs + few >= (1LL << 24)) return ODSD_ERR_UNSUPPORTED;
    p.run_wgs = (int)wgs;
    const unsigned grid = (unsigned)(wgs + few);
    if (N > KV8_LONG) {
        if (!workspace) return ODSD_ERR_NULL;
        if ((uintptr_t)workspace & 3u) return ODSD_ERR_ALIGN;
        if (workspace_bytes < odsd_kv_store_fp8_workspace_bytes(N)) return ODSD_ERR_WORKSPACE;
        p.bitmaps = (uint32_t *)workspace;
        p.n_chunks = (N + KV8_CHUNK - 1) / KV8_CHUNK;
        kv_bitmap_kernel<<<(unsigned)p.n_chunks, KV8_CHUNK, 0, st>>>(p);
    }
    const bool vec = !(((uintptr_t)key | (uintptr_t)value) & 15u) &&
                     !((key_token_stride | key_head_stride | value_token_stride | value_head_stride) & 7);
#define KV8_GO_LONG(T, HDV, VECV)                                                                        \
    do {                                                                                                 \
        if (p.bitmaps) kv_store_fp8_kernel<T, HDV, VECV, true><<<grid, KV8_THREADS, 0, st>>>(p);         \
        else kv_store_fp8_kernel<T, HDV, VECV, false><<<grid, KV8_THREADS, 0, st>>>(p);                  \
    } while (0)
#define KV8_GO(T)                                                                                        \
    do {                                                                                                 \
        if (head_dim == 128) {                                                                           \
            if (vec) KV8_GO_LONG(T, 128, true);                                                          \
            else KV8_GO_LONG(T, 128, false);                                                             \
        } else if (vec) KV8_GO_LONG(T, 64, true);                                                        \
        else KV8_GO_LONG(T, 64, false);                                                                  \
    } while (0)
    if (dtype == ODSD_DT_BF16) KV8_GO(__bf16);
    else KV8_GO(half_t);
#undef KV8_GO
#undef KV8_GO_LONG
    ODSD_CHECK_LAUNCH();
    return ODSD_OK;
}
