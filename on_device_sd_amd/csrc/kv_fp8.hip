// Store of a step's keys and values to the 8-bit paged cache, with one power-of-two scale per block and KV head for K and for V:
//   code = nearest e4m3 of x / s,   s >= amax / 448 over the rows of the block,   K [block][head][token][dim], V [block][head][dim][token]
// Powers of two, so that a row stored earlier keeps its value when a later one raises the scale: the codes are divided by a power of
// two, which only those lose bits by that fall below e4m3's normal numbers.
//
// A (block, head) is written by one workgroup, K and V by one each, so scale and codes need no atomics and the same call gives the same
// bits.  The rows of a block may stand anywhere in slot_mapping: the workgroup of the first of them (the leader) looks through the list
// and notes which row goes to which token of the block (of two with one slot the last).  Rows that follow one of the same block, which
// is what a prompt's are, end at once.
#include "fp8.h"

struct KvFp8Params {
    const uint16_t *key, *value;
    int64_t key_token, key_head, value_token, value_head;      // strides in elements
    uint8_t *k_cache, *v_cache;
    float *scales;                                             // [n_blocks, KVH, 2]
    const int32_t *slots, *src;
    int N, n_src, KVH, HD, bs, n_blocks;
    int per_wg;                                                // list entries of a workgroup
};

template <typename T> __device__ __forceinline__ float kv_value(uint16_t b);
template <> __device__ __forceinline__ float kv_value<__bf16>(uint16_t b) { return bf16_to_f32(b); }
template <> __device__ __forceinline__ float kv_value<half_t>(uint16_t b) { return (float)__builtin_bit_cast(half_t, b); }

template <typename T, bool VEC>
__device__ __forceinline__ void kv_load8(const uint16_t *p, float (&x)[8]) {
    if constexpr (VEC) {
        const uint4_t w = *(const uint4_t *)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = kv_value<T>((uint16_t)(w[i] & 0xffffu));
            x[2 * i + 1] = kv_value<T>((uint16_t)(w[i] >> 16));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = kv_value<T>(p[i]);
    }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void kv_store_fp8_kernel(const KvFp8Params p) {
    __shared__ int row_of[FP8_MAX_BLOCK];      // list entry that goes to a token of the block, -1: none
    __shared__ int present[FP8_MAX_BLOCK];     // tokens that get one
    __shared__ int first, count;
    __shared__ float red[4];
    const int tid = threadIdx.x, h = blockIdx.y;
    const bool is_v = blockIdx.z != 0;
    const uint16_t *x = is_v ? p.value : p.key;
    const int64_t token = is_v ? p.value_token : p.key_token, head = is_v ? p.value_head : p.key_head;
    const int bs = p.bs, HD = p.HD, NP = HD / 8;
    const int begin = blockIdx.x * p.per_wg, end = min(p.N, begin + p.per_wg);
    for (int e = begin; e < end; ++e) {
        const int slot = p.slots[e];
        if (slot < 0) continue;
        const int block = slot / bs, base = block * bs;
        if (block >= p.n_blocks) continue;
        if (e > 0) {
            const int before = p.slots[e - 1];
            if (before >= base && before - base < bs && (!p.src || (p.src[e - 1] >= 0 && p.src[e - 1] < p.n_src))) continue;
        }
        // ---- the block's rows ------------------------------------------------------------------------
        __syncthreads();                        // the arrays are free
        for (int i = tid; i < bs; i += 256) row_of[i] = -1;
        if (tid == 0) {
            first = 0x7fffffff;
            count = 0;
        }
        __syncthreads();
        for (int i = tid; i < p.N; i += 256) {
            const int at = p.slots[i] - base;
            if (p.slots[i] >= base && at < bs && (!p.src || (p.src[i] >= 0 && p.src[i] < p.n_src))) {
                atomicMax(&row_of[at], i);
                atomicMin(&first, i);
            }
        }
        __syncthreads();
        if (first != e) continue;               // (another workgroup's, or a row that does not exist)
        for (int i = tid; i < bs; i += 256)
            if (row_of[i] >= 0) present[atomicAdd(&count, 1)] = i;
        __syncthreads();
        const int rows = count;
        auto source = [&](const int r) {        // the row that goes to token r
            const int i = row_of[r];
            return x + (int64_t)(p.src ? p.src[i] : i) * token + (int64_t)h * head;
        };
        // ---- the scale -------------------------------------------------------------------------------
        float amax = 0.0f;
        for (int i = tid; i < rows * NP; i += 256) {
            float v[8];
            kv_load8<T, VEC>(source(present[i / NP]) + 8 * (i % NP), v);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float a = fabsf(v[j]);
                amax = a <= 3.4028234663852886e38f ? fmaxf(amax, a) : amax;      // infinities and NaN do not count
            }
        }
        amax = wave_max(amax);
        if ((tid & 63) == 0) red[tid >> 6] = amax;
        __syncthreads();
        amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const int64_t bh = (int64_t)block * p.KVH + h;
        float *scale_at = p.scales + 2 * bh + (is_v ? 1 : 0);
        const bool anew = row_of[0] >= 0;       // the block starts: what it held before is given up
        const float old = anew ? 0.0f : *scale_at;
        const float scale = fmaxf(old, fp8_scale_of(amax)), inv = 1.0f / scale;
        uint8_t *codes = (is_v ? p.v_cache : p.k_cache) + bh * bs * HD;
        if (!anew && old < scale) {
            const float ratio = old * inv;      // a power of two (0: the block held nothing, whatever its bytes are)
            for (int i = tid; i < bs * HD / 16; i += 256) {
                uint4_t w = *(const uint4_t *)(codes + 16 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = ratio > 0.0f ? fp8_rescale4(w[j], ratio) : 0u;
                *(uint4_t *)(codes + 16 * i) = w;
            }
        }
        __syncthreads();                        // (every thread has read the scale; the codes are there before the new ones come)
        if (tid == 0) *scale_at = scale;
        // ---- the codes -------------------------------------------------------------------------------
        for (int i = tid; i < rows * NP; i += 256) {
            const int r = present[i / NP], d = 8 * (i % NP);
            float v[8];
            kv_load8<T, VEC>(source(r) + d, v);
            const uint32_t lo = fp8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
            const uint32_t hi = fp8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
            if (!is_v) {
                typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
                *(u32x2 *)(codes + r * HD + d) = u32x2{lo, hi};
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) codes[(d + j) * bs + r] = (uint8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
            }
        }
    }
}

extern "C" int odsd_kv_store_fp8(const void *key, int64_t key_token_stride, int64_t key_head_stride, const void *value,
                                 int64_t value_token_stride, int64_t value_head_stride, void *k_cache, void *v_cache,
                                 float *scales, const int32_t *slot_mapping, const int32_t *src_index, int32_t N,
                                 int32_t n_src, int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int32_t n_blocks,
                                 int32_t dtype, void *stream) {
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
    p.key = (const uint16_t *)key; p.value = (const uint16_t *)value;
    p.key_token = key_token_stride; p.key_head = key_head_stride; p.value_token = value_token_stride; p.value_head = value_head_stride;
    p.k_cache = (uint8_t *)k_cache; p.v_cache = (uint8_t *)v_cache; p.scales = scales;
    p.slots = slot_mapping; p.src = src_index;
    p.N = N; p.n_src = n_src; p.KVH = num_kv_heads; p.HD = head_dim; p.bs = block_size; p.n_blocks = n_blocks;
    // enough workgroups for the chip, no more than 64 entries each
    p.per_wg = (int)max((int64_t)1, min((int64_t)64, (int64_t)N * num_kv_heads / 1024));
    const dim3 grid((unsigned)((N + p.per_wg - 1) / p.per_wg), (unsigned)num_kv_heads, 2);
    const bool vec = !(((uintptr_t)key | (uintptr_t)value) & 15u) &&
                     !((key_token_stride | key_head_stride | value_token_stride | value_head_stride) & 7);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ODSD_DT_BF16) {
        if (vec) kv_store_fp8_kernel<__bf16, true><<<grid, 256, 0, st>>>(p);
        else kv_store_fp8_kernel<__bf16, false><<<grid, 256, 0, st>>>(p);
    } else {
        if (vec) kv_store_fp8_kernel<half_t, true><<<grid, 256, 0, st>>>(p);
        else kv_store_fp8_kernel<half_t, false><<<grid, 256, 0, st>>>(p);
    }
    ODSD_CHECK_LAUNCH();
    return ODSD_OK;
}
