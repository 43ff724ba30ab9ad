// Logits on their way to the verification: penalties for repeated tokens, biases and grammar masks, one pass over the rows.
//   x = logit;   seen (prompt, output or a draft before the row): x = x > 0 ? x / r : x r
//   x = x - (f n + p [n > 0])         n: how often among the output and the drafts before the row
//   x = x + bias;   a mask bit that is clear: x = -inf;   rounded once, to the logits' type
//
// A workgroup has one sequence and a slice of the vocabulary, and goes over it twice.  First all rows are copied, 16 bytes a thread, with -inf where
// the mask forbids: nearly every logit is done then.  (In place and without a mask there is nothing to copy.)  Meanwhile it has
// looked through the sequence's tokens and counted those of its slice in LDS; the tokens that have occurred, are drafted or have a
// bias are listed, and each thread then computes its tokens of the list in all rows, adding to the count the drafts that stand before.  No table of
// counts lives between steps, so drafts that are not kept leave nothing to undo.  The logits are read and written once: that traffic is
// the bound; the tokens (read again by every slice, from L2) and the listed logits (from L2 or the memory-side cache) are little next to it.
#include "common.h"
#include <type_traits>

#define ADJ_SEEN 0x80000000u     // has occurred
#define ADJ_DRAFT 0x40000000u    // is drafted, and may occur in later rows
#define ADJ_BIAS 0x20000000u     // has a bias; the other bits count

struct AdjParams {
    const void *logits;
    void *out;
    int64_t ld, ldo;
    const int32_t *q_lens;                     // [n_seqs] or null: one row each
    const void *tokens;                        // [n_seqs, ..] int32 or int64 (token_bytes), or null
    int64_t token_stride;
    const int32_t *token_lens, *prompt_lens;
    const void *drafts;                        // [n_drafts], or null
    const float *repetition, *frequency, *presence;
    float repetition_all, frequency_all, presence_all;
    const int32_t *bias_tokens;                // [n_seqs, n_bias], or null
    const float *bias_values;
    const int32_t *mask;                       // rows of mask_stride words
    int64_t mask_stride;
    const int32_t *mask_rows;                  // [n_rows] or null
    int n_seqs, n_rows, n_drafts, vocab, token_bytes, max_tokens, n_bias, n_mask, slice, slices;
    int dense, sparse;                         // rows have to be copied; some tokens may differ
};

// 16 bytes at any element
typedef uint32_t raw_t __attribute__((ext_vector_type(4), aligned(2)));

template <typename T> struct AdjIO;
template <> struct AdjIO<float> {
    __device__ static __forceinline__ float get(float v) { return v; }
    __device__ static __forceinline__ float put(float v) { return v; }
};
template <> struct AdjIO<__bf16> {
    __device__ static __forceinline__ float get(__bf16 v) { return (float)v; }
    __device__ static __forceinline__ __bf16 put(float v) { return (__bf16)v; }
};
template <> struct AdjIO<half_t> {
    __device__ static __forceinline__ float get(half_t v) { return (float)v; }
    __device__ static __forceinline__ half_t put(float v) { return (half_t)v; }
};

__device__ __forceinline__ int64_t adj_token(const void *p, const int bytes, const int64_t i) {
    return bytes == 8 ? ((const int64_t *)p)[i] : (int64_t)((const int32_t *)p)[i];
}

template <typename T>
__global__ __launch_bounds__(256) void adjust_logits_kernel(const AdjParams p) {
    extern __shared__ uint32_t lds[];          // counts [slice], the list [slice] in 16 bits
    __shared__ int sums[8], listed;
    uint32_t *counts = lds;
    uint16_t *list = (uint16_t *)(lds + p.slice);
    const int tid = threadIdx.x;
    const int s = blockIdx.x / p.slices, v0 = (blockIdx.x - s * p.slices) * p.slice;
    const int here = min(p.slice, p.vocab - v0);
    if (p.sparse) {
        if (tid == 0) listed = 0;
        for (int i = tid; i < here; i += 256) counts[i] = 0u;
    }
    // the sequence's first row and first draft
    int row = s, draft = 0, rows = 1;
    if (p.q_lens) {
        int r = 0, d = 0;
        for (int i = tid; i < s; i += 256) {
            const int n = max(p.q_lens[i], 0);
            r += n;
            d += max(n - 1, 0);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            r += __shfl_xor(r, o, ODSD_WAVE);
            d += __shfl_xor(d, o, ODSD_WAVE);
        }
        if ((tid & 63) == 0) {
            sums[tid >> 6] = r;
            sums[4 + (tid >> 6)] = d;
        }
        __syncthreads();
        row = __builtin_amdgcn_readfirstlane(sums[0] + sums[1] + sums[2] + sums[3]);
        draft = __builtin_amdgcn_readfirstlane(sums[4] + sums[5] + sums[6] + sums[7]);
        rows = max(p.q_lens[s], 0);
    } else if (p.sparse) {
        __syncthreads();
    }
    rows = min(rows, p.n_rows - row);
    if (rows <= 0) return;
    const int drafts = p.drafts ? max(min(rows - 1, p.n_drafts - draft), 0) : 0;
    if (p.sparse) {
        if (p.tokens) {
            const int len = min(max(p.token_lens ? p.token_lens[s] : p.max_tokens, 0), p.max_tokens);
            const int prompt = p.prompt_lens ? p.prompt_lens[s] : 0;
            for (int i = tid; i < len; i += 256) {
                const int64_t t = adj_token(p.tokens, p.token_bytes, s * p.token_stride + i) - v0;
                if (t >= 0 && t < here) {
                    if (i >= prompt) atomicAdd(&counts[t], 1u);
                    atomicOr(&counts[t], ADJ_SEEN);
                }
            }
        }
        for (int i = tid; i < drafts; i += 256) {
            const int64_t t = adj_token(p.drafts, 8, draft + i) - v0;
            if (t >= 0 && t < here) atomicOr(&counts[t], ADJ_DRAFT);
        }
        for (int i = tid; i < p.n_bias; i += 256) {
            const int t = p.bias_tokens[(int64_t)s * p.n_bias + i];
            if (t >= v0 && t - v0 < here) atomicOr(&counts[t - v0], ADJ_BIAS);
        }
    }
    // ---- all rows, as they are or forbidden ------------------------------------------------------------
    const T *in = (const T *)p.logits + (int64_t)row * p.ld + v0;
    T *to = (T *)p.out + (int64_t)row * p.ldo + v0;
    auto mask_of = [&](const int j) -> const int32_t * {
        const int m = p.mask ? p.mask_rows ? p.mask_rows[row + j] : row + j : -1;
        return m >= 0 && m < p.n_mask ? p.mask + m * p.mask_stride : nullptr;
    };
    if (p.dense) {
        constexpr int TPG = 16 / (int)sizeof(T);           // tokens of a group: 16 bytes, rows at any element
        const int groups = here / TPG;
        for (int j = 0; j < rows; ++j) {
            const T *x = in + j * p.ld;
            T *y = to + j * p.ldo;
            const int32_t *mask = mask_of(j);
            for (int g0 = tid; g0 < groups; g0 += 4 * 256) {
                uint4_t raw[4];
                uint32_t bits[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int g = min(g0 + 256 * u, groups - 1);
                    raw[u] = *(const raw_t *)(x + g * TPG);
                    bits[u] = mask ? (uint32_t)mask[(v0 + g * TPG) >> 5] >> ((v0 + g * TPG) & 31) : ~0u;
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int g = g0 + 256 * u;
                    if (mask) {
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            if constexpr (sizeof(T) == 4) {
                                raw[u][w] = (bits[u] >> w) & 1 ? raw[u][w] : 0xff800000u;
                            } else {
                                constexpr uint32_t INF = std::is_same<T, half_t>::value ? 0xfc00u : 0xff80u;
                                const uint32_t lo = (bits[u] >> (2 * w)) & 1 ? raw[u][w] & 0xffffu : INF;
                                const uint32_t hi = (bits[u] >> (2 * w + 1)) & 1 ? raw[u][w] & 0xffff0000u : INF << 16;
                                raw[u][w] = lo | hi;
                            }
                        }
                    }
                    if (g < groups) *(raw_t *)(y + g * TPG) = raw[u];
                }
            }
            const int i = groups * TPG + tid;              // what is left of a row that is no whole number of groups
            if (i < here) y[i] = !mask || ((mask[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1) ? x[i] : AdjIO<T>::put(-INFINITY);
        }
    }
    if (!p.sparse) return;
    __syncthreads();                           // counts and biases are there, and so are the copies of this workgroup
    for (int i = tid; i < here; i += 256)
        if (counts[i]) list[atomicAdd(&listed, 1)] = (uint16_t)i;
    __syncthreads();
    const float r = p.repetition ? p.repetition[s] : p.repetition_all;
    const float f = p.frequency ? p.frequency[s] : p.frequency_all;
    const float pr = p.presence ? p.presence[s] : p.presence_all;
    for (int k = tid; k < listed; k += 256) {
        const int i = (int)list[k];
        const uint32_t n = counts[i];
        const bool drafted = n & ADJ_DRAFT, biased = n & ADJ_BIAS;
        bool seen = n & ADJ_SEEN;
        uint32_t times = n & (ADJ_BIAS - 1);
        float add = 0.0f;
        if (biased) {                          // the last of the entries that name the token
            int b = p.n_bias - 1;
            while (p.bias_tokens[(int64_t)s * p.n_bias + b] != v0 + i) --b;
            add = p.bias_values[(int64_t)s * p.n_bias + b];
        }
        for (int j = 0; j < rows; ++j) {
            if (drafted && j > 0 && j - 1 < drafts && adj_token(p.drafts, 8, draft + j - 1) == v0 + i) {
                ++times;
                seen = true;
            }
            const int32_t *mask = mask_of(j);
            float x = AdjIO<T>::get(in[j * p.ld + i]);
            if (seen) x = x > 0.0f ? x / r : x * r;
            if (times) x = x - (f * (float)times + pr);
            if (biased) x += add;
            if (mask && !((mask[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1)) x = -INFINITY;
            to[j * p.ldo + i] = AdjIO<T>::put(x);
        }
    }
}

extern "C" int odsd_adjust_logits(const void *logits, int64_t logits_stride, void *out, int64_t out_stride, int32_t dtype,
                                  int32_t n_rows, int32_t vocab, const int32_t *query_lens, int32_t n_seqs,
                                  const void *tokens, int32_t token_bytes, int64_t token_stride, int32_t max_tokens,
                                  const int32_t *token_lens, const int32_t *prompt_lens, const int64_t *draft_tokens,
                                  int32_t n_drafts, const float *repetition, float repetition_all, const float *frequency,
                                  float frequency_all, const float *presence, float presence_all, const int32_t *bias_tokens,
                                  const float *bias_values, int32_t n_bias, const int32_t *mask, int64_t mask_stride,
                                  int32_t n_mask, const int32_t *mask_rows, void *stream) {
    if (n_rows < 0 || vocab <= 0 || n_seqs < 0 || max_tokens < 0 || n_drafts < 0 || n_bias < 0 || n_mask < 0 || logits_stride < vocab ||
        out_stride < vocab || (tokens && token_stride < max_tokens && n_seqs > 1) || (mask && mask_stride < (vocab + 31) / 32) ||
        (!query_lens && n_rows != n_seqs) || !(repetition_all > 0.0f && repetition_all < INFINITY) || !(fabsf(frequency_all) < INFINITY) || !(fabsf(presence_all) < INFINITY))
        return ODSD_ERR_SHAPE;
    if (dtype != ODSD_DT_F32 && dtype != ODSD_DT_BF16 && dtype != ODSD_DT_F16) return ODSD_ERR_DTYPE;
    if (tokens && token_bytes != 4 && token_bytes != 8) return ODSD_ERR_DTYPE;
    if (n_rows == 0 || n_seqs == 0) return ODSD_OK;
    if (!logits || !out || (n_bias && (!bias_tokens || !bias_values)) || (n_drafts && !draft_tokens)) return ODSD_ERR_NULL;
    const uintptr_t e = dtype == ODSD_DT_F32 ? 3u : 1u;
    if (((uintptr_t)logits & e) || ((uintptr_t)out & e) || (tokens && ((uintptr_t)tokens & (uintptr_t)(token_bytes - 1))) ||
        ((uintptr_t)draft_tokens & 7u) || ((uintptr_t)mask & 3u))
        return ODSD_ERR_ALIGN;
    AdjParams p{};
    p.logits = logits; p.out = out; p.ld = logits_stride; p.ldo = out_stride; p.q_lens = query_lens;
    p.tokens = max_tokens ? tokens : nullptr; p.token_bytes = token_bytes; p.token_stride = token_stride; p.max_tokens = max_tokens;
    p.token_lens = token_lens; p.prompt_lens = prompt_lens; p.drafts = draft_tokens; p.n_drafts = n_drafts;
    p.repetition = repetition; p.repetition_all = repetition_all; p.frequency = frequency; p.frequency_all = frequency_all;
    p.presence = presence; p.presence_all = presence_all;
    p.bias_tokens = bias_tokens; p.bias_values = bias_values; p.n_bias = n_bias;
    p.mask = mask; p.mask_stride = mask_stride; p.n_mask = n_mask; p.mask_rows = mask_rows;
    p.n_seqs = n_seqs; p.n_rows = n_rows; p.vocab = vocab;
    // slices: enough workgroups for the chip, of 1024 to 8192 tokens
    int64_t slice = ((int64_t)vocab * n_seqs / 1024 + 255) / 256 * 256;
    slice = max((int64_t)1024, min((int64_t)8192, slice));
    p.slice = (int)slice;
    p.slices = (int)((vocab + slice - 1) / slice);
    if ((int64_t)n_seqs * p.slices >= (1LL << 24) || max_tokens + (int64_t)n_drafts >= (1 << 29)) return ODSD_ERR_UNSUPPORTED;
    p.sparse = p.tokens || n_drafts || n_bias;
    p.dense = out != logits || out_stride != logits_stride || mask;
    if (!p.sparse && !p.dense) return ODSD_OK;
    const unsigned grid = (unsigned)(n_seqs * p.slices);
    const size_t bytes = p.sparse ? (size_t)slice * 6 : 0;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ODSD_DT_F32) adjust_logits_kernel<float><<<grid, 256, bytes, st>>>(p);
    else if (dtype == ODSD_DT_BF16) adjust_logits_kernel<__bf16><<<grid, 256, bytes, st>>>(p);
    else adjust_logits_kernel<half_t><<<grid, 256, bytes, st>>>(p);
    ODSD_CHECK_LAUNCH();
    return ODSD_OK;
}
