// Logits on their way to the verification: penalties for repeated tokens, biases and grammar masks, one pass over the rows.
//   x = logit;   seen (prompt, output or a draft before the row): x = x > 0 ? x / r : x r
//   x = x - (f n + p [n > 0])         n: how often among the output and the drafts before the row
//   x = x + bias;   a mask bit that is clear: x = -inf;   rounded once, to the logits' type
//
// A workgroup has one sequence and a slice of the vocabulary.  It looks through the sequence's tokens once and counts those of its slice
// in LDS (32 bits a token: bit 31 "seen", the others the count), then goes through the sequence's rows, adding to the counts the draft
// that stands before each.  No table of counts lives between steps, so drafts that are not kept leave nothing to undo.  The logits are
// read and written once: 2 bytes of traffic for each, next to which the tokens (read again by every slice, from L2) are little.
#include "common.h"

#define ADJ_SEEN 0x80000000u

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
};

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
    extern __shared__ uint32_t lds[];          // counts [slice], then the last bias entry of a token + 1 [slice]
    __shared__ int sums[8];
    uint32_t *counts = lds, *bias = lds + p.slice;
    const int tid = threadIdx.x;
    const int s = blockIdx.x / p.slices, v0 = (blockIdx.x - s * p.slices) * p.slice;
    const int here = min(p.slice, p.vocab - v0);
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
        row = sums[0] + sums[1] + sums[2] + sums[3];
        draft = sums[4] + sums[5] + sums[6] + sums[7];
        rows = max(p.q_lens[s], 0);
    }
    rows = min(rows, p.n_rows - row);
    if (rows <= 0) return;
    for (int i = tid; i < here; i += 256) {
        counts[i] = 0u;
        if (p.n_bias) bias[i] = 0u;
    }
    __syncthreads();
    if (p.tokens) {
        const int len = min(max(p.token_lens ? p.token_lens[s] : p.max_tokens, 0), p.max_tokens);
        const int prompt = p.prompt_lens ? p.prompt_lens[s] : 0;
        for (int i = tid; i < len; i += 256) {
            const int64_t t = adj_token(p.tokens, p.token_bytes, s * p.token_stride + i) - v0;
            if (t >= 0 && t < here) {
                if (i < prompt) atomicOr(&counts[t], ADJ_SEEN);
                else {
                    atomicAdd(&counts[t], 1u);
                    atomicOr(&counts[t], ADJ_SEEN);
                }
            }
        }
    }
    for (int i = tid; i < p.n_bias; i += 256) {
        const int t = p.bias_tokens[(int64_t)s * p.n_bias + i] - v0;
        if (p.bias_tokens[(int64_t)s * p.n_bias + i] >= v0 && t < here) atomicMax(&bias[t], (uint32_t)i + 1u);
    }
    __syncthreads();
    const float r = p.repetition ? p.repetition[s] : p.repetition_all;
    const float f = p.frequency ? p.frequency[s] : p.frequency_all;
    const float pr = p.presence ? p.presence[s] : p.presence_all;
    for (int j = 0; j < rows; ++j) {
        if (j > 0) {                           // the row has seen the draft before it
            if (p.drafts && draft + j - 1 < p.n_drafts) {
                __syncthreads();
                const int64_t t = adj_token(p.drafts, 8, draft + j - 1) - v0;
                if (tid == 0 && t >= 0 && t < here) counts[t] = (counts[t] + 1u) | ADJ_SEEN;
                __syncthreads();
            }
        }
        const T *from = (const T *)p.logits + (int64_t)(row + j) * p.ld + v0;
        T *to = (T *)p.out + (int64_t)(row + j) * p.ldo + v0;
        const int m = p.mask ? p.mask_rows ? p.mask_rows[row + j] : row + j : -1;
        const int32_t *mask = m >= 0 && m < p.n_mask ? p.mask + m * p.mask_stride : nullptr;
        for (int i = tid; i < here; i += 256) {
            float x = AdjIO<T>::get(from[i]);
            const uint32_t n = counts[i];
            if (n) {
                const uint32_t times = n & ~ADJ_SEEN;
                x = x > 0.0f ? x / r : x * r;
                x = x - (f * (float)times + (times ? pr : 0.0f));
            }
            if (p.n_bias && bias[i]) x += p.bias_values[(int64_t)s * p.n_bias + bias[i] - 1];
            if (mask && !((mask[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1)) x = -INFINITY;
            to[i] = AdjIO<T>::put(x);
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
    if ((int64_t)n_seqs * p.slices >= (1LL << 24)) return ODSD_ERR_UNSUPPORTED;
    const unsigned grid = (unsigned)(n_seqs * p.slices);
    const size_t bytes = (size_t)slice * (n_bias ? 8 : 4);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ODSD_DT_F32) adjust_logits_kernel<float><<<grid, 256, bytes, st>>>(p);
    else if (dtype == ODSD_DT_BF16) adjust_logits_kernel<__bf16><<<grid, 256, bytes, st>>>(p);
    else adjust_logits_kernel<half_t><<<grid, 256, bytes, st>>>(p);
    ODSD_CHECK_LAUNCH();
    return ODSD_OK;
}
