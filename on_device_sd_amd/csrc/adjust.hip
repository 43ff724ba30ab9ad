// Logits on their way to the verification: penalties for repeated tokens, biases and grammar masks, one pass over the rows.
//   x = logit;   seen (prompt, output or a draft before the row): x = x > 0 ? x / r : x r
//   x = x - (f n + p [n > 0])         n: how often among the output and the drafts before the row
//   x = x + bias;   a mask bit that is clear: x = -inf;   rounded once, to the logits' type
//
// A workgroup has one sequence and a share of the vocabulary, every so many granules of 128 tokens (the words that are used most have
// neighbouring numbers).  It looks through the sequence's tokens once, counts its own in LDS and lists those that have occurred, are
// drafted or have a bias.  Then it goes through the sequence's rows, adding to the counts the draft that stands before each: a row's
// share comes in 16 bytes a thread, the listed logits are changed in LDS, and it leaves 16 bytes a thread with -inf where the mask forbids.
// No table of counts lives between steps, so drafts that are not kept leave nothing to undo.  The traffic of the logits, once in and once
// out, is the bound; the tokens (read again for every share, from L2) are little next to it: 449 rows of 131072 in bf16, 4096 tokens a sequence,
// 63 us, 3.9 TB/s (a copy of the rows 45).  Changing the listed logits in memory after a copy took 102: a logit is 2 bytes of the 64 that move.
// Asking for the first rows before the tokens are looked through gains nothing, nor do nontemporal loads or stores (1 to 2 us more).  One row
// a sequence is a chain of some ten waits a workgroup, and LDS for two rows (42 KB) lets a CU have three of them, nearly three rounds for 64
// sequences of 131072; the row is asked for four times (two at a time, two ahead), three of them met by caches: 15 us where the bytes take 7, 18
// with a mask (500 tokens of history), 256 sequences 48 and 57 for 27.  In place and without a mask only the listed logits are read and written.
// Of more than 128 biases in a share every biased token walks all of the sequence's: 300, 3000 and 20000 biases of 64 such rows 21, 223 and
// 10980 us.  A mask is the form for tokens that are forbidden.
#include "common.h"
#include <type_traits>

#define ADJ_SEEN 0x80000000u     // has occurred
#define ADJ_DRAFT 0x40000000u    // is drafted, and may occur in later rows
#define ADJ_BIAS 0x20000000u     // has a bias; the other bits count
#define ADJ_BIASES 128           // biases of a share that are kept in LDS
#define ADJ_GRANULE 128          // tokens, a power of two
#define ADJ_MOST 4096            // tokens of a share at most
#define ADJ_LEAST 1024           // shares are not made smaller; those that are not larger have a kernel with fewer loads (8 sequences of 5 rows of 50257 11.0 / 9.7 us)
#define ADJ_FEW 1024             // workgroups up to which a sequence's rows go to several
#define ADJ_ROWS 64              // rows whose drafts and masks are looked up at a time

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
    int n_seqs, n_rows, n_drafts, vocab, token_bytes, max_tokens, n_bias, n_mask;
    int shares, share_bits, most;              // shares of the vocabulary, a power of two; tokens of a share at most
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

// MOST: tokens of a share at most
template <typename T, bool MASK, int MOST>
__global__ __launch_bounds__(256) void adjust_logits_kernel(const AdjParams p) {
    extern __shared__ uint4_t lds4[];          // two rows of the share (dense), counts [most], the list [most] in 16 bits
    uint32_t *lds = (uint32_t *)lds4 + (p.dense ? 2 * p.most * (int)sizeof(T) / 4 : 0);
    __shared__ int sums[8], listed, biases;
    __shared__ int bias_token[ADJ_BIASES], bias_entry[ADJ_BIASES];       // entries that name a token of the share, in no order
    __shared__ int draft_of[ADJ_ROWS], mask_at[ADJ_ROWS];
    uint32_t *counts = lds;
    uint16_t *list = (uint16_t *)(lds + p.most);
    const int tid = threadIdx.x;
    const int s = blockIdx.x >> p.share_bits, share = blockIdx.x & (p.shares - 1);
    // token i of the share is token at(i) of the vocabulary, from vocab on there is none; mine(t): which of the share's it is, or -1
    auto at = [&](const int i) { return ((i / ADJ_GRANULE << p.share_bits) + share) * ADJ_GRANULE + i % ADJ_GRANULE; };
    auto mine = [&](const int64_t t) -> int {
        if (t < 0 || t >= p.vocab) return -1;
        const int g = (int)t / ADJ_GRANULE;
        return (g & (p.shares - 1)) == share ? (g >> p.share_bits) * ADJ_GRANULE + (int)t % ADJ_GRANULE : -1;
    };
    if (p.sparse) {
        if (tid == 0) listed = biases = 0;
        for (int i = tid; i < p.most / 4; i += 256) ((uint4_t *)counts)[i] = uint4_t{0u, 0u, 0u, 0u};
    }
    // flags of token i of the share; whoever sets the first lists it
    auto mark = [&](const int i, const uint32_t flags) {
        if (atomicOr(&counts[i], flags) == 0u) list[atomicAdd(&listed, 1)] = (uint16_t)i;
    };
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
    // (no row and no draft past those that there are, whatever the lengths say: their sums may have wrapped)
    if (rows == 0 || (uint32_t)row >= (uint32_t)p.n_rows) return;
    rows = min(rows, p.n_rows - row);
    const int drafts = p.drafts && (uint32_t)draft < (uint32_t)p.n_drafts ? min(rows - 1, p.n_drafts - draft) : 0;
    // the rows of this workgroup
    constexpr int R = 2;                       // rows at a time
    const int per_group = ((rows + (int)gridDim.y - 1) / (int)gridDim.y + R - 1) / R * R, from = (int)blockIdx.y * per_group, until = min(rows, from + per_group);
    if (from >= rows) return;
    if (p.sparse) {
        if (p.tokens) {
            const int len = min(max(p.token_lens ? p.token_lens[s] : p.max_tokens, 0), p.max_tokens);
            const int prompt = p.prompt_lens ? p.prompt_lens[s] : 0;
            for (int i0 = tid; i0 < len; i0 += 8 * 256) {      // (eight loads on their way at a time)
                int64_t t[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) t[u] = adj_token(p.tokens, p.token_bytes, s * p.token_stride + min(i0 + 256 * u, len - 1));
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int i = i0 + 256 * u < len ? mine(t[u]) : -1;
                    if (i >= 0) {
                        mark(i, ADJ_SEEN);
                        if (i0 + 256 * u >= prompt) atomicAdd(&counts[i], 1u);
                    }
                }
            }
        }
        for (int i = tid; i < drafts; i += 256) {
            const int t = mine(adj_token(p.drafts, 8, draft + i));
            if (t < 0) continue;
            if (i + 1 >= until) continue;      // (draft i stands before row i + 1)
            mark(t, i + 1 < from ? ADJ_SEEN : ADJ_DRAFT);
            if (i + 1 < from) atomicAdd(&counts[t], 1u);
        }
        for (int i = tid; i < p.n_bias; i += 256) {
            const int t = mine(p.bias_tokens[(int64_t)s * p.n_bias + i]);
            if (t >= 0) {
                mark(t, ADJ_BIAS);
                const int k = atomicAdd(&biases, 1);
                if (k < ADJ_BIASES) {
                    bias_token[k] = t;
                    bias_entry[k] = i;
                }
            }
        }
    }
    const T *in = (const T *)p.logits + (int64_t)row * p.ld;
    T *to = (T *)p.out + (int64_t)row * p.ldo;
    auto mask_row = [&](const int j) {         // of the masks, or -1
        const int m = p.mask_rows ? p.mask_rows[row + j] : row + j;
        return m >= 0 && m < p.n_mask ? m : -1;
    };
    int n_listed = 0;
    if (p.sparse) {
        __syncthreads();                       // counts, list and biases are there
        n_listed = listed;
    }
    const float r = p.repetition ? p.repetition[s] : p.repetition_all;
    const float f = p.frequency ? p.frequency[s] : p.frequency_all;
    const float pr = p.presence ? p.presence[s] : p.presence_all;
    // the bias of token i: the last of the entries that name it
    auto bias_of = [&](const int i) {
        int last = -1;
        if (biases <= ADJ_BIASES) {
            for (int b = 0; b < biases; ++b) last = bias_token[b] == i ? max(last, bias_entry[b]) : last;
        } else {
            const int v = at(i);
            for (int b = 0; b < p.n_bias; ++b) last = p.bias_tokens[(int64_t)s * p.n_bias + b] == v ? b : last;
        }
        return p.bias_values[(int64_t)s * p.n_bias + last];
    };
    auto changed = [&](float x, const uint32_t n, const float add) {
        const uint32_t times = n & (ADJ_BIAS - 1);
        if (n & ADJ_SEEN) x = x > 0.0f ? x / r : x * r;
        if (times) x = x - (f * (float)times + pr);
        return n & ADJ_BIAS ? x + add : x;
    };
    // token i of the share in the workgroup's rows, straight in memory
    auto column = [&](const int i, uint32_t n) {
        const int v = at(i);
        const float add = n & ADJ_BIAS ? bias_of(i) : 0.0f;
        for (int j0 = from; j0 < until; j0 += 4) {         // (four rows' loads on their way at a time)
            T raw[4];
            int64_t before[4];
            bool allowed[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = min(j0 + u, until - 1);
                const int m = MASK ? mask_row(j) : -1;
                raw[u] = in[j * p.ld + v];
                allowed[u] = m < 0 || ((p.mask[m * p.mask_stride + (v >> 5)] >> (v & 31)) & 1);
                before[u] = n & ADJ_DRAFT && j > 0 && j <= drafts ? adj_token(p.drafts, 8, draft + j - 1) : -1;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (j0 + u >= until) break;
                if (before[u] == v) n = (n + 1u) | ADJ_SEEN;
                to[(j0 + u) * p.ldo + v] = AdjIO<T>::put(allowed[u] ? changed(AdjIO<T>::get(raw[u]), n, add) : -INFINITY);
            }
        }
    };
    if (!p.dense) {                            // in place, and no mask: nothing else changes
        for (int k = tid; k < n_listed; k += 256) column(list[k], counts[list[k]]);
        return;
    }
    constexpr int TPG = 16 / (int)sizeof(T);   // tokens of a group: 16 bytes, rows at any element
    constexpr int U = (MOST / TPG + 255) / 256;      // groups of a thread
    // what the vocabulary has behind its last whole group
    const int tail = p.vocab - p.vocab % TPG + tid;
    if (tid < TPG && tail < p.vocab && mine(tail) >= 0) column(mine(tail), p.sparse ? counts[mine(tail)] : 0u);
    if (p.vocab < TPG) return;
    uint4_t raw[R][U], next[R][U];
    uint32_t bits[R][U], next_bits[R][U];
    // of a thread's only token of the list, where no thread has more
    const bool few = n_listed <= 256;
    const int my_i = few && tid < n_listed ? list[tid] : 0, my_v = at(my_i), per = p.most / TPG;
    uint32_t my_n = few && tid < n_listed ? counts[my_i] : 0u;
    const float my_add = my_n & ADJ_BIAS ? bias_of(my_i) : 0.0f;
    for (int c0 = from; c0 < until; c0 += ADJ_ROWS) {
        __syncthreads();                       // nobody reads the last rows' drafts and masks any more
        if (tid < ADJ_ROWS) {
            const int j = c0 + tid;
            const int64_t t = j > 0 && j <= drafts ? adj_token(p.drafts, 8, draft + j - 1) : -1;
            draft_of[tid] = t >= 0 && t < p.vocab ? (int)t : -1;
            mask_at[tid] = MASK && j < rows ? mask_row(j) : -1;
        }
        __syncthreads();
        const int end = min(until, c0 + ADJ_ROWS);
        // (what the next turn needs is requested a turn ahead, loads without branches in between: the compiler then knows how many
        // younger ones it may leave on their way)
        auto load = [&](uint4_t (&w)[R][U], uint32_t (&b)[R][U], const int j) {
#pragma unroll
            for (int q = 0; q < R; ++q) {
                const int jq = min(j + q, end - 1), m = MASK ? mask_at[jq - c0] : -1;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int v = min(at(TPG * (tid + 256 * u)), p.vocab - TPG);
                    w[q][u] = *(const raw_t *)(in + jq * p.ld + v);
                    if constexpr (MASK) b[q][u] = (uint32_t)p.mask[max(m, 0) * p.mask_stride + (v >> 5)] >> (v & 31) | (m < 0 ? ~0u : 0u);
                }
            }
        };
        load(raw, bits, c0);
        for (int j = c0; j < end; j += R) {
            load(next, next_bits, j + R);
            if (n_listed) {
                if (j > c0) __syncthreads();   // the last rows have left LDS
#pragma unroll
                for (int q = 0; q < R; ++q)
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (tid + 256 * u < per) lds4[q * per + tid + 256 * u] = raw[q][u];
                __syncthreads();
                T *one = (T *)lds4;
                if (few) {
#pragma unroll
                    for (int q = 0; q < R; ++q) {
                        if (my_n && draft_of[min(j + q, end - 1) - c0] == my_v && j + q < end) my_n = (my_n + 1u) | ADJ_SEEN;
                        if (my_n) one[q * p.most + my_i] = AdjIO<T>::put(changed(AdjIO<T>::get(one[q * p.most + my_i]), my_n, my_add));
                    }
                } else {
                    for (int k = tid; k < n_listed; k += 256) {
                        const int i = list[k];
                        uint32_t n = counts[i];
                        const float add = n & ADJ_BIAS ? bias_of(i) : 0.0f;
#pragma unroll
                        for (int q = 0; q < R; ++q) {
                            if (j + q < end && draft_of[j + q - c0] == at(i)) counts[i] = n = (n + 1u) | ADJ_SEEN;
                            one[q * p.most + i] = AdjIO<T>::put(changed(AdjIO<T>::get(one[q * p.most + i]), n, add));
                        }
                    }
                }
                __syncthreads();
#pragma unroll
                for (int q = 0; q < R; ++q)
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (tid + 256 * u < per) raw[q][u] = lds4[q * per + tid + 256 * u];
            }
#pragma unroll
            for (int q = 0; q < R; ++q) {
                T *y = to + (j + q) * p.ldo;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = TPG * (tid + 256 * u), v = at(i);
                    if constexpr (MASK) {
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            if constexpr (sizeof(T) == 4) {
                                raw[q][u][w] = (bits[q][u] >> w) & 1 ? raw[q][u][w] : 0xff800000u;
                            } else {
                                constexpr uint32_t INF = std::is_same<T, half_t>::value ? 0xfc00u : 0xff80u;
                                const uint32_t lo = (bits[q][u] >> (2 * w)) & 1 ? raw[q][u][w] & 0xffffu : INF;
                                const uint32_t hi = (bits[q][u] >> (2 * w + 1)) & 1 ? raw[q][u][w] & 0xffff0000u : INF << 16;
                                raw[q][u][w] = lo | hi;
                            }
                        }
                    }
                    if (j + q < end && i < p.most && v + TPG <= p.vocab) *(raw_t *)(y + v) = raw[q][u];
                }
            }
#pragma unroll
            for (int q = 0; q < R; ++q)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    raw[q][u] = next[q][u];
                    if constexpr (MASK) bits[q][u] = next_bits[q][u];
                }
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
    // shares: enough workgroups for the chip, of 1024 to 4096 tokens
    const int64_t granules = ((int64_t)vocab + ADJ_GRANULE - 1) / ADJ_GRANULE;
    auto tokens_of = [&](const int bits) { return ((granules + (1LL << bits) - 1) >> bits) * ADJ_GRANULE; };
    while (tokens_of(p.share_bits) > ADJ_LEAST && (tokens_of(p.share_bits) > ADJ_MOST || ((int64_t)n_seqs << p.share_bits) < 1024)) ++p.share_bits;
    p.shares = 1 << p.share_bits;
    p.most = (int)tokens_of(p.share_bits);
    if ((int64_t)n_seqs * p.shares >= (1LL << 24) || max_tokens + (int64_t)n_drafts >= (1 << 29)) return ODSD_ERR_UNSUPPORTED;
    p.sparse = p.tokens || n_drafts || n_bias;
    p.dense = out != logits || out_stride != logits_stride || mask;
    if (!p.sparse && !p.dense) return ODSD_OK;
    // Few sequences: their rows are dealt out too, two to a workgroup at least, and each looks through the tokens for itself.  (Rows of one
    // workgroup / so, us: one sequence of 5 rows of 50257 fp32 9.2 / 6.5, of 41 35.4 / 11.6; 4 of 5 rows of 131072 bf16 9.9 / 9.3; up to 2048
    // workgroups 16 of 9 rows of 131072 21.2 / 25.3.)
    const int64_t wgs = (int64_t)n_seqs << p.share_bits;
    const int64_t groups = query_lens ? max((int64_t)1, min((int64_t)ADJ_FEW / wgs, ((int64_t)n_rows + 1) / 2)) : 1;
    const dim3 grid((unsigned)wgs, (unsigned)groups);
    const size_t elt = dtype == ODSD_DT_F32 ? 4 : 2, bytes = p.sparse ? (size_t)p.most * (6 + (p.dense ? 2 * elt : 0)) : 0;
    hipStream_t st = (hipStream_t)stream;
#define ADJ_GO(T)                                                                 \
    do {                                                                          \
        if (p.most <= ADJ_LEAST) {                                                \
            if (mask && n_mask) adjust_logits_kernel<T, true, ADJ_LEAST><<<grid, 256, bytes, st>>>(p); \
            else adjust_logits_kernel<T, false, ADJ_LEAST><<<grid, 256, bytes, st>>>(p);         \
        } else if (mask && n_mask) adjust_logits_kernel<T, true, ADJ_MOST><<<grid, 256, bytes, st>>>(p);     \
        else adjust_logits_kernel<T, false, ADJ_MOST><<<grid, 256, bytes, st>>>(p);         \
    } while (0)
    if (dtype == ODSD_DT_F32) ADJ_GO(float);
    else if (dtype == ODSD_DT_BF16) ADJ_GO(__bf16);
    else ADJ_GO(half_t);
#undef ADJ_GO
    ODSD_CHECK_LAUNCH();
    return ODSD_OK;
}
