// Matrix product with bias, activation and residual in its epilogue:
//   y[m][n] = act(sum_k x[m][k] w[n][k] + bias[n]) + residual[m][n]
// the projections around the attention of a layer and the language-model head behind the last one.  Sums in fp32 (the
// matrix cores' accumulators), bias, activation and residual in fp32, one rounding to the output's type.
//
// Every kernel gives the weights as the A operand of the matrix instruction and the tokens as B, so that a lane's
// accumulators are four consecutive n of one token.
#include "attn.h"
#include "w4_gemm.h"

struct LinearParams {
    const void *x, *w, *bias, *res;
    void *out;
    int64_t ldx, ldw, ldr, ldo;    // elements between two rows
    int M, N, K, act;
    int tiles_n, tiles_m, slices, slice_k;   // tile kernel: K in `slices` parts of slice_k columns (a multiple of 64)
    float *part;                   // their sums, [slices][M][part_ld], when there are several
    int64_t part_ld;               // N rounded up to 8
};

// ---- epilogue ------------------------------------------------------------------------------
// exp for the activations.  fp32 outputs: the library's (1 ulp).  16-bit outputs: 2^(v log2 e) by the hardware, off by at
// most |v| 2^-24 log2 e + 2^-22 relative, 1e-5 where it still counts, against half steps of 2^-9 (bf16) and 2^-12 (fp16).
// The reciprocal behind it is the hardware's for both (1 ulp; a correctly rounded quotient is ten instructions a value).  It has
// no subnormal results: where 1 + exp(-v) passes 2^126 (v below -87.3; silu is above -1.1e-36 there) it is 0.
template <bool PRECISE> __device__ __forceinline__ float act_exp(float v) {
    if (PRECISE) return expf(v);
    return __builtin_amdgcn_exp2f(v * 1.44269504088896341f);
}
template <bool PRECISE> __device__ __forceinline__ float act_sigmoid_mul(float y, float v) {   // y / (1 + exp(-v))
    return y * __builtin_amdgcn_rcpf(1.0f + act_exp<PRECISE>(-v));
}
template <bool PRECISE, int ACT> __device__ __forceinline__ float activate(float y) {
    if (ACT == ODSD_ACT_RELU) return y < 0.0f ? 0.0f : y;                  // (NaN stays)
    if (ACT == ODSD_ACT_SILU) return act_sigmoid_mul<PRECISE>(y, y);
    if (ACT == ODSD_ACT_GELU) return 0.5f * y * erfcf(y * -0.70710678118654752f);
    // 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u)): no cancellation for negative u
    if (ACT == ODSD_ACT_GELU_TANH) return act_sigmoid_mul<PRECISE>(y, 1.5957691216057308f * (y + 0.044715f * y * y * y));
    return y;
}

template <typename O> struct Vec8 { typedef O type __attribute__((ext_vector_type(8))); };

// y[m][n .. n + 7] from their sums.  Eight consecutive values are one access at the elements' own alignment (the hardware
// takes any), so neither N nor the rows' distances need be multiples of anything.
template <typename T> __device__ __forceinline__ void load_bias8(const LinearParams &p, int n, float *b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = 0.0f;
    if (!p.bias) return;
    const T *bias = (const T *)p.bias + n;
    if (n + 8 <= p.N) {
        typename Vec8<T>::type v;
        __builtin_memcpy(&v, bias, sizeof v);
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = (float)v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (n + i < p.N) b[i] = (float)bias[i];
    }
}
template <typename T, typename O, int ACT>
__device__ __forceinline__ void finish8(const LinearParams &p, int m, int n, const float *v, const float *b) {
    if (m >= p.M || n >= p.N) return;
    const O *res = p.res ? (const O *)p.res + (int64_t)m * p.ldr + n : nullptr;
    O *out = (O *)p.out + (int64_t)m * p.ldo + n;
    constexpr bool PRECISE = sizeof(O) == 4;
    if (n + 8 <= p.N) {
        typename Vec8<O>::type r, y;
        if (res) __builtin_memcpy(&r, res, sizeof r);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = activate<PRECISE, ACT>(v[i] + b[i]);
            y[i] = (O)(res ? a + (float)r[i] : a);
        }
        __builtin_memcpy(out, &y, sizeof y);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (n + i < p.N) {
            const float a = activate<PRECISE, ACT>(v[i] + b[i]);
            out[i] = (O)(res ? a + (float)res[i] : a);
        }
}
// f with the call's activation as a constant
template <typename F> __device__ __forceinline__ void with_activation(int act, F f) {
    switch (act) {
        case ODSD_ACT_RELU: return f(std::integral_constant<int, ODSD_ACT_RELU>{});
        case ODSD_ACT_SILU: return f(std::integral_constant<int, ODSD_ACT_SILU>{});
        case ODSD_ACT_GELU: return f(std::integral_constant<int, ODSD_ACT_GELU>{});
        case ODSD_ACT_GELU_TANH: return f(std::integral_constant<int, ODSD_ACT_GELU_TANH>{});
        default: return f(std::integral_constant<int, ODSD_ACT_NONE>{});
    }
}
template <typename T, typename O>
__device__ __forceinline__ void finish8(const LinearParams &p, int m, int n, const float *v) {
    with_activation(p.act, [&](auto act) {
        float b[8];
        load_bias8<T>(p, n, b);
        finish8<T, O, decltype(act)::value>(p, m, n, v, b);
    });
}
template <typename T, typename O>
__device__ __forceinline__ void finish1(const LinearParams &p, int m, int n, float v) {
    constexpr bool PRECISE = sizeof(O) == 4;
    if (p.bias) v += (float)((const T *)p.bias)[n];
    with_activation(p.act, [&](auto act) { v = activate<PRECISE, decltype(act)::value>(v); });
    if (p.res) v += (float)((const O *)p.res)[(int64_t)m * p.ldr + n];
    ((O *)p.out)[(int64_t)m * p.ldo + n] = (O)v;
}

// Eight values of a row from column k on, at the elements' own alignment, without a branch before the load: at the row's end
// its last eight, of which clip8() zeroes those in front of k (all, if k is behind the end).  Both operands of a product are
// loaded so, so their columns stay together.  load8_short: K < 8, one by one.
template <typename T> __device__ __forceinline__ uint4_t load8(const T *row, int k, int K) {
    uint4_t v;
    __builtin_memcpy(&v, row + min(k, K - 8), 16);
    return v;
}
template <typename T> __device__ __forceinline__ uint4_t load8_short(const T *row, int k, int K) {
    uint4_t v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint16_t e = 0;
        if (k + i < K) __builtin_memcpy(&e, row + k + i, 2);
        v[i >> 1] |= (uint32_t)e << (16 * (i & 1));
    }
    return v;
}
__device__ __forceinline__ uint4_t clip8(uint4_t v, int k, int K) {
    const int skip = K >= 8 ? k - (K - 8) : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = skip > 2 * i + 1 ? 0u : skip > 2 * i ? v[i] & 0xffff0000u : v[i];
    return v;
}

// ---- few tokens ------------------------------------------------------------------------------
// The weights' bytes bound it.  A workgroup takes 16 rows of w and all of K; its NWV wavefronts share K in blocks of 64
// columns and add their sums up through LDS, so nothing is split over workgroups, there is one launch and no workspace.
// Weights go to registers as the matrix instruction wants them (a lane: 16 consecutive columns of one row), DEPTH blocks of
// them requested at once; a token's columns are used by one wavefront of the workgroup only, so they come to registers, too.
// (Three or four groups of 16 tokens in this form: slower than tiles from 17 tokens on, K 2048, N 5120, M = 40 16.7 / 11.5 us.)
template <typename T, typename O, int NWV, int DEPTH>
__global__ __launch_bounds__(NWV * 64) void linear_rows_kernel(LinearParams p) {
    typedef typename AttnT<T>::V8 V8;
    __shared__ float sums[NWV][16][17];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16;
    const int full = p.K / 64, blocks = (p.K + 63) / 64;       // blocks that lie in K whole; all of them
    const bool token = r < p.M;                                // (columns of the product that nobody stores are not read)
    const T *w = (const T *)p.w + (int64_t)min(n0 + r, p.N - 1) * p.ldw;
    const T *x = (const T *)p.x + (int64_t)min(r, p.M - 1) * p.ldx;
    float4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    uint4_t a[DEPTH][2], c[DEPTH][2];
    auto multiply = [&](int d) {
#pragma unroll
        for (int u = 0; u < 2; ++u) acc = AttnT<T>::mfma(__builtin_bit_cast(V8, a[d][u]), __builtin_bit_cast(V8, c[d][u]), acc);
    };
    int b = wave;
    auto group = [&](auto count) {                             // this many blocks of the wavefront, all of them whole
        constexpr int n = decltype(count)::value;
#pragma unroll
        for (int d = 0; d < n; ++d)
#pragma unroll
            for (int u = 0; u < 2; ++u) __builtin_memcpy(&a[d][u], w + (b + d * NWV) * 64 + g * 16 + u * 8, 16);
#pragma unroll
        for (int d = 0; d < n; ++d)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                c[d][u] = uint4_t{0, 0, 0, 0};
                if (token) __builtin_memcpy(&c[d][u], x + (b + d * NWV) * 64 + g * 16 + u * 8, 16);
            }
#pragma unroll
        for (int d = 0; d < n; ++d) multiply(d);
        b += n * NWV;
    };
    while (b + (DEPTH - 1) * NWV < full) group(std::integral_constant<int, DEPTH>{});
    while (b < full) group(std::integral_constant<int, 1>{});
    if (b < blocks) {                                          // the block that K ends in
        const int k = b * 64 + g * 16;
        if (p.K < 8) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                a[0][u] = load8_short(w, k + u * 8, p.K);
                c[0][u] = load8_short(x, k + u * 8, p.K);
            }
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                a[0][u] = load8(w, k + u * 8, p.K);
                c[0][u] = load8(x, k + u * 8, p.K);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                a[0][u] = clip8(a[0][u], k + u * 8, p.K);
                c[0][u] = clip8(c[0][u], k + u * 8, p.K);
            }
        }
        multiply(0);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[wave][r][g * 4 + e] = acc[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += NWV * 64) {
        const int m = i >> 4, n = i & 15;
        if (m >= p.M || n0 + n >= p.N) continue;
        float v = 0.0f;
#pragma unroll
        for (int q = 0; q < NWV; ++q) v += sums[q][m][n];
        finish1<T, O>(p, m, n0 + n, v);
    }
}

// ---- tiles -----------------------------------------------------------------------------------
// NWN x NWM wavefronts, each FA blocks of 32 n by FB blocks of 32 m on v_mfma_f32_32x32x16; steps of 64 along K.  Both
// operands go to LDS without passing registers (buffer_load ... lds, 16 bytes a lane): STAGES buffers of a step's x, one more of
// w.  A buffer's rows are 128 bytes, whose 16-byte segments are XORed with bits of the row's number: the 16 lanes that read
// together (rows 0-3, 12-15, 20-27 and 4-11, 16-19, 28-31 of a block, one segment) then meet the 16 bank groups.  What is behind
// a row's end, the matrix's last row or the slice's last step is addressed outside the buffer descriptor and arrives as zeros,
// without memory traffic, so every copy is issued whatever follows and a count says which have landed.  KS groups of such
// wavefronts take every KS-th step each, with buffers of their own, and add their sums up at the end: for few tokens, where a
// step is a chain of latencies, and for small tiles, which leave a CU with one workgroup.
template <int NWN, int NWM, int FA, int FB, int STAGES, int KS>
struct LinearTile {
    static constexpr int NW = NWN * NWM, TN = NWN * FA * 32, TM = NWM * FB * 32;
    static constexpr int BK = 64, ROW = BK * 2, SEGS = BK / 8, ROWS = 64 / SEGS;   // bytes and 16-byte segments of a row, rows of a copy
    static constexpr int A_BYTES = TN * ROW, B_BYTES = TM * ROW;
    static constexpr int A_RING = (STAGES + 1) * A_BYTES, B_RING = STAGES * B_BYTES, RING = A_RING + B_RING;
    static constexpr int LA = TN / ROWS / NW, LB = TM / ROWS / NW, L = LA + LB;   // copies of a wavefront per step
    // blocks of n that leave together (one where FB is 3; one block of m at a time and two of n are as fast within 1 %)
    static constexpr int CH = FA < 2 || FB > 2 ? 1 : 2;
    static constexpr int OUT_WAVE = FB * 32 * CH * 32 * 4;
    static constexpr int LDS = KS * (RING > NW * OUT_WAVE ? RING : NW * OUT_WAVE);
    static_assert(LA * ROWS * NW == TN && LB * ROWS * NW == TM && LB >= 1, "every wavefront makes the same number of copies");
    static_assert(NW % 2 == 0, "the swizzle of a copied row does not depend on the copy");
};

__device__ __forceinline__ void copy16_to_lds(uint4_t rsrc, uint32_t off, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :: "s"(lds_addr), "v"(off), "s"(rsrc) : "memory");
}
// the same for what is read once
__device__ __forceinline__ void copy16_to_lds_nt(uint4_t rsrc, uint32_t off, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds"
                 :: "s"(lds_addr), "v"(off), "s"(rsrc) : "memory");
}
__device__ __forceinline__ uint4_t descriptor(const void *base, uint32_t bytes) {
    const uint64_t a = (uint64_t)base;
    uint4_t r;
    r.x = __builtin_amdgcn_readfirstlane((uint32_t)a);
    r.y = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu);
    r.z = __builtin_amdgcn_readfirstlane(bytes);
    r.w = 0x00020000u;
    return r;
}

// What the lanes of a wavefront wrote to LDS before is what its lanes read behind (and the other way round): the hardware keeps
// a wavefront's LDS accesses in order, this keeps the compiler from moving them; no instruction.
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ONCE: the weights are read past the caches
template <typename T, typename O, int NWN, int NWM, int FA, int FB, int STAGES, int KS, bool ONCE>
__global__ __launch_bounds__(NWN * NWM * KS * 64) void linear_tile_kernel(LinearParams p) {
    typedef LinearTile<NWN, NWM, FA, FB, STAGES, KS> C;
    typedef typename AttnT<T>::V8 V8;
    constexpr int BK = C::BK;
    __shared__ __attribute__((aligned(1024))) char lds[C::LDS];
    const int lane = lane_id(), any_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = any_wave % C::NW, part = any_wave / C::NW;      // of a share of K, and which share
    // neighbouring tiles on one XCD (workgroup i is on XCD i % 8), in groups of up to 6 along m that share their weights: 6 x 5
    // of the 32 tiles that its CUs have at once (8 x 4: 8192 x 4096 x 16384 3 % slower, other shapes within 1 %)
    const int total = p.tiles_n * p.tiles_m * p.slices, per = (total + 7) / 8;
    const int b = blockIdx.x, t0 = (b & 7) * per + (b >> 3);
    if ((b >> 3) >= per || t0 >= total) return;
    const int slice = t0 / (p.tiles_n * p.tiles_m), t = t0 - slice * (p.tiles_n * p.tiles_m);
    const int group = t / (6 * p.tiles_n), in_group = t - group * 6 * p.tiles_n;
    const int gm = min(6, p.tiles_m - group * 6);
    const int n0 = in_group / gm * C::TN, m0 = (group * 6 + in_group % gm) * C::TM;

    const int k_begin = slice * p.slice_k, k_end = min(p.K, k_begin + p.slice_k);
    const int steps = (k_end - k_begin + BK * KS - 1) / (BK * KS);   // of a share: every KS-th
    const uint32_t ldw = (uint32_t)p.ldw * 2u, ldx = (uint32_t)p.ldx * 2u;
    const uint4_t rw = descriptor((const char *)p.w + (int64_t)n0 * p.ldw * 2, (uint32_t)(min(C::TN, p.N - n0) - 1) * ldw + p.K * 2);
    const uint4_t rx = descriptor((const char *)p.x + (int64_t)m0 * p.ldx * 2, (uint32_t)(min(C::TM, p.M - m0) - 1) * ldx + p.K * 2);
    // of the row that a lane copies (the same for all its copies: NW is even)
    const int seg = (lane & 7) ^ (((wave & 1) << 2) | (lane >> 4));
    const uint32_t row0 = wave * C::ROWS + lane / C::SEGS;
    const uint32_t off_w = row0 * ldw + seg * 16, off_x = row0 * ldx + seg * 16;
    char *const mine = lds + part * C::RING;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void *)mine;
    struct Place { uint32_t a, b; };                            // of a step's w and x in the rings
    auto copy = [&](int step, Place to, int i) {                // copy i of a step's: first those of w, then those of x
        const int k = k_begin + (step * KS + part) * BK;
        const uint32_t ko = k + seg * 8 < k_end ? (uint32_t)k * 2u : 0x80000000u;
        if (i < C::LA) {
            const uint32_t off = off_w + ko + i * (C::NW * C::ROWS) * ldw, at = lds0 + to.a + (i * C::NW + wave) * 1024;
            if (ONCE) copy16_to_lds_nt(rw, off, at);
            else copy16_to_lds(rw, off, at);
        } else copy16_to_lds(rx, off_x + ko + (i - C::LA) * (C::NW * C::ROWS) * ldx, lds0 + to.b + ((i - C::LA) * C::NW + wave) * 1024);
    };

    const int wn = wave % NWN, wm = wave / NWN;
    const uint32_t frag = (lane & 31) * C::ROW + (((lane >> 5) ^ ((lane >> 1) & 7)) << 4);
    const uint32_t fa0 = wn * FA * 32 * C::ROW + frag, fb0 = wm * FB * 32 * C::ROW + frag;
    float16_t acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    V8 fa[2][FA], fb[2][FB];
    // fragment i of columns 16 j .. of a buffer, in the order in which the products want them: w's first, x's, the rest of w's
    auto read = [&](int par, Place at, int j, int i) {
        if (i > 0 && i <= FB) fb[par][i - 1] = *(const V8 *)(mine + ((at.b + fb0) ^ (j << 5)) + (i - 1) * 32 * C::ROW);
        else fa[par][i ? i - FB : 0] = *(const V8 *)(mine + ((at.a + fa0) ^ (j << 5)) + (i ? i - FB : 0) * 32 * C::ROW);
    };
    // 16 columns: their products, and between those, one by one, the reads of the next 16 columns' fragments and copies.  (The
    // compiler would request a fragment right before its use, and copies in a row stall the wavefront: a CU takes one per 16
    // cycles.)  Copies: in the second 16 columns w of the step that is STAGES ahead, into the buffer that the step before left;
    // behind the barrier its x, into the buffer that this step leaves.  With as many buffers of w as of x, three quarters of a
    // step's copies waited for the barrier and had a step less to arrive: 8192 x 4096 x 16384 890 us, now 856; 1536 x 8192 x 8192
    // 189 and 162.
    constexpr int J = C::BK / 16, NM = FA * FB, NR = FA + FB;
    auto columns = [&](auto jc, int step, Place cur, Place next, uint32_t left) {
        constexpr int j = decltype(jc)::value;
        constexpr bool last = j == J - 1;
        constexpr int NC = last ? C::LB : j == 1 ? C::LA : 0;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            acc[i / FB][i % FB] = AttnT<T>::mfma32(fa[j & 1][i / FB], fb[j & 1][i % FB], acc[i / FB][i % FB]);
            if (last && i == 0) {
                // the next step's copies have landed and this step's last fragments are read: by every wavefront
                ODSD_WAIT_VMCNT_LGKM0((STAGES - 2) * C::L + C::LA);
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            }
#pragma unroll
            for (int r = 0; r < NR; ++r)
                if (r * NM / NR == i) read((j + 1) & 1, last ? next : cur, last ? 0 : j + 1, r);
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (c * NM / (NC ? NC : 1) == i) copy(step + STAGES, Place{left, cur.b}, last ? C::LA + c : c);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

#pragma unroll
    for (int s = 0; s < STAGES; ++s)
#pragma unroll
        for (int i = 0; i < C::L; ++i) copy(s, Place{(uint32_t)(s * C::A_BYTES), (uint32_t)(C::A_RING + s * C::B_BYTES)}, i);
    ODSD_WAIT_VMCNT_LGKM0((STAGES - 1) * C::L);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    Place cur = {0, C::A_RING};
    uint32_t left = C::A_RING - C::A_BYTES;                    // where w of the step before lay
#pragma unroll
    for (int r = 0; r < NR; ++r) read(0, cur, 0, r);
    for (int step = 0; step < steps; ++step) {
        const Place next = {cur.a + C::A_BYTES == C::A_RING ? 0u : cur.a + C::A_BYTES,
                            cur.b + C::B_BYTES == C::RING ? (uint32_t)C::A_RING : cur.b + C::B_BYTES};
        columns(std::integral_constant<int, 0>{}, step, cur, next, left);
        columns(std::integral_constant<int, 1>{}, step, cur, next, left);
        columns(std::integral_constant<int, 2>{}, step, cur, next, left);
        columns(std::integral_constant<int, 3>{}, step, cur, next, left);
        left = cur.a;
        cur = next;
    }
    ODSD_WAIT_VMCNT_LGKM0(0);                  // the copies past the end (zeros) have landed, too
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");

    // The sums leave through LDS (each wavefront its own part): a lane gets eight consecutive n of one token.  16-byte pieces
    // of a token's row are XORed with the token's number.
    constexpr int PIECES = C::CH * 8;          // of 4 sums, per token
    auto swz = [](int m) { return PIECES == 16 ? m & 15 : (m >> 1) & 7; };
    char *stage = lds + any_wave * C::OUT_WAVE;
#pragma unroll
    for (int a0 = 0; a0 < FA; a0 += C::CH) {
#pragma unroll
        for (int a = 0; a < C::CH; ++a)
#pragma unroll
            for (int c = 0; c < FB; ++c)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int m = c * 32 + (lane & 31), piece = a * 8 + q * 2 + (lane >> 5);
                    float4_t v;
#pragma unroll
                    for (int u = 0; u < 4; ++u) v[u] = acc[a0 + a][c][4 * q + u];
                    *(float4_t *)(stage + m * (PIECES * 16) + ((piece ^ swz(m)) << 4)) = v;
                }
        // several shares of K: each adds up its part of the tokens; one: a wavefront's own LDS accesses stay in order
        if (KS > 1) __syncthreads();
        else wave_lds_order();
        constexpr int LANES = PIECES / 2, ROUND = 64 / LANES;  // lanes that share a token's row, rows at a time
        const int pc = lane % LANES * 2, n = n0 + (wn * FA + a0) * 32 + pc * 4;
        auto rows = [&](auto leave) {
#pragma unroll 2                               // (all of them: the largest tile spills)
            for (int i = 0; i < (FB * 32 / ROUND + KS - 1) / KS; ++i) {
                const int r = (i * KS + part) * ROUND + lane / LANES;
                if (r >= FB * 32) return;
                float4_t lo = {0.0f, 0.0f, 0.0f, 0.0f}, hi = lo;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const char *from = KS > 1 ? lds + (s * C::NW + wave) * C::OUT_WAVE : stage;
                    const float4_t a = *(const float4_t *)(from + r * (PIECES * 16) + ((pc ^ swz(r)) << 4));
                    const float4_t b = *(const float4_t *)(from + r * (PIECES * 16) + (((pc + 1) ^ swz(r)) << 4));
                    lo = s ? lo + a : a;
                    hi = s ? hi + b : b;
                }
                float v[8];
                *(float4_t *)v = lo;
                *(float4_t *)(v + 4) = hi;
                leave(m0 + wm * FB * 32 + r, v);
            }
        };
        if (p.slices > 1) {
            rows([&](int m, const float *v) {
                if (m >= p.M || n >= p.N) return;
                float *to = p.part + ((int64_t)slice * p.M + m) * p.part_ld + n;
                *(float4_t *)to = *(const float4_t *)v;
                *(float4_t *)(to + 4) = *(const float4_t *)(v + 4);
            });
        } else {
            float bias[8];
            load_bias8<T>(p, n, bias);
            with_activation(p.act, [&](auto act) { rows([&](int m, const float *v) { finish8<T, O, decltype(act)::value>(p, m, n, v, bias); }); });
        }
        if (KS > 1 && FA > C::CH) __syncthreads();
        else wave_lds_order();
    }
}

// the slices' sums together, in their order, and the epilogue
template <typename T, typename O, int SLICES>
__global__ __launch_bounds__(256) void linear_join_kernel(LinearParams p) {
    const int per_row = (p.N + 7) / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int m = (int)(i / per_row), n = (int)(i - (int64_t)m * per_row) * 8;
    if (m >= p.M) return;
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    float4_t a[SLICES], b[SLICES];             // requested together: the kernel is one latency long
#pragma unroll
    for (int s = 0; s < SLICES; ++s) {
        const float *part = p.part + ((int64_t)min(s, p.slices - 1) * p.M + m) * p.part_ld + n;
        a[s] = *(const float4_t *)part;
        b[s] = *(const float4_t *)(part + 4);
    }
#pragma unroll
    for (int s = 0; s < SLICES; ++s) {
        if (s >= p.slices) break;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] += a[s][e];
            v[4 + e] += b[s][e];
        }
    }
    finish8<T, O>(p, m, n, v);
}

// ---- any shape, any alignment ----------------------------------------------------------------
// 64 x 64 tile, steps of 64 along K, operands through registers into LDS (rows padded by 16 bytes).
template <typename T, typename O>
__global__ __launch_bounds__(256) void linear_any_kernel(LinearParams p) {
    constexpr int LD = 72;
    __shared__ __attribute__((aligned(16))) T ws[64 * LD], xs[64 * LD];
    __shared__ __attribute__((aligned(16))) float ys[64 * 68];
    typedef typename AttnT<T>::V8 V8;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n0 = blockIdx.x * 64, m0 = blockIdx.y * 64;
    const int row = tid >> 3, col = (tid & 7) * 8;       // rows `row` and `row + 32`, 8 values from `col` on
    const T *w = (const T *)p.w, *x = (const T *)p.x;
    uint4_t rw[2], rx[2];
    // (rows past the last: products that nobody stores)
    const T *wr[2], *xr[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        wr[i] = w + (int64_t)min(n0 + row + 32 * i, p.N - 1) * p.ldw;
        xr[i] = x + (int64_t)min(m0 + row + 32 * i, p.M - 1) * p.ldx;
    }
    auto fetch = [&](int k) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            rw[i] = load8(wr[i], k + col, p.K);
            rx[i] = load8(xr[i], k + col, p.K);
        }
    };
    const int wn = (wave & 1) * 32, wm = (wave >> 1) * 32;
    float4_t acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) acc[a][b] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if (p.K >= 8) {
        fetch(0);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            rw[i] = load8_short(wr[i], col, p.K);
            rx[i] = load8_short(xr[i], col, p.K);
        }
    }
    for (int k = 0; k < p.K; k += 64) {
        __syncthreads();
        if (k + 64 > p.K && p.K >= 8) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                rw[i] = clip8(rw[i], k + col, p.K);
                rx[i] = clip8(rx[i], k + col, p.K);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            *(uint4_t *)(ws + (row + 32 * i) * LD + col) = rw[i];
            *(uint4_t *)(xs + (row + 32 * i) * LD + col) = rx[i];
        }
        __syncthreads();
        if (k + 64 < p.K) fetch(k + 64);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            V8 a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[i] = *(const V8 *)(ws + (wn + 16 * i + (lane & 15)) * LD + 32 * s + (lane >> 4) * 8);
                b[i] = *(const V8 *)(xs + (wm + 16 * i + (lane & 15)) * LD + 32 * s + (lane >> 4) * 8);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = AttnT<T>::mfma(a[i], b[j], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
            *(float4_t *)(ys + (wm + 16 * j + (lane & 15)) * 68 + wn + 16 * i + (lane >> 4) * 4) = acc[i][j];
    __syncthreads();
    for (int r = row; r < 64; r += 32) finish8<T, O>(p, m0 + r, n0 + col, ys + r * 68 + col);
}

// Rows of x and of w whose K is no multiple of 8, as rows that are one (zeros behind K): 16 bytes a thread.
template <typename T>
__global__ __launch_bounds__(256) void linear_pack_kernel(LinearParams p, T *x, T *w, int Kp) {
    const int per_row = Kp / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / per_row;
    const int k = (int)(i - row * per_row) * 8;
    if (row >= (int64_t)p.M + p.N) return;
    const T *src = row < p.M ? (const T *)p.x + row * p.ldx : (const T *)p.w + (row - p.M) * p.ldw;
    uint4_t v;
    if (k + 8 <= p.K) __builtin_memcpy(&v, src + k, 16);
    else v = load8_short(src, k, p.K);
    *(uint4_t *)((row < p.M ? x + row * Kp : w + (row - p.M) * Kp) + k) = v;
}

// ---- which kernel ------------------------------------------------------------------------------
// tiles n x m; K4, K2: K shared by groups of wavefronts of the workgroup
enum { LIN_ROWS = 0, LIN_ANY, LIN_TILE_32_64_K4, LIN_TILE_64_32_K2, LIN_TILE_64_64, LIN_TILE_64_64_K2, LIN_TILE_64_128_K2,
       LIN_TILE_128_128, LIN_TILE_128_192, LIN_TILE_128_256, LIN_TILE_256_192, LIN_TILE_256_256, LIN_KINDS };
static const int TILE_N[LIN_KINDS] = {16, 64, 32, 64, 64, 64, 64, 128, 128, 128, 256, 256};
static const int TILE_M[LIN_KINDS] = {16, 64, 64, 32, 64, 64, 128, 128, 192, 256, 192, 256};
static const int THREADS[LIN_KINDS] = {1024, 256, 512, 256, 256, 512, 512, 256, 256, 512, 512, 512};
static const int SHARES[LIN_KINDS] = {1, 1, 4, 2, 1, 2, 2, 1, 1, 1, 1, 1};     // of K in the workgroup
struct LinearPlan {
    int kind, slices, slice_k;
    int64_t part_ld;
    int Kp;            // not 0: x and w are packed into rows of this many columns first
    size_t bytes;      // of workspace
    bool fits;         // a launch has fewer than 2^32 threads
};
static int64_t linear_tiles(int kind, int M, int N) {
    return (int64_t)((uint32_t)(M + TILE_M[kind] - 1) / (uint32_t)TILE_M[kind]) * ((uint32_t)(N + TILE_N[kind] - 1) / (uint32_t)TILE_N[kind]);
}
static LinearPlan linear_plan_of(int kind, int slices, int M, int N, int K) {
    LinearPlan l;
    l.kind = kind;
    const int steps = (K + 63) / 64, per = (steps + slices - 1) / slices;
    l.slice_k = per * 64;
    l.slices = (steps + per - 1) / per;
    l.part_ld = ((int64_t)N + 7) / 8 * 8;
    l.Kp = 0;
    l.fits = (linear_tiles(kind, M, N) * l.slices + 7) * THREADS[kind] < 1LL << 32;
    l.bytes = l.slices > 1 ? (size_t)l.slices * M * l.part_ld * 4 : 0;
    return l;
}
static size_t linear_packed_bytes(int rows, int Kp) { return odsd_round_up((size_t)rows * Kp * 2, 256); }
// For operands whose rows are whole 16-byte segments; *us: about how long it takes.
static LinearPlan linear_plan_aligned(int M, int N, int K, float *us) {
    *us = 0.0f;
    // Few tokens and little work: one pass over the weights' rows, every token's columns read again for 16 of them.  us, rows /
    // the best tile: M = 1: K 4096, N 2048 6.9 / 9.4, K 2048, N 131072 83 / 95; M = 4: K 2048, N 5120 7.8 / 8.2; M = 16: K 1288,
    // N 2056 4.2 / 7.1, K 4096, N 2048 9.6 / 10.2, K 2048, N 5120 10.0 / 9.2, K 4096, N 12288 30 / 20.
    if (M <= 4 || (M <= 16 && (double)M * N * K <= 1.5e8)) return linear_plan_of(LIN_ROWS, 1, M, N, K);
    // Else the shape and the number of parts of K with the least estimated time.  A round of workgroups (256, one per CU; two of
    // 64 x 64, which is for single m tiles: the weights' bytes count there, and how many are on their way) takes a step's time
    // for every 64 columns of a share of K, and its epilogue.  The bytes are a second bound; what the shorter one adds is a root
    // of fourth powers.  Parts of K cost a launch and their sums' way through memory.  The constants are fitted to 913 shapes of
    // 5 to 8192 tokens (bf16, weights from memory), before the rule for weights read past the caches.
    // us of the shape taken / others, K 4096, N 4096: M = 200 (64 x 64, K shared by 2) 17.5 / 20 (64 x 128, 2 parts), 22 (128 x
    // 128, 4 parts); M = 512 (64 x 128) 28 / 31 (128 x 128, 2 parts), 39 (64 x 64); M = 1000 (128 x 128) 40 / 43 (128 x 192), 53
    // (64 x 128); M = 1536 (128 x 192) 52 / 56 (128 x 256), 73 (128 x 128); M = 4096 (256 x 256) 110 / 124 (128 x 256).  K 2048, N
    // 5120: M = 48 (32 x 64) 8.2 / 9.3 (64 x 64), M = 4096 (256 x 192) 85 / 95 (128 x 256), 102 (256 x 256).  K 2048, N 131072, M =
    // 64 (64 x 64) 118 / 130 (the same with K shared by 2).
    static const float STEP[LIN_KINDS] = {0, 0, 0.58f, 0.69f, 0.41f, 0.43f, 0.68f, 0.52f, 0.66f, 0.85f, 1.16f, 1.36f};
    static const float END[LIN_KINDS] = {0, 0, 3.3f, 2.3f, 4.4f, 3.9f, 3.6f, 5.7f, 8.9f, 5.6f, 8.2f, 9.4f};
    const int steps = (K + 63) / 64;
    const float bytes_us = ((float)M * K + (float)N * K + (float)M * N) * 2 / 7.4e6f + 6.7f, bytes2 = bytes_us * bytes_us;
    const float join_us = (float)M * N * 4 / 3.7e6f;           // of a part
    int kind = 0, parts = 1;
    for (int k = LIN_TILE_32_64_K4; k < LIN_KINDS; ++k) {
        if ((k == LIN_TILE_64_32_K2 && M > 32) || (k == LIN_TILE_64_64 && M > 64)) continue;
        const int64_t tiles = linear_tiles(k, M, N);
        for (int slices = 1; slices <= 8; slices *= 2) {
            if (slices > 1 && (tiles * slices > 640 || steps / slices < 4)) break;
            const float rounds = (float)(k == LIN_TILE_64_64 ? (tiles * slices + 511) / 512 : (tiles * slices + 255) / 256);
            const int per_share = ((steps + slices - 1) / slices + SHARES[k] - 1) / SHARES[k];
            const float t = rounds * (per_share * STEP[k] + END[k]);
            const float total = sqrtf(sqrtf(t * t * t * t + bytes2 * bytes2)) + (slices > 1 ? 3.1f + slices * join_us : 0.0f);
            if (*us == 0.0f || total < *us) {
                *us = total;
                kind = k;
                parts = slices;
            }
        }
    }
    return linear_plan_of(kind, parts, M, N, K);
}
static LinearPlan linear_plan(int M, int N, int K, bool aligned) {
    float us;
    if (aligned) return linear_plan_aligned(M, N, K, &us);
    if (M <= 16) return linear_plan_of(LIN_ROWS, 1, M, N, K);
    // Columns that are no whole number of segments: both operands are packed into such rows first, which costs their bytes
    // twice and a launch, where the tiles win more than that over the kernel for any shape (0.8 us a step and round of 512
    // workgroups).  us, that kernel / packed: K 3809: M = 20, N 5000 46 / 33, M = 453, N 768 42 / 25; K 2047: M = 65, N 65536
    // 127 / 172, M = 1000, N 5000 75 / 41; K 4095, M = 8192, N 4096 694 / 255.
    if (K % 8 != 0 && K < (1 << 21) - 8) {
        const int Kp = (K + 7) / 8 * 8;
        LinearPlan l = linear_plan_aligned(M, N, Kp, &us);
        const float pack = 4.0f + ((float)M + (float)N) * K * 4 / 4.5e6f;
        const float any = (float)((linear_tiles(LIN_ANY, M, N) + 511) / 512) * ((K + 63) / 64) * 0.8f;
        if (us + pack < any && l.fits && ((int64_t)M + N) * (Kp / 8) < (1LL << 32) - 256) {
            l.Kp = Kp;
            l.bytes = odsd_round_up(l.bytes, 256) + linear_packed_bytes(M, Kp) + linear_packed_bytes(N, Kp);
            return l;
        }
    }
    return linear_plan_of(LIN_ANY, 1, M, N, K);
}

// One pass over weights of more than a third of the 256 MB cache: nothing of them is there at the next call, so they do not
// displace what is (M = 64, K 2048, N 32768 33.9 -> 31.4 us, M = 33, K 4096, N 65536 107 -> 93, M = 180, K 2048, N 65536 82 ->
// 74).  Smaller ones, called again soon, come out of it (M = 64, K 2048, N 16384 15.0, past it 20.5; not called again 21.1 /
// 19.6), and so do the ends of rows that are no whole lines of 128 bytes (M = 96, K 3000, N 36000 89 / 92).
static bool linear_past_caches(int tile_m, int M, int N, int K, int64_t ldw) {
    return tile_m < 256 && M <= tile_m && (int64_t)N * K * 2 >= (96 << 20) && ldw % 64 == 0;
}

template <typename T, typename O, int NWN, int NWM, int FA, int FB, int STAGES, int KS = 1>
static void launch_tile(LinearParams &p, hipStream_t st) {
    typedef LinearTile<NWN, NWM, FA, FB, STAGES, KS> C;
    p.tiles_n = (p.N + C::TN - 1) / C::TN;
    p.tiles_m = (p.M + C::TM - 1) / C::TM;
    const int64_t total = (int64_t)p.tiles_n * p.tiles_m * p.slices;
    const unsigned grid = (unsigned)((total + 7) / 8 * 8), threads = C::NW * KS * 64;
    if constexpr (C::TM < 256) {
        if (linear_past_caches(C::TM, p.M, p.N, p.K, p.ldw)) {
            linear_tile_kernel<T, O, NWN, NWM, FA, FB, STAGES, KS, true><<<grid, threads, 0, st>>>(p);
            return;
        }
    }
    linear_tile_kernel<T, O, NWN, NWM, FA, FB, STAGES, KS, false><<<grid, threads, 0, st>>>(p);
}

template <typename T, typename O> static int launch_linear(LinearParams &p, const LinearPlan &l, void *workspace, hipStream_t st) {
    if (l.kind == LIN_ROWS) {
        // blocks of 64 columns that each of the 16 wavefronts has: requested together where there are more than two
        const unsigned grid = (unsigned)((p.N + 15) / 16);
        if (p.K > 2048) linear_rows_kernel<T, O, 16, 4><<<grid, 1024, 0, st>>>(p);
        else linear_rows_kernel<T, O, 16, 2><<<grid, 1024, 0, st>>>(p);
        ODSD_CHECK_LAUNCH();
        return ODSD_OK;
    }
    if (l.kind == LIN_ANY) {
        linear_any_kernel<T, O><<<dim3((unsigned)((p.N + 63) / 64), (unsigned)((p.M + 63) / 64)), 256, 0, st>>>(p);
        ODSD_CHECK_LAUNCH();
        return ODSD_OK;
    }
    if (l.Kp) {
        const size_t parts = odsd_round_up(l.slices > 1 ? (size_t)l.slices * p.M * l.part_ld * 4 : 0, 256);
        T *x = (T *)((char *)workspace + parts), *w = (T *)((char *)x + linear_packed_bytes(p.M, l.Kp));
        const int64_t units = ((int64_t)p.M + p.N) * (l.Kp / 8);
        linear_pack_kernel<T><<<(unsigned)((units + 255) / 256), 256, 0, st>>>(p, x, w, l.Kp);
        p.x = x;
        p.w = w;
        p.ldx = p.ldw = p.K = l.Kp;
    }
    p.slices = l.slices;
    p.slice_k = l.slice_k;
    p.part = (float *)workspace;
    p.part_ld = l.part_ld;
    switch (l.kind) {
        case LIN_TILE_32_64_K4: launch_tile<T, O, 1, 2, 1, 1, 3, 4>(p, st); break;
        case LIN_TILE_64_32_K2: launch_tile<T, O, 2, 1, 1, 1, 4, 2>(p, st); break;
        case LIN_TILE_64_64: launch_tile<T, O, 2, 2, 1, 1, 4>(p, st); break;
        case LIN_TILE_64_64_K2: launch_tile<T, O, 2, 2, 1, 1, 3, 2>(p, st); break;
        case LIN_TILE_64_128_K2: launch_tile<T, O, 1, 4, 2, 1, 3, 2>(p, st); break;
        case LIN_TILE_128_128: launch_tile<T, O, 2, 2, 2, 2, 4>(p, st); break;
        case LIN_TILE_128_192: launch_tile<T, O, 2, 2, 2, 3, 3>(p, st); break;
        case LIN_TILE_128_256: launch_tile<T, O, 2, 4, 2, 2, 3>(p, st); break;
        case LIN_TILE_256_192: launch_tile<T, O, 4, 2, 2, 3, 2>(p, st); break;
        default: launch_tile<T, O, 2, 4, 4, 2, 2>(p, st); break;
    }
    if (p.slices > 1) {
        const int64_t units = (int64_t)p.M * ((p.N + 7) / 8);
        const unsigned grid = (unsigned)((units + 255) / 256);
        if (p.slices <= 2) linear_join_kernel<T, O, 2><<<grid, 256, 0, st>>>(p);
        else if (p.slices <= 4) linear_join_kernel<T, O, 4><<<grid, 256, 0, st>>>(p);
        else linear_join_kernel<T, O, 8><<<grid, 256, 0, st>>>(p);
    }
    ODSD_CHECK_LAUNCH();
    return ODSD_OK;
}

// the grid's second dimension and the 32-bit products inside the kernels
static bool linear_sizes_supported(int M, int N, int K) { return M <= 64 * 65535 && N <= 0x7fffffff - 256 && K <= 0x7fffffff - 256; }

extern "C" size_t odsd_linear_workspace_bytes(int32_t M, int32_t N, int32_t K) {
    if (M < 0 || N <= 0 || K <= 0 || !linear_sizes_supported(M, N, K)) return 0;
    const LinearPlan l = linear_plan(M, N, K, K % 8 == 0);      // (pointers that are not aligned need no more)
    return !l.fits ? 0 : l.bytes > 256 ? l.bytes : 256;
}

// rows of whole 16-byte segments, and a tile's rows within 31 bits of bytes
static bool linear_rows_aligned(int K, int64_t ldx, int64_t ldw) { return ((K | ldx | ldw) & 7) == 0 && ldx < (1 << 21) && ldw < (1 << 21); }

extern "C" int odsd_linear_plan(int32_t M, int32_t N, int32_t K, int64_t ldx, int64_t ldw, int32_t aligned, int32_t *plan) {
    if (!plan) return ODSD_ERR_NULL;
    if (M <= 0 || N <= 0 || K <= 0 || ldx < K || ldw < K) return ODSD_ERR_SHAPE;
    if (!linear_sizes_supported(M, N, K)) return ODSD_ERR_UNSUPPORTED;
    const LinearPlan l = linear_plan(M, N, K, aligned && linear_rows_aligned(K, ldx, ldw));
    if (!l.fits) return ODSD_ERR_UNSUPPORTED;
    const bool tiles = l.kind > LIN_ANY;
    plan[0] = tiles ? 2 : l.kind;
    plan[1] = TILE_N[l.kind];
    plan[2] = TILE_M[l.kind];
    plan[3] = SHARES[l.kind];
    plan[4] = l.slices;
    plan[5] = l.Kp;
    plan[6] = tiles && linear_past_caches(TILE_M[l.kind], M, N, l.Kp ? l.Kp : K, l.Kp ? l.Kp : ldw);
    return ODSD_OK;
}

extern "C" int odsd_linear(const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias, const void *residual,
                           int64_t ldr, void *out, int64_t ldo, int32_t M, int32_t N, int32_t K, int32_t dtype,
                           int32_t out_dtype, int32_t act, void *workspace, size_t workspace_bytes, void *stream) {
    if (M < 0 || N <= 0 || K <= 0 || ldx < K || ldw < K || ldo < N || (residual && ldr < N)) return ODSD_ERR_SHAPE;
    if (dtype != ODSD_DT_BF16 && dtype != ODSD_DT_F16) return ODSD_ERR_DTYPE;
    if (out_dtype != dtype && out_dtype != ODSD_DT_F32) return ODSD_ERR_DTYPE;
    if (act < ODSD_ACT_NONE || act > ODSD_ACT_GELU_TANH) return ODSD_ERR_UNSUPPORTED;
    if (!linear_sizes_supported(M, N, K)) return ODSD_ERR_UNSUPPORTED;
    if (M == 0) return ODSD_OK;
    if (!x || !w || !out) return ODSD_ERR_NULL;
    const uintptr_t oe = out_dtype == ODSD_DT_F32 ? 4 : 2;
    if ((((uintptr_t)x | (uintptr_t)w | (uintptr_t)bias) & 1) || (((uintptr_t)out | (uintptr_t)residual) & (oe - 1)) ||
        !odsd_aligned16(workspace)) return ODSD_ERR_ALIGN;
    LinearParams p{x, w, bias, residual, out, ldx, ldw, ldr, ldo, M, N, K, act, 0, 0, 1, 0, nullptr, 0};
    const bool aligned = odsd_aligned16(x) && odsd_aligned16(w) && linear_rows_aligned(K, ldx, ldw);
    const LinearPlan l = linear_plan(M, N, K, aligned);
    if (!l.fits) return ODSD_ERR_UNSUPPORTED;
    if (l.bytes && !workspace) return ODSD_ERR_NULL;
    if (workspace_bytes < l.bytes) return ODSD_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ODSD_DT_BF16)
        return out_dtype == ODSD_DT_F32 ? launch_linear<__bf16, float>(p, l, workspace, st) : launch_linear<__bf16, __bf16>(p, l, workspace, st);
    return out_dtype == ODSD_DT_F32 ? launch_linear<half_t, float>(p, l, workspace, st) : launch_linear<half_t, half_t>(p, l, workspace, st);
}
