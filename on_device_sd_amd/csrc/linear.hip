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
template <typename T, typename O, int ACT>
__device__ __forceinline__ void finish8(const LinearParams &p, int m, int n, const float *v) {
    if (m >= p.M || n >= p.N) return;
    const T *bias = p.bias ? (const T *)p.bias + n : nullptr;
    const O *res = p.res ? (const O *)p.res + (int64_t)m * p.ldr + n : nullptr;
    O *out = (O *)p.out + (int64_t)m * p.ldo + n;
    constexpr bool PRECISE = sizeof(O) == 4;
    if (n + 8 <= p.N) {
        typename Vec8<T>::type b;
        typename Vec8<O>::type r, y;
        if (bias) __builtin_memcpy(&b, bias, sizeof b);
        if (res) __builtin_memcpy(&r, res, sizeof r);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = activate<PRECISE, ACT>(bias ? v[i] + (float)b[i] : v[i]);
            y[i] = (O)(res ? a + (float)r[i] : a);
        }
        __builtin_memcpy(out, &y, sizeof y);
        return;
    }
    for (int i = 0; i < 8 && n + i < p.N; ++i) {
        const float a = activate<PRECISE, ACT>(bias ? v[i] + (float)bias[i] : v[i]);
        out[i] = (O)(res ? a + (float)res[i] : a);
    }
}
template <typename T, typename O>
__device__ __forceinline__ void finish8(const LinearParams &p, int m, int n, const float *v) {
    switch (p.act) {
        case ODSD_ACT_RELU: return finish8<T, O, ODSD_ACT_RELU>(p, m, n, v);
        case ODSD_ACT_SILU: return finish8<T, O, ODSD_ACT_SILU>(p, m, n, v);
        case ODSD_ACT_GELU: return finish8<T, O, ODSD_ACT_GELU>(p, m, n, v);
        case ODSD_ACT_GELU_TANH: return finish8<T, O, ODSD_ACT_GELU_TANH>(p, m, n, v);
        default: return finish8<T, O, ODSD_ACT_NONE>(p, m, n, v);
    }
}

// ---- tiles -----------------------------------------------------------------------------------
// NWN x NWM wavefronts, each FA blocks of 32 n by FB blocks of 32 m on v_mfma_f32_32x32x16; steps of 64 along K.  Both
// operands go to LDS without passing registers (buffer_load ... lds, 16 bytes a lane), STAGES buffers of them; a buffer's
// rows are 128 bytes, whose 16-byte segments are XORed with the row's number, so that the fragment reads (eight lanes, eight
// rows, one segment) meet eight different bank groups.  What is behind a row's end, the matrix's last row or the slice's
// last step is addressed outside the buffer descriptor and arrives as zeros, without memory traffic, so every copy is
// issued whatever follows and a count says which have landed.
template <typename T, typename O, int NWN, int NWM, int FA, int FB, int STAGES>
struct LinearTile {
    static constexpr int NW = NWN * NWM, TN = NWN * FA * 32, TM = NWM * FB * 32;
    static constexpr int A_BYTES = TN * 128, STAGE = (TN + TM) * 128;
    static constexpr int LA = TN / 8 / NW, LB = TM / 8 / NW, L = LA + LB;   // copies of a wavefront per step: 8 rows each
    static constexpr int CH = FA < 2 ? FA : 2;                             // blocks of n that leave together
    static constexpr int OUT_WAVE = FB * 32 * CH * 32 * 4;
    static constexpr int LDS = STAGE * STAGES > NW * OUT_WAVE ? STAGE * STAGES : NW * OUT_WAVE;
    static_assert(LA * 8 * NW == TN && LB * 8 * NW == TM && LB >= 1, "every wavefront copies whole groups of 8 rows");
};

__device__ __forceinline__ void copy16_to_lds(uint4_t rsrc, uint32_t off, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
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

template <typename T, typename O, int NWN, int NWM, int FA, int FB, int STAGES>
__global__ __launch_bounds__(NWN * NWM * 64) void linear_tile_kernel(LinearParams p) {
    typedef LinearTile<T, O, NWN, NWM, FA, FB, STAGES> C;
    typedef typename AttnT<T>::V8 V8;
    __shared__ __attribute__((aligned(1024))) char lds[C::LDS];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // neighbouring tiles on one XCD (workgroup i is on XCD i % 8), in groups of up to 8 along m that share their weights
    const int total = p.tiles_n * p.tiles_m * p.slices, per = (total + 7) / 8;
    const int b = blockIdx.x, t0 = (b & 7) * per + (b >> 3);
    if ((b >> 3) >= per || t0 >= total) return;
    const int slice = t0 / (p.tiles_n * p.tiles_m), t = t0 - slice * (p.tiles_n * p.tiles_m);
    const int group = t / (8 * p.tiles_n), in_group = t - group * 8 * p.tiles_n;
    const int gm = min(8, p.tiles_m - group * 8);
    const int n0 = in_group / gm * C::TN, m0 = (group * 8 + in_group % gm) * C::TM;

    const int k_begin = slice * p.slice_k, k_end = min(p.K, k_begin + p.slice_k);
    const int steps = (k_end - k_begin + 63) / 64;
    const uint32_t ldw = (uint32_t)p.ldw * 2u, ldx = (uint32_t)p.ldx * 2u;
    const uint4_t rw = descriptor((const char *)p.w + (int64_t)n0 * p.ldw * 2, (uint32_t)(min(C::TN, p.N - n0) - 1) * ldw + p.K * 2);
    const uint4_t rx = descriptor((const char *)p.x + (int64_t)m0 * p.ldx * 2, (uint32_t)(min(C::TM, p.M - m0) - 1) * ldx + p.K * 2);
    const int seg = (lane & 7) ^ (lane >> 3);
    const uint32_t row0 = wave * 8 + (lane >> 3);
    const uint32_t off_w = row0 * ldw + seg * 16, off_x = row0 * ldx + seg * 16;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void *)lds;
    auto copy_step = [&](int step, uint32_t buf) {
        const int k = k_begin + step * 64;
        const uint32_t ko = k + seg * 8 < k_end ? (uint32_t)k * 2u : 0x80000000u;
#pragma unroll
        for (int i = 0; i < C::LA; ++i) copy16_to_lds(rw, off_w + ko + i * (C::NW * 8) * ldw, lds0 + buf + (i * C::NW + wave) * 1024);
#pragma unroll
        for (int i = 0; i < C::LB; ++i) copy16_to_lds(rx, off_x + ko + i * (C::NW * 8) * ldx, lds0 + buf + C::A_BYTES + (i * C::NW + wave) * 1024);
    };

    const int wn = wave % NWN, wm = wave / NWN;
    const uint32_t frag = (lane & 31) * 128 + (((lane >> 5) ^ (lane & 7)) << 4);
    const uint32_t fa0 = wn * FA * 4096 + frag, fb0 = C::A_BYTES + wm * FB * 4096 + frag;
    float16_t acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    V8 fa[2][FA], fb[2][FB];
    auto read = [&](int par, uint32_t buf, int j) {
#pragma unroll
        for (int i = 0; i < FB; ++i) fb[par][i] = *(const V8 *)(lds + ((buf + fb0) ^ (j << 5)) + i * 4096);
#pragma unroll
        for (int i = 0; i < FA; ++i) fa[par][i] = *(const V8 *)(lds + ((buf + fa0) ^ (j << 5)) + i * 4096);
    };

    for (int s = 0; s < STAGES; ++s) copy_step(s, s * C::STAGE);
    ODSD_WAIT_VMCNT_LGKM0((STAGES - 1) * C::L);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    uint32_t cur = 0;
    read(0, cur, 0);
    for (int step = 0; step < steps; ++step) {
        uint32_t next = cur + C::STAGE;
        if (next == C::STAGE * STAGES) next = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j == 3) {
                // the next step's copies have landed and this step's last fragments are read: by every wavefront
                __builtin_amdgcn_sched_barrier(0);
                ODSD_WAIT_VMCNT_LGKM0((STAGES - 2) * C::L);
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                read(0, next, 0);
                copy_step(step + STAGES, cur);
            } else {
                read((j + 1) & 1, cur, j + 1);
            }
#pragma unroll
            for (int a = 0; a < FA; ++a)
#pragma unroll
                for (int c = 0; c < FB; ++c) acc[a][c] = AttnT<T>::mfma32(fa[j & 1][a], fb[j & 1][c], acc[a][c]);
        }
        cur = next;
    }
    ODSD_WAIT_VMCNT_LGKM0(0);                  // the copies past the end (zeros) have landed, too
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");

    // The sums leave through LDS (each wavefront its own part): a lane gets eight consecutive n of one token.  16-byte pieces
    // of a token's row are XORed with the token's number.
    constexpr int PIECES = C::CH * 8;          // of 4 sums, per token
    char *stage = lds + wave * C::OUT_WAVE;
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
                    *(float4_t *)(stage + m * (PIECES * 16) + ((piece ^ (m & (PIECES - 1))) << 4)) = v;
                }
        // (a wavefront's own LDS accesses stay in order)
        constexpr int LANES = PIECES / 2;      // lanes that share a token's row
        for (int r = lane / LANES; r < FB * 32; r += 64 / LANES) {
            const int pc = lane % LANES * 2;
            float v[8];
            *(float4_t *)v = *(const float4_t *)(stage + r * (PIECES * 16) + ((pc ^ (r & (PIECES - 1))) << 4));
            *(float4_t *)(v + 4) = *(const float4_t *)(stage + r * (PIECES * 16) + (((pc + 1) ^ (r & (PIECES - 1))) << 4));
            const int m = m0 + wm * FB * 32 + r, n = n0 + (wn * FA + a0) * 32 + pc * 4;
            if (p.slices > 1) {
                if (m < p.M && n < p.N) {
                    float *part = p.part + ((int64_t)slice * p.M + m) * p.part_ld + n;
                    *(float4_t *)part = *(float4_t *)v;
                    *(float4_t *)(part + 4) = *(float4_t *)(v + 4);
                }
            } else {
                finish8<T, O>(p, m, n, v);
            }
        }
        asm volatile("" ::: "memory");
    }
}

// the slices' sums together, in their order, and the epilogue
template <typename T, typename O>
__global__ __launch_bounds__(256) void linear_join_kernel(LinearParams p) {
    const int per_row = (p.N + 7) / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int m = (int)(i / per_row), n = (int)(i - (int64_t)m * per_row) * 8;
    if (m >= p.M) return;
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < p.slices; ++s) {
        const float *part = p.part + ((int64_t)s * p.M + m) * p.part_ld + n;
        const float4_t a = *(const float4_t *)part, b = *(const float4_t *)(part + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] += a[e];
            v[4 + e] += b[e];
        }
    }
    finish8<T, O>(p, m, n, v);
}

// ---- any shape, any alignment ----------------------------------------------------------------
// 64 x 64 tile, steps of 64 along K, operands through registers into LDS (rows padded by 16 bytes).  Eight values of a row
// that lie in K whole are one 16-byte load at the elements' own alignment; the row's end comes element by element.
template <typename T>
__device__ __forceinline__ uint4_t load8_any(const T *row, int k, int K, bool row_ok) {
    uint4_t v = {0, 0, 0, 0};
    if (!row_ok) return v;
    if (k + 8 <= K) {
        __builtin_memcpy(&v, row + k, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint16_t e = 0;
            if (k + i < K) __builtin_memcpy(&e, row + k + i, 2);
            v[i >> 1] |= (uint32_t)e << (16 * (i & 1));
        }
    }
    return v;
}

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
    auto fetch = [&](int k) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int n = n0 + row + 32 * i, m = m0 + row + 32 * i;
            rw[i] = load8_any(w + (int64_t)min(n, p.N - 1) * p.ldw, k + col, p.K, n < p.N);
            rx[i] = load8_any(x + (int64_t)min(m, p.M - 1) * p.ldx, k + col, p.K, m < p.M);
        }
    };
    const int wn = (wave & 1) * 32, wm = (wave >> 1) * 32;
    float4_t acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) acc[a][b] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    fetch(0);
    for (int k = 0; k < p.K; k += 64) {
        __syncthreads();
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

// ---- which kernel ------------------------------------------------------------------------------
struct LinearPlan {
    int tile;          // index of the tile shape below, -1: the kernel for any shape
    int slices, slice_k;
    int64_t part_ld;
    size_t bytes;      // of workspace
    bool fits;         // the launch's workgroups are counted in 31 bits
};
static const int TILE_N[] = {128, 128, 128, 256}, TILE_M[] = {32, 64, 128, 256};

static LinearPlan linear_plan(int M, int N, int K) {
    LinearPlan l;
    l.tile = M <= 32 ? 0 : M <= 64 ? 1 : (int64_t)((M + 255) / 256) * ((N + 255) / 256) >= 192 ? 3 : 2;
    const int64_t tiles = (int64_t)((M + TILE_M[l.tile] - 1) / TILE_M[l.tile]) * ((N + TILE_N[l.tile] - 1) / TILE_N[l.tile]);
    const int steps = (K + 63) / 64;
    int slices = 1;
    while (slices < 16 && tiles * slices * 2 <= 512 && steps / (slices * 2) >= 4) slices *= 2;
    const int per = (steps + slices - 1) / slices;
    l.slice_k = per * 64;
    l.slices = (steps + per - 1) / per;
    l.part_ld = ((int64_t)N + 7) / 8 * 8;
    l.fits = tiles * l.slices <= 0x7ffffff0LL;
    l.bytes = l.slices > 1 ? (size_t)l.slices * M * l.part_ld * 4 : 0;
    return l;
}

template <typename T, typename O, int NWN, int NWM, int FA, int FB, int STAGES>
static void launch_tile(LinearParams &p, hipStream_t st) {
    typedef LinearTile<T, O, NWN, NWM, FA, FB, STAGES> C;
    p.tiles_n = (p.N + C::TN - 1) / C::TN;
    p.tiles_m = (p.M + C::TM - 1) / C::TM;
    const int64_t total = (int64_t)p.tiles_n * p.tiles_m * p.slices;
    linear_tile_kernel<T, O, NWN, NWM, FA, FB, STAGES><<<(unsigned)((total + 7) / 8 * 8), C::NW * 64, 0, st>>>(p);
}

template <typename T, typename O> static int launch_linear(LinearParams &p, const LinearPlan &l, void *workspace, hipStream_t st) {
    // rows of whole 16-byte segments, and a tile's rows within 31 bits of bytes
    const bool aligned = ((p.K | p.ldx | p.ldw) & 7) == 0 && odsd_aligned16(p.x) && odsd_aligned16(p.w) &&
                         p.ldx < (1 << 21) && p.ldw < (1 << 21);
    if (!aligned) {
        linear_any_kernel<T, O><<<dim3((unsigned)((p.N + 63) / 64), (unsigned)((p.M + 63) / 64)), 256, 0, st>>>(p);
        ODSD_CHECK_LAUNCH();
        return ODSD_OK;
    }
    p.slices = l.slices;
    p.slice_k = l.slice_k;
    p.part = (float *)workspace;
    p.part_ld = l.part_ld;
    switch (l.tile) {
        case 0: launch_tile<T, O, 4, 1, 1, 1, 4>(p, st); break;
        case 1: launch_tile<T, O, 4, 1, 1, 2, 3>(p, st); break;
        case 2: launch_tile<T, O, 2, 2, 2, 2, 2>(p, st); break;
        default: launch_tile<T, O, 2, 4, 4, 2, 2>(p, st); break;
    }
    if (p.slices > 1) {
        const int64_t units = (int64_t)p.M * ((p.N + 7) / 8);
        linear_join_kernel<T, O><<<(unsigned)((units + 255) / 256), 256, 0, st>>>(p);
    }
    ODSD_CHECK_LAUNCH();
    return ODSD_OK;
}

extern "C" size_t odsd_linear_workspace_bytes(int32_t M, int32_t N, int32_t K) {
    if (M < 0 || N <= 0 || K <= 0) return 0;
    const LinearPlan l = linear_plan(M, N, K);
    return !l.fits ? 0 : l.bytes > 256 ? l.bytes : 256;
}

extern "C" int odsd_linear(const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias, const void *residual,
                           int64_t ldr, void *out, int64_t ldo, int32_t M, int32_t N, int32_t K, int32_t dtype,
                           int32_t out_dtype, int32_t act, void *workspace, size_t workspace_bytes, void *stream) {
    if (M < 0 || N <= 0 || K <= 0 || ldx < K || ldw < K || ldo < N || (residual && ldr < N)) return ODSD_ERR_SHAPE;
    if (dtype != ODSD_DT_BF16 && dtype != ODSD_DT_F16) return ODSD_ERR_DTYPE;
    if (out_dtype != dtype && out_dtype != ODSD_DT_F32) return ODSD_ERR_DTYPE;
    if (act < ODSD_ACT_NONE || act > ODSD_ACT_GELU_TANH) return ODSD_ERR_UNSUPPORTED;
    // the grid's second dimension and the 32-bit products inside the kernels
    if (M > 64 * 65535 || N > 0x7fffffff - 256 || K > 0x7fffffff - 256) return ODSD_ERR_UNSUPPORTED;
    if (M == 0) return ODSD_OK;
    if (odsd_linear_workspace_bytes(M, N, K) == 0) return ODSD_ERR_UNSUPPORTED;
    if (!x || !w || !out || !workspace) return ODSD_ERR_NULL;
    const uintptr_t oe = out_dtype == ODSD_DT_F32 ? 4 : 2;
    if ((((uintptr_t)x | (uintptr_t)w | (uintptr_t)bias) & 1) || (((uintptr_t)out | (uintptr_t)residual) & (oe - 1)) ||
        !odsd_aligned16(workspace)) return ODSD_ERR_ALIGN;
    if (workspace_bytes < odsd_linear_workspace_bytes(M, N, K)) return ODSD_ERR_WORKSPACE;
    LinearParams p{x, w, bias, residual, out, ldx, ldw, ldr, ldo, M, N, K, act, 0, 0, 1, 0, nullptr, 0};
    const LinearPlan l = linear_plan(M, N, K);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ODSD_DT_BF16)
        return out_dtype == ODSD_DT_F32 ? launch_linear<__bf16, float>(p, l, workspace, st) : launch_linear<__bf16, __bf16>(p, l, workspace, st);
    return out_dtype == ODSD_DT_F32 ? launch_linear<half_t, float>(p, l, workspace, st) : launch_linear<half_t, half_t>(p, l, workspace, st);
}
