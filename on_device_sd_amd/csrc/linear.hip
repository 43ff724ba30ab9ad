// Matrix product with bias, activation and residual in its epilogue:
//   y[m][n] = act(sum_k x[m][k] w[n][k] + bias[n]) + residual[m][n]
// the projections around the attention of a layer and the language-model head behind the last one.  Sums in fp32 (the
// matrix cores' accumulators), bias, activation and residual in fp32, one rounding to the output's type.
//
// Every kernel gives the weights as the A operand of the matrix instruction and the tokens as B, so that a lane's
// accumulators are four consecutive n of one token.
#include "attn.h"

struct LinearParams {
    const void *x, *w, *bias, *res;
    void *out;
    int64_t ldx, ldw, ldr, ldo;    // elements between two rows
    int M, N, K, act;
    int vec_out;                   // four consecutive n of out (and of the residual) are one aligned access
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

template <typename O> struct OutIO;
template <> struct OutIO<float> {
    __device__ static __forceinline__ float load(const float *p) { return *p; }
    __device__ static __forceinline__ void store(float *p, float v) { *p = v; }
    __device__ static __forceinline__ float4_t load4(const float *p) { return *(const float4_t *)p; }
    __device__ static __forceinline__ void store4(float *p, float4_t v) { *(float4_t *)p = v; }
};
template <typename T> struct OutIO16 {
    __device__ static __forceinline__ float load(const T *p) { return (float)*p; }
    __device__ static __forceinline__ void store(T *p, float v) { *p = (T)v; }
    typedef T T4 __attribute__((ext_vector_type(4)));
    __device__ static __forceinline__ float4_t load4(const T *p) { return __builtin_convertvector(*(const T4 *)p, float4_t); }
    __device__ static __forceinline__ void store4(T *p, float4_t v) { *(T4 *)p = __builtin_convertvector(v, T4); }
};
template <> struct OutIO<half_t> : OutIO16<half_t> {};
template <> struct OutIO<__bf16> : OutIO16<__bf16> {};

// y[m][n .. n + 3] from their sums
template <typename T, typename O, int ACT>
__device__ __forceinline__ void finish4(const LinearParams &p, int m, int n, float4_t v) {
    if (m >= p.M || n >= p.N) return;
    const T *bias = (const T *)p.bias;
    const O *res = p.res ? (const O *)p.res + (int64_t)m * p.ldr + n : nullptr;
    O *out = (O *)p.out + (int64_t)m * p.ldo + n;
    constexpr bool PRECISE = sizeof(O) == 4;
    if (p.vec_out && n + 4 <= p.N) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = activate<PRECISE, ACT>(bias ? v[i] + (float)bias[n + i] : v[i]);
        if (res) v += OutIO<O>::load4(res);
        OutIO<O>::store4(out, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (n + i >= p.N) return;
        float y = activate<PRECISE, ACT>(bias ? v[i] + (float)bias[n + i] : v[i]);
        if (res) y += OutIO<O>::load(res + i);
        OutIO<O>::store(out + i, y);
    }
}
template <typename T, typename O>
__device__ __forceinline__ void finish4(const LinearParams &p, int m, int n, float4_t v) {
    switch (p.act) {
        case ODSD_ACT_RELU: return finish4<T, O, ODSD_ACT_RELU>(p, m, n, v);
        case ODSD_ACT_SILU: return finish4<T, O, ODSD_ACT_SILU>(p, m, n, v);
        case ODSD_ACT_GELU: return finish4<T, O, ODSD_ACT_GELU>(p, m, n, v);
        case ODSD_ACT_GELU_TANH: return finish4<T, O, ODSD_ACT_GELU_TANH>(p, m, n, v);
        default: return finish4<T, O, ODSD_ACT_NONE>(p, m, n, v);
    }
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
            finish4<T, O>(p, m0 + wm + 16 * j + (lane & 15), n0 + wn + 16 * i + (lane >> 4) * 4, acc[i][j]);
}

template <typename T, typename O> static int launch_linear(const LinearParams &p, hipStream_t st) {
    const dim3 grid((unsigned)((p.N + 63) / 64), (unsigned)((p.M + 63) / 64));
    linear_any_kernel<T, O><<<grid, 256, 0, st>>>(p);
    ODSD_CHECK_LAUNCH();
    return ODSD_OK;
}

extern "C" size_t odsd_linear_workspace_bytes(int32_t M, int32_t N, int32_t K) {
    if (M < 0 || N <= 0 || K <= 0) return 0;
    return 256;
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
    if (!x || !w || !out || !workspace) return ODSD_ERR_NULL;
    const uintptr_t oe = out_dtype == ODSD_DT_F32 ? 4 : 2;
    if ((((uintptr_t)x | (uintptr_t)w | (uintptr_t)bias) & 1) || (((uintptr_t)out | (uintptr_t)residual) & (oe - 1)) ||
        !odsd_aligned16(workspace)) return ODSD_ERR_ALIGN;
    if (workspace_bytes < odsd_linear_workspace_bytes(M, N, K)) return ODSD_ERR_WORKSPACE;
    LinearParams p{x, w, bias, residual, out, ldx, ldw, ldr, ldo, M, N, K, act, 0};
    const uintptr_t at4 = (uintptr_t)out | (residual ? (uintptr_t)residual : 0) | (uintptr_t)(ldo * oe) |
                          (residual ? (uintptr_t)(ldr * oe) : 0);
    p.vec_out = (at4 & (4 * oe - 1)) == 0;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ODSD_DT_BF16)
        return out_dtype == ODSD_DT_F32 ? launch_linear<__bf16, float>(p, st) : launch_linear<__bf16, __bf16>(p, st);
    return out_dtype == ODSD_DT_F32 ? launch_linear<half_t, float>(p, st) : launch_linear<half_t, half_t>(p, st);
}
