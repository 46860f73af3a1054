// A linear layer with its epilogue, forward and backward:
//
//   z = x W^T + bias,  y = act(z) + residual               x: M x K, W: N x K
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz,  dresidual = dy
//
// Products run on the matrix cores with 32-bit sums. Each result is rounded to its type
// once, from 32 bits. What the backward pass needs of z is kept in 16 bits for the 16-bit
// types, in float16 whatever the type is: its 11 bits keep act'(z) four times nearer than
// bfloat16's 8 would, and act' has its limit long before float16 ends, so larger values
// are kept as its largest.

#include "layers.h"

using namespace drh_rt;

namespace drh_nn {
namespace {

// ---------------------------------------------------------------- activations

// erf for values that are rounded to 16 bits afterwards: Abramowitz and Stegun 7.1.26,
// within 1.5e-7. Results in 32 bits take the library's.
template <bool EXACT>
__device__ inline float erf_of(float x) {
    if constexpr (EXACT) return erff(x);
    const float a = fabsf(x), t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, a, 1.0f));
    float s = fmaf(t, 1.061405429f, -1.453152027f);
    s = fmaf(t, s, 1.421413741f);
    s = fmaf(t, s, -0.284496736f);
    s = fmaf(t, s, 0.254829592f) * t;
    return copysignf(1.0f - s * __expf(-a * a), x);
}

constexpr float SQRT_HALF = 0.70710678118654752f, INV_SQRT_2PI = 0.39894228040143268f;
constexpr float TANH_C = 0.79788456080286536f, TANH_A = 0.044715f;

// 1 / (1 + exp(-v))
template <bool EXACT>
__device__ inline float logistic(float v) {
    return EXACT ? 1.0f / (1.0f + expf(-v)) : __builtin_amdgcn_rcpf(1.0f + __expf(-v));
}

// Far below zero every smooth activation is zero in 32 bits; the bound keeps infinity
// times zero out of the product there. NaN passes.
__device__ inline float not_below(float z, float lo) { return z < lo ? lo : z; }
__device__ inline float not_above(float z, float hi) { return z > hi ? hi : z; }

template <bool EXACT>
__device__ inline float act(int kind, float z) {
    switch (kind) {
        case DRH_ACT_RELU: return z < 0.0f ? 0.0f : z;
        case DRH_ACT_SILU: z = not_below(z, -200.0f); return z * logistic<EXACT>(z);
        case DRH_ACT_GELU: z = not_below(z, -64.0f); return 0.5f * z * (1.0f + erf_of<EXACT>(z * SQRT_HALF));
        case DRH_ACT_GELU_TANH: {
            z = not_below(z, -64.0f);
            const float c = not_above(z, 64.0f);  // (1 + tanh u) / 2 = logistic(2 u)
            return z * logistic<EXACT>(2.0f * TANH_C * fmaf(TANH_A * c * c, c, c));
        }
        default: return z;
    }
}

template <bool EXACT>
__device__ inline float act_slope(int kind, float z) {
    if (kind == DRH_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if (kind == DRH_ACT_NONE) return 1.0f;
    z = not_above(not_below(z, -64.0f), 64.0f);
    if (kind == DRH_ACT_SILU) {
        const float s = logistic<EXACT>(z);
        return s * (1.0f + z * (1.0f - s));
    }
    if (kind == DRH_ACT_GELU)
        return 0.5f * (1.0f + erf_of<EXACT>(z * SQRT_HALF)) + z * INV_SQRT_2PI * (EXACT ? expf(-0.5f * z * z) : __expf(-0.5f * z * z));
    const float s = logistic<EXACT>(2.0f * TANH_C * fmaf(TANH_A * z * z, z, z));
    return s + 2.0f * TANH_C * z * s * (1.0f - s) * (1.0f + 3.0f * TANH_A * z * z);
}

// The type that z is kept in, and its value there: in float16 clamped to the range, and a
// value above zero never becomes zero, where relu's slope turns.
template <class T>
using Kept = std::conditional_t<sizeof(T) == 4, float, f16>;

template <class T>
__device__ inline Kept<T> keep(float z) {
    if constexpr (sizeof(T) == 4) {
        return z;
    } else {
        const f16 h = (f16)not_above(not_below(z, -65504.0f), 65504.0f);
        return (z > 0.0f && h == (f16)0.0f) ? (f16)5.9604645e-8f : h;
    }
}

// ---------------------------------------------------------------- the product

// out[m][n] = epilogue(sum over k of A(m, k) B(n, k)); A(m, k) = a[m * am + k * ak], one of
// am and ak being 1, and B likewise.
struct Gemm {
    const void *a, *b;
    int64_t am, ak, bn, bk;
    int64_t M, N, K;
    const void *bias, *res;  // N; M x N
    void* z;                 // M x N of Kept<T>, or null
    void* out;               // M x N
    int act;
};

template <class T>
using frag16 = std::conditional_t<std::is_same_v<T, bf16>, vec<bf16, 8>, vec<f16, 8>>;
using floatx4 = vec<float, 4>;

// D = A B + C on a wave: lane l gives row l % 16 of A and of B, the 16 bytes of k that
// l / 16 picks, and holds D[4 (l / 16) + i][l % 16]. In 32 bits the four k of a lane go
// through one instruction each: any order of k will do that A and B share.
__device__ inline floatx4 mma(vec<bf16, 8> a, vec<bf16, 8> b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ inline floatx4 mma(vec<f16, 8> a, vec<f16, 8> b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline floatx4 mma(vec<float, 4> a, vec<float, 4> b, floatx4 c) {
#pragma unroll
    for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

template <class T>
__device__ inline void finish_element(const Gemm& p, int64_t m, int64_t n, float v) {
    constexpr bool EXACT = sizeof(T) == 4;
    const int64_t i = m * p.N + n;
    if (p.bias) v += (float)((const T*)p.bias)[n];
    if (p.z) ((Kept<T>*)p.z)[i] = keep<T>(v);
    v = act<EXACT>(p.act, v);
    if (p.res) v += (float)((const T*)p.res)[i];
    ((T*)p.out)[i] = (T)v;
}

// 64 x 64 of the output a workgroup, a quarter each of its four waves; 16-byte chunks of
// k staged through LDS by guarded loads.
template <class T>
__global__ __launch_bounds__(256) void gemm_simple(Gemm p) {
    constexpr int CH = 16 / sizeof(T), BK = 4 * CH, LD = BK + CH;
    __shared__ __align__(16) T sa[64][LD], sb[64][LD];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const int64_t tiles_n = (p.N + 63) / 64;
    const int64_t m0 = blockIdx.x / tiles_n * 64, n0 = blockIdx.x % tiles_n * 64;
    const int wm = (w & 1) * 32, wn = (w >> 1) * 32;
    floatx4 acc[2][2] = {};
    for (int64_t k0 = 0; k0 < p.K; k0 += BK) {
        for (int i = t; i < 64 * BK; i += 256) {
            // consecutive threads along the contiguous dimension
            const int ra = p.ak == 1 ? i / BK : i % 64, ka = p.ak == 1 ? i % BK : i / 64;
            const int rb = p.bk == 1 ? i / BK : i % 64, kb = p.bk == 1 ? i % BK : i / 64;
            sa[ra][ka] = m0 + ra < p.M && k0 + ka < p.K ? ((const T*)p.a)[(m0 + ra) * p.am + (k0 + ka) * p.ak] : (T)0.0f;
            sb[rb][kb] = n0 + rb < p.N && k0 + kb < p.K ? ((const T*)p.b)[(n0 + rb) * p.bn + (k0 + kb) * p.bk] : (T)0.0f;
        }
        __syncthreads();
        using F = vec<T, CH>;
        F fa[2], fb[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            fa[i] = *(const F*)&sa[wm + 16 * i + lane % 16][lane / 16 * CH];
            fb[i] = *(const F*)&sb[wn + 16 * i + lane % 16][lane / 16 * CH];
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] = mma(fb[j], fa[i], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int64_t m = m0 + wm + 16 * i + lane % 16, n = n0 + wn + 16 * j + 4 * (lane / 16) + e;
                if (m < p.M && n < p.N) finish_element<T>(p, m, n, acc[i][j][e]);
            }
}

int gemm(int dtype, const Gemm& p, hipStream_t s) {
    const int64_t tiles = (p.M + 63) / 64 * ((p.N + 63) / 64);
    if (tiles == 0) return DRH_OK;
    if (tiles > INT32_MAX) return fail(DRH_ERR_TOO_LARGE, "more than 2^31 - 1 tiles of 64 x 64 outputs");
    return with_type(dtype, [&](auto t) {
        gemm_simple<decltype(t)><<<dim3((unsigned)tiles), 256, 0, s>>>(p);
        return DRH_OK;
    });
}

// ---------------------------------------------------------------- dz and the bias gradient

// dz = dy act'(z), rounded to its type for the products, and the column sums of the
// unrounded values: a workgroup owns 64 VEC columns of every gridDim.y-th slab of rows,
// its four waves a row each, added in order at the end.
template <class T, int VEC>
__global__ __launch_bounds__(256) void slope_kernel(const T* __restrict__ dy, const Kept<T>* __restrict__ z, int kind,
                                                    int64_t M, int64_t N, T* __restrict__ dz, float* part) {
    constexpr bool EXACT = sizeof(T) == 4;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = ((int64_t)blockIdx.x * 64 + lane) * VEC;
    float sum[VEC] = {};
    if (c < N)
        for (int64_t row = (int64_t)blockIdx.y * 4 + w; row < M; row += (int64_t)gridDim.y * 4) {
            float g[VEC];
            load<VEC>(dy + row * N + c, g);
            if (z) {
                float zz[VEC];
                load<VEC>(z + row * N + c, zz);
#pragma unroll
                for (int i = 0; i < VEC; i++) g[i] *= act_slope<EXACT>(kind, zz[i]);
                store<VEC>(dz + row * N + c, g);
            }
#pragma unroll
            for (int i = 0; i < VEC; i++) sum[i] += g[i];
        }
    if (!part) return;
    __shared__ float sums[4][64 * VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) sums[w][lane * VEC + i] = sum[i];
    __syncthreads();
    for (int k = threadIdx.x; k < 64 * VEC; k += 256) {
        const int64_t col = (int64_t)blockIdx.x * 64 * VEC + k;
        if (col < N) part[(int64_t)blockIdx.y * N + col] = sums[0][k] + sums[1][k] + sums[2][k] + sums[3][k];
    }
}

int64_t slope_groups(int64_t M) {
    const int64_t need = (M + 31) / 32;
    return need < 256 ? need : 256;
}

struct BackwardPlan {
    size_t dz = 0, part = 0, total = 0;
};

BackwardPlan backward_plan(int64_t M, int64_t N, int64_t K, int dtype, int act) {
    BackwardPlan b;
    size_t off = 0;
    b.dz = off;
    if (act != DRH_ACT_NONE) off = up256(off + (size_t)M * N * type_size(dtype));
    b.part = off;
    off = up256(off + (size_t)slope_groups(M) * N * sizeof(float));
    b.total = off;
    return b;
}

int check_linear(drh_ctx* ctx, int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws, int dtype, int act,
                 uint32_t flags) {
    int rc = check_call(ctx, dtype, flags);
    if (rc) return rc;
    if (act < DRH_ACT_NONE || act > DRH_ACT_SILU) return fail(DRH_ERR_INVALID_ARG, "unknown activation " + std::to_string(act));
    if (M < 0 || N <= 0 || K < 0) return fail(DRH_ERR_INVALID_ARG, "rows and inputs must not be negative, outputs positive");
    if (M > INT32_MAX || N > (1 << 30) || K > (1 << 30))
        return fail(DRH_ERR_TOO_LARGE, "more than 2^31 - 1 rows or 2^30 features");
    if ((M > 1 && xs < K) || (N > 1 && ws < K)) return fail(DRH_ERR_INVALID_ARG, "a row stride is less than the row");
    return DRH_OK;
}

}  // namespace
}  // namespace drh_nn

using namespace drh_nn;

extern "C" {

int drh_linear(drh_ctx* ctx, const void* x, const void* weight, const void* bias, const void* residual, int64_t rows,
               int64_t n_out, int64_t n_in, int64_t x_stride, int64_t weight_stride, int dtype, int activation, void* y,
               void* kept, void* stream, uint32_t flags) {
    int rc = check_linear(ctx, rows, n_out, n_in, x_stride, weight_stride, dtype, activation, flags);
    if (rc) return rc;
    if (rows == 0) return DRH_OK;
    if (!y || (n_in > 0 && (!x || !weight))) return fail(DRH_ERR_INVALID_ARG, "x, weight and y must not be NULL");
    DeviceGuard dg(ctx->device);
    hipStream_t s = (hipStream_t)stream;
    Gemm p{};
    p.a = x, p.am = x_stride, p.ak = 1, p.b = weight, p.bn = weight_stride, p.bk = 1;
    p.M = rows, p.N = n_out, p.K = n_in;
    p.bias = bias, p.res = residual, p.out = y, p.act = activation;
    p.z = activation != DRH_ACT_NONE ? kept : nullptr;
    rc = gemm(dtype, p, s);
    return rc ? rc : finish_call(s, flags, "linear");
}

int drh_linear_backward_bytes(int64_t rows, int64_t n_out, int64_t n_in, int dtype, int activation, uint64_t* out_bytes) {
    if (!out_bytes || !known_type(dtype) || rows < 0 || n_out <= 0 || n_in < 0)
        return fail(DRH_ERR_INVALID_ARG, "bad sizes or type, or out_bytes is NULL");
    *out_bytes = backward_plan(rows, n_out, n_in, dtype, activation).total;
    return DRH_OK;
}

int drh_linear_backward(drh_ctx* ctx, const void* x, const void* weight, const void* kept, const void* grad_y,
                        int64_t rows, int64_t n_out, int64_t n_in, int64_t x_stride, int64_t weight_stride, int dtype,
                        int activation, void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                        uint64_t workspace_bytes, void* stream, uint32_t flags) {
    int rc = check_linear(ctx, rows, n_out, n_in, x_stride, weight_stride, dtype, activation, flags);
    if (rc) return rc;
    const int64_t M = rows, N = n_out, K = n_in;
    const bool slope = activation != DRH_ACT_NONE;
    if (M > 0 && (!grad_y || (slope && !kept))) return fail(DRH_ERR_INVALID_ARG, "grad_y and kept must not be NULL");
    if (M > 0 && K > 0 && ((grad_x && !weight) || (grad_weight && !x)))
        return fail(DRH_ERR_INVALID_ARG, "an input pointer is NULL");
    const BackwardPlan plan = backward_plan(M, N, K, dtype, activation);
    if (workspace_bytes < plan.total || (plan.total && !workspace))
        return fail(DRH_ERR_INVALID_ARG, "the backward pass needs " + std::to_string(plan.total) + " bytes of workspace");
    if ((uintptr_t)workspace % 16) return fail(DRH_ERR_INVALID_ARG, "the workspace must be 16-byte aligned");
    DeviceGuard dg(ctx->device);
    hipStream_t s = (hipStream_t)stream;
    const void* dz = grad_y;
    float* part = grad_bias ? (float*)((char*)workspace + plan.part) : nullptr;
    const int64_t groups = slope_groups(M);
    if (M > 0 && (slope || grad_bias)) {
        void* out = slope ? (char*)workspace + plan.dz : nullptr;
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            const int vec = vector_width(dtype, {N}, {grad_y, kept});
            auto go = [&](auto v) {
                const int64_t cols = 64 * v.value;
                slope_kernel<T, v.value><<<dim3((unsigned)((N + cols - 1) / cols), (unsigned)groups), 256, 0, s>>>(
                    (const T*)grad_y, slope ? (const Kept<T>*)kept : nullptr, activation, M, N, (T*)out, part);
            };
            if (vec == 1) go(std::integral_constant<int, 1>());
            else if (sizeof(T) == 2 && vec == 2) go(std::integral_constant<int, 2>());
            else go(std::integral_constant<int, 16 / (int)sizeof(T)>());
            return DRH_OK;
        });
        if (slope) dz = out;
    }
    if (grad_bias) reduce_columns(part, M > 0 ? groups : 0, N, N, grad_bias, nullptr, dtype, s);
    if (grad_x && M > 0 && K > 0) {
        Gemm p{};
        p.a = dz, p.am = N, p.ak = 1, p.b = weight, p.bn = 1, p.bk = weight_stride;
        p.M = M, p.N = K, p.K = N, p.out = grad_x, p.act = DRH_ACT_NONE;
        rc = gemm(dtype, p, s);
        if (rc) return rc;
    }
    if (grad_weight && K > 0) {
        Gemm p{};
        p.a = dz, p.am = 1, p.ak = N, p.b = x, p.bn = 1, p.bk = x_stride;
        p.M = N, p.N = K, p.K = M, p.out = grad_weight, p.act = DRH_ACT_NONE;
        rc = gemm(dtype, p, s);
        if (rc) return rc;
    }
    return finish_call(s, flags, "linear backward");
}

}  // extern "C"
