// A linear layer with its epilogue, forward and backward:
//
//   z = x W^T + bias,  y = act(z) + residual               x: M x K, W: N x K
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz,  dresidual = dy
//
// Products run on the matrix cores with 32-bit sums. Each result is rounded to its type
// once, from 32 bits. The backward pass needs act'(z) alone, so the forward pass, which has
// act's exponential at hand, keeps that and not z: in 16 bits beside the 16-bit types, in
// float16 whatever the type is, since its 11 bits keep a slope eight times nearer than
// bfloat16's 8 would. Slopes are within [-0.13, 1.13]: kept times 2^15 they fill float16's
// range, with all 11 bits down to 2e-9, where the gradients of an activation's tail still count.

#include <algorithm>
#include <cmath>

#include "gemm.h"

using namespace drh_rt;

namespace drh_nn {
namespace {

// ---------------------------------------------------------------- activations

constexpr float LOG2_E = 1.44269504088896341f, SQRT_HALF = 0.70710678118654752f, INV_SQRT_2PI = 0.39894228040143268f;
constexpr float TANH_C = 0.79788456080286536f, TANH_A = 0.044715f;

// EXACT: for results in 32 bits, with the library's functions; else for values that are
// rounded to 16 bits afterwards, by single instructions.

// 1 / (1 + exp(-v))
template <bool EXACT>
__device__ inline float logistic(float v) {
    return EXACT ? 1.0f / (1.0f + expf(-v)) : __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-LOG2_E * v));
}

// One instruction each, which passes NaN.
__device__ inline float not_below(float z, float lo) { return __builtin_elementwise_maximum(z, lo); }
__device__ inline float not_above(float z, float hi) { return __builtin_elementwise_minimum(z, hi); }

// act(z), and act'(z) in `slope`. Below -128 every value and slope is 0 in 32 bits, above 64
// every value z and slope 1; the bounds keep infinity times zero out of the products there.
template <bool EXACT, int ACT>
__device__ inline float act(float z, float& slope) {
    if constexpr (ACT == DRH_ACT_NONE) {
        slope = 1.0f;
        return z;
    } else if constexpr (ACT == DRH_ACT_RELU) {
        slope = z > 0.0f ? 1.0f : 0.0f;
        return z < 0.0f ? 0.0f : z;
    } else {
        z = not_below(z, -128.0f);
        const float c = not_above(z, 64.0f);
        if constexpr (ACT == DRH_ACT_SILU) {
            const float s = logistic<EXACT>(c);
            slope = s * fmaf(c, 1.0f - s, 1.0f);
            return z * s;
        } else if constexpr (ACT == DRH_ACT_GELU_TANH) {
            const float u = TANH_A * c * c, s = logistic<EXACT>(2.0f * TANH_C * fmaf(u, c, c));  // (1 + tanh) / 2
            slope = fmaf(2.0f * TANH_C * c * s * (1.0f - s), fmaf(3.0f, u, 1.0f), s);
            return z * s;
        } else {
            // Phi(c) and exp(-c^2 / 2). Phi is made from its own tail and not as (1 + erf) / 2, which
            // cancels below zero: at -5 that leaves two bits.
            float phi, e;
            if constexpr (EXACT) {
                phi = 0.5f * erfcf(-SQRT_HALF * c);
                e = expf(-0.5f * c * c);
            } else {
                // Phi(-|c|) = e t P(t), t = 1 / (1 + 0.292 |c|), in the manner of Abramowitz and Stegun
                // 7.1.26, with P fitted to stay within 1e-7 of Phi and 6e-5 of its value down to -13
                e = __builtin_amdgcn_exp2f(c * c * (-0.5f * LOG2_E));
                const float t = __builtin_amdgcn_rcpf(fmaf(0.292f, fabsf(c), 1.0f));
                float q = fmaf(t, -0.0867610723f, 0.27079457f);
                q = fmaf(t, q, -0.0762883946f);
                q = fmaf(t, q, 0.170907423f);
                q = fmaf(t, q, 0.103905939f);
                q = fmaf(t, q, 0.117441483f);
                q *= t * e;
                phi = c < 0.0f ? q : 1.0f - q;
            }
            slope = fmaf(c * INV_SQRT_2PI, e, phi);
            return z * phi;
        }
    }
}

// The type that slopes are kept in.
template <class T>
using Kept = std::conditional_t<sizeof(T) == 4, float, f16>;
template <class T>
constexpr float KEPT_SCALE = sizeof(T) == 4 ? 1.0f : 32768.0f;

// ---------------------------------------------------------------- the product's epilogue

// One lane's 4 NV neighbouring outputs of a row: columns() is called before the rows that
// share them.
template <class T, int ACT, int NV>
struct Epilogue {
    static constexpr int W = 4 * NV, CH = 16 / sizeof(T) < W ? 16 / sizeof(T) : W;
    int64_t n = 0;
    float bias[W];

    __device__ void columns(const Gemm& p, int64_t n_) {
        n = n_;
#pragma unroll
        for (int i = 0; i < W; i++) bias[i] = 0.0f;
        if (p.bias && !p.partial)
#pragma unroll
            for (int i = 0; i < W; i++)
                if (n + i < p.N) bias[i] = (float)((const T*)p.bias)[n + i];
    }

    __device__ void row(const Gemm& p, int64_t m, const floatx4 (&v)[NV]) const {
        if (m >= p.M) return;
        const int64_t at = m * p.N + n;
        if (p.partial) {
            float* out = p.partial + (int64_t)blockIdx.y * p.M * p.N + at;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const float o[4] = {v[j][0], v[j][1], v[j][2], v[j][3]};
                if (n + 4 * j < p.N) store_some<4>(out + 4 * j, p.N - n - 4 * j, o);
            }
            return;
        }
        if (n >= p.N) return;
        float o[W];
#pragma unroll
        for (int i = 0; i < W; i++) o[i] = v[i / 4][i % 4] + bias[i];
        apply<W>(p, at, p.N - n, o);
    }

    // From z on: activates, keeps the slope, adds the residual, stores the first `left`. The chunks
    // of a line are stored one right after the other, so that it leaves the L2 whole.
    template <int C>
    static __device__ void apply(const Gemm& p, int64_t at, int64_t left, float (&o)[C]) {
        constexpr int PART = CH < C ? CH : C;
        auto store = [&](auto* to, const float (&x)[C]) {
#pragma unroll
            for (int g = 0; g < C; g += PART) {
                float part[PART];
#pragma unroll
                for (int i = 0; i < PART; i++) part[i] = x[g + i];
                if (g < left) store_some<PART>(to + g, left - g, part);
            }
        };
        if constexpr (ACT != DRH_ACT_NONE) {
            float slope[C];
#pragma unroll
            for (int i = 0; i < C; i++) o[i] = act<sizeof(T) == 4, ACT>(o[i], slope[i]), slope[i] *= KEPT_SCALE<T>;
            if (p.kept) store((Kept<T>*)p.kept + at, slope);
        }
        if (p.res)
#pragma unroll
            for (int g = 0; g < C; g += PART) {
                float r[PART] = {};
                if (g < left) load_some<PART>((const T*)p.res + at + g, left - g, r);
#pragma unroll
                for (int i = 0; i < PART; i++) o[g + i] += r[i];
            }
        store((T*)p.out + at, o);
    }
};

// ---------------------------------------------------------------- the products

template <class T, bool AK, bool BK, int ACT>
__global__ __launch_bounds__(512, 2) void gemm_256_kernel(Gemm p) {
    gemm_256<T, AK, BK, Epilogue<T, ACT, 2>>(p);
}

template <class T, bool AK, bool BK, int ACT, class Math, int TILE, int GROUPS>
__global__ __launch_bounds__(256 * GROUPS, TILE == 64 && GROUPS == 1 ? 3 : 2) void gemm_tile_kernel(Gemm p) {
    gemm_tile<T, AK, BK, Epilogue<T, ACT, TILE / 32>, Math, TILE, GROUPS>(p);
}

// The parts of a split product added in order, and the epilogue: a thread a 16-byte chunk of
// a row of the output. Bound by memory, and the last parts come from the caches: four parts of
// 4096 x 1024 (67 MB) take 13 us, 5.9 TB/s.
template <class T, int ACT>
__global__ __launch_bounds__(256) void join_splits(Gemm p) {
    constexpr int CH = 16 / sizeof(T);
    const uint32_t per = (uint32_t)((p.N + CH - 1) / CH), id = blockIdx.x * 256 + threadIdx.x;
    const int64_t m = id / per, n = (int64_t)(id % per) * CH, at = m * p.N + n, left = p.N - n;
    if (m >= p.M) return;
    float o[CH] = {};
    const int64_t size = p.M * p.N;
    for (int s = 0; s < p.splits; s++) {
        float v[CH] = {};
        load_some<CH>(p.partial + s * size + at, left, v);
#pragma unroll
        for (int i = 0; i < CH; i++) o[i] += v[i];
    }
    if (p.bias) {
        float b[CH] = {};
        load_some<CH>((const T*)p.bias + n, left, b);
#pragma unroll
        for (int i = 0; i < CH; i++) o[i] += b[i];
    }
    Epilogue<T, ACT, 2>::template apply<CH>(p, at, left, o);
}

// Few rows of x (up to 16 MT): the weights are read once and that is what it costs, so
// nothing is staged. A workgroup takes 16 outputs; its eight waves take an eighth of k each,
// straight from memory to the matrix cores (a lane 16 bytes of row l % 16, four lanes 64
// contiguous bytes), and are added through LDS in order. Rows may start anywhere. What bounds it
// is a wave's chain of one load, one product and the sum over LDS: 1500 x 1024 weights in bfloat16
// (3 MB) take 3.9 us for one row, 1280 x 1024 in 32 bits 6.2 for sixteen; the smallest kernel
// of the layers takes 2.6.
template <class T, int MT, int ACT>
__global__ __launch_bounds__(512) void gemm_rows_kernel(Gemm p) {
    constexpr int CH = 16 / sizeof(T), WAVES = 8;
    using F = vec<T, CH>;
    using FU = typename Anywhere<T, CH>::type;
    __shared__ __align__(16) floatx4 part[WAVES][MT][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16, K = p.K;
    const int steps = (int)((K + 4 * CH - 1) / (4 * CH)), s0 = (int)((int64_t)steps * w / WAVES),
              s1 = (int)((int64_t)steps * (w + 1) / WAVES);
    // rows past the end read the last one's values and are not stored
    const T* bp = (const T*)p.b.ptr + (n0 + r < p.N ? n0 + r : p.N - 1) * p.b.ld;
    const T* ap[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) ap[t] = (const T*)p.a.ptr + (16 * t + r < p.M ? 16 * t + r : p.M - 1) * p.a.ld;
    floatx4 acc[MT] = {};
    // eight (four with more rows) steps' loads at once: a wave has little else to wait with
    constexpr int AT_ONCE = MT == 1 ? 8 : 4;
    const int whole = (int)(K / (4 * CH)) < s1 ? (int)(K / (4 * CH)) : s1;
    int s = s0;
    for (; s + AT_ONCE <= whole; s += AT_ONCE) {
        F b[AT_ONCE], a[AT_ONCE][MT];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            const int64_t k = ((int64_t)(s + u) * 4 + q) * CH;
            b[u] = *(const FU*)(bp + k);
#pragma unroll
            for (int t = 0; t < MT; t++) a[u][t] = *(const FU*)(ap[t] + k);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
#pragma unroll
            for (int t = 0; t < MT; t++) acc[t] = mma(b[u], a[u][t], acc[t]);
    }
    auto chunk = [&](const T* row, int64_t k) {
        F v;
        if (k + CH <= K) {
            v = *(const FU*)(row + k);
        } else {
#pragma unroll
            for (int i = 0; i < CH; i++) v[i] = k + i < K ? row[k + i] : (T)0.0f;
        }
        return v;
    };
    for (; s < s1; s++) {
        const int64_t k = ((int64_t)s * 4 + q) * CH;
        const F b = chunk(bp, k);
#pragma unroll
        for (int t = 0; t < MT; t++) acc[t] = mma(b, chunk(ap[t], k), acc[t]);
    }
#pragma unroll
    for (int t = 0; t < MT; t++) part[w][t][lane] = acc[t];
    __syncthreads();
    if (w >= MT) return;
    floatx4 v[1] = {part[0][w][lane]};
#pragma unroll
    for (int i = 1; i < WAVES; i++) v[0] += part[i][w][lane];
    Epilogue<T, ACT, 1> e;
    e.columns(p, n0 + 4 * q);
    e.row(p, 16 * w + r, v);
}

// Any strides and sizes: 64 x 64 of the output a workgroup, a quarter each of its four
// waves, 16-byte chunks of k staged through LDS by guarded loads. Takes what the kernels
// above do not: operands that are not 16-byte aligned or too large for their offsets. Correct
// before fast.
template <class T, int ACT>
__global__ __launch_bounds__(256) void gemm_any_kernel(Gemm p, bool a_kc, bool b_kc) {
    constexpr int CH = 16 / sizeof(T), BK = 4 * CH, LD = BK + CH;
    __shared__ __align__(16) T sa[64][LD], sb[64][LD];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const int64_t tiles_n = (p.N + 63) / 64;
    const int64_t m0 = blockIdx.x / tiles_n * 64, n0 = blockIdx.x % tiles_n * 64;
    const int wm = (w & 1) * 32, wn = (w >> 1) * 32;
    const int64_t am = a_kc ? p.a.ld : 1, ak = a_kc ? 1 : p.a.ld, bn = b_kc ? p.b.ld : 1, bk = b_kc ? 1 : p.b.ld;
    floatx4 acc[2][2] = {};
    for (int64_t k0 = 0; k0 < p.K; k0 += BK) {
        for (int i = t; i < 64 * BK; i += 256) {
            // consecutive threads along the contiguous dimension
            const int ra = a_kc ? i / BK : i % 64, ka = a_kc ? i % BK : i / 64;
            const int rb = b_kc ? i / BK : i % 64, kb = b_kc ? i % BK : i / 64;
            sa[ra][ka] = m0 + ra < p.M && k0 + ka < p.K ? ((const T*)p.a.ptr)[(m0 + ra) * am + (k0 + ka) * ak] : (T)0.0f;
            sb[rb][kb] = n0 + rb < p.N && k0 + kb < p.K ? ((const T*)p.b.ptr)[(n0 + rb) * bn + (k0 + kb) * bk] : (T)0.0f;
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
    for (int j = 0; j < 2; j++) {
        Epilogue<T, ACT, 1> e;
        e.columns(p, n0 + wn + 16 * j + 4 * (lane / 16));
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const floatx4 v[1] = {acc[i][j]};
            e.row(p, m0 + wm + 16 * i + lane % 16, v);
        }
    }
}

// ---------------------------------------------------------------- which kernel

enum Layout { KK, KN, MN };  // A's and B's contiguous dimension: forward, dx, dW

struct GemmPlan {
    int tile = 0;    // 256, 128, 64, or 0: any
    bool rows = false;  // gemm_rows_kernel
    int splits = 1;
    size_t bytes = 0;  // of partial sums
};

constexpr int CUS = 256;
// gemm_rows_kernel's: it reads x from the caches for every 16 outputs, which with more rows and
// a long k costs more than staging. Microseconds in bfloat16, with it and by tiles: 32 rows
// 1280 x 1024 4.8 / 6.5, 4096 x 4096 13.2 / 13.9; 64 rows 4096 x 1024 7.2 / 9.1, 4096 x 4096 21.7 / 14.2.
constexpr int64_t ROWS_FEW = 32, ROWS_MOST = 64, ROWS_MOST_K = 2048;
// Products in 32 bits are split in thirds from this k on: their error, 2^-21 of a term at the
// most (gemm.h says what becomes of terms too small for that), is then below what a 32-bit sum of
// as many terms may lose, k 2^-24, and shorter products are bound by memory either way.
constexpr int64_t THIRDS_LEAST = 64;

// Whether an operand's sizes suit the kernels that load 16-byte chunks through buffers.
bool chunked(int dtype, bool kc, int64_t ld, int64_t rows, int64_t K) {
    const int64_t size = type_size(dtype), ch = 16 / size;
    if (ld % ch || (kc ? K : rows) % ch) return false;
    return kc ? 256 * ld * size < PAST_END : 64 * ld * size < PAST_END;
}

// Microseconds of a product by tiles of 64, 128 or 256 with k in `splits` parts, from what the
// kernels took on an MI355X at 256^2 to 8192 x 4096 outputs and k of 128 to 8192: with `c`
// workgroups on the fullest CU, their start and end, and the `steps` k tiles of 128 bytes. Small
// tiles share a CU at a cost that grows with c, large ones take turns. Joining is a launch more and
// the sums' way to memory and back. For 2048 x 1024 outputs and k = 1024 in bfloat16 it gives 10 and
// 15 us for 64 and 128 (measured 10.0, 14.0), for 4096 x 4096 and k = 2048 98, 73 and 63 for 64, 128
// and 256 (107, 72, 61).
double gemm_time(int dtype, int tile, double tiles, int splits, double steps, double outputs) {
    const double wgs = tiles * splits, c = std::ceil(wgs / CUS);
    double t;
    if (tile == 256) t = c * (11.0 + steps * (1.12 + 0.45 * std::min(1.0, wgs / CUS)));
    else if (dtype == DRH_F32 && tile == 128) t = c > 1 ? 11.0 + 3.5 * c + steps * 1.38 * c : 11.0 + steps * 1.28;
    else if (dtype == DRH_F32) t = c > 1 ? 3.5 + 0.7 * c + steps * (0.25 + 0.42 * c) : 4.5 + steps * 0.54;
    else if (tile == 128) t = c > 1 ? 2.0 + 2.4 * c + steps * 0.475 * c : 6.0 + steps * 0.58;
    else t = c > 1 ? 4.0 + 0.3 * c + steps * std::max(0.21, 0.18 * c) : 3.3 + steps * 0.3;
    return splits > 1 ? t + 6.0 + splits * outputs * 1.45e-6 : t;
}

GemmPlan plan_gemm(int dtype, int64_t M, int64_t N, int64_t K, bool fits) {
    GemmPlan g;
    if (!fits || K == 0 || M == 0) return g;
    const int64_t bk = 128 / (int64_t)type_size(dtype), kt = (K + bk - 1) / bk;
    double best = 1e30;
    for (int tile : {256, 128, 64}) {
        if (tile == 256 && dtype == DRH_F32) continue;
        const int64_t tiles = (M + tile - 1) / tile * ((N + tile - 1) / tile);
        if (tiles > most_groups(tile == 256 ? 512 : 256)) continue;
        for (int64_t s = 1; s <= 64 && s <= kt; s++) {
            const int64_t per = (kt + s - 1) / s;
            if ((kt + per - 1) / per != s) continue;
            if (s > 1 && (double)s * M * N * 4 > 1e9) break;
            const double t = gemm_time(dtype, tile, (double)tiles, (int)s, (double)per, (double)M * N);
            if (t < best) best = t, g.tile = tile, g.splits = (int)s;
        }
    }
    if (g.splits > 1) g.bytes = up256((size_t)g.splits * M * N * sizeof(float));
    return g;
}

template <class F>
int with_act(int act, F&& f) {
    using std::integral_constant;
    switch (act) {
        case DRH_ACT_RELU: return f(integral_constant<int, DRH_ACT_RELU>());
        case DRH_ACT_GELU: return f(integral_constant<int, DRH_ACT_GELU>());
        case DRH_ACT_GELU_TANH: return f(integral_constant<int, DRH_ACT_GELU_TANH>());
        case DRH_ACT_SILU: return f(integral_constant<int, DRH_ACT_SILU>());
        default: return f(integral_constant<int, DRH_ACT_NONE>());
    }
}

bool aligned(const void* p) { return (uintptr_t)p % 16 == 0; }

// Whether a product's launch holds its tiles: a plan's always, gemm_any_kernel's 64 x 64 not
// from 2^36 outputs on.
int check_tiles(const GemmPlan& plan, int64_t M, int64_t N, const void* a, const void* b) {
    if (plan.rows || (plan.tile && aligned(a) && aligned(b))) return DRH_OK;
    if ((M + 63) / 64 * ((N + 63) / 64) <= most_groups(256)) return DRH_OK;
    return fail(DRH_ERR_TOO_LARGE, "more tiles of the output than a launch holds");
}

// p without its plan's fields; `partial` has plan.bytes bytes.
int gemm(int dtype, Layout layout, Gemm p, const GemmPlan& plan, float* partial, hipStream_t s) {
    if (p.M == 0 || p.N == 0) return DRH_OK;
    const int64_t ch = 16 / (int64_t)type_size(dtype);
    const bool fast = plan.tile && aligned(p.a.ptr) && aligned(p.b.ptr);
    const int tile = fast ? plan.tile : 64;  // gemm_any_kernel's too
    const int64_t tiles = (p.M + tile - 1) / tile * ((p.N + tile - 1) / tile);
    p.splits = fast ? plan.splits : 1;
    const int64_t bk = 128 / (int64_t)type_size(dtype), kt = (p.K + bk - 1) / bk;
    p.tiles_per_split = (int)((kt + p.splits - 1) / p.splits);
    p.partial = p.splits > 1 ? partial : nullptr;
    const dim3 grid((unsigned)tiles, (unsigned)p.splits);
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (plan.rows)
            return with_act(p.act, [&](auto a) {
                const dim3 groups((unsigned)((p.N + 15) / 16));
                if (p.M <= 16) gemm_rows_kernel<T, 1, a.value><<<groups, 512, 0, s>>>(p);
                else if (p.M <= 32) gemm_rows_kernel<T, 2, a.value><<<groups, 512, 0, s>>>(p);
                else gemm_rows_kernel<T, 4, a.value><<<groups, 512, 0, s>>>(p);
                return DRH_OK;
            });
        if (!fast)
            return with_act(p.act, [&](auto a) {
                gemm_any_kernel<T, a.value><<<grid, 256, 0, s>>>(p, layout != MN, layout == KK);
                return DRH_OK;
            });
        auto with = [&](auto a, auto math) {
            constexpr int ACT = a.value;
            using Math = decltype(math);
            // 32 bits have no large tile: with thirds one of 256 x 128 in gemm_256's manner was no
            // faster (4096^3 699 us where this one took 684), and 256 x 256 needs more registers
            constexpr bool LARGE = sizeof(T) == 2;
            auto launch = [&](auto ak, auto bk) {
                constexpr bool AK = ak.value, BK = bk.value;
                if constexpr (LARGE)
                    if (tile == 256) gemm_256_kernel<T, AK, BK, ACT><<<grid, 512, 0, s>>>(p);
                // Microseconds with two groups and with one, 256 tiles: 4096 x 1024 outputs and k = 1024
                // in 32 bits 64 / 64, as k by rows 68 / 72; 1024 x 1024 outputs and k = 4096 in bfloat16
                // 23.2 / 30.6. With 512 tiles one is the faster: 2048 x 1024 and k = 1024 10.0 / 10.9
                const bool alone = tiles * p.splits <= CUS;
                if (tile == 128 && alone) gemm_tile_kernel<T, AK, BK, ACT, Math, 128, 2><<<grid, 512, 0, s>>>(p);
                if (tile == 128 && !alone) gemm_tile_kernel<T, AK, BK, ACT, Math, 128, 1><<<grid, 256, 0, s>>>(p);
                if (tile == 64 && alone) gemm_tile_kernel<T, AK, BK, ACT, Math, 64, 2><<<grid, 512, 0, s>>>(p);
                if (tile == 64 && !alone) gemm_tile_kernel<T, AK, BK, ACT, Math, 64, 1><<<grid, 256, 0, s>>>(p);
            };
            if (layout == KK) launch(std::true_type(), std::true_type());
            else if constexpr (ACT == DRH_ACT_NONE) {
                if (layout == KN) launch(std::true_type(), std::false_type());
                else launch(std::false_type(), std::false_type());
            }
            return DRH_OK;
        };
        auto go = [&](auto a) {
            if constexpr (sizeof(T) == 4)
                if (p.K >= THIRDS_LEAST) return with(a, Thirds());
            return with(a, Straight());
        };
        if (!p.partial) return with_act(p.act, go);
        go(std::integral_constant<int, DRH_ACT_NONE>());
        return with_act(p.act, [&](auto a) {
            const int64_t chunks = p.M * ((p.N + ch - 1) / ch);
            join_splits<T, a.value><<<dim3((unsigned)((chunks + 255) / 256)), 256, 0, s>>>(p);
            return DRH_OK;
        });
    });
}

// A row-major operand as the fast kernels take it: as it stands, or copied to rows of K
// elements rounded up to 16 bytes, with zeros behind K.
struct Rows {
    int64_t ld;
    size_t bytes = 0;  // of the copy, 0: none
};

Rows rows_for(int dtype, int64_t rows, int64_t K, int64_t ld) {
    const int64_t ch = 16 / (int64_t)type_size(dtype);
    if (K % ch == 0 && ld % ch == 0) return {ld};
    const int64_t padded = (K + ch - 1) / ch * ch;
    return {padded, up256((size_t)rows * padded * type_size(dtype))};
}

struct PadJob {
    const void* src;
    void* dst;
    int64_t ld, rows;  // rows 0: nothing to copy
};

// Two operands of K columns in one launch, a thread a 16-byte chunk.
template <class T>
__global__ __launch_bounds__(256) void pad_rows(PadJob a, PadJob b, int64_t K, int64_t first) {
    constexpr int CH = 16 / sizeof(T);
    const int64_t per = (K + CH - 1) / CH;
    int64_t i = (first + blockIdx.x) * 256 + threadIdx.x;
    const bool second = i >= a.rows * per;
    if (second) i -= a.rows * per;
    const PadJob& job = second ? b : a;
    if (i >= job.rows * per) return;
    const int64_t row = i / per, c = i % per * CH;
    const Raw v = load_raw<false, false>((const T*)job.src + row * job.ld + c, K - c);
    *(Raw*)((T*)job.dst + row * per * CH + c) = v;
}

void pad(int dtype, const PadJob& a, const PadJob& b, int64_t K, hipStream_t s) {
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t ch = 16 / (int64_t)sizeof(T), chunks = (a.rows + b.rows) * ((K + ch - 1) / ch);
        in_launches((chunks + 255) / 256, most_groups(256), [&](int64_t first, int64_t count) {
            pad_rows<T><<<dim3((unsigned)count), 256, 0, s>>>(a, b, K, first);
        });
        return DRH_OK;
    });
}

// ---------------------------------------------------------------- dz and the bias gradient

// dz = dy act'(z), rounded to its type for the products, in rows of ldz elements with zeros
// behind N, and the column sums of the unrounded values: a workgroup owns 64 chunks of every
// gridDim.y-th slab of rows, its four waves a row each, added in order at the end. Bound by memory:
// 16384 x 4096 in bfloat16 (two arrays read past the caches, one written: 403 MB) take 66 us,
// 6.1 TB/s.
template <class T, bool ONCE>
__global__ __launch_bounds__(256) void slope_kernel(const T* __restrict__ dy, const Kept<T>* __restrict__ slope, int64_t M,
                                                    int64_t N, int64_t ldz, T* __restrict__ dz, float* part) {
    constexpr int CH = 16 / sizeof(T);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = ((int64_t)blockIdx.x * 64 + lane) * CH;
    float sum[CH] = {};
    const int64_t stride = (int64_t)gridDim.y * 4, left = N - c;
    auto fetch = [&](int64_t row, float (&g)[CH], float (&d)[CH]) {
        Raw gr = {}, dr = {};
        if (row < M) {
            gr = load_raw<false, ONCE>(dy + row * N + c, left);
            if (slope) dr = load_raw<false, ONCE>(slope + row * N + c, left);
        }
        const Elements<T> ge = __builtin_bit_cast(Elements<T>, gr);
        const Elements<Kept<T>> de = __builtin_bit_cast(Elements<Kept<T>>, dr);
#pragma unroll
        for (int i = 0; i < CH; i++) g[i] = (float)ge[i], d[i] = slope ? (float)de[i] * (1.0f / KEPT_SCALE<T>) : 1.0f;
    };
    auto finish = [&](int64_t row, float (&g)[CH], const float (&d)[CH]) {
        if (row >= M) return;
#pragma unroll
        for (int i = 0; i < CH; i++) sum[i] += g[i] *= d[i];
        if (dz) store<CH>(dz + row * ldz + c, g);  // ldz is whole chunks
    };
    if (left > 0)
        for (int64_t row = (int64_t)blockIdx.y * 4 + w; row < M; row += 2 * stride) {  // two rows' loads at once
            float g0[CH], d0[CH], g1[CH], d1[CH];
            fetch(row, g0, d0);
            fetch(row + stride, g1, d1);
            finish(row, g0, d0);
            finish(row + stride, g1, d1);
        }
    if (!part) return;
    __shared__ float sums[4][64 * CH];
#pragma unroll
    for (int i = 0; i < CH; i++) sums[w][lane * CH + i] = sum[i];
    __syncthreads();
    for (int k = threadIdx.x; k < 64 * CH; k += 256) {
        const int64_t col = (int64_t)blockIdx.x * 64 * CH + k;
        if (col < N) part[(int64_t)blockIdx.y * N + col] = sums[0][k] + sums[1][k] + sums[2][k] + sums[3][k];
    }
}

// Row groups of slope_kernel: two rows a wave at least, and about 2048 workgroups at most.
int64_t slope_groups(int64_t M, int64_t N, int dtype) {
    const int64_t cols = 64 * (16 / (int64_t)type_size(dtype)), blocks = (N + cols - 1) / cols;
    const int64_t need = (M + 7) / 8, most = std::min<int64_t>(512, std::max<int64_t>(64, 2048 / blocks));
    return std::min(need, most);
}

// A single row has no stride: whatever the caller gives for it must not name rows behind it.
int64_t stride_of(int64_t rows, int64_t stride, int64_t K) { return rows > 1 ? stride : K; }

struct ForwardPlan {
    Rows x, w;
    GemmPlan y;
    size_t x_at = 0, w_at = 0, part_at = 0, total = 0;
};

ForwardPlan forward_plan(int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws, int dtype) {
    ForwardPlan f;
    xs = stride_of(M, xs, K), ws = stride_of(N, ws, K);
    if (K > 0 && (M <= ROWS_FEW || (M <= ROWS_MOST && K <= ROWS_MOST_K)) && (N + 15) / 16 <= most_groups(512)) {
        f.x = {xs}, f.w = {ws}, f.y.rows = true;
        return f;
    }
    f.x = rows_for(dtype, M, K, xs);
    f.w = rows_for(dtype, N, K, ws);
    const int64_t ch = 16 / (int64_t)type_size(dtype), K_pad = (K + ch - 1) / ch * ch;
    f.y = plan_gemm(dtype, M, N, K, chunked(dtype, true, f.x.ld, M, K_pad) && chunked(dtype, true, f.w.ld, N, K_pad));
    if (!f.y.tile) f.x = {xs}, f.w = {ws};
    f.x_at = 0;
    f.w_at = f.x_at + f.x.bytes;
    f.part_at = f.w_at + f.w.bytes;
    f.total = f.part_at + f.y.bytes;
    return f;
}

// x and W padded where dW and dx need them, dz where it is not dy itself or dy needs
// padding, the bias gradient's partial sums, and the larger of the products' partial sums.
struct BackwardPlan {
    Rows x, w;
    bool dz = false;
    int64_t ldz = 0;
    GemmPlan dx, dw;
    size_t x_at = 0, w_at = 0, dz_at = 0, sums_at = 0, part_at = 0, total = 0;
};

BackwardPlan backward_plan(int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws, int dtype, int act) {
    BackwardPlan b;
    xs = stride_of(M, xs, K), ws = stride_of(N, ws, K);
    const int64_t ch = 16 / (int64_t)type_size(dtype), N_pad = (N + ch - 1) / ch * ch, K_pad = (K + ch - 1) / ch * ch;
    b.x = rows_for(dtype, M, K, xs);
    b.w = rows_for(dtype, N, K, ws);
    b.ldz = N_pad;
    b.dz = act != DRH_ACT_NONE || N_pad != N;
    b.dx = plan_gemm(dtype, M, K, N, chunked(dtype, true, b.ldz, M, N_pad) && chunked(dtype, false, b.w.ld, K_pad, N));
    b.dw = plan_gemm(dtype, N, K, M, chunked(dtype, false, b.ldz, N_pad, M) && chunked(dtype, false, b.x.ld, K_pad, M));
    if (!b.dx.tile) b.w = {ws};
    if (!b.dw.tile) b.x = {xs};
    size_t off = b.x.bytes;
    b.w_at = off;
    off += b.w.bytes;
    b.dz_at = off;
    if (b.dz) off += up256((size_t)M * b.ldz * type_size(dtype));
    b.sums_at = off;
    off += up256((size_t)slope_groups(M, N, dtype) * N * sizeof(float));
    b.part_at = off;
    b.total = off + (b.dx.bytes > b.dw.bytes ? b.dx.bytes : b.dw.bytes);
    return b;
}

int check_sizes(int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws) {
    if (M < 0 || N <= 0 || K < 0) return fail(DRH_ERR_INVALID_ARG, "rows and inputs must not be negative, outputs positive");
    if (M > INT32_MAX || N > (1 << 30) || K > (1 << 30))
        return fail(DRH_ERR_TOO_LARGE, "more than 2^31 - 1 rows or 2^30 features");
    if ((M > 1 && xs < K) || (N > 1 && ws < K)) return fail(DRH_ERR_INVALID_ARG, "a row stride is less than the row");
    int rc = check_span(M, xs);
    return rc ? rc : check_span(N, ws);
}

int check_linear(drh_ctx* ctx, int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws, int dtype, int act,
                 uint32_t flags) {
    int rc = check_call(ctx, dtype, flags);
    if (rc) return rc;
    if (act < DRH_ACT_NONE || act > DRH_ACT_SILU) return fail(DRH_ERR_INVALID_ARG, "unknown activation " + std::to_string(act));
    return check_sizes(M, N, K, xs, ws);
}

int check_bytes(int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws, int dtype, const uint64_t* out_bytes) {
    if (!out_bytes || !known_type(dtype)) return fail(DRH_ERR_INVALID_ARG, "unknown element type, or out_bytes is NULL");
    return check_sizes(M, N, K, xs, ws);
}

int check_workspace(size_t need, const void* workspace, uint64_t bytes) {
    if (bytes < need || (need && !workspace))
        return fail(DRH_ERR_INVALID_ARG, "the call needs " + std::to_string(need) + " bytes of workspace");
    if ((uintptr_t)workspace % 16) return fail(DRH_ERR_INVALID_ARG, "the workspace must be 16-byte aligned");
    return DRH_OK;
}

}  // namespace
}  // namespace drh_nn

using namespace drh_nn;

extern "C" {

int drh_linear_bytes(int64_t rows, int64_t n_out, int64_t n_in, int64_t x_stride, int64_t weight_stride, int dtype,
                     uint64_t* out_bytes) {
    int rc = check_bytes(rows, n_out, n_in, x_stride, weight_stride, dtype, out_bytes);
    if (rc) return rc;
    *out_bytes = forward_plan(rows, n_out, n_in, x_stride, weight_stride, dtype).total;
    return DRH_OK;
}

int drh_linear(drh_ctx* ctx, const void* x, const void* weight, const void* bias, const void* residual, int64_t rows,
               int64_t n_out, int64_t n_in, int64_t x_stride, int64_t weight_stride, int dtype, int activation, void* y,
               void* kept, void* workspace, uint64_t workspace_bytes, void* stream, uint32_t flags) {
    int rc = check_linear(ctx, rows, n_out, n_in, x_stride, weight_stride, dtype, activation, flags);
    if (rc) return rc;
    if (rows == 0) return DRH_OK;
    if (!y || (n_in > 0 && (!x || !weight))) return fail(DRH_ERR_INVALID_ARG, "x, weight and y must not be NULL");
    const ForwardPlan plan = forward_plan(rows, n_out, n_in, x_stride, weight_stride, dtype);
    rc = check_workspace(plan.total, workspace, workspace_bytes);
    if (rc) return rc;
    rc = check_tiles(plan.y, rows, n_out, plan.x.bytes ? nullptr : x, plan.w.bytes ? nullptr : weight);
    if (rc) return rc;
    DeviceGuard dg(ctx->device);
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    pad(dtype, {x, ws + plan.x_at, x_stride, plan.x.bytes ? rows : 0},
        {weight, ws + plan.w_at, weight_stride, plan.w.bytes ? n_out : 0}, n_in, s);
    Gemm p{};
    p.a = {plan.x.bytes ? ws + plan.x_at : x, plan.x.ld, rows};
    p.b = {plan.w.bytes ? ws + plan.w_at : weight, plan.w.ld, n_out};
    p.M = rows, p.N = n_out, p.K = n_in;
    p.bias = bias, p.res = residual, p.out = y, p.act = activation;
    p.kept = activation != DRH_ACT_NONE ? kept : nullptr;
    rc = gemm(dtype, KK, p, plan.y, (float*)(ws + plan.part_at), s);
    return rc ? rc : finish_call(s, flags, "linear");
}

int drh_linear_backward_bytes(int64_t rows, int64_t n_out, int64_t n_in, int64_t x_stride, int64_t weight_stride,
                              int dtype, int activation, uint64_t* out_bytes) {
    int rc = check_bytes(rows, n_out, n_in, x_stride, weight_stride, dtype, out_bytes);
    if (rc) return rc;
    *out_bytes = backward_plan(rows, n_out, n_in, x_stride, weight_stride, dtype, activation).total;
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
    const BackwardPlan plan = backward_plan(M, N, K, x_stride, weight_stride, dtype, activation);
    rc = check_workspace(plan.total, workspace, workspace_bytes);
    if (rc) return rc;
    const void* own_dz = plan.dz ? nullptr : grad_y;  // what the call copies stands aligned
    if (grad_x) rc = check_tiles(plan.dx, M, K, own_dz, plan.w.bytes ? nullptr : weight);
    if (!rc && grad_weight) rc = check_tiles(plan.dw, N, K, own_dz, plan.x.bytes ? nullptr : x);
    if (rc) return rc;
    DeviceGuard dg(ctx->device);
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    const bool products = K > 0 && M > 0 && (grad_x || grad_weight), dz_made = plan.dz && products;
    float* sums = grad_bias ? (float*)(ws + plan.sums_at) : nullptr;
    const int64_t groups = slope_groups(M, N, dtype), ldz = plan.ldz;
    const void* dz = dz_made ? ws + plan.dz_at : grad_y;
    if (M > 0 && (dz_made || grad_bias))
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            const int64_t cols = 64 * (16 / (int64_t)sizeof(T));
            auto go = [&](auto once) {
                slope_kernel<T, once.value><<<dim3((unsigned)((N + cols - 1) / cols), (unsigned)groups), 256, 0, s>>>(
                    (const T*)grad_y, slope ? (const Kept<T>*)kept : nullptr, M, N, ldz, dz_made ? (T*)dz : nullptr, sums);
            };
            // dy is read again where it is dz
            if (dz_made && M * N * (int64_t)sizeof(T) >= READ_ONCE_BYTES) go(std::true_type());
            else go(std::false_type());
            return DRH_OK;
        });
    if (grad_bias) reduce_columns(sums, M > 0 ? groups : 0, N, N, grad_bias, nullptr, dtype, s);
    const int64_t ch = 16 / (int64_t)type_size(dtype), N_pad = (N + ch - 1) / ch * ch, K_pad = (K + ch - 1) / ch * ch;
    float* part = (float*)(ws + plan.part_at);
    const bool pad_x = plan.x.bytes && grad_weight && M > 0 && K > 0, pad_w = plan.w.bytes && grad_x && M > 0 && K > 0;
    pad(dtype, {x, ws + plan.x_at, x_stride, pad_x ? M : 0}, {weight, ws + plan.w_at, weight_stride, pad_w ? N : 0}, K, s);
    if (grad_x && M > 0 && K > 0) {
        Gemm p{};
        p.a = {dz, ldz, M}, p.b = {pad_w ? ws + plan.w_at : weight, plan.w.ld, pad_w ? K_pad : K};
        p.M = M, p.N = K, p.K = N, p.out = grad_x, p.act = DRH_ACT_NONE;
        rc = gemm(dtype, KN, p, plan.dx, part, s);
        if (rc) return rc;
    }
    if (grad_weight && K > 0) {
        Gemm p{};
        p.a = {dz, ldz, dz_made ? N_pad : N}, p.b = {pad_x ? ws + plan.x_at : x, plan.x.ld, pad_x ? K_pad : K};
        p.M = N, p.N = K, p.K = M, p.out = grad_weight, p.act = DRH_ACT_NONE;
        rc = gemm(dtype, MN, p, plan.dw, part, s);
        if (rc) return rc;
    }
    return finish_call(s, flags, "linear backward");
}

}  // extern "C"
