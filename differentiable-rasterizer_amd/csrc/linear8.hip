// A linear layer whose operands stand in 8 bits, forward:
//
//   y = act((xq wq^T) s_x s_w + bias) + residual      xq: M x K, s_x: M;  wq: N x K, s_w: N
//
// with e4m3 values and a float32 scale for each row of both (rms_norm.hip makes them). Where y has 16
// bits the product runs on the matrix cores' 8-bit instructions, twice the rate of bfloat16 and half the
// bytes, which lose up to 2^-10 of the terms (mma in gemm.h says how, and why that is taken); for y in 32
// bits, which is how a caller asks for sums in 32 bits, on the bfloat16 ones (Widened in gemm.h). Scales,
// bias, activation and residual follow in 32 bits, and y is rounded once.

#include <algorithm>
#include <cmath>

#include "products.h"

using namespace drh_rt;

namespace drh_nn {
namespace {

// Kernels of 16-bit outputs hold every activation; those of float32, whose functions are long, one each.
constexpr int ANY_ACT = -1;

// f(activation) as a constant.
template <class T, class F>
void with_kernel_act(int kind, F&& f) {
    if constexpr (sizeof(T) == 2) f(std::integral_constant<int, ANY_ACT>());
    else with_act(kind, [&](auto a) { return f(a), DRH_OK; });
}

// One lane's 4 NV neighbouring outputs of a row: columns() is called before the rows that
// share them.
template <class T, int NV, int ACT>
struct Epilogue8 {
    static constexpr int W = 4 * NV, CH = 16 / sizeof(T) < W ? 16 / sizeof(T) : W;
    int64_t n = 0;
    float bias[W], scale[W];

    __device__ void columns(const Gemm& p, int64_t n_) {
        n = n_;
#pragma unroll
        for (int i = 0; i < W; i++) scale[i] = bias[i] = 0.0f;
        if (p.partial || n >= p.N) return;
        load_some<W>(p.col_scale + n, p.N - n, scale);
        if (p.bias) load_some<W>((const T*)p.bias + n, p.N - n, bias);
    }

    // What a row adds at the end, and its scale, loaded ahead: one after the other the rows of a tile would
    // wait for memory each.
    static constexpr bool EARLY = sizeof(T) == 2 && W >= 8;
    struct Ahead {
        Raw res[EARLY ? W / 8 : 1];
        float scale;
    };
    __device__ Ahead ahead(const Gemm& p, int64_t m) const {
        Ahead a = {};
        if (p.partial || m >= p.M || n >= p.N) return a;
        a.scale = p.row_scale[m];
        if (EARLY && p.res)
#pragma unroll
            for (int g = 0; g < W / 8; g++)
                if (n + 8 * g < p.N) a.res[g] = load_raw<false, false>((const T*)p.res + m * p.N + n + 8 * g, p.N - n - 8 * g);
        return a;
    }

    __device__ void row(const Gemm& p, int64_t m, const floatx4 (&v)[NV]) const { row(p, m, v, ahead(p, m)); }
    __device__ void row(const Gemm& p, int64_t m, const floatx4 (&v)[NV], const Ahead& a) const {
        if (m >= p.M || n >= p.N) return;
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
        float o[W], r[W] = {};
#pragma unroll
        for (int i = 0; i < W; i++) o[i] = fmaf(v[i / 4][i % 4] * a.scale, scale[i], bias[i]);
        if constexpr (EARLY) {
#pragma unroll
            for (int i = 0; i < W; i++) r[i] = (float)__builtin_bit_cast(Elements<T>, a.res[i / 8])[i % 8];
        } else if (p.res) {
            load_some<W>((const T*)p.res + at, p.N - n, r);
        }
        apply<W>(p, at, p.N - n, o, r);
    }

    // From z on: activates, adds the residual, stores the first `left`.
    template <int C>
    static __device__ void apply(const Gemm& p, int64_t at, int64_t left, float (&o)[C], const float (&r)[C]) {
        float slope;
#pragma unroll
        for (int i = 0; i < C; i++) o[i] = ACT == ANY_ACT ? act_of<false>(p.act, o[i], slope) : act<true, ACT == ANY_ACT ? 0 : ACT>(o[i], slope);
        if (p.res)
#pragma unroll
            for (int i = 0; i < C; i++) o[i] += r[i];
        constexpr int PART = CH < C ? CH : C;
#pragma unroll
        for (int g = 0; g < C; g += PART) {
            if (g >= left) break;
            float part[PART];
#pragma unroll
            for (int i = 0; i < PART; i++) part[i] = o[g + i];
            store_some<PART>((T*)p.out + at + g, left - g, part);
        }
    }
};

// 16-bit outputs alone. 16384 x 4096 -> 1024 with bias and residual takes 65 us (2.1 PFLOP/s), one tile a
// CU: 42% of the matrix cores' time, its start and its end are covered by nothing.
template <class T, int ACT>
__global__ __launch_bounds__(512, 2) void linear8_256_kernel(Gemm p) {
    gemm_256<e4m3, true, true, Epilogue8<T, 2, ACT>>(p);
}

template <class T, int ACT, int TILE, int GROUPS>
__global__ __launch_bounds__(256 * GROUPS, TILE == 64 && GROUPS == 1 ? 3 : 2) void linear8_tile_kernel(Gemm p) {
    gemm_tile<e4m3, true, true, Epilogue8<T, TILE / 32, ACT>, std::conditional_t<sizeof(T) == 4, Widened, Straight>, TILE, GROUPS>(p);
}

// The parts of a split product added in order, and the epilogue: a thread 16 bytes of a row of y.
template <class T, int ACT>
__global__ __launch_bounds__(256) void linear8_join(Gemm p, int64_t first) {
    constexpr int CH = 16 / sizeof(T);
    const int64_t per = (p.N + CH - 1) / CH, id = (first + blockIdx.x) * 256 + threadIdx.x;
    const int64_t m = id / per, n = id % per * CH, at = m * p.N + n, left = p.N - n;
    if (m >= p.M) return;
    float o[CH] = {};
    for (int s = 0; s < p.splits; s++) {
        float v[CH] = {};
        load_some<CH>(p.partial + (int64_t)s * p.M * p.N + at, left, v);
#pragma unroll
        for (int i = 0; i < CH; i++) o[i] += v[i];
    }
    float b[CH] = {}, c[CH] = {}, r[CH] = {};
    if (p.bias) load_some<CH>((const T*)p.bias + n, left, b);
    if (p.res) load_some<CH>((const T*)p.res + at, left, r);
    load_some<CH>(p.col_scale + n, left, c);
    const float s = p.row_scale[m];
#pragma unroll
    for (int i = 0; i < CH; i++) o[i] = fmaf(o[i] * s, c[i], b[i]);
    Epilogue8<T, 2, ACT>::template apply<CH>(p, at, left, o, r);
}

// Few rows of x (up to 16 MT): the weights are read once and that is what it costs, so nothing is
// staged. A workgroup takes 16 outputs; its eight waves take an eighth of k each, straight from memory
// to the matrix cores (a lane 16 bytes of row l % 16, four lanes 64 contiguous bytes), and are added
// through LDS in order. One row of 1024 -> 4096 with GELU (4.2 MB of weights) takes 3.9 us, of which a
// launch and one wave's chain of loads are most.
template <class T, int ACT, int MT>
__global__ __launch_bounds__(512) void linear8_rows_kernel(Gemm p) {
    constexpr int CH = 16, WAVES = 8, AT_ONCE = MT == 1 ? 4 : 2;  // pairs of steps
    using F = vec<e4m3, CH>;
    using FU = typename Anywhere<e4m3, CH>::type;
    __shared__ __align__(16) floatx4 part[WAVES][MT][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16, K = p.K;
    // steps of 128 values of k: one matrix instruction's
    const int steps = (int)((K + 127) / 128), s0 = (int)((int64_t)steps * w / WAVES),
              s1 = (int)((int64_t)steps * (w + 1) / WAVES);
    // rows past the end read the last one's values and are not stored
    const e4m3* bp = (const e4m3*)p.b.ptr + (n0 + r < p.N ? n0 + r : p.N - 1) * p.b.ld;
    const e4m3* ap[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) ap[t] = (const e4m3*)p.a.ptr + (16 * t + r < p.M ? 16 * t + r : p.M - 1) * p.a.ld;
    auto product = [](const F(&b)[2], const F(&a)[2], floatx4 c) {
        if constexpr (sizeof(T) == 4) return Widened::product(b[1], a[1], Widened::product(b[0], a[0], c));
        else return mma(b[0], b[1], a[0], a[1], c);
    };
    floatx4 acc[MT] = {};
    const int whole = (int)(K / 128) < s1 ? (int)(K / 128) : s1;
    int s = s0;
    for (; s + AT_ONCE <= whole; s += AT_ONCE) {
        F b[AT_ONCE][2], a[AT_ONCE][MT][2];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int64_t k = (int64_t)(s + u) * 128 + h * 64 + q * CH;
                b[u][h] = *(const FU*)(bp + k);
#pragma unroll
                for (int t = 0; t < MT; t++) a[u][t][h] = *(const FU*)(ap[t] + k);
            }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
#pragma unroll
            for (int t = 0; t < MT; t++) acc[t] = product(b[u], a[u][t], acc[t]);
    }
    auto chunk = [&](const e4m3* row, int64_t k) {
        F v;
        if (k + CH <= K) {
            v = *(const FU*)(row + k);
        } else {
#pragma unroll
            for (int i = 0; i < CH; i++) v[i] = k + i < K ? row[k + i] : (e4m3)0;
        }
        return v;
    };
    for (; s < s1; s++) {
        const int64_t k = (int64_t)s * 128 + q * CH;
        const F b[2] = {chunk(bp, k), chunk(bp, k + 64)};
#pragma unroll
        for (int t = 0; t < MT; t++) {
            const F a[2] = {chunk(ap[t], k), chunk(ap[t], k + 64)};
            acc[t] = product(b, a, acc[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; t++) part[w][t][lane] = acc[t];
    __syncthreads();
    if (w >= MT) return;
    floatx4 v[1] = {part[0][w][lane]};
#pragma unroll
    for (int i = 1; i < WAVES; i++) v[0] += part[i][w][lane];
    Epilogue8<T, 1, ACT> e;
    e.columns(p, n0 + 4 * q);
    e.row(p, 16 * w + r, v);
}

// The kernel by gemm_time's bfloat16 figures, whose k tiles have as many bytes: at 15 sizes from 33 x
// 1024 -> 4096 to 16384 x 1024 -> 4096 it takes the fastest tile and number of parts or one within 6% of
// it, for outputs of 16 bits and of 32, but for 128 x 4096 -> 1024 (11.3 us, 10.1 with tiles of 64 unsplit).
GemmPlan plan8(int64_t M, int64_t N, int64_t K, int dtype) {
    GemmPlan g;
    if (few_rows(M, N, K / 2)) {  // half of the bytes that its bound on k means
        g.rows = true;
        return g;
    }
    const int64_t kt = (K + 127) / 128;
    double best = 1e30;
    for (int tile : {256, 128, 64}) {
        if (tile == 256 && dtype == DRH_F32) continue;
        const int64_t tiles = (M + tile - 1) / tile * ((N + tile - 1) / tile);
        if (tiles > most_groups(tile == 256 ? 512 : 256)) continue;
        for (int64_t s = 1; s <= 64 && s <= kt; s++) {
            const int64_t per = (kt + s - 1) / s;
            if ((kt + per - 1) / per != s) continue;
            if (s > 1 && (double)s * M * N * 4 > 1e9) break;
            const double t = gemm_time(DRH_BF16, tile, (double)tiles, (int)s, (double)per, (double)M * N);
            if (t < best) best = t, g.tile = tile, g.splits = (int)s;
        }
    }
    if (g.splits > 1) g.bytes = up256((size_t)g.splits * M * N * sizeof(float));
    return g;
}

int check_sizes8(int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws) {
    if (int rc = check_product_sizes(M, N, K, xs, ws)) return rc;
    xs = stride_of(M, xs, K), ws = stride_of(N, ws, K);
    if (K <= 0 || K % 16 || xs % 16 || ws % 16)
        return fail(DRH_ERR_INVALID_ARG, "8-bit rows are whole 16 bytes, and so are their strides");
    // the loads' offsets within a tile
    if (256 * xs >= PAST_END || 256 * ws >= PAST_END) return fail(DRH_ERR_TOO_LARGE, "a row stride of 2^23 and more");
    return DRH_OK;
}

}  // namespace
}  // namespace drh_nn

using namespace drh_nn;

extern "C" {

int drh_linear_8bit_bytes(int64_t rows, int64_t n_out, int64_t n_in, int64_t x_stride, int64_t weight_stride,
                          int dtype, uint64_t* out_bytes) {
    if (!out_bytes || !known_type(dtype)) return fail(DRH_ERR_INVALID_ARG, "unknown element type, or out_bytes is NULL");
    int rc = check_sizes8(rows, n_out, n_in, x_stride, weight_stride);
    if (rc) return rc;
    *out_bytes = rows > 0 ? plan8(rows, n_out, n_in, dtype).bytes : 0;
    return DRH_OK;
}

int drh_linear_8bit(drh_ctx* ctx, const void* x, const float* x_scale, const void* weight, const float* weight_scale,
                    const void* bias, const void* residual, int64_t rows, int64_t n_out, int64_t n_in, int64_t x_stride,
                    int64_t weight_stride, int dtype, int activation, void* y, void* workspace, uint64_t workspace_bytes,
                    void* stream, uint32_t flags) {
    int rc = check_call(ctx, dtype, flags);
    if (rc || (rc = check_sizes8(rows, n_out, n_in, x_stride, weight_stride))) return rc;
    if (activation < DRH_ACT_NONE || activation > DRH_ACT_SILU)
        return fail(DRH_ERR_INVALID_ARG, "unknown activation " + std::to_string(activation));
    if (rows == 0) return DRH_OK;
    if (!x || !x_scale || !weight || !weight_scale || !y)
        return fail(DRH_ERR_INVALID_ARG, "x, weight, their scales and y must not be NULL");
    if (!aligned(x) || !aligned(weight)) return fail(DRH_ERR_INVALID_ARG, "8-bit operands must be 16-byte aligned");
    const GemmPlan plan = plan8(rows, n_out, n_in, dtype);
    if ((rc = check_workspace(plan.bytes, workspace, workspace_bytes))) return rc;
    if (!plan.rows && !plan.tile) return fail(DRH_ERR_TOO_LARGE, "more tiles of the output than a launch holds");
    DeviceGuard dg(ctx->device);
    hipStream_t s = (hipStream_t)stream;
    Gemm p{};
    p.a = {x, stride_of(rows, x_stride, n_in), rows}, p.b = {weight, stride_of(n_out, weight_stride, n_in), n_out};
    p.M = rows, p.N = n_out, p.K = n_in;
    p.bias = bias, p.res = residual, p.out = y, p.act = activation;
    p.row_scale = x_scale, p.col_scale = weight_scale;
    p.splits = plan.splits;
    p.tiles_per_split = (int)(((n_in + 127) / 128 + p.splits - 1) / p.splits);
    p.partial = p.splits > 1 ? (float*)workspace : nullptr;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        with_kernel_act<T>(activation, [&](auto kind) {
            constexpr int ACT = kind.value;
            if (plan.rows) {
                const dim3 groups((unsigned)((n_out + 15) / 16));
                if (rows <= 16) linear8_rows_kernel<T, ACT, 1><<<groups, 512, 0, s>>>(p);
                else if (rows <= 32) linear8_rows_kernel<T, ACT, 2><<<groups, 512, 0, s>>>(p);
                else linear8_rows_kernel<T, ACT, 4><<<groups, 512, 0, s>>>(p);
                return;
            }
            const int64_t tiles = (rows + plan.tile - 1) / plan.tile * ((n_out + plan.tile - 1) / plan.tile);
            const dim3 grid((unsigned)tiles, (unsigned)p.splits);
            const bool alone = tiles * p.splits <= CUS;
            if constexpr (sizeof(T) == 2)
                if (plan.tile == 256) linear8_256_kernel<T, ACT><<<grid, 512, 0, s>>>(p);
            if (plan.tile == 128 && alone) linear8_tile_kernel<T, ACT, 128, 2><<<grid, 512, 0, s>>>(p);
            if (plan.tile == 128 && !alone) linear8_tile_kernel<T, ACT, 128, 1><<<grid, 256, 0, s>>>(p);
            if (plan.tile == 64 && alone) linear8_tile_kernel<T, ACT, 64, 2><<<grid, 512, 0, s>>>(p);
            if (plan.tile == 64 && !alone) linear8_tile_kernel<T, ACT, 64, 1><<<grid, 256, 0, s>>>(p);
            if (p.partial) {
                const int64_t ch = 16 / (int64_t)sizeof(T);
                in_launches((rows * ((n_out + ch - 1) / ch) + 255) / 256, most_groups(256), [&](int64_t first, int64_t count) {
                    linear8_join<T, ACT><<<dim3((unsigned)count), 256, 0, s>>>(p, first);
                });
            }
        });
        return DRH_OK;
    });
    return finish_call(s, flags, "8-bit linear");
}

}  // extern "C"
