// Layer norm over the last dimension, forward and backward.
//
//   mu = mean(x), v = mean((x - mu)^2), r = 1 / sqrt(v + eps), h = (x - mu) r
//   y  = h w + b
//   dx = r (g w - mean(g w) - h mean(g w h)),  dw = sum over rows of g h,  db = sum over rows of g
//
// Every sum, mean, variance and reciprocal is held in 32 bits; the variance is taken
// about the mean in a second sum over the row's registers, so it does not cancel where
// the mean is large. All of it is bound by memory: the forward pass reads a row once and
// writes it once, the backward pass reads two and writes one.

#include "rows.h"

using namespace drh_rt;

namespace drh_nn {
namespace {

// A row is held in the registers of TPR threads, EPT elements each (with_row), up to
// LN_MAX_COLS elements. Thread t's vectors are t, t + TPR, ...
constexpr int LN_MAX_COLS = 256 * 32;

struct LnArgs {
    const void *x, *w, *b, *g;
    void *y, *dx;
    float *mean, *rstd, *part;
    int64_t rows, xs, gs;
    int cols, wf32;
    float eps;
};

// WHOLE: the columns are whole vectors. 16384 x 1024 in bfloat16 (67 MB) take 14 us, 4.7 TB/s;
// 4099 x 1500 in 32 bits (49 MB) 10.7, 4.6; 32768 x 4096 in bfloat16 (537 MB) 90, 6.0.
template <class T, int EPT, int TPR, int THREADS, bool WHOLE, bool ONCE>
__global__ __launch_bounds__(THREADS) void ln_forward(LnArgs p) {
    constexpr int VEC = 16 / sizeof(T), NV = EPT / VEC, RPB = THREADS / TPR;
    const int t = threadIdx.x % TPR, D = p.cols;
    const int64_t row = (int64_t)blockIdx.x * RPB + __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
    const bool live = row < p.rows;  // a workgroup's last rows may not be there; their waves keep to its barriers
    const T* x = (const T*)p.x + row * p.xs;
    float v[NV][VEC];
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int c = (j * TPR + t) * VEC;
        Raw raw = {};
        if (live && c < D) raw = load_raw<WHOLE, ONCE>(x + c, D - c);
        const Elements<T> e = __builtin_bit_cast(Elements<T>, raw);
#pragma unroll
        for (int i = 0; i < VEC; i++) v[j][i] = (float)e[i];
    }
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int i = 0; i < VEC; i++) s += v[j][i];
    row_sums<TPR, THREADS>(s, q, 0);
    const float mu = s / (float)D;
    q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int left = D - (j * TPR + t) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; i++)
            if (WHOLE ? left > 0 : i < left) q = fmaf(v[j][i] - mu, v[j][i] - mu, q);
    }
    s = 0.0f;
    row_sums<TPR, THREADS>(q, s, 1);
    const float r = 1.0f / sqrtf(q / (float)D + p.eps);
    if (!live) return;
    if (t == 0 && p.mean) {
        p.mean[row] = mu;
        p.rstd[row] = r;
    }
    T* y = (T*)p.y + row * D;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int c = (j * TPR + t) * VEC;
        if (c >= D) continue;
        float o[VEC], w[VEC] = {};
#pragma unroll
        for (int i = 0; i < VEC; i++) o[i] = (v[j][i] - mu) * r;
        if (p.w) {
            load_weight<T, WHOLE>(p.w, p.wf32, c, D, w);
#pragma unroll
            for (int i = 0; i < VEC; i++) o[i] *= w[i];
        }
        if (p.b) {
            load_weight<T, WHOLE>(p.b, p.wf32, c, D, w);
#pragma unroll
            for (int i = 0; i < VEC; i++) o[i] += w[i];
        }
        store_some<VEC>(y + c, WHOLE ? VEC : D - c, o);
    }
}

// A workgroup takes every gridDim-th group of THREADS / TPR rows and keeps its columns' sums
// of g h and g in registers; at the end its row groups are added through LDS in order and go
// to the workgroup's own row of p.part, which reduce_columns adds up. A group's next rows are
// on their way while it works on the present ones: the sums over a row wait for all of it, so
// without that a wave's loads and its arithmetic would take turns. 16384 x 1024 in bfloat16 (101 MB)
// take 20 us, 5.0 TB/s; 4099 x 1500 in 32 bits (74 MB) 16.8, 4.4; 32768 x 4096 in bfloat16 (805 MB)
// 171, 4.7: two waves a SIMD with 24 vector operations an element and a sum over LDS a row do not
// hide all of the loads' latency.
template <class T, int EPT, int TPR, int THREADS, int PER_SIMD, bool WHOLE, bool ONCE>
__global__ __launch_bounds__(THREADS, PER_SIMD) void ln_backward(LnArgs p) {
    constexpr int VEC = 16 / sizeof(T), NV = EPT / VEC, GROUPS = THREADS / TPR;
    const int t = threadIdx.x % TPR, D = p.cols;
    const int grp = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);  // a wave's: rows are addressed by scalars
    float w[NV][VEC], aw[NV][VEC], ab[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int c = (j * TPR + t) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; i++) w[j][i] = 1.0f, aw[j][i] = ab[j][i] = 0.0f;
        if (p.w && c < D) load_weight<T, WHOLE>(p.w, p.wf32, c, D, w[j]);
    }
    const float inv = 1.0f / (float)D;
    // A row as it stands in memory; it is widened where it is used, which costs an operation
    // an element and saves the registers of the next row's loads.
    struct Row {
        Raw x[NV], g[NV];
        float mu, r;
    };
    auto fetch = [&](Row& to, int64_t row) {  // past the last row zeros: no term of a sum
        const bool live = row < p.rows;
        to.mu = live ? p.mean[row] : 0.0f;
        to.r = live ? p.rstd[row] : 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = (j * TPR + t) * VEC;
            to.x[j] = to.g[j] = Raw{};
            if (live && c < D) {
                to.x[j] = load_raw<WHOLE, ONCE>((const T*)p.x + row * p.xs + c, D - c);
                to.g[j] = load_raw<WHOLE, ONCE>((const T*)p.g + row * p.gs + c, D - c);
            }
        }
    };
    const int64_t stride = (int64_t)gridDim.x * GROUPS;
    int slot = 0;
    Row now, next;
    fetch(now, (int64_t)blockIdx.x * GROUPS + grp);
    for (int64_t row0 = (int64_t)blockIdx.x * GROUPS; row0 < p.rows; row0 += stride, slot++) {
        const int64_t row = row0 + grp;
        fetch(next, row + stride);
        float sg = 0.0f, sh = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const Elements<T> xe = __builtin_bit_cast(Elements<T>, now.x[j]), ge = __builtin_bit_cast(Elements<T>, now.g[j]);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                // past the row's end g is zero, and with it every term
                const float h = ((float)xe[i] - now.mu) * now.r, g = (float)ge[i], u = g * w[j][i];
                aw[j][i] = fmaf(g, h, aw[j][i]);
                ab[j][i] += g;
                sg += u;
                sh = fmaf(u, h, sh);
            }
        }
        row_sums<TPR, THREADS>(sg, sh, slot);
        sg *= inv;
        sh *= inv;
        if (row < p.rows && p.dx) {
            T* dx = (T*)p.dx + row * D;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int c = (j * TPR + t) * VEC;
                float o[VEC];
                // what was computed from them above is forgotten, so that it holds no registers
                asm volatile("" : "+v"(now.x[j]), "+v"(now.g[j]));
                const Elements<T> xe = __builtin_bit_cast(Elements<T>, now.x[j]), ge = __builtin_bit_cast(Elements<T>, now.g[j]);
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const float h = ((float)xe[i] - now.mu) * now.r, u = (float)ge[i] * w[j][i];
                    o[i] = now.r * (u - sg - h * sh);
                }
                if (c < D) store_some<VEC>(dx + c, WHOLE ? VEC : D - c, o);
            }
        }
        now = next;
    }
    if (!p.part) return;
    __shared__ float sums[GROUPS][TPR * VEC];
    float* out = p.part + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int which = 0; which < 2; which++) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < VEC; i++) sums[grp][t * VEC + i] = which ? ab[j][i] : aw[j][i];
            __syncthreads();
            for (int k = threadIdx.x; k < TPR * VEC; k += THREADS) {
                const int c = j * TPR * VEC + k;
                if (c >= D) break;
                float s = 0.0f;
                for (int i = 0; i < GROUPS; i++) s += sums[i][k];
                out[which * D + c] = s;
            }
        }
}

// Rows wider than the registers hold: a workgroup a row, the row read again from the
// caches for each sum.
constexpr int WIDE = 1024;

template <class T>
__global__ __launch_bounds__(WIDE) void ln_forward_wide(LnArgs p) {
    const int64_t row = blockIdx.x;
    const int D = p.cols;
    const T* x = (const T*)p.x + row * p.xs;
    T* y = (T*)p.y + row * D;
    float s = 0.0f, q = 0.0f;
    for (int c = threadIdx.x; c < D; c += WIDE) s += (float)x[c];
    row_sums<WIDE, WIDE>(s, q, 0);
    const float mu = s / (float)D;
    q = 0.0f;
    for (int c = threadIdx.x; c < D; c += WIDE) q = fmaf((float)x[c] - mu, (float)x[c] - mu, q);
    s = 0.0f;
    row_sums<WIDE, WIDE>(q, s, 1);
    const float r = 1.0f / sqrtf(q / (float)D + p.eps);
    if (threadIdx.x == 0 && p.mean) {
        p.mean[row] = mu;
        p.rstd[row] = r;
    }
    for (int c = threadIdx.x; c < D; c += WIDE) {
        float o[1] = {((float)x[c] - mu) * r}, w[1];
        if (p.w) load_weight<T, true>(p.w, p.wf32, c, D, w), o[0] *= w[0];
        if (p.b) load_weight<T, true>(p.b, p.wf32, c, D, w), o[0] += w[0];
        store<1>(y + c, o);
    }
}

template <class T>
__global__ __launch_bounds__(WIDE) void ln_backward_wide(LnArgs p) {
    const int64_t row = blockIdx.x;
    const int D = p.cols;
    const T* x = (const T*)p.x + row * p.xs;
    const T* g = (const T*)p.g + row * p.gs;
    const float mu = p.mean[row], r = p.rstd[row];
    float sg = 0.0f, sh = 0.0f, w[1] = {1.0f};
    for (int c = threadIdx.x; c < D; c += WIDE) {
        if (p.w) load_weight<T, true>(p.w, p.wf32, c, D, w);
        const float gw = (float)g[c] * w[0];
        sg += gw;
        sh = fmaf(gw, ((float)x[c] - mu) * r, sh);
    }
    row_sums<WIDE, WIDE>(sg, sh, 0);
    sg /= (float)D;
    sh /= (float)D;
    for (int c = threadIdx.x; c < D; c += WIDE) {
        if (p.w) load_weight<T, true>(p.w, p.wf32, c, D, w);
        ((T*)p.dx)[row * D + c] = (T)(r * ((float)g[c] * w[0] - sg - ((float)x[c] - mu) * r * sh));
    }
}

// The wide rows' column sums: a wave owns 64 columns of every gridDim.y-th row.
template <class T>
__global__ __launch_bounds__(64) void ln_columns_wide(LnArgs p) {
    const int c = blockIdx.x * 64 + threadIdx.x;
    if (c >= p.cols) return;
    float sw = 0.0f, sb = 0.0f;
    for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
        const float g = (float)((const T*)p.g)[row * p.gs + c];
        sw = fmaf(g, ((float)((const T*)p.x)[row * p.xs + c] - p.mean[row]) * p.rstd[row], sw);
        sb += g;
    }
    float* out = p.part + (int64_t)blockIdx.y * 2 * p.cols;
    out[c] = sw;
    out[p.cols + c] = sb;
}

// f(threads per row, elements per thread) as constants, for rows of D elements of T: a wave a
// row as far as it goes, then two, four, and eight for the longest of 32 bits. Few threads with
// much to load each: 4096 of bfloat16 in 128 threads took the backward pass 170 us for 32768
// rows, in 256 threads 183.
template <class T, class F>
void with_row(int64_t D, F&& f) {
    using std::integral_constant;
    constexpr int MOST = sizeof(T) == 4 ? 16 : 32;
    auto ept = [&](auto tpr) {
        const int64_t per = (D + tpr.value - 1) / tpr.value;
        if (per <= 8) f(tpr, integral_constant<int, 8>());
        else if (per <= 16) f(tpr, integral_constant<int, 16>());
        else f(tpr, integral_constant<int, MOST>());
    };
    if (D <= 64 * MOST) ept(integral_constant<int, 64>());
    else if (D <= 128 * MOST) ept(integral_constant<int, 128>());
    else if (D <= 256 * MOST) ept(integral_constant<int, 256>());
    else if constexpr (256 * MOST < LN_MAX_COLS) ept(integral_constant<int, 512>());
}

// Of a backward workgroup: its threads and the waves a SIMD that its registers are to allow.
// Accumulators, weights and two rows of 16 elements or more a thread do not fit 128 registers
// (1024 columns of bfloat16, 16384 rows: 25.6 us with two waves a SIMD, 33.9 with four and
// spills). Rows of several waves take a smaller workgroup, since their barriers hold up all of it.
struct LnShape {
    int threads, per_simd;
};
constexpr LnShape ln_shape(int size, int tpr, int ept) {
    return ept >= 16 ? LnShape{512, 2} : tpr > 64 ? LnShape{512, 4} : LnShape{1024, 4};
}

// Workgroups of the backward pass, each with a row of partial sums: as many as run at once.
int64_t ln_backward_groups(int64_t rows, int64_t cols, int dtype) {
    if (cols > LN_MAX_COLS) return rows < 64 ? rows : 64;
    int64_t per = 1, most = 1;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        with_row<T>(cols, [&](auto tpr, auto ept) {
            constexpr LnShape s = ln_shape(sizeof(T), tpr.value, ept.value);
            per = s.threads / tpr.value;
            most = 256 * (s.per_simd * 256 / s.threads);
        });
        return DRH_OK;
    });
    const int64_t need = (rows + per - 1) / per;
    return need < most ? need : most;
}

// f(p) for p's rows, at most `groups` a launch times `per` rows each.
template <class T, class F>
void row_launches(const LnArgs& p, int64_t groups, int64_t per, F&& f) {
    in_launches(p.rows, groups * per, [&](int64_t first, int64_t count) {
        LnArgs q = p;
        auto at = [&](auto ptr, int64_t n) { return ptr ? ptr + n : ptr; };
        q.x = at((const T*)p.x, first * p.xs), q.g = at((const T*)p.g, first * p.gs);
        q.y = at((T*)p.y, first * p.cols), q.dx = at((T*)p.dx, first * p.cols);
        q.mean = at(p.mean, first), q.rstd = at(p.rstd, first);
        q.rows = count;
        f(q, dim3((unsigned)((count + per - 1) / per)));
    });
}

int check_sizes(int64_t rows, int64_t cols) {
    if (rows < 0 || cols <= 0) return fail(DRH_ERR_INVALID_ARG, "rows must not be negative and cols positive");
    if (rows > INT32_MAX || cols > (1 << 30)) return fail(DRH_ERR_TOO_LARGE, "more than 2^31 - 1 rows or 2^30 columns");
    return DRH_OK;
}

int check_ln(drh_ctx* ctx, int64_t rows, int64_t cols, int dtype, int weight_dtype, uint32_t flags) {
    int rc = check_call(ctx, dtype, flags);
    if (rc) return rc;
    if (weight_dtype != dtype && weight_dtype != DRH_F32)
        return fail(DRH_ERR_INVALID_ARG, "weight and bias stand in the input's element type or in 32 bits");
    return check_sizes(rows, cols);
}

}  // namespace
}  // namespace drh_nn

using namespace drh_nn;

extern "C" {

int drh_layer_norm(drh_ctx* ctx, const void* x, const void* weight, const void* bias, int64_t rows, int64_t cols,
                   int64_t x_stride, int dtype, int weight_dtype, float eps, void* y, float* mean, float* rstd,
                   void* stream, uint32_t flags) {
    int rc = check_ln(ctx, rows, cols, dtype, weight_dtype, flags);
    if (rc) return rc;
    if (!(eps >= 0.0f)) return fail(DRH_ERR_INVALID_ARG, "eps must not be negative");
    if (rows == 0) return DRH_OK;
    if (!x || !y || !mean != !rstd)
        return fail(DRH_ERR_INVALID_ARG, "x and y must not be NULL; mean and rstd come together");
    if (rows > 1 && x_stride < 0) return fail(DRH_ERR_INVALID_ARG, "x_stride must not be negative");
    if ((rc = check_span(rows, x_stride))) return rc;
    DeviceGuard dg(ctx->device);
    hipStream_t s = (hipStream_t)stream;
    LnArgs p{};
    p.x = x, p.w = weight, p.b = bias, p.y = y, p.mean = mean, p.rstd = rstd;
    p.rows = rows, p.cols = (int)cols, p.xs = x_stride, p.eps = eps, p.wf32 = weight_dtype == DRH_F32;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (cols > LN_MAX_COLS) {
            row_launches<T>(p, most_groups(WIDE), 1,
                            [&](const LnArgs& q, dim3 grid) { ln_forward_wide<T><<<grid, WIDE, 0, s>>>(q); });
            return DRH_OK;
        }
        with_row<T>(cols, [&](auto tpr, auto ept) {
            constexpr int THREADS = tpr.value > 256 ? tpr.value : 256, RPB = THREADS / tpr.value;
            with_loads<T>(rows, cols, [&](auto whole, auto once) {
                row_launches<T>(p, most_groups(THREADS), RPB, [&](const LnArgs& q, dim3 grid) {
                    ln_forward<T, ept.value, tpr.value, THREADS, whole.value, once.value><<<grid, THREADS, 0, s>>>(q);
                });
            });
        });
        return DRH_OK;
    });
    return finish_call(s, flags, "layer norm");
}

int drh_layer_norm_backward_bytes(int64_t rows, int64_t cols, int dtype, uint64_t* out_bytes) {
    if (!out_bytes || !known_type(dtype)) return fail(DRH_ERR_INVALID_ARG, "unknown element type, or out_bytes is NULL");
    int rc = check_sizes(rows, cols);
    if (rc) return rc;
    *out_bytes = up256((size_t)ln_backward_groups(rows, cols, dtype) * 2 * (size_t)cols * sizeof(float));
    return DRH_OK;
}

int drh_layer_norm_backward(drh_ctx* ctx, const void* x, const void* weight, const float* mean, const float* rstd,
                            const void* grad_y, int64_t rows, int64_t cols, int64_t x_stride, int64_t grad_stride,
                            int dtype, int weight_dtype, void* grad_x, void* grad_weight, void* grad_bias,
                            void* workspace, uint64_t workspace_bytes, void* stream, uint32_t flags) {
    int rc = check_ln(ctx, rows, cols, dtype, weight_dtype, flags);
    if (rc) return rc;
    const bool sums = grad_weight || grad_bias;
    if (rows > 0 && (!x || !mean || !rstd || !grad_y)) return fail(DRH_ERR_INVALID_ARG, "an input pointer is NULL");
    if (rows > 1 && (x_stride < 0 || grad_stride < 0)) return fail(DRH_ERR_INVALID_ARG, "strides must not be negative");
    if ((rc = check_span(rows, x_stride)) || (rc = check_span(rows, grad_stride))) return rc;
    uint64_t need = 0;
    if (sums) drh_layer_norm_backward_bytes(rows, cols, dtype, &need);
    if (sums && (workspace_bytes < need || (need && !workspace)))
        return fail(DRH_ERR_INVALID_ARG, "the weight's gradient needs " + std::to_string(need) + " bytes of workspace");
    if ((uintptr_t)workspace % 16) return fail(DRH_ERR_INVALID_ARG, "the workspace must be 16-byte aligned");
    DeviceGuard dg(ctx->device);
    hipStream_t s = (hipStream_t)stream;
    const int64_t groups = ln_backward_groups(rows, cols, dtype);
    LnArgs p{};
    p.x = x, p.w = weight, p.g = grad_y, p.dx = grad_x, p.mean = (float*)mean, p.rstd = (float*)rstd;
    p.part = sums ? (float*)workspace : nullptr;
    p.rows = rows, p.cols = (int)cols, p.xs = x_stride, p.gs = grad_stride, p.wf32 = weight_dtype == DRH_F32;
    if (rows > 0 && (grad_x || sums))
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            if (cols > LN_MAX_COLS) {
                if (grad_x)
                    row_launches<T>(p, most_groups(WIDE), 1,
                                    [&](const LnArgs& q, dim3 grid) { ln_backward_wide<T><<<grid, WIDE, 0, s>>>(q); });
                if (sums)
                    ln_columns_wide<T><<<dim3((unsigned)((cols + 63) / 64), (unsigned)groups), 64, 0, s>>>(p);
                return DRH_OK;
            }
            with_row<T>(cols, [&](auto tpr, auto ept) {
                constexpr LnShape sh = ln_shape(sizeof(T), tpr.value, ept.value);
                const dim3 grid((unsigned)groups);
                with_loads<T>(rows, cols, [&](auto whole, auto once) {
                    ln_backward<T, ept.value, tpr.value, sh.threads, sh.per_simd, whole.value, once.value>
                        <<<grid, sh.threads, 0, s>>>(p);
                });
            });
            return DRH_OK;
        });
    if (sums)
        reduce_columns((const float*)workspace, groups, 2 * cols, cols, grad_weight, grad_bias, weight_dtype, s);
    return finish_call(s, flags, "layer norm backward");
}

}  // extern "C"
