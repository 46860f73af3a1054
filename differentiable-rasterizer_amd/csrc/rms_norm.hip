// Root-mean-square norm over the last dimension with the residual's addition in front,
// forward (also with an output in 8 bits) and backward:
//
//   s = x + residual,  r = 1 / sqrt(mean(s^2) + eps),  h = s r,  y = h w
//   q = e4m3(y / t),   t = max(max |y| / 448, 2^-126), a row's scale
//   dx = dresidual = r (g w - h mean(g w h)) + gs,  dw = sum over rows of g h
//
// with g and gs the gradients of y and s. Sums and means are held in 32 bits. y is made from the
// unrounded s; s is rounded to its type where it is stored, and the backward pass reads that (the
// only record of it), so its h is half a step of the type off, and beside bfloat16 dw is 0.0025 of
// itself off where a whole s would leave 0.0018: x and the residual in its place are an array more to
// read, a quarter of what the backward pass moves. All of it is bound by memory: the forward pass
// reads two arrays and writes two, the backward pass reads three and writes one.

#include "e4m3.h"
#include "rows.h"

using namespace drh_rt;

namespace drh_nn {
namespace {

// A row is held in the registers of TPR threads, up to EPT elements each (with_row); thread t's
// vectors are t, t + TPR, ... Longer rows are read again for each sum. Sixteen elements a thread are
// faster than 32 of 16 bits, in twice the threads: 32768 x 4096 in bfloat16 176 and 183 us forward.
constexpr int MOST_EPT = 16;
template <class T>
constexpr int64_t FORWARD_COLS = 1024 * (sizeof(T) == 4 ? MOST_EPT : 2 * MOST_EPT);
constexpr int64_t BACKWARD_COLS = 512 * MOST_EPT;

struct RmsArgs {
    const void *x, *res, *w, *g, *gs;
    void *y, *sum, *dx;
    float *rstd, *scale, *part;
    int64_t rows, xs, rs, gst, gss;  // strides of x (or s), the residual, g, gs
    int cols, wf32;
    bool norm;  // else y = s: rows to 8 bits alone
    float eps;
};

// WHOLE: the columns are whole vectors. CODES: y goes out as e4m3 with a scale a row. ONCE: loads and
// stores past the caches. With a residual 32768 x 4096 in bfloat16 (1.07 GB) take 176 us, 6.1 TB/s (190
// with ordinary stores), 131072 x 512 85, 6.3; 4099 x 1500 in 32 bits, without, 10.7, 4.6.
template <class T, bool CODES, int EPT, int TPR, int THREADS, bool WHOLE, bool ONCE>
__global__ __launch_bounds__(THREADS) void rms_forward(RmsArgs p) {
    constexpr int VEC = 16 / sizeof(T), NV = EPT / VEC, RPB = THREADS / TPR;
    const int t = threadIdx.x % TPR, D = p.cols;
    const int64_t row = (int64_t)blockIdx.x * RPB + __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
    const bool live = row < p.rows;  // a workgroup's last rows may not be there; their waves keep to its barriers
    const T* x = (const T*)p.x + row * p.xs;
    const T* res = (const T*)p.res + row * p.rs;
    Raw xr[NV], rr[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int c = (j * TPR + t) * VEC;
        xr[j] = rr[j] = Raw{};
        if (live && c < D) {
            xr[j] = load_raw<WHOLE, ONCE>(x + c, D - c);
            if (p.res) rr[j] = load_raw<WHOLE, ONCE>(res + c, D - c);
        }
    }
    float v[NV][VEC];
    float q = 0.0f, unused = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const Elements<T> xe = __builtin_bit_cast(Elements<T>, xr[j]), re = __builtin_bit_cast(Elements<T>, rr[j]);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            v[j][i] = p.res ? (float)xe[i] + (float)re[i] : (float)xe[i];
            q = fmaf(v[j][i], v[j][i], q);
        }
    }
    if (p.sum && live) {
        T* sum = (T*)p.sum + row * D;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = (j * TPR + t) * VEC;
            if (c < D) store_once<ONCE, VEC>(sum + c, WHOLE ? VEC : D - c, v[j]);
        }
    }
    if (!CODES || p.norm) {
        row_sums<TPR, THREADS>(q, unused, 0);
        const float r = 1.0f / sqrtf(q / (float)D + p.eps);
        if (live && t == 0 && p.rstd) p.rstd[row] = r;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = (j * TPR + t) * VEC;
            float w[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) w[i] = 1.0f;
            if (p.w && c < D) load_weight<T, WHOLE>(p.w, p.wf32, c, D, w);
#pragma unroll
            for (int i = 0; i < VEC; i++) v[j][i] *= r * w[i];
        }
    }
    if constexpr (CODES) {
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int i = 0; i < VEC; i++) most = fmaxf(most, fabsf(v[j][i]));  // zeros past the row's end
        most = row_max<TPR, THREADS>(most);
        const float scale = fmaxf(most / E4M3_MOST, LEAST_SCALE);
        if (!live) return;
        if (t == 0) p.scale[row] = scale;
        const RowDivisor by(scale);
        uint8_t* y = (uint8_t*)p.y + row * D;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = (j * TPR + t) * VEC;
            uint32_t codes[VEC / 4];
#pragma unroll
            for (int i = 0; i < VEC; i++) v[j][i] = by.of(v[j][i]);
            to_e4m3<VEC>(v[j], codes);
            if (c < D) store_codes<WHOLE, VEC>(y + c, D - c, codes);
        }
    } else {
        if (!live) return;
        T* y = (T*)p.y + row * D;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = (j * TPR + t) * VEC;
            if (c < D) store_once<ONCE, VEC>(y + c, WHOLE ? VEC : D - c, v[j]);
        }
    }
}

// A workgroup takes every gridDim-th group of THREADS / TPR rows and keeps its columns' sums of g h
// in registers; at the end its row groups are added through LDS in order and go to the workgroup's
// own row of p.part, which reduce_columns adds up. A group's next rows are on their way while it
// works on the present ones. With a residual's gradient 32768 x 4096 in bfloat16 (1.07 GB) take 178 us,
// 6.1 TB/s with the column sums' second step, 32768 x 1500 in 32 bits, without, 104, 5.7.
template <class T, int EPT, int TPR, int THREADS, int PER_SIMD, bool WHOLE, bool ONCE>
__global__ __launch_bounds__(THREADS, PER_SIMD) void rms_backward(RmsArgs p) {
    constexpr int VEC = 16 / sizeof(T), NV = EPT / VEC, GROUPS = THREADS / TPR;
    const int t = threadIdx.x % TPR, D = p.cols;
    const int grp = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);  // a wave's: rows are addressed by scalars
    float w[NV][VEC], aw[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int c = (j * TPR + t) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; i++) w[j][i] = 1.0f, aw[j][i] = 0.0f;
        if (p.w && c < D) load_weight<T, WHOLE>(p.w, p.wf32, c, D, w[j]);
    }
    const float inv = 1.0f / (float)D;
    // A row as it stands in memory; it is widened where it is used, which costs an operation
    // an element and saves the registers of the next row's loads.
    struct Row {
        Raw x[NV], g[NV], gs[NV];
        float r;
    };
    auto fetch = [&](Row& to, int64_t row) {  // past the last row zeros: no term of a sum
        const bool live = row < p.rows;
        to.r = live ? p.rstd[row] : 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = (j * TPR + t) * VEC;
            to.x[j] = to.g[j] = to.gs[j] = Raw{};
            if (live && c < D) {
                to.x[j] = load_raw<WHOLE, ONCE>((const T*)p.x + row * p.xs + c, D - c);
                to.g[j] = load_raw<WHOLE, ONCE>((const T*)p.g + row * p.gst + c, D - c);
                if (p.gs) to.gs[j] = load_raw<WHOLE, ONCE>((const T*)p.gs + row * p.gss + c, D - c);
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
        float sh = 0.0f, unused = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const Elements<T> xe = __builtin_bit_cast(Elements<T>, now.x[j]), ge = __builtin_bit_cast(Elements<T>, now.g[j]);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                // past the row's end both are zero
                const float h = (float)xe[i] * now.r, g = (float)ge[i];
                aw[j][i] = fmaf(g, h, aw[j][i]);
                sh = fmaf(g * w[j][i], h, sh);
            }
        }
        if (p.dx) {
            row_sums<TPR, THREADS>(sh, unused, slot);
            const float m = sh * inv * now.r;
            if (row < p.rows) {
                T* dx = (T*)p.dx + row * D;
#pragma unroll
                for (int j = 0; j < NV; j++) {
                    const int c = (j * TPR + t) * VEC;
                    float o[VEC];
                    // what was computed from them above is forgotten, so that it holds no registers
                    asm volatile("" : "+v"(now.x[j]), "+v"(now.g[j]));
                    const Elements<T> xe = __builtin_bit_cast(Elements<T>, now.x[j]), ge = __builtin_bit_cast(Elements<T>, now.g[j]),
                                      se = __builtin_bit_cast(Elements<T>, now.gs[j]);
#pragma unroll
                    for (int i = 0; i < VEC; i++) o[i] = fmaf(now.r, (float)ge[i] * w[j][i] - (float)xe[i] * m, (float)se[i]);
                    if (c < D) store_once<ONCE, VEC>(dx + c, WHOLE ? VEC : D - c, o);
                }
            }
        }
        now = next;
    }
    if (!p.part) return;
    __shared__ float sums[GROUPS][TPR * VEC];
    float* out = p.part + (int64_t)blockIdx.x * D;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VEC; i++) sums[grp][t * VEC + i] = aw[j][i];
        __syncthreads();
        for (int k = threadIdx.x; k < TPR * VEC; k += THREADS) {
            const int c = j * TPR * VEC + k;
            if (c >= D) break;
            float s = 0.0f;
            for (int i = 0; i < GROUPS; i++) s += sums[i][k];
            out[c] = s;
        }
    }
}

// Rows longer than the registers hold: a workgroup a row, the row read again from the caches
// for each sum.
constexpr int WIDE = 1024;

template <class T, bool CODES>
__global__ __launch_bounds__(WIDE) void rms_forward_wide(RmsArgs p) {
    const int64_t row = blockIdx.x;
    const int D = p.cols;
    const T* x = (const T*)p.x + row * p.xs;
    const T* res = (const T*)p.res + row * p.rs;
    auto at = [&](int c) { return p.res ? (float)x[c] + (float)res[c] : (float)x[c]; };
    float r = 1.0f;
    if (!CODES || p.norm) {
        float q = 0.0f, unused = 0.0f;
        for (int c = threadIdx.x; c < D; c += WIDE) q = fmaf(at(c), at(c), q);
        row_sums<WIDE, WIDE>(q, unused, 0);
        r = 1.0f / sqrtf(q / (float)D + p.eps);
        if (threadIdx.x == 0 && p.rstd) p.rstd[row] = r;
    }
    auto value = [&](int c) {
        float w[1] = {1.0f};
        if (p.w) load_weight<T, true>(p.w, p.wf32, c, D, w);
        return at(c) * (r * w[0]);
    };
    float scale = 1.0f;
    if constexpr (CODES) {
        float most = 0.0f;
        for (int c = threadIdx.x; c < D; c += WIDE) most = fmaxf(most, fabsf(value(c)));
        scale = fmaxf(row_max<WIDE, WIDE>(most) / E4M3_MOST, LEAST_SCALE);
        if (threadIdx.x == 0) p.scale[row] = scale;
    }
    const RowDivisor by(scale);
    for (int c = threadIdx.x; c < D; c += WIDE) {
        const float s = at(c), y = value(c);
        if constexpr (CODES)
            ((uint8_t*)p.y)[row * D + c] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(by.of(y), 0.0f, 0, false);
        else
            ((T*)p.y)[row * D + c] = (T)y;
        if (p.sum) ((T*)p.sum)[row * D + c] = (T)s;
    }
}

template <class T>
__global__ __launch_bounds__(WIDE) void rms_backward_wide(RmsArgs p) {
    const int64_t row = blockIdx.x;
    const int D = p.cols;
    const T* x = (const T*)p.x + row * p.xs;
    const T* g = (const T*)p.g + row * p.gst;
    const T* gs = (const T*)p.gs + row * p.gss;
    const float r = p.rstd[row];
    float sh = 0.0f, unused = 0.0f, w[1] = {1.0f};
    for (int c = threadIdx.x; c < D; c += WIDE) {
        if (p.w) load_weight<T, true>(p.w, p.wf32, c, D, w);
        sh = fmaf((float)g[c] * w[0], (float)x[c] * r, sh);
    }
    row_sums<WIDE, WIDE>(sh, unused, 0);
    const float m = sh / (float)D * r;
    for (int c = threadIdx.x; c < D; c += WIDE) {
        if (p.w) load_weight<T, true>(p.w, p.wf32, c, D, w);
        ((T*)p.dx)[row * D + c] = (T)fmaf(r, (float)g[c] * w[0] - (float)x[c] * m, p.gs ? (float)gs[c] : 0.0f);
    }
}

// The wide rows' column sums: a wave owns 64 columns of every gridDim.y-th row.
template <class T>
__global__ __launch_bounds__(64) void rms_columns_wide(RmsArgs p) {
    const int c = blockIdx.x * 64 + threadIdx.x;
    if (c >= p.cols) return;
    float s = 0.0f;
    for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y)
        s = fmaf((float)((const T*)p.g)[row * p.gst + c], (float)((const T*)p.x)[row * p.xs + c] * p.rstd[row], s);
    p.part[(int64_t)blockIdx.y * p.cols + c] = s;
}

// f(threads per row, elements per thread) as constants, for rows of D elements: a wave a row as far
// as it goes, then two, four, eight and (forward) sixteen, of twice the elements for the longest of 16 bits.
template <bool FORWARD, class T, class F>
void with_row(int64_t D, F&& f) {
    using std::integral_constant;
    using Most = integral_constant<int, MOST_EPT>;
    if (D <= 64 * 8) f(integral_constant<int, 64>(), integral_constant<int, 8>());
    else if (D <= 64 * MOST_EPT) f(integral_constant<int, 64>(), Most());
    else if (D <= 128 * MOST_EPT) f(integral_constant<int, 128>(), Most());
    else if (D <= 256 * MOST_EPT) f(integral_constant<int, 256>(), Most());
    else if (D <= 512 * MOST_EPT) f(integral_constant<int, 512>(), Most());
    else if constexpr (FORWARD) {
        if (D <= 1024 * MOST_EPT) f(integral_constant<int, 1024>(), Most());
        else if constexpr (sizeof(T) == 2) f(integral_constant<int, 1024>(), integral_constant<int, 2 * MOST_EPT>());
    }
}

// Of a backward workgroup: its threads and the waves a SIMD that its registers are to allow. Three arrays,
// two rows of them, weights and sums of 16 elements a thread want 150 registers, and with two waves a
// SIMD and half the partial rows it is faster than with three: 32768 x 4096 in bfloat16 183 and 203 us.
struct RmsShape {
    int threads, per_simd;
};
constexpr RmsShape rms_shape(int size, int tpr, int ept) {
    return ept < 16 ? RmsShape{1024, 4} : size == 4 || tpr > 256 ? RmsShape{512, 2} : RmsShape{256, 2};
}

// Workgroups of the backward pass, each with a row of partial sums: as many as run at once.
int64_t rms_backward_groups(int64_t rows, int64_t cols, int dtype) {
    int64_t n = 0;
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (cols > BACKWARD_COLS) {
            n = rows < 64 ? rows : 64;
            return DRH_OK;
        }
        with_row<false, T>(cols, [&](auto tpr, auto ept) {
            constexpr RmsShape s = rms_shape(sizeof(T), tpr.value, ept.value);
            const int64_t per = s.threads / tpr.value, most = 256 * (s.per_simd * 256 / s.threads), need = (rows + per - 1) / per;
            n = need < most ? need : most;
        });
        return DRH_OK;
    });
    return n;
}

// f(p) for p's rows, at most `groups` a launch times `per` rows each.
template <class T, class F>
void row_launches(const RmsArgs& p, bool codes, int64_t groups, int64_t per, F&& f) {
    in_launches(p.rows, groups * per, [&](int64_t first, int64_t count) {
        RmsArgs q = p;
        auto at = [&](auto ptr, int64_t n) { return ptr ? ptr + n : ptr; };
        q.x = at((const T*)p.x, first * p.xs), q.res = at((const T*)p.res, first * p.rs);
        q.g = at((const T*)p.g, first * p.gst), q.gs = at((const T*)p.gs, first * p.gss);
        q.y = at((char*)p.y, first * p.cols * (codes ? 1 : (int64_t)sizeof(T)));
        q.sum = at((T*)p.sum, first * p.cols), q.dx = at((T*)p.dx, first * p.cols);
        q.rstd = at(p.rstd, first), q.scale = at(p.scale, first);
        q.rows = count;
        f(q, dim3((unsigned)((count + per - 1) / per)));
    });
}

int check_sizes(int64_t rows, int64_t cols) {
    if (rows < 0 || cols <= 0) return fail(DRH_ERR_INVALID_ARG, "rows must not be negative and cols positive");
    if (rows > INT32_MAX || cols > (1 << 30)) return fail(DRH_ERR_TOO_LARGE, "more than 2^31 - 1 rows or 2^30 columns");
    return DRH_OK;
}

int check_strides(int64_t rows, std::initializer_list<int64_t> strides) {
    for (int64_t s : strides) {
        if (rows > 1 && s < 0) return fail(DRH_ERR_INVALID_ARG, "strides must not be negative");
        if (int rc = check_span(rows, s)) return rc;
    }
    return DRH_OK;
}

int check_rms(drh_ctx* ctx, int64_t rows, int64_t cols, int dtype, int weight_dtype, uint32_t flags) {
    int rc = check_call(ctx, dtype, flags);
    if (rc) return rc;
    if (weight_dtype != dtype && weight_dtype != DRH_F32)
        return fail(DRH_ERR_INVALID_ARG, "the weight stands in the input's element type or in 32 bits");
    return check_sizes(rows, cols);
}

template <bool CODES>
int forward(const RmsArgs& p, int dtype, hipStream_t s, uint32_t flags, const char* what) {
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (p.cols > FORWARD_COLS<T>) {
            row_launches<T>(p, CODES, most_groups(WIDE), 1,
                            [&](const RmsArgs& q, dim3 grid) { rms_forward_wide<T, CODES><<<grid, WIDE, 0, s>>>(q); });
            return DRH_OK;
        }
        with_row<true, T>(p.cols, [&](auto tpr, auto ept) {
            constexpr int THREADS = tpr.value > 256 ? tpr.value : 256, RPB = THREADS / tpr.value;
            with_loads<T>(p.rows, p.cols, [&](auto whole, auto once) {
                row_launches<T>(p, CODES, most_groups(THREADS), RPB, [&](const RmsArgs& q, dim3 grid) {
                    rms_forward<T, CODES, ept.value, tpr.value, THREADS, whole.value, once.value><<<grid, THREADS, 0, s>>>(q);
                });
            });
        });
        return DRH_OK;
    });
    return finish_call(s, flags, what);
}

}  // namespace
}  // namespace drh_nn

using namespace drh_nn;

extern "C" {

int drh_rms_norm(drh_ctx* ctx, const void* x, const void* residual, const void* weight, int64_t rows, int64_t cols,
                 int64_t x_stride, int64_t residual_stride, int dtype, int weight_dtype, float eps, void* y, void* sum,
                 float* rstd, void* stream, uint32_t flags) {
    int rc = check_rms(ctx, rows, cols, dtype, weight_dtype, flags);
    if (rc) return rc;
    if (!(eps >= 0.0f)) return fail(DRH_ERR_INVALID_ARG, "eps must not be negative");
    if ((rc = check_strides(rows, {x_stride, residual ? residual_stride : 0}))) return rc;
    if (rows == 0) return DRH_OK;
    if (!x || !y) return fail(DRH_ERR_INVALID_ARG, "x and y must not be NULL");
    if (sum && !residual) return fail(DRH_ERR_INVALID_ARG, "there is no sum without a residual");
    DeviceGuard dg(ctx->device);
    RmsArgs p{};
    p.x = x, p.res = residual, p.w = weight, p.y = y, p.sum = sum, p.rstd = rstd;
    p.rows = rows, p.cols = (int)cols, p.xs = x_stride, p.rs = residual_stride;
    p.norm = true, p.eps = eps, p.wf32 = weight_dtype == DRH_F32;
    return forward<false>(p, dtype, (hipStream_t)stream, flags, "rms norm");
}

int drh_rms_norm_8bit(drh_ctx* ctx, const void* x, const void* residual, const void* weight, int64_t rows, int64_t cols,
                      int64_t x_stride, int64_t residual_stride, int dtype, int weight_dtype, float eps, void* y,
                      float* scale, void* sum, void* stream, uint32_t flags) {
    int rc = check_rms(ctx, rows, cols, dtype, weight_dtype, flags);
    if (rc) return rc;
    if (!(eps >= 0.0f)) return fail(DRH_ERR_INVALID_ARG, "eps must not be negative");
    if ((rc = check_strides(rows, {x_stride, residual ? residual_stride : 0}))) return rc;
    if (rows == 0) return DRH_OK;
    if (!x || !y || !scale) return fail(DRH_ERR_INVALID_ARG, "x, y and scale must not be NULL");
    if (sum && !residual) return fail(DRH_ERR_INVALID_ARG, "there is no sum without a residual");
    DeviceGuard dg(ctx->device);
    RmsArgs p{};
    p.x = x, p.res = residual, p.w = weight, p.y = y, p.sum = sum, p.scale = scale;
    p.rows = rows, p.cols = (int)cols, p.xs = x_stride, p.rs = residual_stride;
    p.norm = true, p.eps = eps, p.wf32 = weight_dtype == DRH_F32;
    return forward<true>(p, dtype, (hipStream_t)stream, flags, "rms norm to 8 bits");
}

int drh_quantize_8bit(drh_ctx* ctx, const void* x, int64_t rows, int64_t cols, int64_t x_stride, int dtype, void* y,
                      float* scale, void* stream, uint32_t flags) {
    int rc = check_rms(ctx, rows, cols, dtype, dtype, flags);
    if (rc || (rc = check_strides(rows, {x_stride}))) return rc;
    if (rows == 0) return DRH_OK;
    if (!x || !y || !scale) return fail(DRH_ERR_INVALID_ARG, "x, y and scale must not be NULL");
    DeviceGuard dg(ctx->device);
    RmsArgs p{};
    p.x = x, p.y = y, p.scale = scale, p.rows = rows, p.cols = (int)cols, p.xs = x_stride;
    return forward<true>(p, dtype, (hipStream_t)stream, flags, "rows to 8 bits");
}

int drh_rms_norm_backward_bytes(int64_t rows, int64_t cols, int dtype, uint64_t* out_bytes) {
    if (!out_bytes || !known_type(dtype)) return fail(DRH_ERR_INVALID_ARG, "unknown element type, or out_bytes is NULL");
    int rc = check_sizes(rows, cols);
    if (rc) return rc;
    *out_bytes = up256((size_t)rms_backward_groups(rows, cols, dtype) * (size_t)cols * sizeof(float));
    return DRH_OK;
}

int drh_rms_norm_backward(drh_ctx* ctx, const void* sum, const void* weight, const float* rstd, const void* grad_y,
                          const void* grad_sum, int64_t rows, int64_t cols, int64_t sum_stride, int64_t grad_y_stride,
                          int64_t grad_sum_stride, int dtype, int weight_dtype, void* grad_x, void* grad_weight,
                          void* workspace, uint64_t workspace_bytes, void* stream, uint32_t flags) {
    int rc = check_rms(ctx, rows, cols, dtype, weight_dtype, flags);
    if (rc || (rc = check_strides(rows, {sum_stride, grad_y_stride, grad_sum ? grad_sum_stride : 0}))) return rc;
    if (rows > 0 && (!sum || !rstd || !grad_y)) return fail(DRH_ERR_INVALID_ARG, "an input pointer is NULL");
    uint64_t need = 0;
    if (grad_weight) drh_rms_norm_backward_bytes(rows, cols, dtype, &need);
    if (grad_weight && (workspace_bytes < need || (need && !workspace)))
        return fail(DRH_ERR_INVALID_ARG, "the weight's gradient needs " + std::to_string(need) + " bytes of workspace");
    if ((uintptr_t)workspace % 16) return fail(DRH_ERR_INVALID_ARG, "the workspace must be 16-byte aligned");
    DeviceGuard dg(ctx->device);
    hipStream_t s = (hipStream_t)stream;
    const int64_t groups = rms_backward_groups(rows, cols, dtype);
    RmsArgs p{};
    p.x = sum, p.w = weight, p.g = grad_y, p.gs = grad_sum, p.dx = grad_x, p.rstd = (float*)rstd;
    p.part = grad_weight ? (float*)workspace : nullptr;
    p.rows = rows, p.cols = (int)cols, p.xs = sum_stride, p.gst = grad_y_stride, p.gss = grad_sum_stride;
    p.wf32 = weight_dtype == DRH_F32;
    if (rows > 0 && (grad_x || grad_weight))
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            if (cols > BACKWARD_COLS) {
                if (grad_x)
                    row_launches<T>(p, false, most_groups(WIDE), 1,
                                    [&](const RmsArgs& q, dim3 grid) { rms_backward_wide<T><<<grid, WIDE, 0, s>>>(q); });
                if (grad_weight)
                    rms_columns_wide<T><<<dim3((unsigned)((cols + 63) / 64), (unsigned)groups), 64, 0, s>>>(p);
                return DRH_OK;
            }
            with_row<false, T>(cols, [&](auto tpr, auto ept) {
                constexpr RmsShape sh = rms_shape(sizeof(T), tpr.value, ept.value);
                const dim3 grid((unsigned)groups);
                with_loads<T>(rows, cols, [&](auto whole, auto once) {
                    rms_backward<T, ept.value, tpr.value, sh.threads, sh.per_simd, whole.value, once.value>
                        <<<grid, sh.threads, 0, s>>>(p);
                });
            });
            return DRH_OK;
        });
    if (grad_weight) reduce_columns((const float*)workspace, groups, cols, cols, grad_weight, nullptr, weight_dtype, s);
    return finish_call(s, flags, "rms norm backward");
}

}  // extern "C"
