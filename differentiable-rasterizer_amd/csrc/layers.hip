// What the network layers share on the host, and the second step of their column
// sums (a layer norm's weight gradient, a linear layer's bias gradient).

#include "layers.h"

using namespace drh_rt;

namespace drh_nn {
namespace {

// Sixteen waves a workgroup, 64 columns each, so that a wave reads 256 contiguous
// bytes of a partial row; the waves take every sixteenth row and are added in order. The partial
// sums are 1 to 8 MB and still in the caches: 4 to 5 us, hardly more than a launch.
constexpr int RC_WAVES = 16;
template <class T>
__global__ __launch_bounds__(64 * RC_WAVES) void reduce_columns_kernel(const float* __restrict__ part, int64_t groups,
                                                                       int64_t stride, int64_t cols, int64_t first,
                                                                       T* out_a, T* out_b) {
    __shared__ float sums[RC_WAVES][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t col = first + (int64_t)blockIdx.x * 64 + lane, n = out_b ? 2 * cols : cols;
    float s = 0.0f;
    if (col < n)
#pragma unroll 4
        for (int64_t g = w; g < groups; g += RC_WAVES) s += part[g * stride + col];
    sums[w][lane] = s;
    __syncthreads();
    if (w == 0 && col < n) {
#pragma unroll
        for (int i = 1; i < RC_WAVES; i++) s += sums[i][lane];
        if (col < cols) {
            if (out_a) out_a[col] = (T)s;
        } else {
            out_b[col - cols] = (T)s;
        }
    }
}

}  // namespace

int check_call(drh_ctx* ctx, int dtype, uint32_t flags) {
    if (!ctx) return fail(DRH_ERR_INVALID_ARG, "context is NULL");
    if (!known_type(dtype)) return fail(DRH_ERR_INVALID_ARG, "unknown element type " + std::to_string(dtype));
    if (flags & ~DRH_SYNC)
        return fail(DRH_ERR_INVALID_ARG, "the network layers take device pointers, and DRH_SYNC as their only flag");
    return DRH_OK;
}

int check_span(int64_t rows, int64_t stride) {
    if (rows <= 1 || stride <= (1ll << 48) / rows) return DRH_OK;
    return fail(DRH_ERR_TOO_LARGE, "an array of more than 2^48 elements");
}

int finish_call(hipStream_t s, uint32_t flags, const char* what) {
    HIP_TRY(hipGetLastError(), what);
    return (flags & DRH_SYNC) ? wait_stream(s) : DRH_OK;
}

int reduce_columns(const float* part, int64_t groups, int64_t stride, int64_t cols, void* out_a, void* out_b,
                   int out_dtype, hipStream_t s) {
    const int64_t n = out_b ? 2 * cols : cols;
    if (n == 0) return DRH_OK;
    return with_type(out_dtype, [&](auto t) {
        using T = decltype(t);
        in_launches((n + 63) / 64, most_groups(64 * RC_WAVES), [&](int64_t first, int64_t count) {
            reduce_columns_kernel<T><<<dim3((unsigned)count), 64 * RC_WAVES, 0, s>>>(part, groups, stride, cols, first * 64,
                                                                                     (T*)out_a, (T*)out_b);
        });
        return DRH_OK;
    });
}

}  // namespace drh_nn
