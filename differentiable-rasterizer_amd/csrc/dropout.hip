// Dropout whose mask is never stored: both passes draw it again from a counter-based
// generator.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2,
// 3", 2011): ten rounds over the counter (element / 8, offset) with the key `seed` give
// four 32-bit words, and element i takes the 16-bit half i % 2 of word (i % 8) / 2. It is
// dropped where that number is below t = round(p 2^16); what stays is multiplied by
// 2^16 / (2^16 - t), the inverse of the probability that is really applied, so the mean is
// kept exactly. 16 bits a draw, not 32: a thread's 16-byte vector of 16-bit elements then
// takes one evaluation (about 60 integer operations, a third of them at a quarter rate),
// which memory hides.

#include <cmath>

#include "layers.h"

using namespace drh_rt;

namespace drh_nn {
namespace {

__device__ inline void philox(uint64_t block, uint64_t offset, uint64_t seed, uint32_t (&out)[4]) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    out[0] = c0, out[1] = c1, out[2] = c2, out[3] = c3;
}

// A thread takes the eight elements of one counter.
template <class T>
__global__ __launch_bounds__(256) void dropout_kernel(const T* __restrict__ x, const T* __restrict__ res, int64_t n,
                                                      uint32_t threshold, float scale, uint64_t seed, uint64_t offset,
                                                      T* __restrict__ y) {
    constexpr int VEC = 16 / sizeof(T);
    const int64_t block = (int64_t)blockIdx.x * 256 + threadIdx.x, i0 = block * 8;
    if (i0 >= n) return;
    uint32_t w[4];
    philox((uint64_t)block, offset, seed, w);
#pragma unroll
    for (int j = 0; j < 8; j += VEC) {
        if (i0 + j >= n) break;
        float a[VEC] = {}, r[VEC] = {};
        load_some<VEC>(x + i0 + j, n - i0 - j, a);
        if (res) load_some<VEC>(res + i0 + j, n - i0 - j, r);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const int e = i + j;
            const uint32_t bits = (e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu;
            a[i] = bits >= threshold ? a[i] * scale : 0.0f;
            if (res) a[i] += r[i];
        }
        store_some<VEC>(y + i0 + j, n - i0 - j, a);
    }
}

}  // namespace
}  // namespace drh_nn

using namespace drh_nn;

extern "C" int drh_dropout(drh_ctx* ctx, const void* x, const void* residual, int64_t n, int dtype, double p,
                           uint64_t seed, uint64_t offset, void* y, void* stream, uint32_t flags) {
    int rc = check_call(ctx, dtype, flags);
    if (rc) return rc;
    if (!(p >= 0.0 && p < 1.0)) return fail(DRH_ERR_INVALID_ARG, "p must be in [0, 1)");
    if (n < 0) return fail(DRH_ERR_INVALID_ARG, "n must not be negative");
    if (n > ((int64_t)1 << 40)) return fail(DRH_ERR_TOO_LARGE, "more than 2^40 elements");
    if (n == 0) return DRH_OK;
    if (!x || !y) return fail(DRH_ERR_INVALID_ARG, "x and y must not be NULL");
    // p just below one keeps one draw in 2^16
    uint32_t t = (uint32_t)lrint(p * 65536.0);
    if (t > 65535u) t = 65535u;
    const float scale = (float)(65536.0 / (65536.0 - t));
    DeviceGuard dg(ctx->device);
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)((n + 2047) / 2048));
    with_type(dtype, [&](auto ty) {
        using T = decltype(ty);
        dropout_kernel<T><<<grid, 256, 0, s>>>((const T*)x, (const T*)residual, n, t, scale, seed, offset, (T*)y);
        return DRH_OK;
    });
    return finish_call(s, flags, "dropout");
}
