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

// A thread takes 16 bytes: the eight elements of a counter, or in 32 bits four of them. Two
// threads then evaluate the same counter, which costs less than the half-used lines of 32
// bytes a thread (16384 x 4096 in 32 bits with a residual: 116 us so, 202 with those). Bound by
// memory: in bfloat16 that size takes 63 us with the residual (403 MB, 6.4 TB/s) and 43 without.
template <class T, bool ONCE>
__global__ __launch_bounds__(256) void dropout_kernel(const T* __restrict__ x, const T* __restrict__ res, int64_t n,
                                                      int64_t first, uint32_t threshold, float scale, uint64_t seed, uint64_t offset,
                                                      T* __restrict__ y) {
    constexpr int VEC = 16 / sizeof(T);
    const int64_t i0 = first + ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC, left = n - i0;
    if (left <= 0) return;
    const Raw xr = load_raw<false, ONCE>(x + i0, left);
    Raw rr = {};
    if (res) rr = load_raw<false, ONCE>(res + i0, left);
    uint32_t w[4];
    philox((uint64_t)i0 >> 3, offset, seed, w);
    if (i0 & 4) w[0] = w[2], w[1] = w[3];  // the counter's second half
    const Elements<T> xe = __builtin_bit_cast(Elements<T>, xr), re = __builtin_bit_cast(Elements<T>, rr);
    float a[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        const uint32_t bits = (e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu;
        a[e] = bits >= threshold ? (float)xe[e] * scale : 0.0f;
        if (res) a[e] += (float)re[e];
    }
    store_some<VEC>(y + i0, left, a);
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
    with_type(dtype, [&](auto ty) {
        using T = decltype(ty);
        constexpr int64_t PER = 256 * (16 / (int64_t)sizeof(T));
        auto go = [&](auto once) {
            in_launches((n + PER - 1) / PER, most_groups(256), [&](int64_t first, int64_t count) {
                dropout_kernel<T, once.value><<<dim3((unsigned)count), 256, 0, s>>>(
                    (const T*)x, (const T*)residual, n, first * PER, t, scale, seed, offset, (T*)y);
            });
        };
        if (n * (int64_t)sizeof(T) >= READ_ONCE_BYTES) go(std::true_type());
        else go(std::false_type());
        return DRH_OK;
    });
    return finish_call(s, flags, "dropout");
}
