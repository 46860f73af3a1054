// Values in 8 bits: e4m3 (a sign, four bits of exponent, three of mantissa, up to 448, no
// infinities), the type of the matrix cores' 8-bit products.
#pragma once

#include "layers.h"

namespace drh_nn {

constexpr float E4M3_MOST = 448.0f, LEAST_SCALE = 0x1p-126f;

// N values as e4m3, rounded to nearest even; |v| may pass 448 by a rounding.
template <int N>
__device__ inline void to_e4m3(const float (&v)[N], uint32_t (&out)[(N + 3) / 4]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        int word = __builtin_amdgcn_cvt_pk_fp8_f32(v[i], v[i + 1], 0, false);
        out[i / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[i + 2], v[i + 3], word, true);
    }
}

// The first `left` of N codes at any address.
template <bool WHOLE, int N>
__device__ inline void store_codes(uint8_t* p, int64_t left, const uint32_t (&w)[N / 4]) {
    if (WHOLE || left >= N) {
        vec<uint32_t, N / 4> v;
#pragma unroll
        for (int i = 0; i < N / 4; i++) v[i] = w[i];
        typedef vec<uint32_t, N / 4> any __attribute__((aligned(1)));
        *reinterpret_cast<any*>(p) = v;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < left) p[i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
    }
}

// Four codes at any address; of fewer the others are zero.
__device__ inline uint32_t load_codes(const uint8_t* p, int64_t left) {
    typedef uint32_t any __attribute__((aligned(1)));
    if (left >= 4) return *reinterpret_cast<const any*>(p);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 3; i++)
        if (i < left) w |= (uint32_t)p[i] << (8 * i);
    return w;
}

// Four codes as floats.
__device__ inline void from_e4m3(uint32_t w, float (&out)[4]) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    out[0] = lo[0], out[1] = lo[1], out[2] = hi[0], out[3] = hi[1];
}

// Quotients by one divisor, as a division rounds them: a reciprocal corrected once, and each quotient by its own
// remainder (Markstein, 1990). What is rounded to few bits afterwards goes by the last one now and then: a value
// half way between two codes, or random bits that just reach the upper one. 32768 x 4096 bfloat16 numbers take
// 63 us to their codes so, 76 with a division for each, 61 with a product (whose ties are wrong).
struct Divisor {
    float d, r;
    __device__ explicit Divisor(float by) : d(by) {
        const float e = __builtin_amdgcn_rcpf(by);
        r = fmaf(fmaf(-by, e, 1.0f), e, e);
    }
    __device__ float of(float x) const {
        const float q = x * r;
        return fmaf(fmaf(-q, d, x), r, q);
    }
};

// The same by a row's scale, which may be tiny (remainders lose bits below 2^-126) or infinite (finite
// numbers are nothing of it, others NaN). A zero keeps its sign, which the correction would drop.
struct RowDivisor {
    float up;
    Divisor by;
    __device__ explicit RowDivisor(float scale)
        : up(scale < 0x1p-64f ? 0x1p64f : scale < __builtin_inff() ? 1.0f : 0.0f), by(up > 0.0f ? scale * up : 1.0f) {}
    __device__ float of(float x) const { return __builtin_copysignf(by.of(x * up), x); }
};

}  // namespace drh_nn
