// Shared by the norms over rows (layer_norm.hip, rms_norm.hip): weights, sums over the
// threads that hold a row, and how a row is loaded.
#pragma once

#include "layers.h"

namespace drh_nn {

// Weights from column c on; they may stand in 32 bits beside activations in 16.
template <class T, bool WHOLE, int VEC>
__device__ inline void load_weight(const void* w, bool wf32, int c, int D, float (&out)[VEC]) {
    if (wf32)
        load_some<VEC>((const float*)w + c, WHOLE ? VEC : D - c, out);
    else
        load_some<VEC>((const T*)w + c, WHOLE ? VEC : D - c, out);
}

// Sums of a and b over a row's threads, in all of them. `slot` alternates between
// calls, so that one barrier a call is enough.
template <int TPR, int THREADS>
__device__ inline void row_sums(float& a, float& b, int slot) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (TPR > 64) {
        __shared__ float2 part[2][THREADS / 64];
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) part[slot & 1][w] = make_float2(a, b);
        __syncthreads();
        const int first = w & ~(TPR / 64 - 1);
        a = b = 0.0f;
#pragma unroll
        for (int i = 0; i < TPR / 64; i++) {
            const float2 p = part[slot & 1][first + i];
            a += p.x;
            b += p.y;
        }
    }
}

// The largest v of a row's threads, in all of them; NaN is passed over. Called once by a kernel.
template <int TPR, int THREADS>
__device__ inline float row_max(float v) {
    v = wave_max(v);
    if constexpr (TPR > 64) {
        __shared__ float part[THREADS / 64];
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) part[w] = v;
        __syncthreads();
        const int first = w & ~(TPR / 64 - 1);
#pragma unroll
        for (int i = 0; i < TPR / 64; i++) v = fmaxf(v, part[first + i]);
    }
    return v;
}

// f(WHOLE, ONCE) as constants.
template <class T, class F>
void with_loads(int64_t rows, int64_t cols, F&& f) {
    if (cols % (16 / (int64_t)sizeof(T))) f(std::false_type(), std::false_type());
    else if (rows * cols * (int64_t)sizeof(T) < READ_ONCE_BYTES) f(std::true_type(), std::false_type());
    else f(std::true_type(), std::true_type());
}

}  // namespace drh_nn
