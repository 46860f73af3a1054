// Shared by the network layers (layer_norm.hip, linear.hip, dropout.hip): element
// types, vector access, wave sums and the second step of column sums.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <initializer_list>
#include <string>
#include <type_traits>

#include "diffrast_hip.h"
#include "runtime.h"

namespace drh_nn {

using bf16 = __bf16;
using f16 = _Float16;

template <class T, int N>
using vec = T __attribute__((ext_vector_type(N)));

// N elements at p, aligned to their whole size where N > 1.
template <int N, class T>
__device__ inline void load(const T* p, float (&out)[N]) {
    if constexpr (N == 1) {
        out[0] = (float)*p;
    } else {
        const vec<T, N> v = *reinterpret_cast<const vec<T, N>*>(p);
#pragma unroll
        for (int i = 0; i < N; i++) out[i] = (float)v[i];
    }
}

// Rounds to T once, to nearest even.
template <int N, class T>
__device__ inline void store(T* p, const float (&v)[N]) {
    if constexpr (N == 1) {
        *p = (T)v[0];
    } else {
        vec<T, N> r;
#pragma unroll
        for (int i = 0; i < N; i++) r[i] = (T)v[i];
        *reinterpret_cast<vec<T, N>*>(p) = r;
    }
}

__device__ inline float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// f(T()) for the C element type of a DRH_* dtype.
template <class F>
int with_type(int dtype, F&& f) {
    if (dtype == DRH_F32) return f(float());
    if (dtype == DRH_BF16) return f(bf16());
    return f(f16());
}

inline size_t type_size(int dtype) { return dtype == DRH_F32 ? 4 : 2; }
inline bool known_type(int dtype) { return dtype == DRH_F32 || dtype == DRH_BF16 || dtype == DRH_F16; }
inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// The widest vector (16 bytes, then 4, then one element) that divides every one
// of the strides and addresses given.
inline int vector_width(int dtype, std::initializer_list<int64_t> strides, std::initializer_list<const void*> ptrs) {
    const int size = (int)type_size(dtype);
    for (int bytes : {16, 4}) {
        if (bytes < size) break;
        bool ok = true;
        for (int64_t s : strides) ok = ok && s % (bytes / size) == 0;
        for (const void* p : ptrs) ok = ok && (uintptr_t)p % bytes == 0;
        if (ok) return bytes / size;
    }
    return 1;
}

// Checks that every layer call makes; the flags a layer knows are DRH_SYNC alone.
int check_call(drh_ctx* ctx, int dtype, uint32_t flags);
// After the last launch: its error, and DRH_SYNC's wait.
int finish_call(hipStream_t s, uint32_t flags, const char* what);

// out_a[c] = sum over g of part[g * stride + c] for c < cols, and out_b likewise
// from part + cols on (either may be null). Each sum is made in a fixed order.
int reduce_columns(const float* part, int64_t groups, int64_t stride, int64_t cols, void* out_a, void* out_b,
                   int out_dtype, hipStream_t s);

}  // namespace drh_nn
