// Shared by the network layers (layer_norm.hip, linear.hip, dropout.hip): element
// types, vector access, wave sums and the second step of column sums.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>
#include <type_traits>

#include "diffrast_hip.h"
#include "runtime.h"

namespace drh_nn {

using bf16 = __bf16;
using f16 = _Float16;

template <class T, int N>
using vec = T __attribute__((ext_vector_type(N)));

// The same vector at any address that suits one element: global memory takes 16 bytes a
// lane from and to any of them, at no cost where the address is a multiple of 16.
template <class T, int N>
struct Anywhere {
    typedef vec<T, N> type __attribute__((aligned(sizeof(T))));
};

// N elements at p.
template <int N, class T>
__device__ inline void load(const T* p, float (&out)[N]) {
    const vec<T, N> v = *reinterpret_cast<const typename Anywhere<T, N>::type*>(p);
#pragma unroll
    for (int i = 0; i < N; i++) out[i] = (float)v[i];
}

// The first `left` of N elements at p; the others keep their values.
template <int N, class T>
__device__ inline void load_some(const T* p, int64_t left, float (&out)[N]) {
    if (left >= N) {
        load<N>(p, out);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < left) out[i] = (float)p[i];
    }
}

// Sixteen bytes of T as they stand in memory. Words and not a vector of T: 16-bit elements that
// live across branches would each take a register.
using Raw = vec<uint32_t, 4>;
template <class T>
using Elements = vec<T, 16 / sizeof(T)>;

// Arrays of this size and more are read past the caches (ONCE below): the last one holds 256
// MiB, so nothing of them would be there when it is read again, and what else it holds stays.
// Layer norm 32768 x 4096 in bfloat16 (268 MB) takes 88 us so, 98 with ordinary loads; 16384 x
// 1024 (34 MB) 16.0 and 13.8.
constexpr int64_t READ_ONCE_BYTES = 128ll << 20;

// The 16 bytes at p where WHOLE; else the first `left` elements, zeros behind.
template <bool WHOLE, bool ONCE, class T>
__device__ inline Raw load_raw(const T* p, int64_t left) {
    constexpr int N = 16 / sizeof(T);
    if (WHOLE || left >= N) {
        const auto q = reinterpret_cast<const typename Anywhere<T, N>::type*>(p);
        return __builtin_bit_cast(Raw, ONCE ? (Elements<T>)__builtin_nontemporal_load(q) : (Elements<T>)*q);
    }
    Elements<T> v;
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = i < left ? p[i] : (T)0.0f;
    return __builtin_bit_cast(Raw, v);
}

// Rounds to T once, to nearest even.
template <int N, class T>
__device__ inline void store(T* p, const float (&v)[N]) {
    vec<T, N> r;
#pragma unroll
    for (int i = 0; i < N; i++) r[i] = (T)v[i];
    *reinterpret_cast<typename Anywhere<T, N>::type*>(p) = r;
}

template <int N, class T>
__device__ inline void store_some(T* p, int64_t left, const float (&v)[N]) {
    if (left >= N) {
        store<N>(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < left) p[i] = (T)v[i];
    }
}

// store_some, past the caches where ONCE.
template <bool ONCE, int N, class T>
__device__ inline void store_once(T* p, int64_t left, const float (&v)[N]) {
    if (ONCE && left >= N) {
        vec<T, N> r;
#pragma unroll
        for (int i = 0; i < N; i++) r[i] = (T)v[i];
        __builtin_nontemporal_store(r, reinterpret_cast<typename Anywhere<T, N>::type*>(p));
    } else {
        store_some<N>(p, left, v);
    }
}

__device__ inline float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ inline float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
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

// A launch has fewer threads than this in x; what needs more takes several launches.
constexpr int64_t LAUNCH_THREADS = 1ll << 32;
constexpr int64_t most_groups(int64_t threads) { return (LAUNCH_THREADS - 1) / threads; }

// f(first, count) for n units, `most` at a time.
template <class F>
void in_launches(int64_t n, int64_t most, F&& f) {
    for (int64_t first = 0; first < n; first += most) f(first, n - first < most ? n - first : most);
}

// Checks that every layer call makes; the flags a layer knows are DRH_SYNC alone.
int check_call(drh_ctx* ctx, int dtype, uint32_t flags);
// Rows `stride` elements apart: no more than an address space holds, so that no offset passes 64 bits.
int check_span(int64_t rows, int64_t stride);
// After the last launch: its error, and DRH_SYNC's wait.
int finish_call(hipStream_t s, uint32_t flags, const char* what);

// out_a[c] = sum over g of part[g * stride + c] for c < cols, and out_b likewise
// from part + cols on (either may be null). Each sum is made in a fixed order.
int reduce_columns(const float* part, int64_t groups, int64_t stride, int64_t cols, void* out_a, void* out_b,
                   int out_dtype, hipStream_t s);

}  // namespace drh_nn
