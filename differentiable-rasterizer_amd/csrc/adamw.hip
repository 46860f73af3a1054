// One AdamW step (Loshchilov and Hutter, 2019) over many tensors at once:
//
//   t = step + 1
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in 32 bits, the bias corrections in 64; p is rounded to its type once. The states m and v stand
// in 32 bits, or in 8: then m and sqrt(v) are e4m3 with a scale for each 256 elements, the block's
// largest magnitude / 448. What is stored is rounded up or down at random, up with the probability
// of the part that is missing. To the nearest the averages would stand still: a step moves v by
// (1 - b2) of it, 0.001, and e4m3's neighbours are 1/16 to 1/8 apart. sqrt(v) and not v, since
// e4m3 spans 2^18 and v the square of what g does; and where v is not zero its code is not either,
// or m would be divided by eps alone. p is made from the m and v before they are rounded.
//
// Bound by memory: an element in 32 bits is read as 16 bytes and written as 12, with 8-bit states
// as 10 and 6.

#include <algorithm>
#include <cmath>
#include <vector>

#include "e4m3.h"
#include "philox.h"

using namespace drh_rt;

namespace drh_nn {
namespace {

constexpr int STATE_BLOCK = 256;     // elements that share a scale
constexpr int TENSORS = 48;          // of a launch; their table goes with its arguments (under 4 KB)
constexpr int THREADS = 256, VEC = 4, GROUPS = 2;  // a thread takes GROUPS vectors a round
constexpr int ROUND = THREADS * VEC * GROUPS;

struct Tensor {
    void* p;
    const void* g;
    void *m, *v;
    float *ms, *vs;
    int64_t* step;
    int64_t n;
    uint32_t first, blocks;  // of the launch's workgroups, those that work on it
};

struct StepArgs {
    Tensor t[TENSORS];
    int count;
    int rounds;     // ROUNDs of elements a workgroup takes
    uint32_t base;  // the first tensor's number in the call
    float lr, b1, b2, eps, keep;  // keep: 1 - lr wd
    float c1, c2;                 // 1 - b1, 1 - b2 (in 64 bits, then rounded)
    double beta1, beta2;
    uint64_t seed;
};

// b^t in 64 bits, by squaring.
__device__ inline double power(double b, uint32_t t) {
    double r = 1.0;
    for (; t; t >>= 1) {
        if (t & 1) r *= b;
        b *= b;
    }
    return r;
}

// |x| <= 448 rounded to e4m3's grid, up where the 16 random bits, as a fraction, pass what is
// missing; not below `least` unless x is zero.
__device__ inline float round_at_random(float x, uint32_t bits, float least) {
    const float a = fabsf(x);
    // the step of the grid at a: 2^(exponent - 3), 2^-9 from 2^-6 down
    const int e = (int)((__builtin_bit_cast(uint32_t, a) >> 23) & 0xff);
    const int es = e < 121 ? 118 : e > 135 ? 132 : e - 3;
    const float step = __builtin_bit_cast(float, (uint32_t)es << 23), inv = __builtin_bit_cast(float, (uint32_t)(254 - es) << 23);
    float q = fminf(floorf(fmaf(a, inv, (float)bits * 0x1p-16f)) * step, E4M3_MOST);
    if (a > 0.0f) q = fmaxf(q, least);
    return a != a ? x : copysignf(q, x);
}

// A workgroup takes a tensor's next `rounds` rounds; a wave's vector is the 256 elements of one
// 8-bit block. Neighbouring lanes share a counter's eight draws: each evaluates the counter of one
// of its two vectors and hands the neighbour its half.
template <class T, bool SMALL>
__global__ __launch_bounds__(THREADS) void adamw_kernel(StepArgs a) {
    const int lane = threadIdx.x & 63;
    // the tensor: the last one whose first workgroup is not past this one
    const bool reached = lane < a.count && a.t[lane < a.count ? lane : 0].first <= blockIdx.x;
    const int id = __builtin_amdgcn_readfirstlane(__popcll(__ballot(reached)) - 1);
    const Tensor& t = a.t[id];
    const uint32_t step = (uint32_t)__hip_atomic_load(t.step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
    const float rate = a.lr / (float)(1.0 - power(a.beta1, step));
    const float root = 1.0f / (float)sqrt(1.0 - power(a.beta2, step));
    const int64_t n = t.n, begin = (int64_t)(blockIdx.x - t.first) * a.rounds * ROUND;
    for (int round = 0; round < a.rounds; round++) {
        const int64_t at0 = begin + (int64_t)round * ROUND;
        if (at0 >= n) break;
        float g[GROUPS][VEC], p[GROUPS][VEC], m[GROUPS][VEC], v[GROUPS][VEC];
        uint32_t mc[GROUPS], vc[GROUPS];
        float ms[GROUPS], vs[GROUPS];
        int64_t left[GROUPS];
#pragma unroll
        for (int k = 0; k < GROUPS; k++) {
            const int64_t i = at0 + (int64_t)k * THREADS * VEC + threadIdx.x * VEC;
            left[k] = n - i;
            mc[k] = vc[k] = 0, ms[k] = vs[k] = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; e++) g[k][e] = p[k][e] = m[k][e] = v[k][e] = 0.0f;
            if (left[k] <= 0) continue;
            load_some<VEC>((const T*)t.g + i, left[k], g[k]);
            load_some<VEC>((const T*)t.p + i, left[k], p[k]);
            if constexpr (SMALL) {
                mc[k] = load_codes((const uint8_t*)t.m + i, left[k]);
                vc[k] = load_codes((const uint8_t*)t.v + i, left[k]);
                ms[k] = t.ms[i / STATE_BLOCK], vs[k] = t.vs[i / STATE_BLOCK];
            } else {
                load_some<VEC>((const float*)t.m + i, left[k], m[k]);
                load_some<VEC>((const float*)t.v + i, left[k], v[k]);
            }
        }
        uint32_t draws[GROUPS][2];  // four 16-bit draws a vector
        if constexpr (SMALL) {
            const int odd = lane & 1;
            const int64_t i = at0 + (int64_t)odd * THREADS * VEC + threadIdx.x * VEC;
            uint32_t w[4];
            philox((uint64_t)i >> 3, (uint64_t)step | (uint64_t)(a.base + id) << 32, a.seed, w);
            // lane 2j has its first vector's counter, lane 2j + 1 its second's: words 0 and 1 are the even lane's
            const uint32_t s0 = odd ? w[0] : w[2], s1 = odd ? w[1] : w[3];
            const uint32_t r0 = __shfl_xor(s0, 1, 64), r1 = __shfl_xor(s1, 1, 64);
            draws[0][0] = odd ? r0 : w[0], draws[0][1] = odd ? r1 : w[1];
            draws[1][0] = odd ? w[2] : r0, draws[1][1] = odd ? w[3] : r1;
        }
#pragma unroll
        for (int k = 0; k < GROUPS; k++) {
            const int64_t i = at0 + (int64_t)k * THREADS * VEC + threadIdx.x * VEC;
            float r[VEC];
            if constexpr (SMALL) {
                from_e4m3(mc[k], m[k]);
                from_e4m3(vc[k], v[k]);
#pragma unroll
                for (int e = 0; e < VEC; e++) m[k][e] *= ms[k], v[k][e] *= vs[k], v[k][e] *= v[k][e];
            }
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                m[k][e] = fmaf(a.b1, m[k][e], a.c1 * g[k][e]);
                v[k][e] = fmaf(a.b2, v[k][e], a.c2 * g[k][e] * g[k][e]);
                r[e] = sqrtf(v[k][e]);
                p[k][e] = fmaf(p[k][e], a.keep, -rate * (m[k][e] / fmaf(r[e], root, a.eps)));
            }
            if constexpr (SMALL) {
                float mm = 0.0f, mv = 0.0f;
#pragma unroll
                for (int e = 0; e < VEC; e++)
                    if (e < left[k]) mm = fmaxf(mm, fabsf(m[k][e])), mv = fmaxf(mv, r[e]);
                mm = fmaxf(wave_max(mm) / E4M3_MOST, LEAST_SCALE);
                mv = fmaxf(wave_max(mv) / E4M3_MOST, LEAST_SCALE);
                if (left[k] <= 0) continue;
                if (lane == 0) t.ms[i / STATE_BLOCK] = mm, t.vs[i / STATE_BLOCK] = mv;
                const float im = 1.0f / mm, iv = 1.0f / mv;
                float qm[VEC], qv[VEC];
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const uint32_t bits = (e & 1) ? draws[k][e >> 1] >> 16 : draws[k][e >> 1] & 0xffffu;
                    qm[e] = round_at_random(m[k][e] * im, bits, 0.0f);
                    qv[e] = round_at_random(r[e] * iv, (bits >> 8) | (bits & 0xffu) << 8, 0x1p-9f);
                }
                uint32_t cm[1], cv[1];
                to_e4m3<VEC>(qm, cm);
                to_e4m3<VEC>(qv, cv);
                store_codes<false, VEC>((uint8_t*)t.m + i, left[k], cm);
                store_codes<false, VEC>((uint8_t*)t.v + i, left[k], cv);
            } else {
                if (left[k] <= 0) continue;
                store_some<VEC>((float*)t.m + i, left[k], m[k]);
                store_some<VEC>((float*)t.v + i, left[k], v[k]);
            }
            store_some<VEC>((T*)t.p + i, left[k], p[k]);
        }
    }
    // The tensor's last workgroup counts the step. Until then the upper half of the number counts
    // the workgroups that are done, each of which has read the lower half.
    __syncthreads();
    if (threadIdx.x == 0) {
        const int64_t before = __hip_atomic_fetch_add(t.step, (int64_t)1 << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if ((uint32_t)(before >> 32) == t.blocks - 1)
            __hip_atomic_store(t.step, (int64_t)step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

int check_tensors(const drh_adamw_tensor* tensors, int64_t count, int dtype, bool small) {
    std::vector<const void*> params, steps;
    for (int64_t i = 0; i < count; i++) {
        const drh_adamw_tensor& t = tensors[i];
        if (t.n < 0) return fail(DRH_ERR_INVALID_ARG, "a tensor has a negative number of elements");
        if (t.n > (int64_t)1 << 40) return fail(DRH_ERR_TOO_LARGE, "a tensor of more than 2^40 elements");
        if (!t.step) return fail(DRH_ERR_INVALID_ARG, "a tensor has no step count");
        if (t.n > 0 && (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq)) return fail(DRH_ERR_INVALID_ARG, "a pointer of a tensor is NULL");
        if (t.n > 0 && small != (t.exp_avg_scale != nullptr && t.exp_avg_sq_scale != nullptr))
            return fail(DRH_ERR_INVALID_ARG, "8-bit states, and no others, come with scales");
        const uintptr_t e = type_size(dtype);
        if ((uintptr_t)t.param % e || (uintptr_t)t.grad % e || (uintptr_t)t.step % 8 ||
            (!small && ((uintptr_t)t.exp_avg % 4 || (uintptr_t)t.exp_avg_sq % 4)) ||
            (small && ((uintptr_t)t.exp_avg_scale % 4 || (uintptr_t)t.exp_avg_sq_scale % 4)))
            return fail(DRH_ERR_INVALID_ARG, "a pointer of a tensor is not aligned to its elements");
        if (t.n > 0) params.push_back(t.param);
        steps.push_back(t.step);
    }
    for (auto* v : {&params, &steps}) {
        std::sort(v->begin(), v->end());
        if (std::adjacent_find(v->begin(), v->end()) != v->end())
            return fail(DRH_ERR_INVALID_ARG, "two tensors share a parameter or a step count");
    }
    return DRH_OK;
}

}  // namespace
}  // namespace drh_nn

using namespace drh_nn;

extern "C" int drh_adamw(drh_ctx* ctx, const drh_adamw_tensor* tensors, int64_t count, int dtype, int state_bits, double lr,
                         double beta1, double beta2, double eps, double weight_decay, uint64_t seed, void* stream,
                         uint32_t flags) {
    int rc = check_call(ctx, dtype, flags);
    if (rc) return rc;
    if (state_bits != 32 && state_bits != 8) return fail(DRH_ERR_INVALID_ARG, "states have 32 or 8 bits");
    if (!(lr >= 0.0 && eps >= 0.0 && weight_decay >= 0.0) || std::isinf(lr) || std::isinf(eps) || std::isinf(weight_decay))
        return fail(DRH_ERR_INVALID_ARG, "lr, eps and weight_decay must be finite and not negative");
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0))
        return fail(DRH_ERR_INVALID_ARG, "beta1 and beta2 must be in [0, 1)");
    if (count < 0 || (count > 0 && !tensors)) return fail(DRH_ERR_INVALID_ARG, "tensors must not be NULL, nor count negative");
    if (count > INT32_MAX) return fail(DRH_ERR_TOO_LARGE, "more than 2^31 - 1 tensors");
    const bool small = state_bits == 8;
    if ((rc = check_tensors(tensors, count, dtype, small))) return rc;
    if (count == 0) return DRH_OK;
    DeviceGuard dg(ctx->device);
    hipStream_t s = (hipStream_t)stream;
    StepArgs a;
    a.lr = (float)lr, a.b1 = (float)beta1, a.b2 = (float)beta2, a.eps = (float)eps, a.keep = (float)(1.0 - lr * weight_decay);
    a.c1 = (float)(1.0 - beta1), a.c2 = (float)(1.0 - beta2), a.beta1 = beta1, a.beta2 = beta2, a.seed = seed;
    for (int64_t from = 0; from < count; from += TENSORS) {
        a.count = (int)std::min<int64_t>(TENSORS, count - from);
        a.base = (uint32_t)from;
        int64_t rounds = 0;
        for (int i = 0; i < a.count; i++) rounds += (tensors[from + i].n + ROUND - 1) / ROUND;
        // Eight rounds a workgroup where that leaves some for every CU's waves, and more where a
        // launch would not hold their number
        const int64_t per = std::max(std::min<int64_t>(8, std::max<int64_t>(1, rounds / 2048)), (rounds >> 22) + 1);
        a.rounds = (int)per;
        uint32_t first = 0;
        for (int i = 0; i < a.count; i++) {
            const drh_adamw_tensor& t = tensors[from + i];
            const int64_t need = (t.n + per * ROUND - 1) / (per * ROUND);
            const uint32_t blocks = (uint32_t)std::max<int64_t>(1, need);  // one to count the step
            a.t[i] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.exp_avg_scale, t.exp_avg_sq_scale, t.step, t.n, first, blocks};
            first += blocks;
        }
        with_type(dtype, [&](auto ty) {
            using T = decltype(ty);
            if (small) adamw_kernel<T, true><<<dim3(first), THREADS, 0, s>>>(a);
            else adamw_kernel<T, false><<<dim3(first), THREADS, 0, s>>>(a);
            return DRH_OK;
        });
    }
    return finish_call(s, flags, "AdamW");
}
