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
// or m would be divided by eps alone. It is the root that keeps its mean: v gains the rounding's variance at
// each step, so that with normal gradients and b2 = 0.999 it is 3 to 5% above that of 32 bits and deviates by a
// third of itself (its root by a sixth). In a block of unlike elements a v whose root is below 2^-15 of the largest is
// 15% high and more, and no root falls below 2^-18 of it: such elements take shorter steps. p is made from the m
// and v before they are rounded.
//
// Bound by memory: an element in 32 bits is read as 16 bytes and written as 12, with 8-bit states
// as 10 and 6. 203 M float32 parameters with 8-bit states (3.3 GB) take 553 us, 5.9 TB/s; 25 M bfloat16
// with 32-bit states, odd and unaligned (555 MB), 106 us, 5.2. The 8-bit states' arithmetic comes next, a hundred
// instructions an element at first and 581 us: the rounding instruction, roots by one correction, the blocks'
// maxima side by side and whole rounds without their ends brought it below the memory's time. ONCE, for arrays
// past the caches' size: loads and stores that leave the caches alone (609 and 119 us without, of 569 and 110).

#include <algorithm>
#include <cmath>
#include <iterator>
#include <new>
#include <utility>
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
    const int64_t* step;
    int64_t n;
    uint32_t first;  // of the launch's workgroups, the first that works on it
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

// The square roots of a vector's values, rounded right: with the reciprocal root's unit in the last place one
// correction does (checked for each value from 2^-100 to 2^102), beyond that sqrtf's dozen instructions more.
template <int N>
__device__ inline void roots(const float (&v)[N], float (&r)[N]) {
    float least = v[0], most = v[0];
#pragma unroll
    for (int i = 1; i < N; i++) least = fminf(least, v[i]), most = fmaxf(most, v[i]);
    if (least >= 0x1p-100f && most <= 0x1p100f) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float y = __builtin_amdgcn_rsqf(v[i]), s = v[i] * y;
            r[i] = fmaf(fmaf(-s, s, v[i]), 0.5f * y, s);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) r[i] = sqrtf(v[i]);
    }
}

// Four values as e4m3 codes, each rounded up where its draw, 16 random bits in its word's upper half, as a
// fraction, and what the grid leaves of the magnitude make a whole step. The instruction adds the word's upper
// 20 bits to the 20 that it cuts: what a rounding put past 448, by less than 16 units in the last place, stays 448.
__device__ inline uint32_t to_e4m3_at_random(const float (&v)[4], uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
    int w = __builtin_amdgcn_cvt_sr_fp8_f32(v[0], (int)r0, 0, 0);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(v[1], (int)r1, w, 1);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(v[2], (int)r2, w, 2);
    return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(v[3], (int)r3, w, 3);
}

// The largest v >= 0 of the wave, of N at once (a step waits for the one before it); none is NaN, so that
// their bits have their order.
template <int N>
__device__ inline void wave_most(float (&v)[N]) {
    uint32_t x[N];
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = __builtin_bit_cast(uint32_t, v[i]);
    auto step = [&](auto ctrl) {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = std::max(x[i], (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x[i], ctrl.value, 0xf, 0xf, true));
    };
    // one, two, four and eight lanes down within 16, then lane 15's to the next 16 and 31's to the
    // upper half: lane 63 has all
    step(std::integral_constant<int, 0x111>());
    step(std::integral_constant<int, 0x112>());
    step(std::integral_constant<int, 0x114>());
    step(std::integral_constant<int, 0x118>());
    step(std::integral_constant<int, 0x142>());
    step(std::integral_constant<int, 0x143>());
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = __builtin_bit_cast(float, __builtin_amdgcn_readlane((int)x[i], 63));
}

// The first `left` of N elements at p, in a state's or a parameter's type; zeros behind.
template <int N, bool ONCE, class T>
__device__ inline void fetch(const T* p, int64_t left, float (&out)[N]) {
    if (left >= N) {
        const auto q = reinterpret_cast<const typename Anywhere<T, N>::type*>(p);
        const vec<T, N> v = ONCE ? (vec<T, N>)__builtin_nontemporal_load(q) : (vec<T, N>)*q;
#pragma unroll
        for (int i = 0; i < N; i++) out[i] = (float)v[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) out[i] = i < left ? (float)p[i] : 0.0f;
    }
}

// A workgroup takes a tensor's next `rounds` rounds (one, but for tensors that a launch would not hold);
// a wave's vector is the 256 elements of one
// 8-bit block. Neighbouring lanes share a counter's eight draws: each evaluates the counter of one
// of its two vectors and hands the neighbour its half.
template <class T, bool SMALL, bool ONCE>
__global__ __launch_bounds__(THREADS) void adamw_kernel(StepArgs a) {
    const int lane = threadIdx.x & 63;
    // the tensor: the last one whose first workgroup is not past this one (one of no elements has none, and
    // stands before the tensor with the same first)
    const bool reached = lane < a.count && a.t[lane < a.count ? lane : 0].first <= blockIdx.x;
    const int id = __builtin_amdgcn_readfirstlane(__popcll(__ballot(reached)) - 1);
    const Tensor& t = a.t[id];
    const uint32_t step = (uint32_t)*t.step + 1;
    const int64_t n = t.n, begin = (int64_t)(blockIdx.x - t.first) * a.rounds * ROUND;
    float rate = 0.0f, root = 0.0f;
    // a round that the tensor fills has no ends to look for
    auto update = [&](auto whole, int64_t at0, bool first) {
        float g[GROUPS][VEC], p[GROUPS][VEC], m[GROUPS][VEC], v[GROUPS][VEC];
        uint32_t mc[GROUPS], vc[GROUPS];
        float ms[GROUPS], vs[GROUPS];
        int64_t left[GROUPS];
#pragma unroll
        for (int k = 0; k < GROUPS; k++) {
            const int64_t i = at0 + (int64_t)k * THREADS * VEC + threadIdx.x * VEC;
            left[k] = whole ? VEC : n - i;
            mc[k] = vc[k] = 0, ms[k] = vs[k] = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; e++) g[k][e] = p[k][e] = m[k][e] = v[k][e] = 0.0f;
            if (left[k] <= 0) continue;
            fetch<VEC, ONCE>((const T*)t.g + i, left[k], g[k]);
            fetch<VEC, ONCE>((const T*)t.p + i, left[k], p[k]);
            if constexpr (SMALL) {
                mc[k] = load_codes((const uint8_t*)t.m + i, left[k]);
                vc[k] = load_codes((const uint8_t*)t.v + i, left[k]);
                ms[k] = t.ms[i / STATE_BLOCK], vs[k] = t.vs[i / STATE_BLOCK];
            } else {
                fetch<VEC, ONCE>((const float*)t.m + i, left[k], m[k]);
                fetch<VEC, ONCE>((const float*)t.v + i, left[k], v[k]);
            }
        }
        if (first) {  // while the first loads are on their way
            rate = a.lr / (float)(1.0 - power(a.beta1, step));
            root = 1.0f / (float)sqrt(1.0 - power(a.beta2, step));
        }
        uint32_t draws[GROUPS][2];  // four 16-bit draws a vector
        if constexpr (SMALL) {
            const int odd = lane & 1;
            const int64_t i = at0 + (int64_t)odd * THREADS * VEC + threadIdx.x * VEC;
            uint32_t w[4];
            philox((uint64_t)i >> 3, (uint64_t)step | (uint64_t)(a.base + id) << 32, a.seed, w);
            // lane 2j has its first vector's counter, lane 2j + 1 its second's: words 0 and 1 are the even lane's
            const uint32_t s0 = odd ? w[0] : w[2], s1 = odd ? w[1] : w[3];
            constexpr int SWAP = 0xb1;  // lanes 1, 0, 3, 2 of each four
            const uint32_t r0 = __builtin_amdgcn_update_dpp(0, s0, SWAP, 0xf, 0xf, false),
                           r1 = __builtin_amdgcn_update_dpp(0, s1, SWAP, 0xf, 0xf, false);
            draws[0][0] = odd ? r0 : w[0], draws[0][1] = odd ? r1 : w[1];
            draws[1][0] = odd ? w[2] : r0, draws[1][1] = odd ? w[3] : r1;
        }
        float r[GROUPS][VEC], scale[2 * GROUPS];
#pragma unroll
        for (int k = 0; k < GROUPS; k++) {
            if constexpr (SMALL) {
                from_e4m3(mc[k], m[k]);
                from_e4m3(vc[k], v[k]);
#pragma unroll
                for (int e = 0; e < VEC; e++) m[k][e] *= ms[k], v[k][e] *= vs[k], v[k][e] *= v[k][e];
            }
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                m[k][e] = a.b1 * m[k][e] + a.c1 * g[k][e];
                v[k][e] = a.b2 * v[k][e] + a.c2 * g[k][e] * g[k][e];
            }
            roots<VEC>(v[k], r[k]);
#pragma unroll
            for (int e = 0; e < VEC; e++)
                p[k][e] = fmaf(p[k][e], a.keep, -rate * (m[k][e] * __builtin_amdgcn_rcpf(fmaf(r[k][e], root, a.eps))));
            float mm = 0.0f, mv = 0.0f;  // zeros past the tensor's end: g and the codes are
#pragma unroll
            for (int e = 0; e < VEC; e++) mm = fmaxf(mm, fabsf(m[k][e])), mv = fmaxf(mv, r[k][e]);
            scale[2 * k] = mm, scale[2 * k + 1] = mv;
        }
        if constexpr (SMALL) {
            wave_most<2 * GROUPS>(scale);
#pragma unroll
            for (int k = 0; k < 2 * GROUPS; k++) scale[k] = fmaxf(scale[k] * (1.0f / E4M3_MOST), LEAST_SCALE);
        }
#pragma unroll
        for (int k = 0; k < GROUPS; k++) {
            const int64_t i = at0 + (int64_t)k * THREADS * VEC + threadIdx.x * VEC;
            if (left[k] <= 0) break;
            if constexpr (SMALL) {
                if (lane == 0) t.ms[i / STATE_BLOCK] = scale[2 * k], t.vs[i / STATE_BLOCK] = scale[2 * k + 1];
                const Divisor dm(scale[2 * k]), dv(scale[2 * k + 1]);
                float qm[VEC], qv[VEC];
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    qm[e] = dm.of(m[k][e]), qv[e] = dv.of(r[k][e]);
                    if (r[k][e] > 0.0f) qv[e] = fmaxf(qv[e], 0x1p-9f);
                }
                uint32_t cm[1], cv[1];
                cm[0] = to_e4m3_at_random(qm, draws[k][0] << 16, draws[k][0] & 0xffff0000u, draws[k][1] << 16, draws[k][1] & 0xffff0000u);
                // v takes its draws' two bytes the other way round
                const uint32_t w0 = draws[k][0], w1 = draws[k][1];
                cv[0] = to_e4m3_at_random(qv, __builtin_amdgcn_perm(0, w0, 0x00010c0c), __builtin_amdgcn_perm(0, w0, 0x02030c0c),
                                          __builtin_amdgcn_perm(0, w1, 0x00010c0c), __builtin_amdgcn_perm(0, w1, 0x02030c0c));
                store_codes<false, VEC>((uint8_t*)t.m + i, left[k], cm);
                store_codes<false, VEC>((uint8_t*)t.v + i, left[k], cv);
            } else {
                store_once<ONCE, VEC>((float*)t.m + i, left[k], m[k]);
                store_once<ONCE, VEC>((float*)t.v + i, left[k], v[k]);
            }
            store_once<ONCE, VEC>((T*)t.p + i, left[k], p[k]);
        }
    };
    for (int round = 0; round < a.rounds; round++) {
        const int64_t at0 = begin + (int64_t)round * ROUND;
        if (at0 >= n) break;
        if (n - at0 >= ROUND) update(std::true_type(), at0, round == 0);
        else update(std::false_type(), at0, round == 0);
    }
}

// The steps are counted behind the kernels that read them. (By each tensor's last workgroup, found by
// an atomic count, 12000 workgroups took 460 us to be counted: one address takes an atomic every 37 ns.)
constexpr int COUNTS = 448;
struct CountArgs {
    int64_t* step[COUNTS];
    int count;
};
__global__ __launch_bounds__(64) void count_steps(CountArgs a) {
    const int i = blockIdx.x * 64 + threadIdx.x;
    if (i < a.count) *a.step[i] += 1;
}

int check_tensors(const drh_adamw_tensor* tensors, int64_t count, int dtype, bool small) {
    std::vector<std::pair<uintptr_t, uintptr_t>> written;  // each array's first byte and the one behind its last
    auto writes = [&](const void* p, int64_t bytes) { written.emplace_back((uintptr_t)p, (uintptr_t)p + (uint64_t)bytes); };
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
        writes(t.step, 8);
        if (t.n == 0) continue;
        writes(t.param, t.n * (int64_t)e);
        for (const void* state : {t.exp_avg, t.exp_avg_sq}) writes(state, t.n * (small ? 1 : 4));
        if (small)
            for (const void* scale : {t.exp_avg_scale, t.exp_avg_sq_scale}) writes(scale, (t.n + STATE_BLOCK - 1) / STATE_BLOCK * 4);
    }
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); i++)
        if (written[i].first < written[i - 1].second)
            return fail(DRH_ERR_INVALID_ARG, "two parameters, states, scales or step counts share memory");
    for (int64_t i = 0; i < count; i++) {  // a workgroup must not read as a gradient what another one writes
        const uintptr_t begin = (uintptr_t)tensors[i].grad, end = begin + (uint64_t)tensors[i].n * type_size(dtype);
        const auto next = std::lower_bound(written.begin(), written.end(), std::make_pair(end, (uintptr_t)0));
        if (tensors[i].n > 0 && next != written.begin() && std::prev(next)->second > begin)
            return fail(DRH_ERR_INVALID_ARG, "a gradient and a parameter, state, scale or step count share memory");
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
    try {
        rc = check_tensors(tensors, count, dtype, small);
    } catch (const std::bad_alloc&) {
        return fail(DRH_ERR_TOO_LARGE, "no memory to check so many tensors");
    }
    if (rc) return rc;
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
        // One round a workgroup, more only where a launch would not hold their number: with eight, 203 M
        // parameters with 8-bit states took 672 us, with one 609
        const int64_t per = (rounds >> 23) + 1;
        a.rounds = (int)per;
        uint32_t first = 0;
        for (int i = 0; i < a.count; i++) {
            const drh_adamw_tensor& t = tensors[from + i];
            a.t[i] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.exp_avg_scale, t.exp_avg_sq_scale, t.step, t.n, first};
            first += (uint32_t)((t.n + per * ROUND - 1) / (per * ROUND));
        }
        if (first == 0) continue;
        with_type(dtype, [&](auto ty) {
            using T = decltype(ty);
            auto go = [&](auto once) {
                if (small) adamw_kernel<T, true, once.value><<<dim3(first), THREADS, 0, s>>>(a);
                else adamw_kernel<T, false, once.value><<<dim3(first), THREADS, 0, s>>>(a);
            };
            if (rounds * ROUND * (int64_t)(2 * sizeof(T) + (small ? 2 : 8)) >= READ_ONCE_BYTES) go(std::true_type());
            else go(std::false_type());
            return DRH_OK;
        });
    }
    for (int64_t from = 0; from < count; from += COUNTS) {
        CountArgs c;
        c.count = (int)std::min<int64_t>(COUNTS, count - from);
        for (int i = 0; i < c.count; i++) c.step[i] = tensors[from + i].step;
        count_steps<<<dim3((unsigned)((c.count + 63) / 64)), 64, 0, s>>>(c);
    }
    return finish_call(s, flags, "AdamW");
}
