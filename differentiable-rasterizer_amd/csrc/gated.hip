// A gated linear layer (the first half of a gated feed-forward block), forward and backward:
//
//   zg = x Wg^T + bg,  zu = x Wu^T + bu,  y = act(zg) zu          x: M x K, W = [Wg; Wu]: 2 N x K
//   dzg = dy zu act'(zg),  dzu = dy act(zg),  dz = [dzg dzu]: M x 2 N
//   dx = dz W,  dW = dz^T x,  db = sum over rows of dz
//
// The forward pass is one product of 2 N columns whose tiles take the same outputs' rows of both
// halves (GatedLoader in gemm.h), so that the activation and the product are made where both sums
// are, in registers, and z is never stored. Sums and activations are held in 32 bits, y is rounded
// once. The backward pass needs act(zg) and zu act'(zg); the forward pass has both at hand and keeps
// them, not z, which would have to be activated again. They are unbounded, so float16 will not do,
// and bfloat16's 8 bits would cost the gradients as much again as the rounding of dz does (which is
// an operand of two products): beside bfloat16 they are kept in 20 bits, beside float16 in 24, float32
// cut off to 12 and 16 bits of precision, 16 times finer than dz is rounded.

#include "products.h"

using namespace drh_rt;

namespace drh_nn {
namespace {

// ---------------------------------------------------------------- what is kept

// M x N pairs (act(zg), zu act'(zg)) in planes of M x N. For 16-bit types the upper 16 bits of the
// first and of the second, and then what is left of both: for float16 16 bits, a byte each, the first's
// below, for bfloat16 8, four each. The rest is cut off and not rounded, which would take twice the
// instructions; a NaN has its mantissa's upper bit.
template <class T>
constexpr int PAIR_BYTES = sizeof(T) == 4 ? 8 : std::is_same_v<T, bf16> ? 5 : 6;

// N bytes at any address.
template <int N>
struct AnyWords {
    typedef vec<uint32_t, N / 4> type __attribute__((aligned(1)));
};

template <class T, int C>
struct Pairs {
    static __device__ void keep(void* kept, int64_t size, int64_t at, int64_t left, const float (&a)[C], const float (&b)[C]) {
        if constexpr (sizeof(T) == 2) {
            using Words = vec<uint32_t, C / 2>;
            constexpr bool NIBBLES = PAIR_BYTES<T> == 5;
            Words ha, hb;
            vec<uint32_t, NIBBLES ? C / 4 : C / 2> lo;
#pragma unroll
            for (int i = 0; i < C; i += 2) {
                const uint32_t a0 = __builtin_bit_cast(uint32_t, a[i]), a1 = __builtin_bit_cast(uint32_t, a[i + 1]);
                const uint32_t b0 = __builtin_bit_cast(uint32_t, b[i]), b1 = __builtin_bit_cast(uint32_t, b[i + 1]);
                ha[i / 2] = __builtin_amdgcn_perm(a1, a0, 0x07060302);
                hb[i / 2] = __builtin_amdgcn_perm(b1, b0, 0x07060302);
                // bytes 1 of both numbers, of the first's and the second's
                const uint32_t la = __builtin_amdgcn_perm(a1, a0, 0x0c0c0501), lb = __builtin_amdgcn_perm(b1, b0, 0x0c0c0501);
                if constexpr (NIBBLES) {
                    const uint32_t two = ((la >> 4) & 0x0f0fu) | (lb & 0xf0f0u);
                    lo[i / 4] = i % 4 ? lo[i / 4] | two << 16 : two;
                } else {
                    lo[i / 2] = __builtin_amdgcn_perm(lb, la, 0x05010400);
                }
            }
            char* p = (char*)kept;
            put<2 * C>(p + at * 2, left, ha), put<2 * C>(p + (size + at) * 2, left, hb);
            put<(NIBBLES ? 1 : 2) * C>(p + size * 4 + at * (NIBBLES ? 1 : 2), left, lo);
        } else {
            store_some<C>((float*)kept + at, left, a);
            store_some<C>((float*)kept + size + at, left, b);
        }
    }
    // The first `left` of C parts of v's N bytes.
    template <int N>
    static __device__ void put(char* p, int64_t left, const vec<uint32_t, N / 4>& v) {
        if (left >= C) {
            *reinterpret_cast<typename AnyWords<N>::type*>(p) = v;
        } else {
            constexpr int PER = N / C;
#pragma unroll
            for (int i = 0; i < N; i++)
                if (i / PER < left) p[i] = (char)(v[i / 4] >> (8 * (i % 4)));
        }
    }
    // C pairs as they were read: a, b.
    static __device__ void open(const Raw& ha, const Raw& hb, const Raw& lo, float (&a)[C], float (&b)[C]) {
        static_assert(C == 16 / sizeof(T), "16 bytes of a plane");
#pragma unroll
        for (int i = 0; i < C; i++) {
            if constexpr (sizeof(T) == 4) {
                a[i] = __builtin_bit_cast(vec<float, 4>, ha)[i], b[i] = __builtin_bit_cast(vec<float, 4>, hb)[i];
            } else {
                const uint32_t ua = i % 2 ? ha[i / 2] & 0xffff0000u : ha[i / 2] << 16,
                               ub = i % 2 ? hb[i / 2] & 0xffff0000u : hb[i / 2] << 16;
                if constexpr (PAIR_BYTES<T> == 5) {
                    const uint32_t byte = lo[i / 4] >> (8 * (i % 4));
                    a[i] = __builtin_bit_cast(float, ua | (byte & 0x0fu) << 12);
                    b[i] = __builtin_bit_cast(float, ub | (byte & 0xf0u) << 8);
                } else {
                    const uint32_t half = lo[i / 2] >> (16 * (i % 2));
                    a[i] = __builtin_bit_cast(float, ua | (half & 0xffu) << 8);
                    b[i] = __builtin_bit_cast(float, ub | (half & 0xff00u));
                }
            }
        }
    }
    // The plane of what is left, the first `left` of C parts; zeros behind.
    static __device__ Raw rest(const void* kept, int64_t size, int64_t at, int64_t left) {
        Raw r = {};
        if constexpr (sizeof(T) == 2) {
            constexpr int PER = PAIR_BYTES<T> - 4, N = PER * C;
            const char* p = (const char*)kept + size * 4 + at * PER;
            if (left >= C) {
                const vec<uint32_t, N / 4> v = *reinterpret_cast<const typename AnyWords<N>::type*>(p);
#pragma unroll
                for (int i = 0; i < N / 4; i++) r[i] = v[i];
            } else {
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (i / PER < left) r[i / 4] |= (uint32_t)(uint8_t)p[i] << (8 * (i % 4));
            }
        }
        return r;
    }
};

// ---------------------------------------------------------------- the product's epilogue

// One lane's 2 NV neighbouring outputs of a row, from NV / 2 fragments of either half: columns()
// is called before the rows that share them.
template <class T, int NV>
struct GatedEpilogue {
    static constexpr int W = 2 * NV;
    int64_t n = 0;
    float bg[W], bu[W];

    __device__ void columns(const Gemm& p, int64_t n_) {
        n = n_;
#pragma unroll
        for (int i = 0; i < W; i++) bg[i] = bu[i] = 0.0f;
        if (p.bias && !p.partial && n < p.N) {
            load_some<W>((const T*)p.bias + n, p.N - n, bg);
            load_some<W>((const T*)p.bias + p.N + n, p.N - n, bu);
        }
    }

    __device__ void row(const Gemm& p, int64_t m, const floatx4 (&v)[NV]) const {
        if (m >= p.M || n >= p.N) return;
        if (p.partial) {
            float* out = p.partial + ((int64_t)blockIdx.y * p.M + m) * 2 * p.N + n;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const float o[4] = {v[j][0], v[j][1], v[j][2], v[j][3]};
                const int c = j % (NV / 2) * 4;
                if (n + c < p.N) store_some<4>(out + (j < NV / 2 ? 0 : p.N) + c, p.N - n - c, o);
            }
            return;
        }
        float g[W], u[W];
#pragma unroll
        for (int i = 0; i < W; i++) g[i] = v[i / 4][i % 4], u[i] = v[NV / 2 + i / 4][i % 4];
        if (p.bias)
#pragma unroll
            for (int i = 0; i < W; i++) g[i] += bg[i], u[i] += bu[i];
        apply<W>(p, m * p.N + n, p.N - n, g, u);
    }

    // From z on: the first `left` of C outputs.
    template <int C>
    static __device__ void apply(const Gemm& p, int64_t at, int64_t left, float (&g)[C], const float (&u)[C]) {
        float y[C], b[C];
#pragma unroll
        for (int i = 0; i < C; i++) {
            float slope;
            g[i] = act_of<sizeof(T) == 4>(p.act, g[i], slope);
            y[i] = g[i] * u[i], b[i] = u[i] * slope;
        }
        constexpr int CH = 16 / sizeof(T) < C ? 16 / sizeof(T) : C;
#pragma unroll
        for (int c = 0; c < C; c += CH) {
            if (c >= left) break;
            float part[CH], pa[CH], pb[CH];
#pragma unroll
            for (int i = 0; i < CH; i++) part[i] = y[c + i], pa[i] = g[c + i], pb[i] = b[c + i];
            store_some<CH>((T*)p.out + at + c, left - c, part);
            if (p.kept) Pairs<T, CH>::keep(p.kept, p.M * p.N, at + c, left - c, pa, pb);
        }
    }
};

// ---------------------------------------------------------------- the products

// 16384 x 1024 -> 4096 in bfloat16 takes 258 us without the pairs (1.06 PFLOP/s), 314 with them: 335 MB
// more that are written at the rate of memory, beside products that run at the power limit. So neither
// starting CUs one after the other nor starting the next tile's loads before a tile's end (312) nor two
// workgroups of 128 a CU (379) covers them, and stores past the caches, half lines each, take 44 more.
template <class T>
__global__ __launch_bounds__(512, 2) void gated_256_kernel(Gemm p) {
    gemm_256<T, true, true, GatedEpilogue<T, 4>, true>(p);
}

// Smaller outputs, and 32 bits (thirds): 4096 x 1024 -> 1024 in 32 bits takes 116 us (148 TFLOP/s, what a
// large 32-bit product of the library reaches), 1531 x 75 -> 1501 in f16 14 us.
template <class T, class Math, int TILE, int GROUPS>
__global__ __launch_bounds__(256 * GROUPS, TILE == 64 && GROUPS == 1 ? 3 : 2) void gated_tile_kernel(Gemm p) {
    gemm_tile<T, true, true, GatedEpilogue<T, TILE / 32>, Math, TILE, GROUPS, true>(p);
}

// The parts of a split product added in order, and the epilogue: a thread 16 bytes of a row of y.
template <class T>
__global__ __launch_bounds__(256) void gated_join(Gemm p, int64_t first) {
    constexpr int CH = 16 / sizeof(T);
    const int64_t per = (p.N + CH - 1) / CH, id = (first + blockIdx.x) * 256 + threadIdx.x;
    const int64_t m = id / per, n = id % per * CH, left = p.N - n;
    if (m >= p.M) return;
    float z[2][CH] = {};
#pragma unroll
    for (int h = 0; h < 2; h++) {
        for (int s = 0; s < p.splits; s++) {
            float v[CH] = {};
            load_some<CH>(p.partial + ((int64_t)s * p.M + m) * 2 * p.N + h * p.N + n, left, v);
#pragma unroll
            for (int i = 0; i < CH; i++) z[h][i] += v[i];
        }
        if (p.bias) {
            float b[CH] = {};
            load_some<CH>((const T*)p.bias + h * p.N + n, left, b);
#pragma unroll
            for (int i = 0; i < CH; i++) z[h][i] += b[i];
        }
    }
    GatedEpilogue<T, 4>::template apply<CH>(p, m * p.N + n, left, z[0], z[1]);
}

// Few rows of x (up to 16 MT): the weights are read once and that is what it costs, so nothing is
// staged. A workgroup takes 16 outputs, 32 rows of W; its eight waves take an eighth of k each,
// straight from memory to the matrix cores, and are added through LDS in order. One row of 1024 -> 4096
// in bfloat16 (16.8 MB of weights, from the caches when repeated) takes 5.2 us, 3.2 TB/s.
template <class T, int MT>
__global__ __launch_bounds__(512) void gated_rows_kernel(Gemm p) {
    constexpr int CH = 16 / sizeof(T), WAVES = 8;
    using F = vec<T, CH>;
    using FU = typename Anywhere<T, CH>::type;
    __shared__ __align__(16) floatx4 part[WAVES][2 * MT][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16, K = p.K;
    const int steps = (int)((K + 4 * CH - 1) / (4 * CH)), s0 = (int)((int64_t)steps * w / WAVES),
              s1 = (int)((int64_t)steps * (w + 1) / WAVES);
    // rows past the end read the last one's values and are not stored
    const T* bp[2];
    bp[0] = (const T*)p.b.ptr + (n0 + r < p.N ? n0 + r : p.N - 1) * p.b.ld;
    bp[1] = bp[0] + p.N * p.b.ld;
    const T* ap[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) ap[t] = (const T*)p.a.ptr + (16 * t + r < p.M ? 16 * t + r : p.M - 1) * p.a.ld;
    floatx4 acc[2][MT] = {};
    constexpr int AT_ONCE = MT == 1 ? 4 : 2;  // steps' loads: a wave has little else to wait with
    const int whole = (int)(K / (4 * CH)) < s1 ? (int)(K / (4 * CH)) : s1;
    int s = s0;
    for (; s + AT_ONCE <= whole; s += AT_ONCE) {
        F b[AT_ONCE][2], a[AT_ONCE][MT];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            const int64_t k = ((int64_t)(s + u) * 4 + q) * CH;
#pragma unroll
            for (int h = 0; h < 2; h++) b[u][h] = *(const FU*)(bp[h] + k);
#pragma unroll
            for (int t = 0; t < MT; t++) a[u][t] = *(const FU*)(ap[t] + k);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int h = 0; h < 2; h++) acc[h][t] = mma(b[u][h], a[u][t], acc[h][t]);
    }
    auto chunk = [&](const T* row, int64_t k) {
        F v;
        if (k + CH <= K) {
            v = *(const FU*)(row + k);
        } else {
#pragma unroll
            for (int i = 0; i < CH; i++) v[i] = k + i < K ? row[k + i] : (T)0.0f;
        }
        return v;
    };
    for (; s < s1; s++) {
        const int64_t k = ((int64_t)s * 4 + q) * CH;
        const F b0 = chunk(bp[0], k), b1 = chunk(bp[1], k);
#pragma unroll
        for (int t = 0; t < MT; t++) {
            const F a = chunk(ap[t], k);
            acc[0][t] = mma(b0, a, acc[0][t]);
            acc[1][t] = mma(b1, a, acc[1][t]);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
        for (int h = 0; h < 2; h++) part[w][2 * t + h][lane] = acc[h][t];
    __syncthreads();
    if (w >= MT) return;
    floatx4 v[2] = {part[0][2 * w][lane], part[0][2 * w + 1][lane]};
#pragma unroll
    for (int i = 1; i < WAVES; i++) v[0] += part[i][2 * w][lane], v[1] += part[i][2 * w + 1][lane];
    GatedEpilogue<T, 2> e;
    e.columns(p, n0 + 4 * q);
    e.row(p, 16 * w + r, v);
}

// Any strides and sizes: 64 rows by 32 outputs a workgroup, 32 by 16 of them each of its four waves,
// 16-byte chunks of k staged through LDS by guarded loads. Takes what the kernels above do not:
// operands that are not 16-byte aligned or too large for their offsets. Correct before fast.
template <class T>
__global__ __launch_bounds__(256) void gated_any_kernel(Gemm p) {
    constexpr int CH = 16 / sizeof(T), BK = 4 * CH, LD = BK + CH;
    __shared__ __align__(16) T sa[64][LD], sb[64][LD];  // sb: 32 rows of the gate, 32 of the other half
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const int64_t tiles_n = (p.N + 31) / 32;
    const int64_t m0 = blockIdx.x / tiles_n * 64, n0 = blockIdx.x % tiles_n * 32;
    const int wm = (w & 1) * 32, wn = (w >> 1) * 16;
    floatx4 acc[2][2] = {};
    for (int64_t k0 = 0; k0 < p.K; k0 += BK) {
        for (int i = t; i < 64 * BK; i += 256) {
            const int row = i / BK, k = i % BK;
            const int64_t n = n0 + row % 32;
            sa[row][k] = m0 + row < p.M && k0 + k < p.K ? ((const T*)p.a.ptr)[(m0 + row) * p.a.ld + k0 + k] : (T)0.0f;
            sb[row][k] = n < p.N && k0 + k < p.K ? ((const T*)p.b.ptr)[((row < 32 ? 0 : p.N) + n) * p.b.ld + k0 + k] : (T)0.0f;
        }
        __syncthreads();
        using F = vec<T, CH>;
        F fa[2], fb[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            fa[i] = *(const F*)&sa[wm + 16 * i + lane % 16][lane / 16 * CH];
            fb[i] = *(const F*)&sb[wn + 32 * i + lane % 16][lane / 16 * CH];
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] = mma(fb[j], fa[i], acc[i][j]);
        __syncthreads();
    }
    GatedEpilogue<T, 2> e;
    e.columns(p, n0 + wn + 4 * (lane / 16));
#pragma unroll
    for (int i = 0; i < 2; i++) e.row(p, m0 + wm + 16 * i + lane % 16, acc[i]);
}

// p without its plan's fields; `partial` has plan.bytes bytes.
int gated_gemm(int dtype, Gemm p, const GemmPlan& plan, float* partial, hipStream_t s) {
    const int64_t ch = 16 / (int64_t)type_size(dtype), bk = 8 * ch, kt = (p.K + bk - 1) / bk;
    const bool fast = plan.tile && aligned(p.a.ptr) && aligned(p.b.ptr);
    const int tile = fast ? plan.tile : 64;  // gated_any_kernel's too
    const int64_t tiles = (p.M + tile - 1) / tile * ((p.N + tile / 2 - 1) / (tile / 2));
    p.splits = fast ? plan.splits : 1;
    p.tiles_per_split = (int)((kt + p.splits - 1) / p.splits);
    p.partial = p.splits > 1 ? partial : nullptr;
    const dim3 grid((unsigned)tiles, (unsigned)p.splits);
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (plan.rows) {
            const dim3 groups((unsigned)((p.N + 15) / 16));
            if (p.M <= 16) gated_rows_kernel<T, 1><<<groups, 512, 0, s>>>(p);
            else if (p.M <= 32) gated_rows_kernel<T, 2><<<groups, 512, 0, s>>>(p);
            else gated_rows_kernel<T, 4><<<groups, 512, 0, s>>>(p);
            return DRH_OK;
        }
        if (!fast) {
            gated_any_kernel<T><<<grid, 256, 0, s>>>(p);
            return DRH_OK;
        }
        auto launch = [&](auto math) {
            using Math = decltype(math);
            const bool alone = tiles * p.splits <= CUS;
            if constexpr (sizeof(T) == 2)
                if (tile == 256) gated_256_kernel<T><<<grid, 512, 0, s>>>(p);
            if (tile == 128 && alone) gated_tile_kernel<T, Math, 128, 2><<<grid, 512, 0, s>>>(p);
            if (tile == 128 && !alone) gated_tile_kernel<T, Math, 128, 1><<<grid, 256, 0, s>>>(p);
            if (tile == 64 && alone) gated_tile_kernel<T, Math, 64, 2><<<grid, 512, 0, s>>>(p);
            if (tile == 64 && !alone) gated_tile_kernel<T, Math, 64, 1><<<grid, 256, 0, s>>>(p);
        };
        if constexpr (sizeof(T) == 4) {
            if (p.K >= THIRDS_LEAST) launch(Thirds());
            else launch(Straight());
        } else {
            launch(Straight());
        }
        if (p.partial)
            in_launches((p.M * ((p.N + ch - 1) / ch) + 255) / 256, most_groups(256), [&](int64_t first, int64_t count) {
                gated_join<T><<<dim3((unsigned)count), 256, 0, s>>>(p, first);
            });
        return DRH_OK;
    });
}

// ---------------------------------------------------------------- dz and the bias gradient

// dz = [dy zu act'(zg), dy act(zg)], rounded to its type for the products, in rows of ldz elements
// with zeros behind 2 N, and the column sums of the unrounded values: a workgroup owns 64 chunks of
// every gridDim.y-th slab of rows, its four waves a row each, added in order at the end. Bound by memory:
// 16384 x 4096 in bfloat16 (740 MB) take 130 us, 5.7 TB/s; ONCE: loads and stores past the caches, without
// which forward and backward of that size take 34 us more.
template <class T, bool ONCE>
__global__ __launch_bounds__(256) void gate_slopes(const T* __restrict__ dy, const void* __restrict__ kept, int64_t M, int64_t N,
                                                   int64_t ldz, T* __restrict__ dz, float* part) {
    constexpr int CH = 16 / sizeof(T);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = ((int64_t)blockIdx.x * 64 + lane) * CH;
    float sum[2][CH] = {};
    const int64_t stride = (int64_t)gridDim.y * 4, left = N - c;
    struct Row {
        Raw g, a, b, lo;
    };
    auto fetch = [&](int64_t row, Row& to) {
        to = Row{};
        if (row >= M) return;
        const int64_t at = row * N + c;
        to.g = load_raw<false, ONCE>(dy + at, left);
        to.a = load_raw<false, ONCE>((const T*)kept + at, left);
        to.b = load_raw<false, ONCE>((const T*)kept + M * N + at, left);
        to.lo = Pairs<T, CH>::rest(kept, M * N, at, left);
    };
    auto finish = [&](int64_t row, const Row& from) {
        if (row >= M) return;
        const Elements<T> ge = __builtin_bit_cast(Elements<T>, from.g);
        float dg[CH], du[CH], a[CH], b[CH];
        Pairs<T, CH>::open(from.a, from.b, from.lo, a, b);
#pragma unroll
        for (int i = 0; i < CH; i++) {
            du[i] = (float)ge[i] * a[i], dg[i] = (float)ge[i] * b[i];
            sum[0][i] += dg[i], sum[1][i] += du[i];
        }
        if (dz) {
            store_once<ONCE, CH>(dz + row * ldz + c, left, dg);
            store_once<ONCE, CH>(dz + row * ldz + N + c, left, du);
            if (left <= CH)  // the last chunk's lane
                for (int64_t i = 2 * N; i < ldz; i++) dz[row * ldz + i] = (T)0.0f;
        }
    };
    if (left > 0)
        for (int64_t row = (int64_t)blockIdx.y * 4 + w; row < M; row += 2 * stride) {  // two rows' loads at once
            Row r0, r1;
            fetch(row, r0);
            fetch(row + stride, r1);
            finish(row, r0);
            finish(row + stride, r1);
        }
    if (!part) return;
    __shared__ float sums[4][64 * CH];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < CH; i++) sums[w][lane * CH + i] = sum[h][i];
        __syncthreads();
        for (int k = threadIdx.x; k < 64 * CH; k += 256) {
            const int64_t col = (int64_t)blockIdx.x * 64 * CH + k;
            if (col < N) part[(int64_t)blockIdx.y * 2 * N + h * N + col] = sums[0][k] + sums[1][k] + sums[2][k] + sums[3][k];
        }
    }
}

// ---------------------------------------------------------------- plans

struct ForwardPlan {
    Rows x, w;
    GemmPlan y;
    size_t x_at = 0, w_at = 0, part_at = 0, total = 0;
};

ForwardPlan forward_plan(int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws, int dtype) {
    ForwardPlan f;
    xs = stride_of(M, xs, K);
    if (few_rows(M, N, K)) {
        f.x = {xs}, f.w = {ws}, f.y.rows = true;
        return f;
    }
    f.x = rows_for(dtype, M, K, xs);
    f.w = rows_for(dtype, 2 * N, K, ws);
    const int64_t ch = 16 / (int64_t)type_size(dtype), K_pad = (K + ch - 1) / ch * ch;
    f.y = plan_gemm(dtype, M, 2 * N, K, chunked(dtype, true, f.x.ld, M, K_pad) && chunked(dtype, true, f.w.ld, N, K_pad));
    if (!f.y.tile) f.x = {xs}, f.w = {ws};
    f.w_at = f.x.bytes;
    f.part_at = f.w_at + f.w.bytes;
    f.total = f.part_at + f.y.bytes;
    return f;
}

int check_gated_sizes(int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws) {
    if (N > (1 << 29)) return fail(DRH_ERR_TOO_LARGE, "more than 2^29 outputs");
    return check_product_sizes(M, 2 * N, K, xs, ws);
}

int check_gated(drh_ctx* ctx, int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws, int dtype, uint32_t flags) {
    int rc = check_call(ctx, dtype, flags);
    return rc ? rc : check_gated_sizes(M, N, K, xs, ws);
}

int check_bytes(int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws, int dtype, const uint64_t* out_bytes) {
    if (!out_bytes || !known_type(dtype)) return fail(DRH_ERR_INVALID_ARG, "unknown element type, or out_bytes is NULL");
    return check_gated_sizes(M, N, K, xs, ws);
}

// dz is always made: the linear layer's plan for an activation.
BackwardPlan gated_backward_plan(int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws, int dtype) {
    return backward_plan(M, 2 * N, K, xs, ws, dtype, DRH_ACT_RELU);
}

}  // namespace
}  // namespace drh_nn

using namespace drh_nn;

extern "C" {

int drh_gated_linear_bytes(int64_t rows, int64_t n_out, int64_t n_in, int64_t x_stride, int64_t weight_stride, int dtype,
                           uint64_t* out_bytes) {
    int rc = check_bytes(rows, n_out, n_in, x_stride, weight_stride, dtype, out_bytes);
    if (rc) return rc;
    *out_bytes = forward_plan(rows, n_out, n_in, x_stride, weight_stride, dtype).total;
    return DRH_OK;
}

int drh_gated_linear(drh_ctx* ctx, const void* x, const void* weight, const void* bias, int64_t rows, int64_t n_out,
                     int64_t n_in, int64_t x_stride, int64_t weight_stride, int dtype, int activation, void* y, void* kept,
                     void* workspace, uint64_t workspace_bytes, void* stream, uint32_t flags) {
    int rc = check_gated(ctx, rows, n_out, n_in, x_stride, weight_stride, dtype, flags);
    if (rc) return rc;
    if (activation < DRH_ACT_NONE || activation > DRH_ACT_SILU)
        return fail(DRH_ERR_INVALID_ARG, "unknown activation " + std::to_string(activation));
    if (rows == 0) return DRH_OK;
    if (!y || (n_in > 0 && (!x || !weight))) return fail(DRH_ERR_INVALID_ARG, "x, weight and y must not be NULL");
    if (!aligned(kept)) return fail(DRH_ERR_INVALID_ARG, "kept must be 16-byte aligned");
    const ForwardPlan plan = forward_plan(rows, n_out, n_in, x_stride, weight_stride, dtype);
    rc = check_workspace(plan.total, workspace, workspace_bytes);
    if (rc) return rc;
    rc = check_tiles(plan.y, rows, 2 * n_out, plan.x.bytes ? nullptr : x, plan.w.bytes ? nullptr : weight);
    if (rc) return rc;
    DeviceGuard dg(ctx->device);
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    pad(dtype, {x, ws + plan.x_at, x_stride, plan.x.bytes ? rows : 0},
        {weight, ws + plan.w_at, weight_stride, plan.w.bytes ? 2 * n_out : 0}, n_in, s);
    Gemm p{};
    p.a = {plan.x.bytes ? ws + plan.x_at : x, plan.x.ld, rows};
    p.b = {plan.w.bytes ? ws + plan.w_at : weight, plan.w.ld, n_out};
    p.M = rows, p.N = n_out, p.K = n_in;
    p.bias = bias, p.out = y, p.kept = kept, p.act = activation;
    rc = gated_gemm(dtype, p, plan.y, (float*)(ws + plan.part_at), s);
    return rc ? rc : finish_call(s, flags, "gated linear");
}

int drh_gated_linear_backward_bytes(int64_t rows, int64_t n_out, int64_t n_in, int64_t x_stride, int64_t weight_stride,
                                    int dtype, uint64_t* out_bytes) {
    int rc = check_bytes(rows, n_out, n_in, x_stride, weight_stride, dtype, out_bytes);
    if (rc) return rc;
    *out_bytes = gated_backward_plan(rows, n_out, n_in, x_stride, weight_stride, dtype).total;
    return DRH_OK;
}

int drh_gated_linear_backward(drh_ctx* ctx, const void* x, const void* weight, const void* kept, const void* grad_y,
                              int64_t rows, int64_t n_out, int64_t n_in, int64_t x_stride, int64_t weight_stride, int dtype,
                              void* grad_x, void* grad_weight, void* grad_bias, void* workspace, uint64_t workspace_bytes,
                              void* stream, uint32_t flags) {
    int rc = check_gated(ctx, rows, n_out, n_in, x_stride, weight_stride, dtype, flags);
    if (rc) return rc;
    const int64_t M = rows, N = n_out, K = n_in;
    if (M > 0 && (!grad_y || !kept)) return fail(DRH_ERR_INVALID_ARG, "grad_y and kept must not be NULL");
    if (!aligned(kept)) return fail(DRH_ERR_INVALID_ARG, "kept must be 16-byte aligned");
    if (M > 0 && K > 0 && ((grad_x && !weight) || (grad_weight && !x)))
        return fail(DRH_ERR_INVALID_ARG, "an input pointer is NULL");
    const BackwardPlan plan = gated_backward_plan(M, N, K, x_stride, weight_stride, dtype);
    rc = check_workspace(plan.total, workspace, workspace_bytes);
    if (rc) return rc;
    if (grad_x) rc = check_tiles(plan.dx, M, K, nullptr, plan.w.bytes ? nullptr : weight);
    if (!rc && grad_weight) rc = check_tiles(plan.dw, 2 * N, K, nullptr, plan.x.bytes ? nullptr : x);
    if (rc) return rc;
    DeviceGuard dg(ctx->device);
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    const bool dz_made = K > 0 && M > 0 && (grad_x || grad_weight);
    float* sums = grad_bias ? (float*)(ws + plan.sums_at) : nullptr;
    const int64_t groups = slope_groups(M, 2 * N, dtype), ldz = plan.ldz;
    void* dz = ws + plan.dz_at;
    if (M > 0 && (dz_made || grad_bias))
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            const int64_t cols = 64 * (16 / (int64_t)sizeof(T));
            auto go = [&](auto once) {
                gate_slopes<T, once.value><<<dim3((unsigned)((N + cols - 1) / cols), (unsigned)groups), 256, 0, s>>>(
                    (const T*)grad_y, kept, M, N, ldz, dz_made ? (T*)dz : nullptr, sums);
            };
            if (M * N * (int64_t)sizeof(T) >= READ_ONCE_BYTES) go(std::true_type());
            else go(std::false_type());
            return DRH_OK;
        });
    if (grad_bias) reduce_columns(sums, M > 0 ? groups : 0, 2 * N, 2 * N, grad_bias, nullptr, dtype, s);
    const int64_t ch = 16 / (int64_t)type_size(dtype), N_pad = (2 * N + ch - 1) / ch * ch, K_pad = (K + ch - 1) / ch * ch;
    float* part = (float*)(ws + plan.part_at);
    const bool pad_x = plan.x.bytes && grad_weight && M > 0 && K > 0, pad_w = plan.w.bytes && grad_x && M > 0 && K > 0;
    pad(dtype, {x, ws + plan.x_at, x_stride, pad_x ? M : 0}, {weight, ws + plan.w_at, weight_stride, pad_w ? 2 * N : 0}, K, s);
    if (grad_x && M > 0 && K > 0) {
        Gemm p{};
        p.a = {dz, ldz, M}, p.b = {pad_w ? ws + plan.w_at : weight, plan.w.ld, pad_w ? K_pad : K};
        p.M = M, p.N = K, p.K = 2 * N, p.out = grad_x, p.act = DRH_ACT_NONE;
        rc = gemm(dtype, KN, p, plan.dx, part, s);
        if (rc) return rc;
    }
    if (grad_weight && K > 0) {
        Gemm p{};
        p.a = {dz, ldz, N_pad}, p.b = {pad_x ? ws + plan.x_at : x, plan.x.ld, pad_x ? K_pad : K};
        p.M = 2 * N, p.N = K, p.K = M, p.out = grad_weight, p.act = DRH_ACT_NONE;
        rc = gemm(dtype, MN, p, plan.dw, part, s);
        if (rc) return rc;
    }
    return finish_call(s, flags, "gated linear backward");
}

}  // extern "C"
