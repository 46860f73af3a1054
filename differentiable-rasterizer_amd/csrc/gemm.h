// The matrix product of the linear layer on gfx950's matrix cores:
//   out[m][n] = epilogue(sum over k of A(m, k) B(n, k)),
// each operand with either k or its rows contiguous in memory.
//
// Operands go from memory to LDS without passing registers (buffer loads with LDS as their
// destination, 16 bytes a lane) in units of 128 rows by 128 bytes of k. The buffer's bounds
// check fills rows and k past the end with zeros, so no shape needs a case of its own as long
// as 16-byte chunks do not straddle an edge. In LDS a unit keeps its layout in memory, with
// its 16-byte chunks permuted by an exclusive or that spreads a wave's reads over the banks;
// the permutation is made on the loads' addresses, since a wave's load writes LDS linearly.
#pragma once

#include "layers.h"

namespace drh_nn {

using floatx4 = vec<float, 4>;

struct Operand {
    const void* ptr;
    int64_t ld;    // elements between rows (k contiguous) or between values of k (rows contiguous)
    int64_t rows;  // M or N; with rows contiguous up to the end of the last 16-byte chunk
};

struct Gemm {
    Operand a, b;
    int64_t M, N, K;
    const void *bias, *res;  // N; M x N
    void* kept;              // M x N of Kept<T>: the activation's slopes, scaled; or null
    void* out;               // M x N
    float* partial;          // splits x M x N sums instead of `out`, or null
    int act;
    int splits;              // the k range in this many parts, grid.y
    int tiles_per_split;     // tiles of k in each
};

// D = A B + C on a wave: lane l gives row l % 16 of A and of B, the 16 bytes of k that
// l / 16 picks, and holds D[4 (l / 16) + i][l % 16]. In 32 bits the four k of a lane go
// through one instruction each: any order of k will do that A and B share.
__device__ inline floatx4 mma(vec<bf16, 8> a, vec<bf16, 8> b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ inline floatx4 mma(vec<f16, 8> a, vec<f16, 8> b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline floatx4 mma(vec<float, 4> a, vec<float, 4> b, floatx4 c) {
#pragma unroll
    for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

constexpr int UNIT_BYTES = 16384;  // of 128 rows
constexpr uint32_t PAST_END = 0x7ffffff0u;  // an offset that no buffer here reaches

using lds_char = __attribute__((address_space(3))) char;

// Which of a wave's fragments of 16 rows hold which rows of a unit. Fragments of A take
// 16 rows in order. Those of B are interleaved by fours, so that a lane's results (four
// rows of each of NF fragments) are 4 NF neighbours in the output.
template <bool B, int NF>
__device__ inline int frag_row(int f, int r) {
    return B ? (r >> 2) * (4 * NF) + f * 4 + (r & 3) : f * 16 + r;
}

// The chunk permutation: by row where k is contiguous (eight chunks a row), by k where the
// rows are (sixteen chunks a value of k for 128 rows, 32 in 32 bits).
template <class T, bool KC, bool B, int NF, int ROWS>
__device__ inline int swizzle(int i) {
    constexpr int PER = ROWS * (int)sizeof(T) / 16;  // chunks a value of k
    if constexpr (KC) {
        return B ? (i & 3) | ((i / (4 * NF)) & 1) << 2 : i & 7;
    } else if constexpr (sizeof(T) == 2) {
        return (B ? 4 * (i & 3) : 2 * ((i & 3) | ((i >> 3) & 1) << 2)) & (PER - 1);
    } else {
        return (B ? 8 * ((i >> 2) & 1) + ((i >> 3) & 1) : 4 * ((i >> 2) & 3)) & (PER - 1);
    }
}

// One operand of a workgroup's tile: UNITS units of ROWS rows; row R of unit u is row
// u * ROWS + R of the tile. On B's side with two units and k contiguous it is (R / 32) * 64
// + u * 32 + R % 32 instead, so that a wave's 32 rows of both units are neighbours in the
// output; with rows contiguous that would read half lines.
template <class T, bool KC, bool B, int UNITS, int NF, int WAVES, int ROWS = 128>
struct Loader {
    static constexpr int CH = 16 / sizeof(T), BK = 8 * CH, LOADS = ROWS / 8 / WAVES;
    const char* base;
    uint64_t step;          // bytes per tile of k
    uint64_t span;          // KC: bytes from the base to the end of the tile's last row
    int64_t K;
    uint32_t row_bytes, tail_bytes;  // rows contiguous: bytes between values of k; from a row's start to its end
    uint32_t off[UNITS][LOADS];
    int kc;                 // KC: first k of the lane's chunk in a tile

    __device__ void init(const Operand& o, int64_t row0, int64_t K_) {
        const int lane = threadIdx.x & 63, w = (threadIdx.x >> 6) % WAVES;
        K = K_;
        const int64_t ld = o.ld;
        const int64_t valid = o.rows - row0 < ROWS * UNITS ? o.rows - row0 : ROWS * UNITS;
        if constexpr (KC) {
            base = (const char*)o.ptr + row0 * ld * (int64_t)sizeof(T);
            step = 128;
            span = ((valid - 1) * ld + (K + CH - 1) / CH * CH) * (int64_t)sizeof(T);  // whole chunks
        } else {
            base = (const char*)o.ptr + row0 * (int64_t)sizeof(T);
            step = BK * ld * (int64_t)sizeof(T);
            row_bytes = (uint32_t)(ld * sizeof(T));
            const int64_t tail = (o.rows - row0 < 512 ? o.rows - row0 : 512) * (int64_t)sizeof(T);
            tail_bytes = (uint32_t)tail;
        }
        kc = 0;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int pos = (i * WAVES + w) * 64 + lane;  // chunk of the unit that this load fills
#pragma unroll
            for (int u = 0; u < UNITS; u++) {
                if constexpr (KC) {
                    const int R = pos >> 3, chunk = (pos & 7) ^ swizzle<T, KC, B, NF, ROWS>(R);
                    off[u][i] = (uint32_t)(tile_row(u, R) * ld * sizeof(T)) + chunk * 16;
                    kc = chunk * CH;
                } else {
                    constexpr int PER = ROWS / CH;
                    const int k = pos / PER, R = ((pos % PER) ^ swizzle<T, KC, B, NF, ROWS>(k)) * CH;
                    const int64_t row = tile_row(u, R);
                    off[u][i] = row0 + row < o.rows ? (uint32_t)(k * ld * sizeof(T) + row * sizeof(T)) : PAST_END;
                }
            }
        }
    }

    static __device__ int64_t tile_row(int u, int R) {
        return B && KC && UNITS == 2 ? (R / 32) * 64 + u * 32 + R % 32 : u * ROWS + R;
    }

    // Starts the loads of unit u of k tile kt into LDS at `lds`; past the last tile they
    // fill it with zeros and touch no memory, so that every tile has the same loads.
    __device__ void issue(int u, int64_t kt, uint32_t lds) const {
        const int w = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) % WAVES);
        const int64_t left = K - kt * BK;
        const char* p = base + kt * step;
        uint32_t bytes;
        if constexpr (KC) {
            bytes = left > 0 ? (uint32_t)(span - kt * 128) : 0u;
        } else {
            const int rows = left >= BK ? BK : left > 0 ? (int)left : 0;
            bytes = rows ? (uint32_t)(rows - 1) * row_bytes + tail_bytes : 0u;
        }
        vec<uint32_t, 4> rsrc = {(uint32_t)(uintptr_t)p, (uint32_t)((uintptr_t)p >> 32) & 0xffffu, bytes, 0x00020000u};
#pragma unroll
        for (int i = 0; i < 4; i++) rsrc[i] = __builtin_amdgcn_readfirstlane(rsrc[i]);
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const uint32_t dst = __builtin_amdgcn_readfirstlane(lds + (i * WAVES + w) * 1024);
            uint32_t o = off[u][i];
            if constexpr (KC) o = kc < left ? o : PAST_END;
            // m0, the destination, is a reserved register: the compiler keeps nothing in it, and a
            // clobber list may not name it
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst), "v"(o),
                         "s"(rsrc)
                         : "memory");
        }
    }
};

template <int N>
__device__ inline void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}
// Nothing of this wave's is on its way to LDS or from it.
__device__ inline void wait_all() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
__device__ inline void wg_barrier() { asm volatile("s_barrier" ::: "memory"); }

// A wave's fragments of one unit, NF of 16 rows from row r0 on, both halves of the k tile.
template <class T, bool KC, bool B, int NF, int ROWS = 128>
struct Frags {
    static constexpr int CH = 16 / sizeof(T);
    using F = vec<T, CH>;
    F f[NF][2];

    // unit: the unit in LDS
    __device__ void read(const char* unit, int r0) {
        const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
#pragma unroll
        for (int i = 0; i < NF; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if constexpr (KC) {
                    const int R = r0 + frag_row<B, NF>(i, r);
                    f[i][h] = *(const F*)(unit + R * 128 + (((h * 4 + q) ^ swizzle<T, KC, B, NF, ROWS>(R)) * 16));
                } else if constexpr (sizeof(T) == 2) {
                    // A transposing read: sixteen lanes give the addresses of four rows' pieces
                    // for four values of k, and each gets its row's four values.
                    using S4 = vec<short, 4>;
                    union {
                        S4 s[2];
                        F v;
                    } x;
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int k = h * 32 + q * 8 + e * 4 + (r >> 2), R = r0 + frag_row<B, NF>(i, (r & 3) * 4);
                        const char* p = unit + k * (ROWS * 2) + (((R >> 3) ^ swizzle<T, KC, B, NF, ROWS>(k)) * 16) + (R & 7) * 2;
                        x.s[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) S4*)p);
                    }
                    f[i][h] = x.v;
                } else {
                    const int R = r0 + frag_row<B, NF>(i, r);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int k = h * 16 + q * 4 + e;
                        f[i][h][e] = *(const float*)(unit + k * (ROWS * 4) + (((R >> 2) ^ swizzle<T, KC, B, NF, ROWS>(k)) * 16) + (R & 3) * 4);
                    }
                }
            }
    }
};

// How a k tile's fragments are multiplied.
//
// Straight: with the instructions of the operands' own type.
//
// Thirds, for 32 bits: v = v1 + v2 + v3 in bfloat16, each the first eight bits of what is left,
// is exact (3 x 8 bits) from about 2^-111 on, above bfloat16's smallest number, 2^-133, by all of
// them; a tile where what smaller numbers lose could count is made again (gemm_tile's second pass). a b is a1 b1 + a1 b2
// + a2 b1 + a2 b2 + a1 b3 + a3 b1 but for less than 2^-21 |a b|, 2^-24 in the mean; thirds have
// their value's sign, so what is dropped of a product has the product's. Six bfloat16 products
// take 96 cycles of the matrix core where the 32-bit instructions take 256, and splitting costs six
// vector operations an element, four to five behind each matrix instruction of a 64 x 64 quarter.
// (Rounding each third to the nearest is as many operations, but the conversion is a slow one.)
// Alone, a matrix instruction and four such operations take 12 ns with one wave a SIMD and 10 with
// two, 8 and 7 without them: the two kinds overlap in part. 4096^3 takes 680 to 760 us (190
// TFLOP/s in 32 bits, 1.15 P in bfloat16, where the power limit has the clock) however the splits
// are placed; 4096 x 1024 outputs and k = 1024 64 us, of which gathering what is lost is three.
// Infinities come out as NaN: see gemm_tile's second pass.
struct Straight {
    template <class FA, class FB, int NA, int NB>
    static __device__ inline void multiply(const FA& a, const FB& b, floatx4 (&acc)[NA][NB]) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < NA; i++)
#pragma unroll
                for (int j = 0; j < NB; j++) acc[i][j] = mma(b.f[j][h], a.f[i][h], acc[i][j]);
    }
};

struct Thirds {
    struct Held {
        vec<uint32_t, 4> third[3];
    };
    // A third of the work of splitting pair i of a fragment's values: three parts in turn, with
    // `r` and `m` handed on.
    struct Pair {
        uint32_t r[2], m[2];
        __device__ void less(int i) {
            r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, r[i]) - __builtin_bit_cast(float, m[i]));
        }
    };
    // `lost` gathers what the last third leaves in its lower 16 bits.
    template <class F>
    static __device__ inline void split(const F (&f)[2], Held& to, int i, int part, Pair& p, uint32_t& lost) {
        if (part == 0)
#pragma unroll
            for (int e = 0; e < 2; e++) p.r[e] = __builtin_bit_cast(uint32_t, (float)f[i / 2][2 * (i % 2) + e]);
        if (part == 1) p.less(1);
        if (part == 2) {
            p.less(0), p.less(1);
            lost |= p.r[0] | p.r[1];
            asm volatile("" : "+v"(lost));  // here, so that nothing of the pairs is kept for it
        }
        uint32_t both = __builtin_amdgcn_perm(p.r[1], p.r[0], 0x07060302);  // the upper halves
        asm volatile("" : "+v"(both));  // here, not where it is used
        to.third[part][i] = both;
        if (part < 2)
#pragma unroll
            for (int e = 0; e < 2; e++) p.m[e] = p.r[e] & 0xffff0000u;
        if (part == 0) p.less(0);
    }
    template <class F>
    static __device__ inline void split(const F (&f)[2], Held& to, uint32_t& lost) {
        Pair p;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int part = 0; part < 3; part++) split(f, to, i, part, p, lost);
    }
    static __device__ inline vec<bf16, 8> term(const Held& h, int third) {
        return __builtin_bit_cast(vec<bf16, 8>, h.third[third]);
    }
    // A fragment of A by all of B's, the smallest terms first; between the matrix instructions
    // the parts of SPLITS splits, v0 to h0 and v1 to h1.
    template <int SPLITS, int NF, class FA, class FB>
    static __device__ inline void row(const Held& a, const Held (&b)[NF], floatx4 (&acc)[NF], const FA& v0, Held& h0,
                                      const FB& v1, Held& h1, uint32_t& lost) {
        constexpr int PA[6] = {2, 0, 1, 1, 0, 0}, PB[6] = {0, 2, 1, 0, 1, 0}, PARTS = 4 / NF;
        Pair p;
#pragma unroll
        for (int m = 0; m < 6 * NF; m++) {
            acc[m % NF] = mma(term(b[m % NF], PB[m / NF]), term(a, PA[m / NF]), acc[m % NF]);
#pragma unroll
            for (int e = 0; e < PARTS; e++) {
                const int n = m * PARTS + e;
                if (n < 12 && SPLITS > 0) split(v0, h0, n / 3, n % 3, p, lost);
                if (n >= 12 && SPLITS > 1) split(v1, h1, (n - 12) / 3, n % 3, p, lost);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// The tile that a workgroup takes. Workgroups go to the eight XCDs in turn and each XCD
// has an L2 of its own: an XCD gets a run of neighbouring tiles, in bands eight tiles high.
__device__ inline void pick_tile(int64_t tiles_m, int64_t tiles_n, int64_t& tm, int64_t& tn) {
    const uint32_t total = gridDim.x, b = blockIdx.x, xcd = b & 7, in = b >> 3;
    const uint32_t per = total >> 3, extra = total & 7;
    const uint32_t id = xcd * per + (xcd < extra ? xcd : extra) + in;
    constexpr uint32_t BAND = 8;
    const uint32_t band = id / (uint32_t)(BAND * tiles_n), first = band * BAND;
    const uint32_t high = tiles_m - first < BAND ? (uint32_t)tiles_m - first : BAND;
    const uint32_t rest = id - band * (uint32_t)(BAND * tiles_n);
    tm = first + rest % high;
    tn = rest / high;
}

// 256 x 256 of the output by eight waves, 128 x 64 each, in quarters of 64 x 32: one unit
// of A by one of B. LDS holds two k tiles (128 KiB), so one workgroup fills a CU, two waves
// a SIMD. The waves of a SIMD are of two groups that run half a step apart: while one reads
// its fragments and starts loads, the other has the matrix cores. A k tile is four steps, each
// reading at most one unit's fragments and starting one unit's loads, six steps ahead of
// their use (five units in flight). A unit is overwritten two steps after both groups have
// read it at the earliest.
//
// 8192^3 in bfloat16 takes 765 us, 1.43 PFLOP/s: the matrix cores are busy for 75% of the cycles
// at the 1.8 GHz that the power limit leaves, so it is power that bounds it. With k of 1024 and
// less a tile's start and end, about 10 us that nothing covers, count as well: 16384 x 4096
// outputs and k = 1024 take 132 us (1.04 PFLOP/s), 16384 x 1024 and k = 4096 103 us (1.33). A CU that
// is given 128 x 128 tiles instead reads an operand twice as often: 72 and 61 us at 4096^2 and k = 2048.
template <class T, bool AK, bool BK_, class Epilogue>
__device__ inline void gemm_256(const Gemm& p) {
    __shared__ __align__(1024) char lds[8 * UNIT_BYTES];
    using LA = Loader<T, AK, false, 2, 4, 8>;
    using LB = Loader<T, BK_, true, 2, 2, 8>;
    int64_t tm, tn;
    pick_tile((p.M + 255) / 256, (p.N + 255) / 256, tm, tn);
    const int64_t m0 = tm * 256, n0 = tn * 256;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = w >> 2, wn = w & 3;
    const int64_t tiles = (p.K + LA::BK - 1) / LA::BK, first = (int64_t)blockIdx.y * p.tiles_per_split;
    const int64_t last = first + p.tiles_per_split < tiles ? first + p.tiles_per_split : tiles;
    LA la;
    LB lb;
    la.init(p.a, m0, p.K);
    lb.init(p.b, n0, p.K);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char*)lds;
    // units of a buffer: A0, A1, B0, B1
    auto at = [&](int64_t kt, int unit) { return (uint32_t)(((kt - first) & 1) * 4 + unit) * UNIT_BYTES; };
    auto load_a = [&](int u, int64_t kt) { la.issue(u, kt, lds0 + at(kt, u)); };
    auto load_b = [&](int u, int64_t kt) { lb.issue(u, kt, lds0 + at(kt, 2 + u)); };

    floatx4 acc[2][2][4][2] = {};
    Frags<T, AK, false, 4> fa;
    Frags<T, BK_, true, 2> fb[2];
    load_b(0, first);
    load_a(0, first);
    load_b(1, first);
    load_a(1, first);
    load_b(0, first + 1);
    load_a(0, first + 1);
    load_b(1, first + 1);
    wait_vm<10>();
    wg_barrier();
    fb[0].read(lds + at(first, 2), wn * 32);
    if (wm == 1) wg_barrier();

    auto step = [&](int ua, int ub) {
        wait_vm<10>();
        __builtin_amdgcn_sched_barrier(0);
        wg_barrier();
        __builtin_amdgcn_s_setprio(1);
        Straight::multiply(fa, fb[ub], acc[ua][ub]);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        wg_barrier();
    };
    for (int64_t kt = first; kt < last; kt++) {
        fa.read(lds + at(kt, 0), wm * 64);
        load_a(1, kt + 1);
        step(0, 0);
        fb[1].read(lds + at(kt, 3), wn * 32);
        load_b(0, kt + 2);
        step(0, 1);
        fa.read(lds + at(kt, 1), wm * 64);
        load_a(0, kt + 2);
        step(1, 0);
        fb[0].read(lds + at(kt + 1, 2), wn * 32);
        load_b(1, kt + 2);
        step(1, 1);
    }
    if (wm == 0) wg_barrier();
    wait_vm<0>();  // LDS is given up with no load on its way there
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int nu = BK_ ? 32 : 128;
    Epilogue e0, e1;
    e0.columns(p, n0 + wn * (BK_ ? 64 : 32) + q * 8);
    e1.columns(p, n0 + wn * (BK_ ? 64 : 32) + nu + q * 8);
#pragma unroll
    for (int ua = 0; ua < 2; ua++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t m = m0 + ua * 128 + wm * 64 + i * 16 + r;
            e0.row(p, m, acc[ua][0][i]);
            e1.row(p, m, acc[ua][1][i]);
        }
}

// TILE x TILE (128 or 64) by GROUPS groups of four waves, a quarter of the output each, two k
// tiles in LDS for each group. With one group a CU takes two workgroups with tiles of 128, five
// with 64, which cover each other's waits: more k tiles in LDS were slower for both (4096^2
// outputs, k = 2048 in bfloat16: 72 us with two of 128, 111 with four; 107 with two of 64, 105 with
// three, 124 with four). A workgroup that is alone on its CU has two groups that cover each
// other's waits: they take the k tiles in turn, and add their sums through LDS at the end.
template <class T, bool AK, bool BK_, class Epilogue, class Math, int TILE, int GROUPS>
__device__ inline void gemm_tile(const Gemm& p) {
    constexpr int NF = TILE / 32, UNIT = TILE * 128;
    __shared__ __align__(1024) char lds[GROUPS * 4 * UNIT];
    using LA = Loader<T, AK, false, 1, NF, 4, TILE>;
    using LB = Loader<T, BK_, true, 1, NF, 4, TILE>;
    using FA = Frags<T, AK, false, NF, TILE>;
    using FB = Frags<T, BK_, true, NF, TILE>;
    int64_t tm, tn;
    pick_tile((p.M + TILE - 1) / TILE, (p.N + TILE - 1) / TILE, tm, tn);
    const int64_t m0 = tm * TILE, n0 = tn * TILE;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3, group = GROUPS == 2 ? wave >> 2 : 0;
    const int wm = (w >> 1) * (TILE / 2), wn = (w & 1) * (TILE / 2);
    const int64_t tiles = (p.K + LA::BK - 1) / LA::BK, start = (int64_t)blockIdx.y * p.tiles_per_split;
    const int64_t last = start + p.tiles_per_split < tiles ? start + p.tiles_per_split : tiles;
    const int64_t first = start + group, steps = (last - start + GROUPS - 1) / GROUPS;  // the group's tiles
    LA la;
    LB lb;
    la.init(p.a, m0, p.K);
    lb.init(p.b, n0, p.K);
    char* mine = lds + group * 4 * UNIT;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char*)mine;
    auto load = [&](int64_t step, int stage) {
        const uint32_t b = (uint32_t)stage * 2 * UNIT;
        la.issue(0, first + step * GROUPS, lds0 + b);
        lb.issue(0, first + step * GROUPS, lds0 + b + UNIT);
    };
    floatx4 acc[NF][NF] = {};
    auto walk = [&](auto use) {  // use(fragments of A, of B) for each tile
        load(0, 0);
        for (int64_t i = 0; i < steps; i++) {
            const int stage = (int)i & 1;
            const char* b = mine + stage * 2 * UNIT;
            wait_all();
            wg_barrier();  // this tile is there, and the other buffer read by every wave
            load(i + 1, stage ^ 1);
            if (GROUPS == 1 || first + i * GROUPS < last) {
                FA fa;
                FB fb;
                fa.read(b, wm);
                fb.read(b + UNIT, wn);
                use(fa, fb);
            }
        }
        wait_all();  // LDS is given up, or used again, with no load on its way there
    };
    auto straight = [&] { walk([&](const FA& fa, const FB& fb) { Straight::multiply(fa, fb, acc); }); };
    if constexpr (std::is_same_v<Math, Straight>) {
        straight();
    } else {
        // While a tile is multiplied, the next one's fragments are read and split. ha[0] holds a
        // tile's first fragment of A when its turn comes, fa the others as they were read.
        FA fa;
        FB fb;
        Thirds::Held ha[2], even[NF], odd[NF];
        uint32_t lost = 0;
        load(0, 0);
        load(1, 1);
        wait_vm<LA::LOADS + LB::LOADS>();
        wg_barrier();
        fa.read(mine, wm);
        fb.read(mine + UNIT, wn);
#pragma unroll
        for (int j = 0; j < NF; j++) Thirds::split(fb.f[j], even[j], lost);
        Thirds::split(fa.f[0], ha[0], lost);
        auto multiply = [&](const char* b, const Thirds::Held (&now)[NF], Thirds::Held (&next)[NF], auto more) {
            constexpr bool MORE = more.value;
            if (MORE) fb.read(b + UNIT, wn);
#pragma unroll
            for (int r = 0; r < NF - 1; r++)
                Thirds::row<MORE ? 2 : 1>(ha[r & 1], now, acc[r], fa.f[r + 1], ha[(r + 1) & 1], fb.f[r], next[r], lost);
            if (MORE) fa.read(b, wm);
            Thirds::row<MORE ? 2 : 0>(ha[1], now, acc[NF - 1], fb.f[NF - 1], next[NF - 1], fa.f[0], ha[0], lost);
        };
        auto step = [&](int64_t i, const Thirds::Held (&now)[NF], Thirds::Held (&next)[NF]) {
            const int stage = (int)i & 1;
            wait_all();
            wg_barrier();  // the next tile is there, and this one read by every wave
            load(i + 2, stage);
            const char* b = mine + (stage ^ 1) * 2 * UNIT;
            const int64_t kt = first + i * GROUPS;
            // The last tile has no next one; where registers are short it takes the code of the others
            if (kt + GROUPS < last || (NF == 4 && GROUPS == 1)) multiply(b, now, next, std::true_type());
            else if (GROUPS == 1 || kt < last) multiply(b, now, next, std::false_type());
        };
        for (int64_t i = 0; i < steps; i += 2) {
            step(i, even, odd);
            if (i + 1 < steps) step(i + 1, odd, even);
        }
        wait_all();
        // A result that is not finite comes from an infinity, a NaN or an overflow. The thirds turn
        // the first into NaN, so the tile is made again with instructions that do not.
        float zero = 0.0f;
#pragma unroll
        for (int i = 0; i < NF * NF; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) zero = fmaf(acc[i / NF][i % NF][e], 0.0f, zero);
        bool again = !(zero == 0.0f);
        // So it is where the thirds lost bits that count. A number loses less than 2^-133, so a sum
        // is off by that times k times the largest numbers; 2^-21 of the sum is what thirds may cost.
        // A few numbers of a GELU's tail, say, are no reason: they are found by reading the tiles once
        // more, a third of the time of making them again.
        if (__syncthreads_or(lost & 0xffffu)) {
            float most = 0.0f;
            auto largest = [&](const auto& f) {
#pragma unroll
                for (int i = 0; i < NF; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf(f.f[i][e / 4][e % 4]));
            };
            walk([&](const FA& fa, const FB& fb) { largest(fa), largest(fb); });
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
            const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
            const float least = most * (float)(steps * LA::BK) * 0x1p-111f;
#pragma unroll
            for (int i = 0; i < NF * NF; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool there = m0 + wm + i / NF * 16 + r < p.M && n0 + wn + q * (4 * NF) + i % NF * 4 + e < p.N;
                    again |= there && !(fabsf(acc[i / NF][i % NF][e]) >= least);
                }
        }
        if (__syncthreads_or(again)) {
#pragma unroll
            for (int i = 0; i < NF * NF; i++) acc[i / NF][i % NF] = floatx4{};
            straight();
        }
    }
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    Epilogue epilogue;
    epilogue.columns(p, n0 + wn + q * (4 * NF));
    if constexpr (GROUPS == 1) {
#pragma unroll
        for (int i = 0; i < NF; i++) epilogue.row(p, m0 + wm + i * 16 + r, acc[i]);
    } else {
        // Each group finishes half of the rows, with the other's sums of them.
        constexpr int HALF = NF / 2;
        floatx4* to = (floatx4*)lds + (wave ^ 4) * (HALF * NF * 64) + lane;
        const floatx4* from = (const floatx4*)lds + wave * (HALF * NF * 64) + lane;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < HALF * NF; i++) to[i * 64] = group ? acc[i / NF][i % NF] : acc[HALF + i / NF][i % NF];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < HALF; i++) {
            floatx4 sum[NF];
#pragma unroll
            for (int j = 0; j < NF; j++) sum[j] = (group ? acc[HALF + i][j] : acc[i][j]) + from[(i * NF + j) * 64];
            epilogue.row(p, m0 + wm + (group * HALF + i) * 16 + r, sum);
        }
    }
}

}  // namespace drh_nn
