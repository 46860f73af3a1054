// The products behind the layers (linear.hip), as its neighbours call them: plans, workspaces,
// padded operands.
#pragma once

#include "activation.h"
#include "gemm.h"

namespace drh_nn {

constexpr int CUS = 256;

enum Layout { KK, KN, MN };  // A's and B's contiguous dimension: forward, dx, dW

struct GemmPlan {
    int tile = 0;    // 256, 128, 64, or 0: any
    bool rows = false;  // gemm_rows_kernel
    int splits = 1;
    size_t bytes = 0;  // of partial sums
};

// gemm_rows_kernel's: it reads x from the caches for every 16 outputs, which with more rows and
// a long k costs more than staging. Microseconds in bfloat16, with it and by tiles: 32 rows
// 1280 x 1024 4.8 / 6.5, 4096 x 4096 13.2 / 13.9; 64 rows 4096 x 1024 7.2 / 9.1, 4096 x 4096 21.7 / 14.2.
constexpr int64_t ROWS_FEW = 32, ROWS_MOST = 64, ROWS_MOST_K = 2048;
inline bool few_rows(int64_t M, int64_t N, int64_t K) {
    return K > 0 && (M <= ROWS_FEW || (M <= ROWS_MOST && K <= ROWS_MOST_K)) && (N + 15) / 16 <= most_groups(512);
}
// Products in 32 bits are split in thirds from this k on: their error, 2^-21 of a term at the
// most (gemm.h says what becomes of terms too small for that), is then below what a 32-bit sum of
// as many terms may lose, k 2^-24, and shorter products are bound by memory either way.
constexpr int64_t THIRDS_LEAST = 64;
// Microseconds of a product by tiles of 64, 128 or 256 with k in `splits` parts.
double gemm_time(int dtype, int tile, double tiles, int splits, double steps, double outputs);
// The kernel for M x N outputs; `fits`: the operands are chunked.
GemmPlan plan_gemm(int dtype, int64_t M, int64_t N, int64_t K, bool fits);
// Whether an operand's sizes suit the kernels that load 16-byte chunks through buffers.
bool chunked(int dtype, bool kc, int64_t ld, int64_t rows, int64_t K);
inline bool aligned(const void* p) { return (uintptr_t)p % 16 == 0; }
// Whether a product's launch holds its tiles: a plan's always, gemm_any_kernel's 64 x 64 not
// from 2^36 outputs on.
int check_tiles(const GemmPlan& plan, int64_t M, int64_t N, const void* a, const void* b);
// p without its plan's fields; `partial` has plan.bytes bytes.
int gemm(int dtype, Layout layout, Gemm p, const GemmPlan& plan, float* partial, hipStream_t s);

// A row-major operand as the fast kernels take it: as it stands, or copied to rows of K
// elements rounded up to 16 bytes, with zeros behind K.
struct Rows {
    int64_t ld;
    size_t bytes = 0;  // of the copy, 0: none
};

Rows rows_for(int dtype, int64_t rows, int64_t K, int64_t ld);

struct PadJob {
    const void* src;
    void* dst;
    int64_t ld, rows;  // rows 0: nothing to copy
};

// Copies two operands of K columns to padded rows, in one launch.
void pad(int dtype, const PadJob& a, const PadJob& b, int64_t K, hipStream_t s);

// Row groups of a pass over M x N slopes: two rows a wave at least, and about 2048 workgroups at most.
int64_t slope_groups(int64_t M, int64_t N, int dtype);

// A single row has no stride: whatever the caller gives for it must not name rows behind it.
inline int64_t stride_of(int64_t rows, int64_t stride, int64_t K) { return rows > 1 ? stride : K; }

// x and W padded where dW and dx need them, dz where it is not dy itself or dy needs
// padding, the bias gradient's partial sums, and the larger of the products' partial sums.
struct BackwardPlan {
    Rows x, w;
    bool dz = false;
    int64_t ldz = 0;
    GemmPlan dx, dw;
    size_t x_at = 0, w_at = 0, dz_at = 0, sums_at = 0, part_at = 0, total = 0;
};

BackwardPlan backward_plan(int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws, int dtype, int act);

// x rows x n_in and weight n_out x n_in: sizes and strides that a layer takes.
int check_product_sizes(int64_t M, int64_t N, int64_t K, int64_t xs, int64_t ws);
int check_workspace(size_t need, const void* workspace, uint64_t bytes);

}  // namespace drh_nn
