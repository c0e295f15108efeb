// Products of rows in 8 bits (gfx950): what its kernels share.
//
//   y[m, n] = xs[m] ws[n] sum_k x[m, k] w[n, k] + bias[n]
//
// Sums are whole numbers in 32 bits, exact for K up to 131071 (128 * 128 * K <
// 2^31), so the order and the split of a sum change nothing; one conversion, two
// multiplications and an addition in float32 follow, then the rounding to the
// result's type.  x and w are both contiguous along k, rows on 16 bytes, and a
// 16-byte group of k is what a lane hands to v_mfma_i32_16x16x64_i8 (lane l: row
// l % 16, k 16 (l / 16) .. + 15; both operands alike, so any fixed order of k
// would do).  w is the first operand: a lane's four sums are four neighbouring
// columns of y.
#pragma once

#include "pe_rows.h"

namespace pe {
namespace q8 {

using ssm::BF16;

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

struct Q8Args {
    const int8_t *x, *w;              // (x of another type where the kernel for few rows takes that)
    const float *xs, *ws;
    const void* bias;
    void* y;
    int64_t x_ms, w_ns;
    int32_t M, N, K;
    int32_t bias_f32;
    int32_t tiles_m, tiles_n;
};

// Scale and bias of four neighbouring columns (past the end: of the last one).
struct Column {
    float scale[4], bias[4];
};
template <typename E>
__device__ __forceinline__ Column column(const Q8Args& g, int n) {
    Column c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int at = min(n + i, g.N - 1);
        c.scale[i] = g.ws[at];
        c.bias[i] = !g.bias ? 0.0f : g.bias_f32 ? static_cast<const float*>(g.bias)[at]
                                                : E::to_f32(static_cast<const typename E::T*>(g.bias)[at]);
    }
    return c;
}

// Column r of those in float32, from its sum and its row's scale.  A sum, at most 2^31,
// times a scale of 2^96 stays in float32, and times a small one, whichever it is, loses
// no more than a rounding: above 2^-126 that is one, below it the product, a whole
// number of the scale's last bits, is exact.  So a larger row's scale comes behind the
// column's, and nothing but the result leaves the range.  (Rows with such scales are
// rare: a branch of the wave for its rows, `value` for the others.)
__device__ __forceinline__ float value(const Column& c, float sx, int r, int32_t sum) {
    return fmaf(float(sum) * sx, c.scale[r], c.bias[r]);
}
__device__ __forceinline__ bool large(float sx) { return fabsf(sx) > 0x1p96f; }
__device__ __forceinline__ float value_of_large(const Column& c, float sx, int r, int32_t sum) {
    return large(sx) ? fmaf(float(sum) * c.scale[r], sx, c.bias[r]) : value(c, sx, r, sum);
}

// These columns of row m of y from their sums.
template <typename E>
__device__ __forceinline__ void finish(const Q8Args& g, const Column& c, float sx, int m, int n, i32x4 acc) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = value_of_large(c, sx, i, acc[i]);
    if (n < g.N) ssm::store_f32<E, 4>(static_cast<typename E::T*>(g.y) + int64_t(m) * g.N + n, g.N - n, v);
}

// Whether the kernel for few rows takes these to 8 bits itself, and the launch for x
// of y's type (rows of x as they are in g.x, x_ms in elements).
bool rows_take_own(int64_t m, int64_t k);
int rows_launch_own(int dtype, const Q8Args& g, hipStream_t stream);
int rows_launch(int y_dtype, const Q8Args& g, hipStream_t stream);
// kernel: 0 chooses a tile, 2 + i takes the i-th.
constexpr int kTileKernels = 7;
int tile_launch(int y_dtype, const Q8Args& g, int kernel, hipStream_t stream);

}  // namespace q8
}  // namespace pe
