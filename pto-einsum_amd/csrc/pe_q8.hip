// Entry point of the product of rows in 8 bits (pe_q8.h).
#include "pe_q8.h"

#include <algorithm>

namespace pe {
namespace q8 {
namespace {

constexpr int64_t kMostK = 131071;

// Whether the kernel for few rows is the one to take.
//   Up to 64 rows of x, and more where one round of blocks of 64 x 64 holds the
// product, whose waves share K: 256 x 4096 x 4096 11.3 us (tiles of the other
// kernel 17.2), 512 x 2048 x 8192 17.1 (31.8); with two rounds 512 x 4096 x 4096
// 21.0 (20.3) and 256 x 8192 x 2048 15.9 (12.1).
//   Fewer channels than a launch of its blocks, 256 threads for 64 of them, has room for;
// of the other kernel's tiles, 256 of them each, it has for all that there may be.
bool few_rows(const pe_q8_desc* d) {
    if (d->kernel) return d->kernel == 1;
    if (ceil_div(d->N, 64) >= int64_t(1) << 24) return false;
    return d->M <= 64 || ceil_div(d->M, 64) * ceil_div(d->N, 64) <= cu_count();
}

// Whether it takes x to 8 bits itself.
bool own_rows(const pe_q8_desc* d) {
    return d->x_dtype == d->y_dtype && d->K > 0 && rows_take_own(d->M, d->K) && few_rows(d);
}

// The workspace: x's rows in 8 bits and, from `scales` on, their scales, where x comes
// in another type.
struct Space {
    int64_t scales = 0, bytes = 0;
};
Space space_of(const pe_q8_desc* d) {
    Space s;
    if (d->x_dtype != PE_I8 && !own_rows(d)) {
        s.scales = ceil_div(d->M * rows::row_pitch(d->K), 256) * 256;
        s.bytes = s.scales + ceil_div(4 * d->M, 256) * 256;
    }
    return s;
}

int check(const pe_q8_desc* d) {
    if (!d) return fail(PE_ERR_INVALID, "matmul_q8: null descriptor");
    if (d->x_dtype != PE_I8 && !ssm::dtype_ok(d->x_dtype))
        return fail(PE_ERR_UNSUPPORTED, "matmul_q8: x must be PE_I8, PE_F32, PE_F16 or PE_BF16");
    if (!ssm::dtype_ok(d->y_dtype)) return fail(PE_ERR_UNSUPPORTED, "matmul_q8: y must be PE_F32, PE_F16 or PE_BF16");
    if (d->bias_dtype != d->y_dtype && d->bias_dtype != PE_F32)
        return fail(PE_ERR_UNSUPPORTED, "matmul_q8: the bias must have y's dtype or be PE_F32");
    if (d->kernel < 0 || d->kernel > 1 + kTileKernels) return fail(PE_ERR_INVALID, "matmul_q8: no such kernel");
    if (d->M < 0 || d->N < 0 || d->K < 0) return fail(PE_ERR_INVALID, "matmul_q8: negative extent");
    if (d->K > kMostK) return fail(PE_ERR_UNSUPPORTED, "matmul_q8: K above 131071 may overflow sums of 32 bits");
    const int64_t big = (int64_t(1) << 31) - 4096;
    if (d->M > big || d->N > big) return fail(PE_ERR_UNSUPPORTED, "matmul_q8: an extent of 2^31 or more");
    const int64_t whole = rows::row_bytes(d->K);         // (16-byte groups are read whole)
    const int64_t far = int64_t(1) << 23;                // 256 rows within 32-bit offsets
    if (d->x_dtype == PE_I8) {
        if (d->x_ms % 16 || (d->M > 1 && d->x_ms < whole) || d->x_ms > far)
            return fail(PE_ERR_UNSUPPORTED, "matmul_q8: rows of x must start every 16 bytes, at least K and at most 2^23 apart");
        if (d->K && !ssm::within({{d->M, d->x_ms}, {whole, 1}}, d->x_numel)) return fail(PE_ERR_BOUNDS, "matmul_q8: strides address past x");
    } else if (!ssm::within({{d->M, d->x_ms}, {d->K, 1}}, d->x_numel)) {
        return fail(PE_ERR_BOUNDS, "matmul_q8: strides address past x");
    }
    if (d->w_ns % 16 || (d->N > 1 && d->w_ns < whole) || d->w_ns > far)
        return fail(PE_ERR_UNSUPPORTED, "matmul_q8: rows of w must start every 16 bytes, at least K and at most 2^23 apart");
    if (d->K && !ssm::within({{d->N, d->w_ns}, {whole, 1}}, d->w_numel)) return fail(PE_ERR_BOUNDS, "matmul_q8: strides address past w");
    return PE_OK;
}

}  // namespace
}  // namespace q8
}  // namespace pe

using namespace pe;
using namespace pe::q8;

extern "C" int64_t pe_matmul_q8_workspace_bytes(const pe_q8_desc* d) {
    return check(d) == PE_OK ? space_of(d).bytes : 0;
}

extern "C" int pe_matmul_q8(const pe_q8_desc* d, const void* x, const float* x_scales, const void* w,
                            const float* w_scales, const void* bias, void* y, void* ws, int64_t ws_bytes,
                            void* stream) {
    if (int rc = check(d)) return rc;
    if (d->M == 0 || d->N == 0) return PE_OK;
    const bool whole = d->x_dtype == PE_I8;
    if (!y || !w_scales || (whole && !x_scales) || (d->K && (!x || !w))) return fail(PE_ERR_INVALID, "matmul_q8: null pointer");
    if (d->K && (!aligned(w, 16) || (whole && !aligned(x, 16))))
        return fail(PE_ERR_UNSUPPORTED, "matmul_q8: rows in 8 bits must start on 16 bytes");
    const Space space = space_of(d);
    if (space.bytes && (!ws || ws_bytes < space.bytes || !aligned(ws, 16)))
        return fail(PE_ERR_WORKSPACE, "matmul_q8: workspace missing, too small or not on 16 bytes");
    const auto s = static_cast<hipStream_t>(stream);
    Q8Args g{};
    g.x = static_cast<const int8_t*>(x);
    g.x_ms = d->x_ms;
    g.xs = x_scales;
    g.w = static_cast<const int8_t*>(w);
    g.w_ns = d->w_ns;
    g.ws = w_scales;
    g.bias = bias;
    g.bias_f32 = d->bias_dtype == PE_F32;
    g.y = y;
    g.M = int32_t(d->M); g.N = int32_t(d->N); g.K = int32_t(d->K);
    if (!whole) {
        if (own_rows(d)) return rows_launch_own(d->y_dtype, g, s);
        int8_t* q = static_cast<int8_t*>(ws);
        float* qs = reinterpret_cast<float*>(static_cast<char*>(ws) + space.scales);
        pe_rows_desc r{};
        r.dtype = d->x_dtype;
        r.rows0 = 1; r.rows1 = d->M; r.D = d->K; r.groups = 1;
        r.x_s1 = d->x_ms;
        r.x_numel = d->x_numel;
        r.q_ms = rows::row_pitch(d->K);
        if (int rc = pe_quantize_q8(&r, x, q, qs, stream)) return rc;
        g.x = q;
        g.xs = qs;
        g.x_ms = r.q_ms;
    }
    return few_rows(d) ? rows_launch(d->y_dtype, g, s) : tile_launch(d->y_dtype, g, d->kernel, s);
}
