// Entry points of the norms between blocks and of rows in 8 bits (kernels and
// formulas: pe_norm.h, pe_rows.h).
#include "pe_rows.h"

#include <algorithm>

namespace pe {
namespace rows {
namespace {

constexpr int kMostParts = 8192;      // groups of a norm whose rows go to 8 bits: 32 KB of LDS

// Checks what the three operators share and fills the arguments.
int arguments(const char* what, const pe_rows_desc* d, const void* x, bool gate, bool residual, bool q8, NormArgs& a) {
    const std::string name(what);
    if (!d) return fail(PE_ERR_INVALID, name + ": null descriptor");
    if (!ssm::dtype_ok(d->dtype)) return fail(PE_ERR_UNSUPPORTED, name + ": dtype must be PE_F32, PE_F16 or PE_BF16");
    if (d->rows0 < 0 || d->rows1 < 0 || d->D < 0) return fail(PE_ERR_INVALID, name + ": negative extent");
    if (d->groups < 1 || d->D % d->groups) return fail(PE_ERR_INVALID, name + ": D is not a whole number of groups");
    if (!(d->eps >= 0.0f)) return fail(PE_ERR_INVALID, name + ": eps must be 0 or more");
    const int64_t big = (int64_t(1) << 31) - 32768;
    if (d->D > big) return fail(PE_ERR_UNSUPPORTED, name + ": rows of 2^31 elements or more");
    // (in two steps: the three extents' product may pass 128 bits)
    const __int128 rows = __int128(d->rows0) * d->rows1;
    if (d->rows0 && d->rows1 && (rows > big || rows * d->groups > big)) return fail(PE_ERR_UNSUPPORTED, name + ": 2^31 rows or more");
    if (!ssm::within({{d->rows0, d->x_s0}, {d->rows1, d->x_s1}, {d->D, 1}}, d->x_numel))
        return fail(PE_ERR_BOUNDS, name + ": strides address past x");
    if (gate && !ssm::within({{d->rows0, d->g_s0}, {d->rows1, d->g_s1}, {d->gate_row ? 1 : d->D, 1}}, d->g_numel))
        return fail(PE_ERR_BOUNDS, name + ": strides address past the gate");
    if (residual) {
        if (d->res_dtype != d->dtype && d->res_dtype != PE_F32)
            return fail(PE_ERR_UNSUPPORTED, name + ": the residual must have x's dtype or be PE_F32");
        if (!ssm::within({{d->rows0, d->r_s0}, {d->rows1, d->r_s1}, {d->D, 1}}, d->r_numel))
            return fail(PE_ERR_BOUNDS, name + ": strides address past the residual");
    }
    if (q8 && (d->q_ms < row_bytes(d->D) || d->q_ms % 16 || d->q_ms > ceil_div(d->D, 128) * 128))
        return fail(PE_ERR_INVALID, name + ": q_ms must be a multiple of 16 from D to D rounded up to 128");
    if (q8 && d->groups > kMostParts) return fail(PE_ERR_UNSUPPORTED, name + ": more than 8192 groups in 8 bits");
    if (d->rows0 && d->rows1 && d->D && !x) return fail(PE_ERR_INVALID, name + ": null pointer");
    a.x = x;
    a.x0 = d->x_s0; a.x1 = d->x_s1;
    a.g0 = d->g_s0; a.g1 = d->g_s1;
    a.r0 = d->r_s0; a.r1 = d->r_s1;
    a.q_ms = d->q_ms;
    // Rows in 8 bits have one scale: their groups stay together.
    const int64_t apart = q8 ? 1 : d->groups;
    a.units = uint32_t(d->rows0 * d->rows1 * apart);
    a.inner = FastDiv(uint32_t(d->rows1));
    a.groups = FastDiv(uint32_t(apart));
    a.D = int32_t(d->D / apart);
    // (of rows without elements there is nothing to share out)
    a.parts = int32_t(q8 && d->D ? d->groups : 1);
    a.per = 1.0f / float(d->D / d->groups);
    a.g_ds = d->gate_row ? 0 : 1;
    a.norm_first = d->norm_first;
    a.eps = d->eps;
    a.scale = d->scale;
    return PE_OK;
}

int launch(Op op, bool q8, const pe_rows_desc* d, const NormArgs& a, void* stream) {
    const auto s = static_cast<hipStream_t>(stream);
    const bool wide = op == kResidual && d->res_dtype == PE_F32;
    switch (d->dtype) {
        case PE_F16: return norm_launch_f16(op, q8, wide, a, s);
        case PE_BF16: return norm_launch_bf16(op, q8, wide, a, s);
        default: return norm_launch_f32(op, q8, wide, a, s);
    }
}

}  // namespace
}  // namespace rows
}  // namespace pe

using namespace pe;
using namespace pe::rows;

extern "C" int pe_quantize_q8(const pe_rows_desc* d, const void* x, int8_t* q, float* scales, void* stream) {
    NormArgs a{};
    if (int rc = arguments("quantize_q8", d, x, false, false, true, a)) return rc;
    if (a.units == 0) return PE_OK;
    if (!scales || (a.D && !q)) return fail(PE_ERR_INVALID, "quantize_q8: null pointer");
    a.parts = 1;
    a.q = q;
    a.qs = scales;
    return launch(kQuantize, true, d, a, stream);
}

extern "C" int pe_gated_norm(const pe_rows_desc* d, const void* x, const void* weight, const void* z, void* y,
                             int8_t* q, float* scales, void* stream) {
    NormArgs a{};
    const bool q8 = scales != nullptr;
    if (int rc = arguments("gated_norm", d, x, z != nullptr, false, q8, a)) return rc;
    if (z && d->gate_row) return fail(PE_ERR_INVALID, "gated_norm: z has a value for each element");
    if (a.units == 0) return PE_OK;
    if (a.D && (q8 ? !q : !y)) return fail(PE_ERR_INVALID, "gated_norm: null pointer");
    if (a.D == 0 && !q8) return PE_OK;
    a.w = weight; a.g = z; a.y = y; a.q = q; a.qs = scales;
    return launch(kGated, q8, d, a, stream);
}

extern "C" int pe_residual_norm(const pe_rows_desc* d, const void* x, const void* residual, const void* weight,
                                const void* post_weight, const void* gate, void* y, void* new_residual, int8_t* q,
                                float* scales, void* stream) {
    NormArgs a{};
    const bool q8 = scales != nullptr;
    if (int rc = arguments("residual_norm", d, x, gate != nullptr, true, q8, a)) return rc;
    if (d->groups != 1) return fail(PE_ERR_INVALID, "residual_norm: has no groups");
    if (a.units == 0 || (a.D == 0 && !q8)) return PE_OK;
    if (a.D && (!residual || !new_residual || (q8 ? !q : !y))) return fail(PE_ERR_INVALID, "residual_norm: null pointer");
    a.w = weight; a.pw = post_weight; a.g = gate; a.res = residual;
    a.y = y; a.r = new_residual; a.q = q; a.qs = scales;
    return launch(kResidual, q8, d, a, stream);
}
