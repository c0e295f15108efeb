// Entry points of the selective scan: checks, and the choice of kernel.
#include "pe_scan.h"

namespace pe {
namespace ssm {
namespace {

int check(const pe_scan_desc* d, bool step, bool packed, const void* z) {
    if (!d) return fail(PE_ERR_INVALID, "selective_scan: null descriptor");
    if (!dtype_ok(d->dtype)) return fail(PE_ERR_UNSUPPORTED, "selective_scan: dtype must be PE_F32, PE_F16 or PE_BF16");
    if (d->dt_dtype != d->dtype && d->dt_dtype != PE_F32)
        return fail(PE_ERR_UNSUPPORTED, "selective_scan: dt must be of x's dtype or PE_F32");
    if (d->reserved != 0) return fail(PE_ERR_INVALID, "selective_scan: reserved field must be 0");
    if (d->nseq < 0 || d->H < 0 || d->P < 0 || d->N < 0 || (!step && d->T < 0) || (step && d->nslots < 0))
        return fail(PE_ERR_INVALID, "selective_scan: negative extent");
    if (d->G < 1 || d->H % d->G != 0) return fail(PE_ERR_INVALID, "selective_scan: H is no multiple of G");
    if (d->N > PE_SCAN_MAX_N)
        return fail(PE_ERR_UNSUPPORTED, "selective_scan: N above " + std::to_string(PE_SCAN_MAX_N));
    const int64_t big = int64_t(1) << 31;
    if (d->nseq >= big || d->H >= big || d->P >= big || (!step && d->T >= big))
        return fail(PE_ERR_UNSUPPORTED, "selective_scan: an extent of 2^31 or more");
    const int64_t T = step ? 1 : d->T, seqs = packed ? 1 : d->nseq;
    auto in = [&](int64_t bs, int64_t ts, int64_t hs, int64_t heads, int64_t inner, int64_t numel) {
        return within({{seqs, bs}, {T, ts}, {heads, hs}, {inner, 1}}, numel);
    };
    if (!in(d->x_bs, d->x_ts, d->x_hs, d->H, d->P, d->x_numel) ||
        (z && !in(d->z_bs, d->z_ts, d->z_hs, d->H, d->P, d->z_numel)) ||
        !in(d->dt_bs, d->dt_ts, d->dt_hs, d->H, 1, d->dt_numel) ||
        !in(d->b_bs, d->b_ts, d->b_gs, d->G, d->N, d->b_numel) ||
        !in(d->c_bs, d->c_ts, d->c_gs, d->G, d->N, d->c_numel))
        return fail(PE_ERR_BOUNDS, "selective_scan: strides address past an operand");
    return PE_OK;
}

ScanArgs arguments(const pe_scan_desc& d, const void* x, const void* dt, const float* A, const void* B, const void* C,
                   const float* D, const void* z, const float* dt_bias) {
    ScanArgs g{};
    g.x = x; g.dt = dt; g.A = A; g.B = B; g.C = C; g.D = D; g.z = z; g.dt_bias = dt_bias;
    g.x_bs = d.x_bs; g.x_ts = d.x_ts; g.x_hs = d.x_hs;
    g.z_bs = d.z_bs; g.z_ts = d.z_ts; g.z_hs = d.z_hs;
    g.dt_bs = d.dt_bs; g.dt_ts = d.dt_ts; g.dt_hs = d.dt_hs;
    g.b_bs = d.b_bs; g.b_ts = d.b_ts; g.b_gs = d.b_gs;
    g.c_bs = d.c_bs; g.c_ts = d.c_ts; g.c_gs = d.c_gs;
    g.nseq = int32_t(d.nseq); g.H = int32_t(d.H); g.P = int32_t(d.P); g.G = int32_t(d.G); g.N = int32_t(d.N);
    g.dt_f32 = d.dt_dtype == PE_F32;
    g.softplus = d.softplus;
    return g;
}

}  // namespace
}  // namespace ssm
}  // namespace pe

using namespace pe;
using namespace pe::ssm;

extern "C" int64_t pe_selective_scan_workspace_bytes(const pe_scan_desc* d, int packed) {
    (void)d;
    (void)packed;
    return 0;
}

extern "C" int pe_selective_scan(const pe_scan_desc* d, const void* x, const void* dt, const float* A, const void* B,
                                 const void* C, const float* D, const void* z, const float* dt_bias,
                                 const float* state_in, const int32_t* cu, void* y, float* state_out, void* ws,
                                 int64_t ws_bytes, void* stream) {
    if (int rc = check(d, false, cu != nullptr, z)) return rc;
    if (cu && d->nseq < 1) return fail(PE_ERR_INVALID, "selective_scan: packed tokens without a sequence");
    if (d->nseq == 0 || d->H == 0 || d->P == 0) return PE_OK;
    if (!A || (d->T > 0 && (!x || !dt || !y || (d->N > 0 && (!B || !C)))))
        return fail(PE_ERR_INVALID, "selective_scan: null pointer");
    (void)ws;
    (void)ws_bytes;
    ScanArgs g = arguments(*d, x, dt, A, B, C, D, z, dt_bias);
    g.cu = cu; g.T = d->T; g.y = y; g.state_in = state_in; g.state_out = state_out;
    g.nslots = d->nseq;
    return launch_rows(d->dtype, g, static_cast<hipStream_t>(stream));
}

extern "C" int pe_selective_scan_step(const pe_scan_desc* d, const void* x, const void* dt, const float* A,
                                      const void* B, const void* C, const float* D, const void* z,
                                      const float* dt_bias, float* state, const int32_t* slots, void* y,
                                      void* stream) {
    if (int rc = check(d, true, false, z)) return rc;
    if (d->nseq == 0 || d->H == 0 || d->P == 0) return PE_OK;
    if (!A || !x || !dt || !y || (d->N > 0 && (!B || !C || !state)))
        return fail(PE_ERR_INVALID, "selective_scan_step: null pointer");
    if (!slots && d->nslots < d->nseq) return fail(PE_ERR_BOUNDS, "selective_scan_step: fewer states than rows");
    ScanArgs g = arguments(*d, x, dt, A, B, C, D, z, dt_bias);
    g.T = 1; g.y = y; g.state_in = state; g.state_out = state; g.slots = slots;
    g.nslots = d->nslots;
    return launch_rows(d->dtype, g, static_cast<hipStream_t>(stream));
}
