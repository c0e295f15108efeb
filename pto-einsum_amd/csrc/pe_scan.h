// Arguments and entry points of the selective scan's kernels.
#pragma once

#include "pe_ssm.h"

namespace pe {
namespace ssm {

struct ScanArgs {
    const void *x, *dt, *B, *C, *z;
    const float *A, *D, *dt_bias;
    const float* state_in;
    float* state_out;
    const int32_t *cu, *slots;
    void* y;
    int64_t x_bs, x_ts, x_hs, z_bs, z_ts, z_hs, dt_bs, dt_ts, dt_hs, b_bs, b_ts, b_gs, c_bs, c_ts, c_gs;
    int64_t T;           // tokens of a sequence (dense) or of the buffer (packed)
    int64_t nslots;
    int32_t nseq, H, P, G, N;
    int32_t dt_f32, softplus;
};

template <typename E>
__device__ __forceinline__ float load_dt(const ScanArgs& g, int64_t at) {
    return g.dt_f32 ? static_cast<const float*>(g.dt)[at] : E::to_f32(static_cast<const typename E::T*>(g.dt)[at]);
}

// The step size of head h for the raw value v.
__device__ __forceinline__ float step_size(const ScanArgs& g, float v, float bias) {
    v += bias;
    return g.softplus ? softplus(v) : v;
}

// One wave holds whole rows of the state and walks its sequence token by token:
// single tokens (slots), and prompts (rows_kernel in pe_scan_rows.hip).
int launch_rows(int dtype, const ScanArgs& g, hipStream_t stream);

}  // namespace ssm
}  // namespace pe
