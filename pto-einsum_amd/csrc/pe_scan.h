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
__device__ __forceinline__ uint32_t dt_bits(const ScanArgs& g, const void* dt, int64_t at) {
    if (E::kBytes == 4 || g.dt_f32) return static_cast<const uint32_t*>(dt)[at];
    return static_cast<const uint16_t*>(dt)[at];
}
template <typename E>
__device__ __forceinline__ float dt_of(const ScanArgs& g, uint32_t bits) {
    if constexpr (E::kBytes == 2) {
        if (!g.dt_f32) return E::to_f32(__builtin_bit_cast(typename E::T, uint16_t(bits)));
    }
    return __uint_as_float(bits);
}

// The step size of head h for the raw value v.
__device__ __forceinline__ float step_size(const ScanArgs& g, float v, float bias) {
    v += bias;
    return g.softplus ? softplus(v) : v;
}

// Outputs of tokens before the first packed sequence and after the last: zeros.
template <typename E>
__device__ __forceinline__ void clear_outside(const ScanArgs& g, int64_t thread, int64_t threads) {
    typename E::T* y = static_cast<typename E::T*>(g.y);
    const int64_t row = int64_t(g.H) * g.P, first = offset_of(g.cu, 0, g.T) * row;
    for (int64_t i = thread; i < first; i += threads) y[i] = typename E::T(0.0f);
    for (int64_t i = offset_of(g.cu, g.nseq, g.T) * row + thread; i < g.T * row; i += threads) y[i] = typename E::T(0.0f);
}

// One wave holds whole rows of the state and walks its sequence token by token:
// single tokens (slots), and prompts (rows_kernel in pe_scan_rows.hip).
int launch_rows(int dtype, const ScanArgs& g, hipStream_t stream);

}  // namespace ssm
}  // namespace pe
