// Shared by the state-space operators and the 4-bit product: element types
// (bfloat16 beside the contractions' two), vectors at element alignment,
// activations, and which tokens belong to which sequence.
#pragma once

#include "pe_common.h"

#include <initializer_list>
#include <type_traits>
#include <utility>

namespace pe {
namespace ssm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct BF16 {
    using T = __bf16;
    static constexpr int kBytes = 2;
    __device__ __forceinline__ static float to_f32(__bf16 x) { return (float)x; }
};

// V elements, loaded and stored at element alignment (gfx950 takes vector
// accesses at any address; aligned ones cost no more this way).
template <typename E, int V>
struct Vec {
    typedef typename E::T type __attribute__((ext_vector_type(V)));
    typedef typename E::T utype __attribute__((ext_vector_type(V), aligned(E::kBytes)));
};

// n of V consecutive elements in float32 (n < V: the rest 0, not read).
template <typename E, int V>
__device__ __forceinline__ void load_f32(const typename E::T* p, int n, float (&o)[V]) {
    if (n >= V) {
        const typename Vec<E, V>::utype v = *reinterpret_cast<const typename Vec<E, V>::utype*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = E::to_f32(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = i < n ? E::to_f32(p[i]) : 0.0f;
    }
}

template <typename E, int V>
__device__ __forceinline__ void store_f32(typename E::T* p, int n, const float (&v)[V]) {
    if (n >= V) {
        typename Vec<E, V>::utype o;
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = (typename E::T)v[i];
        *reinterpret_cast<typename Vec<E, V>::utype*>(p) = o;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) p[i] = (typename E::T)v[i];
    }
}

// v / (1 + exp(-v)); -0 for v far below 0, where exp(-v) is infinite.  Through
// the hardware's 2^x and reciprocal, good to a unit each (the exponent's own
// rounding counts where the result is small): the library's exp and divide made
// the convolution of a large prompt compute longer than its memory takes.
__device__ __forceinline__ float silu(float v) {
    return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * v));
}

// log(1 + exp(v)) without overflow; exp(-|v|) below 2^-24 leaves max(v, 0).
__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v))); }

// Between LDS writes and reads of other lanes of the same wave: a wave's LDS
// operations are carried out in order, and the compiler must keep them so.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Offset i of packed sequences, clamped to the buffer's tokens.
__device__ __forceinline__ int64_t offset_of(const int32_t* cu, int64_t i, int64_t total) {
    const int64_t v = cu[i];
    return v < 0 ? 0 : v > total ? total : v;
}

// Calls f with the element type of `dtype`.
template <typename F>
int with_type(int dtype, F f) {
    switch (dtype) {
        case PE_F32: return f(F32{});
        case PE_F16: return f(F16{});
        default: return f(BF16{});
    }
}

inline bool dtype_ok(int dtype) { return dtype == PE_F32 || dtype == PE_F16 || dtype == PE_BF16; }

inline int hip_status_of_launch(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? PE_OK : hip_status(e, what);
}

// Whether a tensor of the given extents and strides stays within numel
// elements (extents of 0: nothing is addressed).
inline bool within(std::initializer_list<std::pair<int64_t, int64_t>> axes, int64_t numel) {
    __int128 last = 0;
    for (const auto& [n, stride] : axes) {
        if (n == 0) return true;
        if (n < 0 || stride < 0) return false;
        last += __int128(n - 1) * stride;
    }
    return last < numel;
}

}  // namespace ssm
}  // namespace pe
