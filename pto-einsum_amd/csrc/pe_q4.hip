// Products of few rows with 4-bit weights and group scales:
//
//   y[m, n] = sum_k x[m, k] s[n, k / group] (q[n, k] - z[n, k / group])
//
// Reading the weights once bounds it, half a byte each.  A wave owns 16 weight
// rows and a range of K, the block's waves split K and add their parts in LDS
// in a fixed order.  Weights become matrix-core operands without an inexact
// step: q is a whole number, exact in float16 and bfloat16, so a group's sum
// Q = sum q x and X = sum x (a product with ones) come from the matrix cores in
// float32 and s (Q - z X) is added to the running sum: scales never meet a
// 16-bit rounding.  float32 x is cut into three bfloat16 terms, exactly.
//
//   float16:  0x6400 | q is 1024 + q; minus 1032, q - 8 exactly.
//   others:   q through float32, whose upper half is q in bfloat16.
#include "pe_ssm.h"

#include <algorithm>

namespace pe {
namespace ssm {
namespace {

constexpr int kMaxWaves = 8;

struct Q4Args {
    const void* x;
    const uint8_t* packed;
    const void *scales, *zeros;
    void* y;
    int64_t x_ms;
    int32_t M, N, K, groups, row_bytes;
    int32_t steps;       // K steps of 128 of a wave
};

// 16-bit matrix-core operand vectors and products of a type.
template <typename E>
struct Mma {
    using V8 = bf16x8;
    static constexpr int kTerms = 1;
    static constexpr bool kSigned = false;
};
template <>
struct Mma<F16> {
    using V8 = f16x8;
    static constexpr int kTerms = 1;
    static constexpr bool kSigned = true;   // weights are q - 8
};
template <>
struct Mma<F32> {
    using V8 = bf16x8;
    static constexpr int kTerms = 3;
    static constexpr bool kSigned = false;
};

__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Eight weights of a word, k ascending from the lowest nibble.
__device__ __forceinline__ void weights(uint32_t w, f16x8& o) {
    // nibble pairs (k, k + 4) share a masked word; the words are put in order
    // by x, whose elements take the same places (order()).
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    union { uint32_t u[4]; f16x2 h[4]; f16x8 v; } t;
    const f16x2 off = {(_Float16)1032.0f, (_Float16)1032.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        t.u[i] = ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u;
        t.h[i] = t.h[i] - off;
    }
    o = t.v;
}
__device__ __forceinline__ void weights(uint32_t w, bf16x8& o) {
    union { uint32_t u[4]; bf16x8 v; } t;
    const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = float((even >> (8 * i)) & 0xff), b = float((odd >> (8 * i)) & 0xff);
        t.u[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    }
    o = t.v;
}

// Eight elements of x as operand terms, in the order of weights().
__device__ __forceinline__ void operand(const float (&x)[8], f16x8 (&o)[1]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        o[0][2 * i] = (_Float16)x[i];
        o[0][2 * i + 1] = (_Float16)x[i + 4];
    }
}
__device__ __forceinline__ void operand(const float (&x)[8], bf16x8 (&o)[1]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[0][i] = (__bf16)x[i];
}
__device__ __forceinline__ void operand(const float (&x)[8], bf16x8 (&o)[3]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float v = x[i];
        o[0][i] = (__bf16)v;
        v -= (float)o[0][i];
        o[1][i] = (__bf16)v;
        v -= (float)o[1][i];
        o[2][i] = (__bf16)v;
    }
}

// The 4 bytes of a row at byte `at`, bytes past the row's end 0.
__device__ __forceinline__ uint32_t load_word(const uint8_t* row, int at, int row_bytes) {
    typedef uint32_t u1 __attribute__((aligned(1)));
    if (at + 4 <= row_bytes) return *reinterpret_cast<const u1*>(row + at);
    uint32_t w = 0;
    for (int i = 0; at + i < row_bytes && i < 4; ++i) w |= uint32_t(row[at + i]) << (8 * i);
    return w;
}

// S steps of 32 k share a group's scale; MT tiles of 16 rows of x.
template <typename E, int S, int MT>
__global__ __launch_bounds__(64 * kMaxWaves) void q4_kernel(Q4Args g) {
    using T = typename E::T;
    using V8 = typename Mma<E>::V8;
    constexpr int NT = Mma<E>::kTerms;
    __shared__ float part[kMaxWaves][16 * MT][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int lr = lane & 15, lg = lane >> 4;
    const int n0 = int(blockIdx.x) * 16, m0 = int(blockIdx.y) * 16 * MT;
    const uint8_t* wrow = g.packed + int64_t(min(n0 + lr, g.N - 1)) * g.row_bytes;
    f32x4 acc[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[j] = f32x4{0, 0, 0, 0};
    V8 ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = (typename std::remove_reference<decltype(ones[0])>::type)1.0f;
    const bool with_x = g.zeros || !Mma<E>::kSigned;

    const int k_begin = wave * g.steps * 128, k_end = min(k_begin + g.steps * 128, g.K);
    for (int k = k_begin; k < k_end; k += 32 * S) {
        f32x4 q[MT], xs[MT];
#pragma unroll
        for (int j = 0; j < MT; ++j) q[j] = xs[j] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int kk = k + 32 * s + 8 * lg;
            V8 w;
            weights(load_word(wrow, kk >> 1, g.row_bytes), w);
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                float xv[8];
                const int m = m0 + 16 * j + lr;
                load_f32<E, 8>(static_cast<const T*>(g.x) + int64_t(min(m, g.M - 1)) * g.x_ms + kk,
                               m < g.M ? max(0, g.K - kk) : 0, xv);
                V8 o[NT];
                operand(xv, o);
#pragma unroll
                for (int i = NT - 1; i >= 0; --i) {
                    q[j] = mma(w, o[i], q[j]);
                    if (with_x) xs[j] = mma(ones, o[i], xs[j]);
                }
            }
        }
        const int group = k / (32 * S);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t at = int64_t(min(n0 + 4 * lg + i, g.N - 1)) * g.groups + group;
            const float sc = E::to_f32(static_cast<const T*>(g.scales)[at]);
            float zero = g.zeros ? E::to_f32(static_cast<const T*>(g.zeros)[at]) : 8.0f;
            if (Mma<E>::kSigned) zero -= 8.0f;
#pragma unroll
            for (int j = 0; j < MT; ++j)
                acc[j][i] = __builtin_fmaf(sc, with_x ? __builtin_fmaf(-zero, xs[j][i], q[j][i]) : q[j][i], acc[j][i]);
        }
    }
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[wave][16 * j + lr][4 * lg + i] = acc[j][i];
    __syncthreads();
    for (int at = threadIdx.x; at < 256 * MT; at += blockDim.x) {
        const int m = at >> 4, n = at & 15;
        float v = 0.0f;
        for (int w = 0; w < waves; ++w) v += part[w][m][n];
        if (m0 + m < g.M && n0 + n < g.N) static_cast<T*>(g.y)[int64_t(m0 + m) * g.N + n0 + n] = (T)v;
    }
}

template <typename E, int S>
void launch(const Q4Args& g, dim3 grid, int threads, int mt, hipStream_t stream) {
    if (mt == 1) q4_kernel<E, S, 1><<<grid, threads, 0, stream>>>(g);
    else if (mt == 2) q4_kernel<E, S, 2><<<grid, threads, 0, stream>>>(g);
    else q4_kernel<E, S, 4><<<grid, threads, 0, stream>>>(g);
}

}  // namespace
}  // namespace ssm
}  // namespace pe

using namespace pe;
using namespace pe::ssm;

extern "C" int pe_matvec_q4(const pe_q4_desc* d, const void* x, const void* packed, const void* scales,
                            const void* zeros, void* y, void* stream) {
    if (!d) return fail(PE_ERR_INVALID, "matvec_q4: null descriptor");
    if (!dtype_ok(d->dtype)) return fail(PE_ERR_UNSUPPORTED, "matvec_q4: dtype must be PE_F32, PE_F16 or PE_BF16");
    if (d->group != 32 && d->group != 64 && d->group != 128)
        return fail(PE_ERR_UNSUPPORTED, "matvec_q4: group must be 32, 64 or 128");
    if (d->M < 0 || d->N < 0 || d->K < 0) return fail(PE_ERR_INVALID, "matvec_q4: negative extent");
    const int64_t big = (int64_t(1) << 31) - 4096;
    if (d->M > big || d->N > big || d->K > big) return fail(PE_ERR_UNSUPPORTED, "matvec_q4: an extent of 2^31 or more");
    if (!within({{d->M, d->x_ms}, {d->K, 1}}, d->x_numel))
        return fail(PE_ERR_BOUNDS, "matvec_q4: strides address past x");
    if (d->M == 0 || d->N == 0) return PE_OK;
    if (!y || (d->K > 0 && (!x || !packed || !scales))) return fail(PE_ERR_INVALID, "matvec_q4: null pointer");
    Q4Args g{};
    g.x = x; g.packed = static_cast<const uint8_t*>(packed); g.scales = scales; g.zeros = zeros; g.y = y;
    g.x_ms = d->x_ms; g.M = int32_t(d->M); g.N = int32_t(d->N); g.K = int32_t(d->K);
    g.groups = int32_t(ceil_div(d->K, d->group));
    g.row_bytes = int32_t(ceil_div(d->K, 2));
    const int ksteps = int(ceil_div(d->K, 128)), waves = std::max(1, std::min(kMaxWaves, ksteps));
    g.steps = int(ceil_div(ksteps, waves));
    const int mt = d->M <= 16 ? 1 : d->M <= 32 ? 2 : 4;
    const int64_t rows = ceil_div(d->M, 16 * mt), cols = ceil_div(d->N, 16);
    if (rows > 65535 || rows * cols * 64 * waves >= (int64_t(1) << 32))
        return fail(PE_ERR_UNSUPPORTED, "matvec_q4: too many rows");
    const dim3 grid{uint32_t(cols), uint32_t(rows)};
    return with_type(d->dtype, [&](auto e) {
        using E = decltype(e);
        auto s = static_cast<hipStream_t>(stream);
        if (d->group == 32) launch<E, 1>(g, grid, 64 * waves, mt, s);
        else if (d->group == 64) launch<E, 2>(g, grid, 64 * waves, mt, s);
        else launch<E, 4>(g, grid, 64 * waves, mt, s);
        return hip_status_of_launch("matvec_q4");
    });
}
