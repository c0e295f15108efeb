// Products of few rows with 4-bit weights and group scales:
//
//   y[m, n] = sum_k x[m, k] s[n, k / group] (q[n, k] - z[n, k / group])
//
// Reading the weights once bounds it, half a byte each.  A wave owns 16 NT weight
// rows and a range of K; the block's waves split K and add their parts in LDS in
// a fixed order.  A step covers 256 k: a lane loads a quarter of each group of
// one row (4, 8 or 16 bytes) for all of them at once, so that a step's weights,
// scales and x are in flight together and matrix-core operands are whole words of
// what was loaded; the order of k inside a group is the same for x.
//
// Weights become operands without an inexact step: q is a whole number, exact in
// 16 bits, so a group's sum Q = sum q x and X = sum x (a product with ones, once
// for the NT tiles) come from the matrix cores in float32 and s (Q - z X) is added
// to the running sum: scales never meet a 16-bit rounding.
//
//   float16:  0x6400 | q is 1024 + q; minus 1032, q - 8 exactly.
//   bfloat16: 0x4300 | q is 128 + q, used as it is, with z + 128: what the float32
//             sums lose by it, 2^-24 of 136 |x| a product, is far below the
//             result's own rounding.
//   float32:  q through float32, whose upper half is q in bfloat16; x is cut into
//             three bfloat16 terms, exactly.
#include "pe_ssm.h"

#include <algorithm>

namespace pe {
namespace ssm {
namespace {

// Waves of a block: 16 where a wave's registers (128 then) hold a step.
// Whether registers hold two steps.
template <typename E, int MT, int NT>
constexpr bool kPairs = E::kBytes == 2 && MT * NT >= 2 && MT < 4;
template <typename E, int MT, int NT>
constexpr int kWaves = MT * NT == 1 ? 16 : 8;
// k of a step: a float32 step of 256 would be twice the code and registers.
template <typename E>
constexpr int kStep = E::kBytes == 4 ? 128 : 256;
#ifndef PE_Q4_TILES
#define PE_Q4_TILES 4
#endif

struct Q4Args {
    const void* x;
    const uint8_t* packed;
    const void *scales, *zeros;
    void* y;
    int64_t x_ms;
    int32_t M, N, K, groups, row_bytes;
    int32_t steps;       // of a wave
};

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Operand vectors and terms of a type, and what its weights are: q + kOffset.
template <typename E>
struct Mma {  // BF16
    using V8 = bf16x8;
    static constexpr int kTerms = 1;
    static constexpr float kOffset = 128.0f;
};
template <>
struct Mma<F16> {
    using V8 = f16x8;
    static constexpr int kTerms = 1;
    static constexpr float kOffset = -8.0f;
};
template <>
struct Mma<F32> {
    using V8 = bf16x8;
    static constexpr int kTerms = 3;
    static constexpr float kOffset = 0.0f;
};

__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The eight weights of a word; 16-bit types take them in the order 0, 4, 1, 5, 2,
// 6, 3, 7 (nibbles i and i + 4 share a masked word), as does x.
__device__ __forceinline__ f16x8 weights(F16, uint32_t w) {
    u32x4 t;
    const f16x2 off = {(_Float16)1032.0f, (_Float16)1032.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        t[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u) - off);
    return __builtin_bit_cast(f16x8, t);
}
__device__ __forceinline__ bf16x8 weights(BF16, uint32_t w) {
    u32x4 t;
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
    return __builtin_bit_cast(bf16x8, t);
}
__device__ __forceinline__ bf16x8 weights(F32, uint32_t w) {
    u32x4 t;
    const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = float((even >> (8 * i)) & 0xff), b = float((odd >> (8 * i)) & 0xff);
        t[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    }
    return __builtin_bit_cast(bf16x8, t);
}

// Eight elements of x as loaded, and as operand terms in the weights' order.
template <typename E>
struct XVec {
    u32x4 v;
    __device__ __forceinline__ void load(const typename E::T* p) {
        typedef u32x4 uv __attribute__((aligned(2)));
        v = *reinterpret_cast<const uv*>(p);
    }
    // The first `by` elements dropped, zeros moved in.
    __device__ __forceinline__ void drop(int by) {
        if (by & 1)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (v[i] >> 16) | (i < 3 ? v[(i + 1) & 3] << 16 : 0u);
        if (by & 2) v = u32x4{v[1], v[2], v[3], 0};
        if (by & 4) v = u32x4{v[2], v[3], 0, 0};
        if (by & 8) v = u32x4{0, 0, 0, 0};
    }
    __device__ __forceinline__ void set(int i, typename E::T x) {
        const uint32_t b = __builtin_bit_cast(uint16_t, x);
        v[i / 2] = (i & 1) ? (v[i / 2] & 0xffffu) | (b << 16) : (v[i / 2] & 0xffff0000u) | b;
    }
    __device__ __forceinline__ void operand(typename Mma<E>::V8 (&o)[1]) const {
        u32x4 t;
#pragma unroll
        for (int i = 0; i < 4; ++i)   // elements i and i + 4
            t[i] = __builtin_amdgcn_perm(v[2 + i / 2], v[i / 2], (i & 1) ? 0x07060302u : 0x05040100u);
        o[0] = __builtin_bit_cast(typename Mma<E>::V8, t);
    }
};
template <>
struct XVec<F32> {
    float v[8];
    __device__ __forceinline__ void load(const float* p) {
        typedef f32x4 uv __attribute__((aligned(4)));
        const f32x4 a = *reinterpret_cast<const uv*>(p), b = *reinterpret_cast<const uv*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = a[i];
            v[4 + i] = b[i];
        }
    }
    __device__ __forceinline__ void drop(int by) {
#pragma unroll
        for (int s = 1; s <= 8; s *= 2)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (by & s) ? (i + s < 8 ? v[(i + s) & 7] : 0.0f) : v[i];
    }
    __device__ __forceinline__ void set(int i, float x) { v[i] = x; }
    __device__ __forceinline__ void operand(bf16x8 (&o)[3]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float r = v[i];
            o[0][i] = (__bf16)r;
            r -= (float)o[0][i];
            o[1][i] = (__bf16)r;
            r -= (float)o[1][i];
            o[2][i] = (__bf16)r;
        }
    }
};

// The word at byte `at` of a row; bytes past its end are anything.
__device__ __forceinline__ uint32_t last_word(const uint8_t* row, int at, int bytes) {
    typedef uint32_t u1 __attribute__((aligned(1)));
    if (bytes >= 4) {
        const int from = min(at, bytes - 4);
        return *reinterpret_cast<const u1*>(row + from) >> (8 * min(3, at - from));
    }
    uint32_t v = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) v |= uint32_t(row[min(at + b, bytes - 1)]) << (8 * b);
    return v;
}

// One step's operands.  GW words of a row's group belong to a lane.
template <typename E, int GROUP, int MT, int NT>
struct Step {
    using T = typename E::T;
    static constexpr int kGroups = kStep<E> / GROUP, GW = GROUP / 32;
    typedef uint32_t Words __attribute__((ext_vector_type(GW)));
    typedef uint32_t LooseWords __attribute__((ext_vector_type(GW), aligned(1)));
    Words w[NT][kGroups];
    // Scales and zero points, packed as they lie in memory.
    static constexpr int kSW = kGroups * E::kBytes / 4;
    typedef uint32_t Pack __attribute__((ext_vector_type(kSW)));
    typedef uint32_t LoosePack __attribute__((ext_vector_type(kSW), aligned(E::kBytes)));
    Pack scale[NT], zero[NT];
    __device__ __forceinline__ static float value(const Pack& p, int j) {
        if constexpr (E::kBytes == 4) return __uint_as_float(p[j]);
        else return E::to_f32(__builtin_bit_cast(T, uint16_t(p[j / 2] >> (16 * (j & 1)))));
    }
    __device__ __forceinline__ static Pack gather(const T* p, int64_t row, int g0, int groups) {
        Pack o = {};
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
            const T v = p[row + min(g0 + j, groups - 1)];
            if constexpr (E::kBytes == 4) o[j] = __float_as_uint(v);
            else o[j / 2] |= uint32_t(__builtin_bit_cast(uint16_t, v)) << (16 * (j & 1));
        }
        return o;
    }
    // x of one tile comes with the weights; of several, a vector at a time as it
    // is used (the registers would not hold it).
    static constexpr bool kAhead = MT == 1;
    XVec<E> x[kAhead ? kGroups : 1][kAhead ? GW : 1];

    // FULL: all of the step's k are there.  Loads take clamped addresses else,
    // and x is 0 past K (a weight there does not count then, nor does a scale).
    template <bool FULL>
    __device__ __forceinline__ void load(const Q4Args& g, const uint8_t* const (&wrow)[NT], const int64_t (&srow)[NT],
                                         const T* const (&xrow)[MT], const bool (&there)[MT], int k0, int lg) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < kGroups; ++j) {
                const int at = (k0 + j * GROUP) / 2 + lg * (GROUP / 8);
                if constexpr (FULL) {
                    w[t][j] = *reinterpret_cast<const LooseWords*>(wrow[t] + at);
                } else {
#pragma unroll
                    for (int i = 0; i < GW; ++i) w[t][j][i] = last_word(wrow[t], at + 4 * i, g.row_bytes);
                }
            }
        const int g0 = k0 / GROUP;
        const T *sp = static_cast<const T*>(g.scales), *zp = static_cast<const T*>(g.zeros);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            zero[t] = Pack{};
            if constexpr (FULL) {
                scale[t] = *reinterpret_cast<const LoosePack*>(sp + srow[t] + g0);
                if (zp) zero[t] = *reinterpret_cast<const LoosePack*>(zp + srow[t] + g0);
            } else {
                scale[t] = gather(sp, srow[t], g0, g.groups);
                if (zp) zero[t] = gather(zp, srow[t], g0, g.groups);
            }
        }
        if constexpr (kAhead)
#pragma unroll
            for (int j = 0; j < kGroups; ++j)
#pragma unroll
                for (int i = 0; i < GW; ++i) load_x<FULL>(g, x[j][i], xrow[0], there[0], k0, j, i, lg);
    }

    template <bool FULL>
    __device__ __forceinline__ static void load_x(const Q4Args& g, XVec<E>& v, const T* row, bool there, int k0, int j,
                                                  int i, int lg) {
        const int k = k0 + j * GROUP + lg * (GROUP / 4) + 8 * i;
        if constexpr (FULL) {
            v.load(row + k);
        } else {
            // A vector that starts earlier, moved into place; or element by element.
            if (g.K >= 8) {
                const int from = min(k, g.K - 8);
                v.load(row + from);
                v.drop(there ? min(8, k - from) : 8);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const T u = row[min(k + e, g.K - 1)];
                    v.set(e, there && k + e < g.K ? u : T(0.0f));
                }
            }
        }
    }

    // acc[m][t]: rows m = 4 lg + element, column n = lr.
    template <bool FULL>
    __device__ __forceinline__ void apply(const Q4Args& g, const T* const (&xrow)[MT], const bool (&there)[MT], int k0,
                                          int lg, f32x4 (&acc)[MT][NT]) const {
        using V8 = typename Mma<E>::V8;
        constexpr int kTerms = Mma<E>::kTerms;
        V8 ones;
#pragma unroll
        for (int i = 0; i < 8; ++i) ones[i] = (typename std::remove_reference<decltype(ones[0])>::type)1.0f;
        const bool with_x = g.zeros || Mma<E>::kOffset != -8.0f;
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
            f32x4 q[MT][NT], xs[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                xs[m] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < NT; ++t) q[m][t] = f32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int i = 0; i < GW; ++i) {
                V8 o[MT][kTerms];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    if constexpr (kAhead) {
                        x[j][i].operand(o[m]);
                    } else {
                        XVec<E> v;
                        load_x<FULL>(g, v, xrow[m], there[m], k0, j, i, lg);
                        v.operand(o[m]);
                    }
                    if (with_x)
#pragma unroll
                        for (int c = kTerms - 1; c >= 0; --c) xs[m] = mma(o[m][c], ones, xs[m]);
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const V8 wv = weights(E{}, w[t][j][i]);
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int c = kTerms - 1; c >= 0; --c) q[m][t] = mma(o[m][c], wv, q[m][t]);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float s = value(scale[t], j);
                const float z = (g.zeros ? value(zero[t], j) : 8.0f) + Mma<E>::kOffset;
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = with_x ? __builtin_fmaf(-z, xs[m][e], q[m][t][e]) : q[m][t][e];
                        acc[m][t][e] = __builtin_fmaf(s, v, acc[m][t][e]);
                    }
            }
            // One group's operands at a time: unpacked ahead, they do not fit.
            if constexpr (MT * NT > 1) __builtin_amdgcn_sched_barrier(0);
        }
    }
};

template <typename E, int GROUP, int MT, int NT>
__global__ __launch_bounds__(64 * (kWaves<E, MT, NT>)) void q4_kernel(Q4Args g) {
    using T = typename E::T;
    constexpr int kPitch = 16 * NT + 1;
    __shared__ float part[kWaves<E, MT, NT>][16 * MT][kPitch];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = int(blockDim.x) >> 6, lr = lane & 15, lg = lane >> 4;
    const int n0 = int(blockIdx.x) * 16 * NT, m0 = int(blockIdx.y) * 16 * MT;
    const uint8_t* wrow[NT];
    int64_t srow[NT];
    const T* xrow[MT];
    bool there[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t n = min(n0 + 16 * t + lr, g.N - 1);
        wrow[t] = g.packed + n * g.row_bytes;
        srow[t] = n * g.groups;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        there[m] = m0 + 16 * m + lr < g.M;
        xrow[m] = static_cast<const T*>(g.x) + int64_t(min(m0 + 16 * m + lr, g.M - 1)) * g.x_ms;
    }
    f32x4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0, 0, 0, 0};

    const int first = wave * g.steps, all = (g.K + kStep<E> - 1) / kStep<E>, last = min(first + g.steps, all);
    const int full = min(last, g.K / kStep<E>);
    Step<E, GROUP, MT, NT> s;
    if constexpr (kPairs<E, MT, NT>) {
        // While a step is worked on, the next one's operands are on their way.
        Step<E, GROUP, MT, NT> u;
        if (first < full) s.template load<true>(g, wrow, srow, xrow, there, first * kStep<E>, lg);
        for (int i = first; i < full; i += 2) {
            if (i + 1 < full) u.template load<true>(g, wrow, srow, xrow, there, (i + 1) * kStep<E>, lg);
            s.template apply<true>(g, xrow, there, i * kStep<E>, lg, acc);
            if (i + 1 >= full) break;
            if (i + 2 < full) s.template load<true>(g, wrow, srow, xrow, there, (i + 2) * kStep<E>, lg);
            u.template apply<true>(g, xrow, there, (i + 1) * kStep<E>, lg, acc);
        }
    } else {
        for (int i = first; i < full; ++i) {
            s.template load<true>(g, wrow, srow, xrow, there, i * kStep<E>, lg);
            s.template apply<true>(g, xrow, there, i * kStep<E>, lg, acc);
        }
    }
    if (full < last && full >= first) {
        s.template load<false>(g, wrow, srow, xrow, there, full * kStep<E>, lg);
        s.template apply<false>(g, xrow, there, full * kStep<E>, lg, acc);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[wave][16 * m + 4 * lg + e][16 * t + lr] = acc[m][t][e];
    __syncthreads();
    for (int at = threadIdx.x; at < 256 * MT * NT; at += blockDim.x) {
        const int m = at / (16 * NT), n = at % (16 * NT);
        float v = 0.0f;
        for (int w = 0; w < waves; ++w) v += part[w][m][n];
        if (m0 + m < g.M && n0 + n < g.N) static_cast<T*>(g.y)[int64_t(m0 + m) * g.N + n0 + n] = (T)v;
    }
}

template <typename E, int GROUP>
int launch(Q4Args g, hipStream_t stream) {
    // Tiles of 16 rows of x, and weight rows for each x that is loaded: as many as
    // leave a block for each CU.
    const int mt = g.M <= 16 ? 1 : g.M <= 32 ? 2 : 4;
    const int64_t tall = ceil_div(g.M, 16 * mt);
    int nt = 1;
    while (2 * nt * mt <= PE_Q4_TILES && ceil_div(g.N, 32 * nt) * tall >= cu_count()) nt *= 2;
    auto run = [&](auto m, auto n) {
        constexpr int MT = m(), NT = n();
        const int steps = int(ceil_div(g.K, kStep<E>));
        g.steps = std::max(1, int(ceil_div(steps, kWaves<E, MT, NT>)));
        const int waves = std::max(1, int(ceil_div(steps, g.steps)));
        const int64_t cols = ceil_div(g.N, 16 * NT);
        if (tall > 65535 || tall * cols * 64 * waves >= (int64_t(1) << 32))
            return fail(PE_ERR_UNSUPPORTED, "matvec_q4: too many rows");
        q4_kernel<E, GROUP, MT, NT><<<dim3{uint32_t(cols), uint32_t(tall)}, 64 * waves, 0, stream>>>(g);
        return hip_status_of_launch("matvec_q4");
    };
    using std::integral_constant;
    const integral_constant<int, 1> one{};
    const integral_constant<int, 2> two{};
    const integral_constant<int, 4> four{};
    if (mt == 1) return nt == 1 ? run(one, one) : nt == 2 ? run(one, two) : run(one, four);
    if (mt == 2) return nt == 1 ? run(two, one) : run(two, two);
    return run(four, one);
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
    return with_type(d->dtype, [&](auto e) {
        using E = decltype(e);
        auto s = static_cast<hipStream_t>(stream);
        return d->group == 32 ? launch<E, 32>(g, s) : d->group == 64 ? launch<E, 64>(g, s) : launch<E, 128>(g, s);
    });
}
