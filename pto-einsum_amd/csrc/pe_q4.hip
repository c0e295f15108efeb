// Products of few rows with 4-bit weights and group scales:
//
//   y[m, n] = sum_k x[m, k] s[n, k / group] (q[n, k] - z[n, k / group])
//
// Reading the weights once bounds it, half a byte each.  A wave owns 16 NT weight
// rows and a range of K; the block's waves split K and add their parts in LDS in
// a fixed order.  A step covers 128 k: its weights, scales and x are loaded as they
// lie, 16 bytes a lane and rows contiguous over lanes, while the step before is
// worked on, and pass through LDS of the wave's own to the lanes that feed them to
// the matrix cores.  (Loaded straight in that order, where neighbouring lanes have
// different rows, every lane's 8 bytes cost a look-up of their own: 16 tokens
// 16384 x 8192 took 34 us.)
//
// Weights become operands without an inexact step: q is a whole number, exact in
// 16 bits, so a group's sum Q = sum q x and X = sum x (a product with ones, once
// for the NT tiles) come from the matrix cores in float32 and s (Q - z X) is added
// to the running sum: scales never meet a 16-bit rounding.
//
//   float16:  0x6400 | q is 1024 + q; minus 1032, q - 8 exactly.
//   bfloat16: 0x4300 | q is 128 + q, used as it is, with z + 128: what the float32
//             sums lose by it, 2^-24 of (128 + q) |s x| a product, is far below the
//             result's own rounding, except where a row's weights are all 0: then
//             the result is that small, not 0.
//   float32:  q through float32, whose upper half is q in bfloat16; x is cut into
//             three bfloat16 terms, exactly: of 2^24 x, since bfloat16 has no bits below
//             2^-133 and the matrix cores lose subnormals (x of 2^-124: 6e-4 of the
//             result as it is).
//
// Outputs that end as an infinity or NaN are formed again one by one, whole weights
// times x (whole_weights).
//
// 16 tokens, 16384 x 8192 bfloat16 in groups of 64, three sets of weights in turn:
// 20.8 us, 3.7 TB/s (75 with 4-byte loads and no step ahead; 24 with a branch
// around the loads ahead and a stretch of K for each wave); eight sets, which no
// cache holds: 30 us, 2.2 TB/s, one token 27.  One block of eight waves a CU has
// too little on its way for more.  One token, 4096 x 4096: 6.6 us of a call of
// 9.5, which the host's part bounds.
#include "pe_ssm.h"

#include <algorithm>

namespace pe {
namespace ssm {
namespace {

constexpr int kStep = 128;
// Waves of a block: what its LDS holds.
template <typename E, int MT, int NT>
constexpr int kWaves = E::kBytes == 4 ? (MT == 1 ? 8 : 4) : MT * NT == 1 ? 16 : 8;

struct Q4Args {
    const void* x;
    const uint8_t* packed;
    const void *scales, *zeros;
    void* y;
    int64_t x_ms;
    int32_t M, N, K, groups, row_bytes;
};

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Operand vectors and terms of a type, what its weights are, q + kOffset, and what
// x enters the products times.
template <typename E>
struct Mma {  // BF16
    using V8 = bf16x8;
    static constexpr int kTerms = 1;
    static constexpr float kOffset = 128.0f, kScale = 1.0f;
};
template <>
struct Mma<F16> {
    using V8 = f16x8;
    static constexpr int kTerms = 1;
    static constexpr float kOffset = -8.0f, kScale = 1.0f;
};
template <>
struct Mma<F32> {
    using V8 = bf16x8;
    static constexpr int kTerms = 3;
    static constexpr float kOffset = 0.0f, kScale = 0x1p24f;
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

// Eight elements of x as operand terms in the weights' order.
__device__ __forceinline__ void operand(const _Float16* p, f16x8 (&o)[1]) {
    const u32x4 v = *reinterpret_cast<const u32x4*>(p);
    u32x4 t;
#pragma unroll
    for (int i = 0; i < 4; ++i)   // elements i and i + 4
        t[i] = __builtin_amdgcn_perm(v[2 + i / 2], v[i / 2], (i & 1) ? 0x07060302u : 0x05040100u);
    o[0] = __builtin_bit_cast(f16x8, t);
}
__device__ __forceinline__ void operand(const __bf16* p, bf16x8 (&o)[1]) {
    f16x8 t[1];
    operand(reinterpret_cast<const _Float16*>(p), t);
    o[0] = __builtin_bit_cast(bf16x8, t[0]);
}
__device__ __forceinline__ void operand(const float* p, bf16x8 (&o)[3]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
    u32x4 t[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // two at a time: one conversion
        f32x2 r = i < 2 ? f32x2{a[(2 * i) & 3], a[(2 * i + 1) & 3]} : f32x2{b[(2 * i) & 3], b[(2 * i + 1) & 3]};
#pragma unroll
        for (int c = 0; c < 3; ++c) {
            t[c][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
            r[0] -= __uint_as_float(t[c][i] << 16);
            r[1] -= __uint_as_float(t[c][i] & 0xffff0000u);
        }
    }
#pragma unroll
    for (int c = 0; c < 3; ++c) o[c] = __builtin_bit_cast(bf16x8, t[c]);
}

// 16 bytes of a row at byte `at`, those past its end 0.
typedef u32x4 LooseVec __attribute__((aligned(1)));
__device__ __forceinline__ u32x4 last_vec(const uint8_t* row, int64_t at, int64_t bytes) {
    u32x4 v = {0, 0, 0, 0};
    if (bytes >= 16) {
        // a vector that starts earlier, moved into place
        const int64_t from = min(at, bytes - 16);
        const int by = int(min(int64_t(16), at - from));
        v = *reinterpret_cast<const LooseVec*>(row + from);
        if (by & 16) v = u32x4{0, 0, 0, 0};
        if (by & 8) v = u32x4{v[2], v[3], 0, 0};
        if (by & 4) v = u32x4{v[1], v[2], v[3], 0};
        const int bits = 8 * (by & 3);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = uint32_t((uint64_t(v[i]) | (i < 3 ? uint64_t(v[(i + 1) & 3]) << 32 : 0)) >> bits);
        return v;
    }
    for (int b = 0; b < 16; ++b)
        if (at + b < bytes) v[b / 4] |= uint32_t(row[at + b]) << (8 * (b & 3));
    return v;
}

template <typename E, int GROUP, int MT, int NT>
struct Wave {
    using T = typename E::T;
    static constexpr int kGroups = kStep / GROUP, GW = GROUP / 32, kRows = 16 * NT, kXRows = 16 * MT;
    static constexpr int kWP = kStep / 2 + 16, kXP = kStep + 16 / E::kBytes;   // pitches: bytes, elements
    static constexpr int kXVecs = kStep * E::kBytes / 16;                      // of a row of x
    static constexpr int kXEach = kXRows * kXVecs / 64;
    // Scales and zero points of a row: kGroups of each.
    typedef typename Vec<E, kGroups>::utype LooseScales;

    struct Lds {
        alignas(16) uint8_t w[kRows * kWP];
        alignas(16) T x[kXRows * kXP];
        float scale[kGroups][kRows], zero[kGroups][kRows];
    };

    // A step's weights and scales in registers.  Lane l: weight rows l / 4 + 16 t,
    // 16 bytes each; scales and zero points of row l.
    struct Weights {
        u32x4 w[NT];
        typename Vec<E, kGroups>::type scale, zero;
    };
    u32x4 x[kXEach];

    template <bool FULL>
    __device__ __forceinline__ static void load(Weights& o, const Q4Args& g, int n0, int k0, int lane) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint8_t* row = g.packed + int64_t(min(n0 + 16 * t + lane / 4, g.N - 1)) * g.row_bytes;
            const int at = k0 / 2 + 16 * (lane & 3);
            if constexpr (FULL) o.w[t] = *reinterpret_cast<const LooseVec*>(row + at);
            else o.w[t] = last_vec(row, at, g.row_bytes);
        }
        // (Without zero points the scales are read in their place, so that there is
        // no branch around a load.)
        const int64_t at = int64_t(min(n0 + min(lane, kRows - 1), g.N - 1)) * g.groups + k0 / GROUP;
        const T *sp = static_cast<const T*>(g.scales) + at, *zp = static_cast<const T*>(g.zeros ? g.zeros : g.scales) + at;
        if constexpr (FULL) {
            o.scale = *reinterpret_cast<const LooseScales*>(sp);
            o.zero = *reinterpret_cast<const LooseScales*>(zp);
        } else {
#pragma unroll
            for (int j = 0; j < kGroups; ++j) {
                const int i = min(j, g.groups - 1 - k0 / GROUP);
                o.scale[j] = sp[i];
                o.zero[j] = zp[i];
            }
        }
    }

    template <bool FULL>
    __device__ __forceinline__ void load_x(const Q4Args& g, int m0, int k0, int lane) {
#pragma unroll
        for (int i = 0; i < kXEach; ++i) {
            const int v = lane + 64 * i, m = m0 + v / kXVecs, vec = v % kXVecs;
            const int64_t at = int64_t(k0) * E::kBytes + vec * 16;
            const uint8_t* row = reinterpret_cast<const uint8_t*>(static_cast<const T*>(g.x) +
                                                                  int64_t(min(m, g.M - 1)) * g.x_ms);
            if constexpr (FULL) x[i] = *reinterpret_cast<const LooseVec*>(row + at);
            else x[i] = last_vec(row, at, int64_t(g.K) * E::kBytes);
        }
    }

    // Rows of x past M stay 0.
    __device__ __forceinline__ static void clear(const Q4Args& g, Lds& m, int m0, int lane) {
        constexpr int kVecs = kXRows * kXP * E::kBytes / 16;
        if (m0 + kXRows > g.M)
            for (int i = lane; i < kVecs; i += 64) reinterpret_cast<u32x4*>(m.x)[i] = u32x4{0, 0, 0, 0};
    }

    __device__ __forceinline__ void store(const Weights& o, const Q4Args& g, Lds& m, int m0, int lane) const {
#pragma unroll
        for (int t = 0; t < NT; ++t)
            *reinterpret_cast<u32x4*>(m.w + (16 * t + lane / 4) * kWP + 16 * (lane & 3)) = o.w[t];
        if (lane < kRows)
#pragma unroll
            for (int j = 0; j < kGroups; ++j) {
                m.scale[j][lane] = E::to_f32(o.scale[j]);
                m.zero[j][lane] = (g.zeros ? E::to_f32(o.zero[j]) : 8.0f) + Mma<E>::kOffset;
            }
#pragma unroll
        for (int i = 0; i < kXEach; ++i) {
            const int v = lane + 64 * i;
            u32x4 xv = x[i];
            if constexpr (Mma<E>::kScale != 1.0f)
#pragma unroll
                for (int e = 0; e < 4; ++e) xv[e] = __float_as_uint(__uint_as_float(xv[e]) * Mma<E>::kScale);
            if (m0 + v / kXVecs < g.M)
                *reinterpret_cast<u32x4*>(m.x + v / kXVecs * kXP + v % kXVecs * (16 / E::kBytes)) = xv;
        }
    }

    // acc[m][t]: rows m = 4 lg + element, column n = lr.
    __device__ __forceinline__ static void apply(const Lds& l, int lane, f32x4 (&acc)[MT][NT]) {
        using V8 = typename Mma<E>::V8;
        constexpr int kTerms = Mma<E>::kTerms;
        const int lr = lane & 15, lg = lane >> 4;
        V8 ones;
#pragma unroll
        for (int i = 0; i < 8; ++i) ones[i] = (typename std::remove_reference<decltype(ones[0])>::type)1.0f;
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
            typedef uint32_t Words __attribute__((ext_vector_type(GW)));
            f32x4 q[MT][NT], xs[MT];
            Words w[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t)
                w[t] = *reinterpret_cast<const Words*>(l.w + (16 * t + lr) * kWP + j * (GROUP / 2) + lg * (GROUP / 8));
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
                    operand(l.x + (16 * m + lr) * kXP + j * GROUP + lg * (GROUP / 4) + 8 * i, o[m]);
#pragma unroll
                    for (int c = kTerms - 1; c >= 0; --c) xs[m] = mma(o[m][c], ones, xs[m]);
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const V8 wv = weights(E{}, w[t][i]);
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int c = kTerms - 1; c >= 0; --c) q[m][t] = mma(o[m][c], wv, q[m][t]);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float s = l.scale[j][16 * t + lr], z = l.zero[j][16 * t + lr];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[m][t][e] = __builtin_fmaf(s, __builtin_fmaf(-z, xs[m][e], q[m][t][e]), acc[m][t][e]);
            }
            // One group's operands at a time: unpacked ahead, they do not fit.
            if constexpr (kGroups > 1) __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// One output by its definition, whole weights times x.  Sums of q x and of x apart
// are not it where x is infinite (inf - inf, 0 inf) or so large that one of them
// passes float32's range while s (q - z) x does not, and such sums never end
// finite: outputs that are not finite are formed again this way, ends included.
template <typename E, int GROUP>
__device__ __forceinline__ float whole_weights(const Q4Args& g, int64_t m, int64_t n) {
    using T = typename E::T;
    const T* x = static_cast<const T*>(g.x) + m * g.x_ms;
    const uint8_t* w = g.packed + n * g.row_bytes;
    float v = 0.0f;
    for (int64_t k = 0; k < g.K && v == v; k += 32) {   // a NaN stays one
        const int64_t at = n * g.groups + k / GROUP;
        const float s = E::to_f32(static_cast<const T*>(g.scales)[at]);
        const float z = g.zeros ? E::to_f32(static_cast<const T*>(g.zeros)[at]) : 8.0f;
        const u32x4 q = last_vec(w, k / 2, g.row_bytes);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float o[8];
            const int left = int(min(int64_t(8), g.K - k - 8 * i));
            load_f32<E, 8>(x + k + 8 * i, left, o);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v = j < left ? __builtin_fmaf(o[j], s * (float((q[i] >> (4 * j)) & 15) - z), v) : v;
        }
    }
    return v;
}

template <typename E, int GROUP, int MT, int NT>
__global__ __launch_bounds__(64 * (kWaves<E, MT, NT>)) void q4_kernel(Q4Args g) {
    using T = typename E::T;
    using W = Wave<E, GROUP, MT, NT>;
    constexpr int kPitch = 16 * NT + 1;
    __shared__ union {
        typename W::Lds wave[kWaves<E, MT, NT>];
        float part[kWaves<E, MT, NT>][16 * MT][kPitch];
    } m;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = int(blockDim.x) >> 6, lr = lane & 15, lg = lane >> 4;
    const int n0 = int(blockIdx.x) * 16 * NT, m0 = int(blockIdx.y) * 16 * MT;
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0, 0, 0, 0};

    // This wave's steps: every waves-th, so that the block reads whole stretches of
    // its rows at a time.  The last of all may be one of less than kStep.
    const int last = (g.K + kStep - 1) / kStep;
    W s;
    typename W::Weights even, odd;
    auto load = [&](typename W::Weights& o, int i) __attribute__((always_inline)) {
        if (i >= last) return;
        if ((i + 1) * int64_t(kStep) <= g.K) W::template load<true>(o, g, n0, i * kStep, lane);
        else W::template load<false>(o, g, n0, i * kStep, lane);
    };
    auto load_x = [&](int i) __attribute__((always_inline)) {
        if (i >= last) return;
        if ((i + 1) * int64_t(kStep) <= g.K) s.template load_x<true>(g, m0, i * kStep, lane);
        else s.template load_x<false>(g, m0, i * kStep, lane);
    };
    // One step, with what comes after it loaded: weights two steps ahead (memory
    // answers later than a step takes), x, which comes from a cache, one.  AHEAD: both
    // are there, whole; the loads then lie on one path, and what they are waited for
    // by can be counted (on several, a step waited for the weights of the next two).
    auto step = [&](typename W::Weights& o, int i, auto ahead) __attribute__((always_inline)) {
        s.store(o, g, m.wave[wave], m0, lane);
        if constexpr (ahead()) {
            s.template load_x<true>(g, m0, (i + waves) * kStep, lane);
            W::template load<true>(o, g, n0, (i + 2 * waves) * kStep, lane);
        } else {
            load_x(i + waves);
            load(o, i + 2 * waves);
        }
        wave_sync();
        W::apply(m.wave[wave], lane, acc);
        wave_sync();
    };
    load(even, wave);
    load_x(wave);
    load(odd, wave + waves);
    W::clear(g, m.wave[wave], m0, lane);
    wave_sync();
    int i = wave;
    for (; i + 3 * waves < g.K / kStep; i += 2 * waves) {
        step(even, i, std::true_type{});
        step(odd, i + waves, std::true_type{});
    }
    for (; i < last; i += 2 * waves) {
        step(even, i, std::false_type{});
        if (i + waves < last) step(odd, i + waves, std::false_type{});
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) m.part[wave][16 * i + 4 * lg + e][16 * t + lr] = acc[i][t][e];
    __syncthreads();
    for (int at = threadIdx.x; at < 256 * MT * NT; at += blockDim.x) {
        const int row = at / (16 * NT), n = at % (16 * NT);
        float v = 0.0f;
        for (int w = 0; w < waves; ++w) v += m.part[w][row][n];
        v *= 1.0f / Mma<E>::kScale;
        if (m0 + row < g.M && n0 + n < g.N) {
            if (!(fabsf(v) <= 3.4028235e38f)) v = whole_weights<E, GROUP>(g, m0 + row, n0 + n);
            static_cast<T*>(g.y)[int64_t(m0 + row) * g.N + n0 + n] = (T)v;
        }
    }
}

template <typename E, int GROUP>
int launch(const Q4Args& g, hipStream_t stream) {
    // Tiles of 16 rows of x, and weight rows for each x that is loaded: as many as
    // leave a block for each CU.
    const int mt = g.M <= 16 ? 1 : g.M <= 32 ? 2 : 4;
    const int64_t tall = ceil_div(g.M, 16 * mt);
    int nt = 1;
    while (2 * nt * mt <= 4 && ceil_div(g.N, 32 * nt) * tall >= cu_count()) nt *= 2;
    auto run = [&](auto m, auto n) {
        constexpr int MT = m(), NT = n();
        const int steps = int(ceil_div(g.K, kStep));
        const int each = std::max(1, int(ceil_div(steps, kWaves<E, MT, NT>)));   // of a wave
        const int waves = std::max(1, int(ceil_div(steps, each)));
        const int64_t cols = ceil_div(g.N, 16 * NT);
        // Rows of x that a launch holds (65535 tiles along an axis, fewer than 2^32
        // threads), and as many launches as they need.
        const int64_t tiles = std::min<int64_t>(65535, ((int64_t(1) << 32) - 1) / (cols * 64 * waves));
        if (tiles < 1) return fail(PE_ERR_UNSUPPORTED, "matvec_q4: too many weight rows");
        for (int64_t m = 0; m < g.M; m += tiles * 16 * MT) {
            Q4Args part = g;
            part.x = static_cast<const typename E::T*>(g.x) + m * g.x_ms;
            part.y = static_cast<typename E::T*>(g.y) + m * g.N;
            part.M = int32_t(std::min<int64_t>(g.M - m, tiles * 16 * MT));
            q4_kernel<E, GROUP, MT, NT><<<dim3{uint32_t(cols), uint32_t(ceil_div(part.M, 16 * MT))}, 64 * waves, 0, stream>>>(part);
        }
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
