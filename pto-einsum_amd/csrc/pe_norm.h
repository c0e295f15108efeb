// Norms between blocks and rows in 8 bits (gfx950): one pass over each row.
//
//   quantize:  q, scale of x                                (pe_rows.h)
//   gated:     u = x silu(z), y = u / sqrt(mean u^2 + eps) w, or with norm_first
//              y = x / sqrt(mean x^2 + eps) w silu(z); the mean over each group
//   residual:  u = x, or x / sqrt(mean x^2 + eps) pw;  r = res + scale gate u;
//              y = r / sqrt(mean r^2 + eps) w; y comes of r before r is rounded
//
// y is rounded once to the type, or goes to rows in 8 bits from float32.  What
// bounds these is memory: each value is read once into registers, the sums go
// over the lanes of a row's threads, and the row is written from the registers.
// TPR threads take a row, NV chunks of eight elements each; a wave alone needs no
// barrier, and short rows share a block.  Rows too long for the registers, and
// rows in 8 bits of a grouped norm (whose scale spans the groups) unless its groups are
// whole 512 elements, go to a kernel that reads the row again for each step: from the
// caches, mostly (4096 rows of 4096: 8 groups 22 us here, 16 groups 60 there).
#pragma once

#include "pe_rows.h"

namespace pe {
namespace rows {
namespace {

using ssm::silu;
using ssm::store_f32;

// Sum, and maximum of magnitudes, over the TPR threads of a row.
template <int TPR>
struct Across {
    static constexpr int WAVES = TPR / 64;
    uint32_t* slots;                  // two sets of WAVES words, used in turn
    int turn = 0;
    template <typename F>
    __device__ __forceinline__ uint32_t over(uint32_t v, F f) {
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) v = f(v, uint32_t(__shfl_xor(int(v), m)));
        if constexpr (WAVES > 1) {
            uint32_t* s = slots + turn * WAVES;
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
            __syncthreads();
            v = s[0];
#pragma unroll
            for (int i = 1; i < WAVES; ++i) v = f(v, s[i]);
        }
        return v;
    }
    __device__ __forceinline__ float sum(float v) {
        return __uint_as_float(over(__float_as_uint(v), [](uint32_t a, uint32_t b) {
            return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
        }));
    }
    __device__ __forceinline__ uint32_t most(uint32_t v) {
        return over(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
    }
};

// Sums of squares that float32 does not hold, beyond its range (values from about 1e19
// on) or of squares that it holds in too few bits or not at all (1e-15 and less, where
// eps is as small): the row is taken once more, with its values times a power of two.
// Which one, as a number that a wave's lanes share, so that other rows only pass a
// branch of the wave.
enum Far { kNear, kLarge, kSmall };
__device__ __forceinline__ bool lifted(int far) { return __builtin_expect(far != kNear, 0); }
__device__ __forceinline__ float lift(int far) { return far == kLarge ? 0x1p-80f : far == kSmall ? 0x1p100f : 1.0f; }
__device__ __forceinline__ int far_of(float mean) {
    constexpr uint32_t kLeast = (127u - 100u) << 23;                 // 2^-100
    const uint32_t bits = __float_as_uint(mean);
    const bool held = bits - kLeast < 0x7f800000u - kLeast;          // (below infinity)
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(int(held)), 1)) return kNear;
    return __builtin_amdgcn_readfirstlane(bits < kLeast ? kSmall : kLarge);
}

// The mean of squares of which `sum` is the sum, of values times lift(far); `per` is one
// divided by their number.
__device__ __forceinline__ float mean_of(float sum, float per, float eps, int far) {
    if (lifted(far)) eps = eps * lift(far) * lift(far);
    return fmaf(sum, per, eps);
}

// 1 / sqrt(mean).  Of a near one, neither 0 nor infinite, through the hardware's, which
// is good to a unit, and a step of Newton's: off by less than the division's and the
// root's two roundings, without the 20 instructions that a row would wait for.
__device__ __forceinline__ float factor_of(float mean, int far) {
    if (lifted(far)) return 1.0f / sqrtf(mean);
    const float r = __builtin_amdgcn_rsqf(mean);
    return fmaf(0.5f * r, fmaf(-mean * r, r, 1.0f), r);
}

// Where a unit's values start.
struct Place {
    int64_t x, g, r, y;               // y: in the contiguous outputs
    int64_t row;
    int32_t w;                        // first element of the unit in its row
    __device__ __forceinline__ Place(const NormArgs& a, uint32_t unit) {
        uint32_t rw, gr, o, i;
        a.groups.divmod(unit, rw, gr);
        a.inner.divmod(rw, o, i);
        row = rw;
        w = int32_t(gr) * a.D;
        x = int64_t(o) * a.x0 + int64_t(i) * a.x1 + w;
        g = int64_t(o) * a.g0 + int64_t(i) * a.g1 + (a.g_ds ? w : 0);
        r = int64_t(o) * a.r0 + int64_t(i) * a.r1 + w;
        y = int64_t(unit) * a.D;
    }
};

// What values are multiplied by, lift(far) and then inv.
struct Factor {
    float inv = 1.0f;
    int far = kNear;
    // Both in one float32: of lifted ones the sign is set, and a part of the lift brings
    // inv, 2^-48 to 2^24 of large ones and 2^-50 to 2^50 of small ones, below 1 or above;
    // and what else a value is multiplied by.
    __device__ __forceinline__ float packed() const { return inv * (far == kNear ? 1.0f : far == kLarge ? -0x1p-60f : -0x1p60f); }
    __device__ __forceinline__ static float rest(float f) { return f >= 0.0f ? 1.0f : f > -1.0f ? -0x1p-20f : -0x1p40f; }
};

// What a wave's chunk holds: a grouped norm whose groups are whole ones of these needs
// no second reading for rows in 8 bits.
constexpr int kSegment = 64 * kChunk;

template <typename E, typename R, int OP, bool Q, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_kernel(NormArgs a) {
    constexpr int THREADS = TPR < 256 ? 256 : TPR, RPB = THREADS / TPR;
    __shared__ uint32_t slots[2 * (TPR / 64)];
    __shared__ float segments[OP == kGated && Q ? RPB * NV * (TPR / 64) : 1];
    Across<TPR> across{slots};
    const int tid = threadIdx.x % TPR;
    const bool gate = a.g != nullptr, post = a.pw != nullptr, scaled = a.w != nullptr;
    // What the row's values are lifted by: for a residual x's and then the sum's, for
    // groups within a row each chunk's; and whether it is taken once more.
    constexpr int FAR = OP == kResidual ? 2 : OP == kGated && Q ? NV : 1;
    int far[FAR] = {};
    bool again = false;
    for (uint64_t unit = uint64_t(blockIdx.x) * RPB + threadIdx.x / TPR; unit < a.units;
         unit += again ? 0 : uint64_t(gridDim.x) * RPB) {
        const Place at(a, uint32_t(unit));
        // (The length as the compiler cannot see through: the masks of a row's end,
        // one for each element, are the same for every row, and taken out of the loop
        // they filled the scalar registers and went through lanes of vector ones.  The
        // residual's kernels of four chunks still put 42 or 52 there.)
        int len = a.D;
        asm volatile("" : "+s"(len));
        Raw<E> x[NV], g[NV], w[NV], pw[NV];
        Raw<R> res[NV];
        float one = 1.0f;             // the row's own gate
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = kChunk * (tid + j * TPR), n = len - e;
            x[j].load(a.x, at.x + e, n);
            if constexpr (OP == kResidual) res[j].load(a.res, at.r + e, n);
            if (OP != kQuantize && gate && a.g_ds) g[j].load(a.g, at.g + e, n);
            if (OP == kResidual && post) pw[j].load(a.pw, e, n);
            if (OP != kQuantize && scaled) w[j].load(a.w, at.w + e, n);
        }
        if (OP == kResidual && gate && !a.g_ds) one = E::to_f32(static_cast<const typename E::T*>(a.g)[at.g]);
        float v[NV][kChunk];
        int found = kNear;            // what is to be lifted is not yet, here or (groups within a row) in another wave
        if constexpr (OP == kResidual) {
            float inv = 1.0f, raised = 1.0f;
            if (post) {
                float ss = 0.0f;
                raised = lift(far[0]);
                if (lifted(far[0])) {
#pragma unroll
                    for (int j = 0; j < NV; ++j)
#pragma unroll
                        for (int i = 0; i < kChunk; ++i) ss = fmaf(x[j][i] * raised, x[j][i] * raised, ss);
                } else {
#pragma unroll
                    for (int j = 0; j < NV; ++j)
#pragma unroll
                        for (int i = 0; i < kChunk; ++i) ss = fmaf(x[j][i], x[j][i], ss);
                }
                const float mean = mean_of(across.sum(ss), a.per, a.eps, far[0]);
                inv = factor_of(mean, far[0]);
                if (!lifted(far[0])) found = far_of(mean);
            }
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int e = kChunk * (tid + j * TPR), n = len - e;
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    float u = x[j][i];
                    if (post) u = u * raised * inv * pw[j][i];
                    if (gate) u *= a.g_ds ? g[j][i] : one;
                    v[j][i] = res[j][i] + a.scale * u;
                    // (Lanes past the row hold x = 0, but a gate or a norm of
                    // its own may be infinite.)
                    if (n < kChunk && i >= n) v[j][i] = 0.0f;
                }
                store_f32<R, kChunk>(static_cast<typename R::T*>(a.r) + at.y + e, n, v[j]);
            }
            if (lifted(far[FAR - 1])) {
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int i = 0; i < kChunk; ++i) v[j][i] *= lift(far[FAR - 1]);
            }
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) ss = fmaf(v[j][i], v[j][i], ss);
            const float mean = mean_of(across.sum(ss), a.per, a.eps, far[FAR - 1]);
            // (of a row whose x is to be lifted, the sum written above is not yet it)
            far[0] |= found;
            if (!lifted(found) && !lifted(far[FAR - 1])) {
                found = far_of(mean);
                far[FAR - 1] = found;
            }
            inv = factor_of(mean, far[FAR - 1]);
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    v[j][i] *= inv;
                    if (scaled) v[j][i] *= w[j][i];
                }
        } else if constexpr (OP == kGated) {
            const bool first = gate && !a.norm_first;
            float ss[NV], inv[NV];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                ss[j] = 0.0f;
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    v[j][i] = x[j][i];
                    if (first) v[j][i] *= silu(g[j][i]);
                }
                if (lifted(far[FAR == 1 ? 0 : j]))
#pragma unroll
                    for (int i = 0; i < kChunk; ++i) v[j][i] *= lift(far[FAR == 1 ? 0 : j]);
#pragma unroll
                for (int i = 0; i < kChunk; ++i) ss[j] = fmaf(v[j][i], v[j][i], ss[j]);
            }
            if (Q && a.parts > 1) {
                // Groups of whole segments, the 512 elements that a wave's chunk holds:
                // each segment's sum to LDS, and there those of its group together.
                constexpr int WAVES = TPR / 64;
                const int wave = tid >> 6, each = len / a.parts / kSegment;
                float* mine = segments + threadIdx.x / TPR * (NV * WAVES);
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const float sum = Across<64>{nullptr}.sum(ss[j]);
                    if ((tid & 63) == 0) mine[j * WAVES + wave] = sum;
                }
                if constexpr (WAVES > 1) __syncthreads();
                else ssm::wave_sync();
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int from = (j * WAVES + wave) / each * each;
                    float sum = 0.0f;
                    for (int i = from; i < min(from + each, NV * WAVES); ++i) sum += mine[i];
                    const float mean = mean_of(sum, a.per, a.eps, far[FAR == 1 ? 0 : j]);
                    inv[j] = factor_of(mean, far[FAR == 1 ? 0 : j]);
                    // (a wave's chunk past the row takes no part)
                    if (!lifted(far[FAR == 1 ? 0 : j]) && kSegment * (j * WAVES + wave) < len) {
                        const int f = far_of(mean);
                        far[FAR == 1 ? 0 : j] = f;
                        found |= f;
                    }
                }
                // (across.most below lies between these reads and the next row's sums)
                if constexpr (WAVES == 1) ssm::wave_sync();
            } else {
                float all = 0.0f;
#pragma unroll
                for (int j = 0; j < NV; ++j) all += ss[j];
                const float mean = mean_of(across.sum(all), a.per, a.eps, far[0]);
                inv[0] = factor_of(mean, far[0]);
                if (!lifted(far[0])) found = far_of(mean);
#pragma unroll
                for (int j = 0; j < FAR; ++j) far[j] |= found;
#pragma unroll
                for (int j = 1; j < NV; ++j) inv[j] = inv[0];
            }
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    v[j][i] *= inv[j];
                    if (scaled) v[j][i] *= w[j][i];
                    if (gate && a.norm_first) v[j][i] *= silu(g[j][i]);
                }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) v[j][i] = x[j][i];
        }
        if constexpr (Q) {
            // (above any magnitude, where a wave finds a group that is to be lifted)
            constexpr uint32_t kBeyond = 0x80000000u;
            uint32_t top = lifted(found) ? kBeyond : 0u;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    // (values past the row count for nothing, whatever they are)
                    if (kChunk * (tid + j * TPR) + i >= len) v[j][i] = 0.0f;
                    const uint32_t b = magnitude(v[j][i]);
                    top = b > top ? b : top;
                }
            top = across.most(top);
            if (OP != kQuantize && __builtin_expect(__builtin_amdgcn_readfirstlane(int(top >= kBeyond)), 0)) {
                again = true;
                continue;
            }
            const Quant qt(top);
            if (tid == 0) a.qs[at.row] = qt.scale();
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int e = kChunk * (tid + j * TPR);
                if (e < a.q_ms) *reinterpret_cast<u32x2*>(a.q + at.row * a.q_ms + e) = eight(qt, v[j]);
            }
        } else {
            again = lifted(found);
            if (again) continue;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int e = kChunk * (tid + j * TPR);
                store_f32<E, kChunk>(static_cast<typename E::T*>(a.y) + at.y + e, len - e, v[j]);
            }
        }
        again = false;
#pragma unroll
        for (int j = 0; j < FAR; ++j) far[j] = kNear;
    }
}

// Any length: the values are formed again for each step, a chunk at a time.  `parts`
// groups within the unit (rows in 8 bits of a grouped norm), whose factors lie in LDS.
constexpr int kLongThreads = 512;

// (Three blocks a CU, which the lifted path would otherwise leave at two: 4096 rows of
// 20480, residual to 8 bits, 276 us with two and 234 with three.)
template <typename E, typename R, int OP, bool Q>
__global__ __launch_bounds__(kLongThreads, OP == kResidual && R::kBytes == 4 ? 5 : 6) void norm_long_kernel(NormArgs a) {
    __shared__ uint32_t slots[2 * (kLongThreads / 64)];
    extern __shared__ float factor[];  // [parts] where there are several, packed
    Across<kLongThreads> across{slots};
    const int tid = threadIdx.x;
    const int part = a.D / a.parts;
    const bool gate = a.g != nullptr, post = a.pw != nullptr, scaled = a.w != nullptr;
    for (uint64_t unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        const Place at(a, uint32_t(unit));
        const float one = OP == kResidual && gate && !a.g_ds ? E::to_f32(static_cast<const typename E::T*>(a.g)[at.g]) : 1.0f;
        Factor norm, whole;           // of x, in the residual, and of what is normed, undivided
        // n values from e on, as the norm takes them (past those 0).
        auto values = [&](int e, int n, float (&v)[kChunk]) {
            Raw<E> x, g, pw;
            Raw<R> res;
            x.load(a.x, at.x + e, n);
            if (OP != kQuantize && gate && a.g_ds && !(OP == kGated && a.norm_first)) g.load(a.g, at.g + e, n);
            if constexpr (OP == kResidual) {
                res.load(a.res, at.r + e, n);
                if (post) pw.load(a.pw, e, n);
            }
#pragma unroll
            for (int i = 0; i < kChunk; ++i) v[i] = x[i];
            if (OP == kResidual && lifted(norm.far))
#pragma unroll
                for (int i = 0; i < kChunk; ++i) v[i] *= lift(norm.far);
#pragma unroll
            for (int i = 0; i < kChunk; ++i) {
                float u = v[i];
                if constexpr (OP == kResidual) {
                    if (post) u = u * norm.inv * pw[i];
                    if (gate) u *= a.g_ds ? g[i] : one;
                    u = res[i] + a.scale * u;
                } else if constexpr (OP == kGated) {
                    if (gate && !a.norm_first) u *= silu(g[i]);
                }
                v[i] = i < n ? u : 0.0f;
            }
        };
        // The factor of n values that f(e, v) gives by chunks, dealt to the
        // threads of `over`, of which this is number `thread`: twice where they are
        // to be lifted.
        auto formed = [&](int n, int thread, auto& over, auto f) {
            constexpr int kThreads = std::decay_t<decltype(over)>::WAVES * 64;
            for (int far = kNear;;) {
                float ss = 0.0f;
                for (int e = kChunk * thread; e < n; e += kChunk * kThreads) {
                    float v[kChunk];
                    f(e, v);
                    if (lifted(far))
#pragma unroll
                        for (int i = 0; i < kChunk; ++i) v[i] *= lift(far);
#pragma unroll
                    for (int i = 0; i < kChunk; ++i) ss = fmaf(v[i], v[i], ss);
                }
                const float mean = mean_of(over.sum(ss), a.per, a.eps, far);
                const int found = lifted(far) ? kNear : far_of(mean);
                if (found == kNear) return Factor{factor_of(mean, far), far};
                far = found;
            }
        };
        if constexpr (OP == kResidual) {
            if (post)
                norm = formed(a.D, tid, across, [&](int e, float (&v)[kChunk]) {
                    Raw<E> x;
                    x.load(a.x, at.x + e, a.D - e);
#pragma unroll
                    for (int i = 0; i < kChunk; ++i) v[i] = x[i];
                });
        }
        if constexpr (OP != kQuantize) {
            if (a.parts == 1) {
                whole = formed(a.D, tid, across, [&](int e, float (&v)[kChunk]) {
                    values(e, a.D - e, v);
                    if constexpr (OP == kResidual) store_f32<R, kChunk>(static_cast<typename R::T*>(a.r) + at.y + e, a.D - e, v);
                });
            } else {
                Across<64> wave{nullptr};
                for (int p = tid >> 6; p < a.parts; p += kLongThreads / 64) {
                    const Factor f = formed(part, tid & 63, wave, [&](int e, float (&v)[kChunk]) {
                        values(p * part + e, part - e, v);
                    });
                    if ((tid & 63) == 0) factor[p] = f.packed();
                }
                __syncthreads();
            }
        }
        auto results = [&](int e, float (&v)[kChunk]) {
            const int n = a.D - e;
            values(e, n, v);
            if constexpr (OP != kQuantize) {
                Raw<E> w, g;
                if (scaled) w.load(a.w, at.w + e, n);
                if (OP == kGated && gate && a.norm_first) g.load(a.g, at.g + e, n);
                if (a.parts == 1) {
                    if (lifted(whole.far))
#pragma unroll
                        for (int i = 0; i < kChunk; ++i) v[i] *= lift(whole.far);
#pragma unroll
                    for (int i = 0; i < kChunk; ++i) v[i] *= whole.inv;
                } else {
                    const int p0 = e / part, left0 = (p0 + 1) * part - e;
                    auto factors = [&](auto f) {
                        int p = p0, left = left0;
#pragma unroll
                        for (int i = 0; i < kChunk; ++i) {
                            if (i < n && left-- == 0) {
                                ++p;
                                left = part - 1;
                            }
                            f(v[i], factor[p]);
                        }
                    };
                    uint32_t signs = 0;
                    factors([&](float& u, float f) {
                        u *= f;
                        signs |= __float_as_uint(f);
                    });
                    if (__builtin_expect(__any(int(signs) < 0), 0)) factors([](float& u, float f) { u *= Factor::rest(f); });
                }
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    if (scaled) v[i] *= w[i];
                    if (OP == kGated && gate && a.norm_first) v[i] *= silu(g[i]);
                }
            }
        };
        if constexpr (Q) {
            uint32_t top = 0;
            float v[kChunk];
            for (int e = kChunk * tid; e < a.D; e += kChunk * kLongThreads) {
                results(e, v);
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    const uint32_t b = e + i < a.D ? magnitude(v[i]) : 0u;
                    top = b > top ? b : top;
                }
            }
            const Quant qt(across.most(top));
            if (tid == 0) a.qs[at.row] = qt.scale();
            for (int e = kChunk * tid; e < a.q_ms; e += kChunk * kLongThreads) {
                if (e < a.D) results(e, v);
#pragma unroll
                for (int i = 0; i < kChunk; ++i)
                    if (e + i >= a.D) v[i] = 0.0f;
                *reinterpret_cast<u32x2*>(a.q + at.row * a.q_ms + e) = eight(qt, v);
            }
        } else {
            for (int e = kChunk * tid; e < a.D; e += kChunk * kLongThreads) {
                float v[kChunk];
                results(e, v);
                store_f32<E, kChunk>(static_cast<typename E::T*>(a.y) + at.y + e, a.D - e, v);
            }
        }
        // (the next unit's factors are written behind this unit's reads)
        __syncthreads();
    }
}

// Rows of at most this many elements pass through registers.
constexpr int kLongest = 2048 * kChunk;
constexpr int64_t kMostBlocks = int64_t(1) << 20;

template <typename E, typename R, int OP, bool Q>
int launch(const NormArgs& a, hipStream_t stream) {
    if (a.D > kLongest || (a.parts > 1 && a.D / a.parts % kSegment)) {
        const uint32_t grid = uint32_t(std::min<int64_t>(a.units, kMostBlocks));
        norm_long_kernel<E, R, OP, Q><<<grid, kLongThreads, sizeof(float) * a.parts, stream>>>(a);
        return ssm::hip_status_of_launch("norm");
    }
    auto go = [&](auto t, auto v) {
        constexpr int TPR = t(), NV = v(), THREADS = TPR < 256 ? 256 : TPR;
        const uint32_t grid = uint32_t(std::min<int64_t>(ceil_div(a.units, THREADS / TPR), kMostBlocks));
        norm_kernel<E, R, OP, Q, TPR, NV><<<grid, THREADS, 0, stream>>>(a);
        return ssm::hip_status_of_launch("norm");
    };
    using std::integral_constant;
    // Threads and chunks of a row: a wave while its registers do, then 256 threads,
    // which leave the other rows of a CU something to do at each barrier (rows of
    // 8192 to 8 bits: 256 threads with four chunks 42 us, 512 with two 48, 1024 with
    // one 84; 16384: 512 with four 44, 1024 with two 63).
    const integral_constant<int, 1> one{};
    const integral_constant<int, 2> two{};
    const integral_constant<int, 4> four{};
    const integral_constant<int, 64> wave{};
    const integral_constant<int, 256> block{};
    if (a.D <= 64 * kChunk) return go(wave, one);
    if (a.D <= 128 * kChunk) return go(wave, two);
    if (a.D <= 256 * kChunk) return go(block, one);
    if (a.D <= 512 * kChunk) return go(block, two);
    if (a.D <= 1024 * kChunk) return go(block, four);
    return go(integral_constant<int, 512>{}, four);
}

template <typename E>
int launch_type(Op op, bool q8, bool wide, const NormArgs& a, hipStream_t stream) {
    if (op == kQuantize) return launch<E, E, kQuantize, true>(a, stream);
    if (op == kGated) return q8 ? launch<E, E, kGated, true>(a, stream) : launch<E, E, kGated, false>(a, stream);
    if (wide) return q8 ? launch<E, F32, kResidual, true>(a, stream) : launch<E, F32, kResidual, false>(a, stream);
    return q8 ? launch<E, E, kResidual, true>(a, stream) : launch<E, E, kResidual, false>(a, stream);
}

}  // namespace
}  // namespace rows
}  // namespace pe
