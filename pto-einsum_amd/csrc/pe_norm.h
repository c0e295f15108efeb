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
// caches, mostly (4096 rows of 4096, 8 groups: 25 us here, 51 there).
#pragma once

#include "pe_rows.h"

namespace pe {
namespace rows {
namespace {

using ssm::load_f32;
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

__device__ __forceinline__ float inv_rms(float sum, float D, float eps) { return 1.0f / sqrtf(sum / D + eps); }

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
    for (uint64_t unit = uint64_t(blockIdx.x) * RPB + threadIdx.x / TPR; unit < a.units;
         unit += uint64_t(gridDim.x) * RPB) {
        const Place at(a, uint32_t(unit));
        // (The length as the compiler cannot see through: the masks of a row's end,
        // one for each element, are the same for every row, and taken out of the loop
        // they filled the scalar registers and went through lanes of vector ones.)
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
        if constexpr (OP == kResidual) {
            float inv = 1.0f;
            if (post) {
                float ss = 0.0f;
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int i = 0; i < kChunk; ++i) ss = fmaf(x[j][i], x[j][i], ss);
                inv = inv_rms(across.sum(ss), float(len), a.eps);
            }
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int e = kChunk * (tid + j * TPR), n = len - e;
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    float u = x[j][i];
                    if (post) u = u * inv * pw[j][i];
                    if (gate) u *= a.g_ds ? g[j][i] : one;
                    v[j][i] = res[j][i] + a.scale * u;
                    // (Lanes past the row hold x = 0, but a gate or a norm of
                    // its own may be infinite.)
                    if (n < kChunk && i >= n) v[j][i] = 0.0f;
                    ss = fmaf(v[j][i], v[j][i], ss);
                }
                store_f32<R, kChunk>(static_cast<typename R::T*>(a.r) + at.y + e, n, v[j]);
            }
            inv = inv_rms(across.sum(ss), float(len), a.eps);
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
                    ss[j] = fmaf(v[j][i], v[j][i], ss[j]);
                }
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
                    inv[j] = inv_rms(sum, float(len / a.parts), a.eps);
                }
                // (across.most below lies between these reads and the next row's sums)
                if constexpr (WAVES == 1) ssm::wave_sync();
            } else {
                float all = 0.0f;
#pragma unroll
                for (int j = 0; j < NV; ++j) all += ss[j];
                inv[0] = inv_rms(across.sum(all), float(len), a.eps);
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
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    // (values past the row count for nothing, whatever they are)
                    if (kChunk * (tid + j * TPR) + i >= len) v[j][i] = 0.0f;
                    const uint32_t b = magnitude(v[j][i]);
                    top = b > top ? b : top;
                }
            const Quant qt(across.most(top));
            if (tid == 0) a.qs[at.row] = qt.scale();
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int e = kChunk * (tid + j * TPR);
                if (e < a.q_ms) *reinterpret_cast<u32x2*>(a.q + at.row * a.q_ms + e) = eight(qt, v[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int e = kChunk * (tid + j * TPR);
                store_f32<E, kChunk>(static_cast<typename E::T*>(a.y) + at.y + e, len - e, v[j]);
            }
        }
    }
}

// Any length: the values are formed again for each step, a chunk at a time.  `parts`
// groups within the unit (rows in 8 bits of a grouped norm), whose factors lie in LDS.
constexpr int kLongThreads = 512;

template <typename E, typename R, int OP, bool Q>
__global__ __launch_bounds__(kLongThreads) void norm_long_kernel(NormArgs a) {
    __shared__ uint32_t slots[2 * (kLongThreads / 64)];
    extern __shared__ float factor[];  // [parts]
    Across<kLongThreads> across{slots};
    const int tid = threadIdx.x;
    const int part = a.D / a.parts;
    const bool gate = a.g != nullptr, post = a.pw != nullptr, scaled = a.w != nullptr;
    for (uint64_t unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        const Place at(a, uint32_t(unit));
        const float one = OP == kResidual && gate && !a.g_ds ? E::to_f32(static_cast<const typename E::T*>(a.g)[at.g]) : 1.0f;
        float inv0 = 1.0f;            // of the norm of x, in the residual
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
            for (int i = 0; i < kChunk; ++i) {
                float u = x[i];
                if constexpr (OP == kResidual) {
                    if (post) u = u * inv0 * pw[i];
                    if (gate) u *= a.g_ds ? g[i] : one;
                    u = res[i] + a.scale * u;
                } else if constexpr (OP == kGated) {
                    if (gate && !a.norm_first) u *= silu(g[i]);
                }
                v[i] = i < n ? u : 0.0f;
            }
        };
        auto squares = [](const float (&v)[kChunk], float ss) {
#pragma unroll
            for (int i = 0; i < kChunk; ++i) ss = fmaf(v[i], v[i], ss);
            return ss;
        };
        if constexpr (OP == kResidual) {
            if (post) {
                float ss = 0.0f;
                for (int e = kChunk * tid; e < a.D; e += kChunk * kLongThreads) {
                    Raw<E> x;
                    x.load(a.x, at.x + e, a.D - e);
                    float v[kChunk];
#pragma unroll
                    for (int i = 0; i < kChunk; ++i) v[i] = x[i];
                    ss = squares(v, ss);
                }
                inv0 = inv_rms(across.sum(ss), float(a.D), a.eps);
            }
        }
        if constexpr (OP != kQuantize) {
            float v[kChunk];
            if (a.parts == 1) {
                float ss = 0.0f;
                for (int e = kChunk * tid; e < a.D; e += kChunk * kLongThreads) {
                    values(e, a.D - e, v);
                    if constexpr (OP == kResidual) store_f32<R, kChunk>(static_cast<typename R::T*>(a.r) + at.y + e, a.D - e, v);
                    ss = squares(v, ss);
                }
                const float inv = inv_rms(across.sum(ss), float(a.D), a.eps);
                if (tid == 0) factor[0] = inv;
            } else {
                for (int p = tid >> 6; p < a.parts; p += kLongThreads / 64) {
                    float ss = 0.0f;
                    for (int e = kChunk * (tid & 63); e < part; e += kChunk * 64) {
                        values(p * part + e, part - e, v);
                        ss = squares(v, ss);
                    }
                    const float inv = inv_rms(Across<64>{nullptr}.sum(ss), float(part), a.eps);
                    if ((tid & 63) == 0) factor[p] = inv;
                }
            }
            __syncthreads();
        }
        auto results = [&](int e, float (&v)[kChunk]) {
            const int n = a.D - e;
            values(e, n, v);
            if constexpr (OP != kQuantize) {
                Raw<E> w, g;
                if (scaled) w.load(a.w, at.w + e, n);
                if (OP == kGated && gate && a.norm_first) g.load(a.g, at.g + e, n);
                int p = a.parts == 1 ? 0 : e / part, left = a.parts == 1 ? a.D : (p + 1) * part - e;
#pragma unroll
                for (int i = 0; i < kChunk; ++i) {
                    if (a.parts > 1 && i < n && left-- == 0) {
                        ++p;
                        left = part - 1;
                    }
                    v[i] *= factor[p];
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
