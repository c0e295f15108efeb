// Rows in 8 bits: which whole number stands for a value, shared by the row
// quantiser and the norms that answer with such rows.
//
//   a = max |v| of the row,  scale = a / 127 (rounded once to float32),
//   q = 127 v / a rounded to the nearest whole number, ties to even.
//
// The rounding is that of the exact quotient, not of some float32 form of it:
// half-way values are common (v = a / 2 is always one, 63.5), and forms that
// differ by a unit in the last place would answer 63 here and 64 there.
#pragma once

#include "pe_ssm.h"

namespace pe {
namespace rows {

using ssm::BF16;

constexpr int kChunk = 8;             // elements a lane takes at once: 16 bytes of 16-bit types

// A chunk as it lies in memory, so that loads go out together and take half the
// registers in 16 bits.
template <typename E>
struct Raw {
    typename ssm::Vec<E, kChunk>::type v;
    __device__ __forceinline__ void load(const void* base, int64_t at, int n) {
        const typename E::T* p = static_cast<const typename E::T*>(base) + at;
        if (n >= kChunk) {
            v = *reinterpret_cast<const typename ssm::Vec<E, kChunk>::utype*>(p);
        } else if (n > 0) {
            // (the last one again where the row has ended: no load behind it, and no
            // branch for each)
#pragma unroll
            for (int i = 0; i < kChunk; ++i) {
                const typename E::T t = p[min(i, n - 1)];
                v[i] = i < n ? t : (typename E::T)0.0f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kChunk; ++i) v[i] = (typename E::T)0.0f;
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return E::to_f32(v[i]); }
};

// A row's largest absolute value is kept as the bits of |v|: whole numbers order
// like the values, infinities above them and NaN above those, so neither gets
// lost in the maximum.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct Quant {
    float given, amax, inv, lift;     // amax = given * lift, inv = 127 / amax, rounded
    uint32_t keep;
    __device__ __forceinline__ explicit Quant(uint32_t bits) {
        given = __uint_as_float(bits);
        // Rows far from 1 are multiplied by a power of two first, so that neither
        // 127 / amax nor 127 v leaves float32's range and v's last bits stay (of a
        // large row, what those lose rounds to 0).
        lift = given < 0x1p-60f ? 0x1p90f : given > 0x1p100f ? 0x1p-60f : 1.0f;
        amax = given * lift;
        const bool none = bits == 0 || bits >= 0x7f800000u;
        inv = none ? 0.0f : 127.0f / amax;
        keep = none ? 0u : 0xffffffffu;
    }
    // NaN for a row that holds one or an infinity, so that no finite result comes
    // of it.
    __device__ __forceinline__ float scale() const {
        return __float_as_uint(given) >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : given / 127.0f;
    }
};

// Eight values as bytes.  Added to 1.5 * 2^23, a value is rounded to a whole number
// that stands in the last bits.  v * inv is off by less than 127 * 2^-24 = 7.6e-6, so
// only where it lies that close to a half can the exact quotient round elsewhere.
// There the sign of 127 v - h amax decides, h the half: 127 v is the sum of two
// floats, and h amax, a multiple of half amax's last bit as 127 v next to it is,
// differs from the first by a float.  (One branch for eight values: with one for
// each of a thread's 32 the scalar registers spilled.)
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u32x2 eight(const Quant& qt, const float (&v)[kChunk]) {
    constexpr float kRound = 12582912.0f;
    float u[kChunk], w[kChunk], d[kChunk], far = 0.0f;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) u[i] = v[i];
    if (__builtin_expect(qt.lift != 1.0f, 0)) {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) u[i] *= qt.lift;
    }
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
        w[i] = fmaf(u[i], qt.inv, kRound);
        d[i] = fmaf(u[i], qt.inv, kRound - w[i]);
        far = fmaxf(far, fabsf(d[i]));
    }
    if (__builtin_expect(far > 0.5f - 1.0f / 65536.0f, 0)) {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            const float n = w[i] - kRound, up = copysignf(1.0f, d[i]), h = n + 0.5f * up, p = 127.0f * u[i];
            const float beyond = (fmaf(-h, qt.amax, p) + fmaf(127.0f, u[i], -p)) * up;
            w[i] = kRound + (beyond > 0.0f ? n + up : beyond == 0.0f ? 2.0f * rintf(0.5f * h) : n);
        }
    }
    u32x2 o;
    // (the low byte of each of four words)
#pragma unroll
    for (int i = 0; i < 2; ++i)
        o[i] = (__builtin_amdgcn_perm(__float_as_uint(w[4 * i + 1]), __float_as_uint(w[4 * i]), 0x0c0c0400u) |
                __builtin_amdgcn_perm(__float_as_uint(w[4 * i + 3]), __float_as_uint(w[4 * i + 2]), 0x04000c0cu)) & qt.keep;
    return o;
}

// Bytes of a row in 8 bits that the product reads, in groups of 16, and from one
// row to the next where this library lays them out: long rows on whole lines, since
// a 64-byte piece that straddles two costs both (1203 x 5001 x 2500 29.3 us with
// both operands on lines, 35.8 on every 16 bytes).
inline int64_t row_bytes(int64_t k) { return ceil_div(k, 16) * 16; }
inline int64_t row_pitch(int64_t k) { return k < 1024 ? row_bytes(k) : ceil_div(k, 128) * 128; }

// What the operators are (pe_norm.hip): rows in 8 bits, a norm with a gate, and a
// norm behind a residual sum.
enum Op { kQuantize, kGated, kResidual };

struct NormArgs {
    const void *x, *w, *pw, *g, *res;  // g: z of the gated norm, the gate of the residual one
    void *y, *r;
    int8_t* q;
    float* qs;
    int64_t x0, x1, g0, g1, r0, r1;   // strides of the two leading axes
    int64_t q_ms;
    uint32_t units;                   // rows times groups
    FastDiv inner, groups;            // extent of the second leading axis; groups a unit is one of
    int32_t D;                        // elements of a unit
    int32_t parts;                    // groups within a unit (rows in 8 bits of a grouped norm)
    int32_t g_ds;                     // 0: one gate for a row
    int32_t norm_first;
    float per;                        // one divided by a group's elements
    float eps, scale;
};

int norm_launch_f16(Op op, bool q8, bool wide, const NormArgs& a, hipStream_t stream);
int norm_launch_bf16(Op op, bool q8, bool wide, const NormArgs& a, hipStream_t stream);
int norm_launch_f32(Op op, bool q8, bool wide, const NormArgs& a, hipStream_t stream);

}  // namespace rows
}  // namespace pe
