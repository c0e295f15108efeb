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
        } else {
#pragma unroll
            for (int i = 0; i < kChunk; ++i) v[i] = i < n ? p[i] : (typename E::T)0.0f;
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return E::to_f32(v[i]); }
};

// A row's largest absolute value is kept as the bits of |v|: whole numbers order
// like the values, infinities above them and NaN above those, so neither gets
// lost in the maximum.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct Quant {
    float amax, inv;                  // inv = 127 / amax, rounded
    bool none, exactly;
    __device__ __forceinline__ explicit Quant(uint32_t bits) {
        none = bits == 0 || bits >= 0x7f800000u;
        amax = __uint_as_float(bits);
        // (where 127 / amax overflows float32 every value goes the long way)
        exactly = amax < 1e-36f;
        inv = none || exactly ? 0.0f : 127.0f / amax;
    }
    // NaN for a row that holds one or an infinity, so that no finite result comes
    // of it.
    __device__ __forceinline__ float scale() const {
        return __float_as_uint(amax) >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : amax / 127.0f;
    }
    // The whole number of v in the low byte.  Added to 1.5 * 2^23, a value is rounded
    // to a whole number that stands in the last bits.  v * inv is off by less than
    // 127 * 2^-24 = 7.6e-6, so only where it lies that close to a half can the exact
    // quotient round elsewhere; there 127 v and half * amax are compared in 64 bits,
    // which hold both exactly.
    __device__ __forceinline__ uint32_t of(float v) const {
        constexpr float kRound = 12582912.0f;
        float n = fmaf(v, inv, kRound) - kRound;
        const float d = fmaf(v, inv, -n);
        if (__builtin_expect(fabsf(d) > 0.5f - 1.0f / 65536.0f, 0)) {
            const float up = copysignf(1.0f, d);
            const double beyond = (127.0 * double(v) - double(n + 0.5f * up) * double(amax)) * double(up);
            if (beyond > 0.0 || (beyond == 0.0 && (int(n) & 1))) n += up;
        }
        return __float_as_uint(n + kRound);
    }
    __device__ __forceinline__ uint32_t slowly(float v) const {
        return none ? 0u : uint32_t(int(rint(127.0 * double(v) / double(amax)))) & 255u;
    }
};

// Eight values as bytes at q (8-byte aligned).
__device__ __forceinline__ void store_q8(int8_t* q, const Quant& qt, const float (&v)[kChunk]) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    u32x2 o;
    if (__builtin_expect(qt.none || qt.exactly, 0)) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            o[i] = qt.slowly(v[4 * i]) | qt.slowly(v[4 * i + 1]) << 8 | qt.slowly(v[4 * i + 2]) << 16 | qt.slowly(v[4 * i + 3]) << 24;
    } else {
        // (the low byte of each of four words)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            o[i] = __builtin_amdgcn_perm(qt.of(v[4 * i + 1]), qt.of(v[4 * i]), 0x0c0c0400u) |
                   __builtin_amdgcn_perm(qt.of(v[4 * i + 3]), qt.of(v[4 * i + 2]), 0x04000c0cu);
    }
    *reinterpret_cast<u32x2*>(q) = o;
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
    float eps, scale;
};

int norm_launch_f16(Op op, bool q8, bool wide, const NormArgs& a, hipStream_t stream);
int norm_launch_bf16(Op op, bool q8, bool wide, const NormArgs& a, hipStream_t stream);
int norm_launch_f32(Op op, bool q8, bool wide, const NormArgs& a, hipStream_t stream);

}  // namespace rows
}  // namespace pe
