// Selective scan of prompts in chunks of Q tokens on the matrix cores.
//
// Within a chunk, with run_t = sum_{r <= t} A d_r from the chunk's start, G = C
// B^T and S the state at the start,
//
//   y_t = exp(run_t) C_t S + sum_{s <= t} G_ts exp(run_t - run_s) d_s x_s
//   S'  = exp(run_Q) S + sum_s B_s exp(run_Q - run_s) d_s x_s^T
//
// so all work but the state's hand-over from chunk to chunk is products.  A
// block walks a piece of a sequence for one head and 16 WAVES rows p of it.
// Each wave keeps its 16 columns of S^T [N x 16] in matrix-core accumulators all
// the way; in an accumulator a lane holds four n of one p, which is an operand
// fragment of C S^T when the order of n in that product is chosen to match, so S
// moves through neither LDS nor other lanes.  G^T is computed once a block, a
// wave per 16 tokens t, weighted in registers (a lane holds one t) and passed
// through LDS; B and x reach the products over s by transposing LDS reads.
//
// With few sequences and heads, sequences are cut into pieces that run at once:
// a first launch forms each piece's contribution to the state (the second line
// alone), carry_kernel the states at the pieces' starts, and the main launch
// the outputs.
//
// Rounding: the products take 16-bit operands, so a float32 value enters as a
// sum of terms, each the 16-bit value nearest to what the earlier ones left:
//   bfloat16  state's input three bfloat16 terms (2^-24), S and the weighted
//             scores, which only reach the bfloat16 output, two (2^-16)
//   float16   two float16 terms (2^-21) of the value times a power of two that
//             puts a column's (row's) largest at 2^14: float16's range is not
//             met, and what is lost is below 2^-38 of the largest
//   float32   three bfloat16 terms of everything, products of terms i + j <= 2
// Operands of 16 bits enter as they are.  So a float16 scan's new states are good to
// 2^-21 of their inputs (their sums are float32), and float32 values below 2^-110
// lose bits: the last term of 2^-120 lies under what the matrix cores keep, 6e-4.
// Sums are float32; run_t is summed in 64 bits and kept as two float32, since
// differences of large sums count.
//
// Infinities and NaN spread through terms and through weights of 0 to tokens and
// elements that the recurrence keeps clear of them, and C B^T can pass float32's
// range where the recurrence does not; nothing of the kind ends in finite outputs.  So
// a wave that finds an output (before its gate), or a piece's contribution, not finite
// runs its piece again by the recurrence.
//
// What bounds it is vector work, not memory or the matrix cores: a wave spends some
// 600 vector instructions on a chunk (splitting S and the weighted x into terms,
// fading S, weights, gates) beside 40 matrix instructions, three waves a SIMD.  Two
// prompts of 4096 tokens, 64 heads of 64 x 128, float16: contributions 40 us, states
// 9, outputs 126, a call of 155; 1 x 16384, 24 heads, bfloat16: 32, 11, 88, a call
// of 119 to 129 (token by token 15.2 and 55.6 ms).  Chunks of 64 tokens halve what is done
// once a chunk but leave two waves a SIMD: 17 % longer.
#pragma once

#include "pe_scan.h"

#include <algorithm>

namespace pe {
namespace ssm {

struct ChunkArgs {
    ScanArgs s;
    float* ws_state;     // [pieces][H][ptiles][columns of 16 p][NT / 16][64 lanes][4], or null: one piece each
    float* ws_decay;     // [pieces][H]
    uint32_t piece;      // tokens
    uint32_t pieces;     // in all
    uint32_t per_seq;    // dense: of a sequence
    uint32_t ptiles;
    uint32_t blocks;     // pieces * H * ptiles
    int32_t state4;      // rows of the states are whole aligned 16-byte vectors
};

constexpr int kScanTailBlocks = 64;

// A piece of a sequence: its tokens [t0, t1) and where it stands.
struct Piece {
    int64_t t0, t1;
    int32_t seq;
    bool last;
};

// Piece `id`.  Packed pieces end at multiples of g.piece of the buffer and at
// sequences' ends: the one of sequence s in stretch j of the buffer is j + s,
// which grows from piece to piece.
__device__ __forceinline__ bool find_piece(const ChunkArgs& g, uint32_t id, Piece& o) {
    const ScanArgs& a = g.s;
    if (!a.cu) {
        o.seq = int32_t(id / g.per_seq);
        const uint32_t j = id - uint32_t(o.seq) * g.per_seq;
        o.t0 = int64_t(j) * g.piece;
        o.t1 = min(a.T, o.t0 + int64_t(g.piece));
        o.last = j + 1 == g.per_seq;
        return true;
    }
    int32_t lo = 0, hi = a.nseq;
    while (hi - lo > 1) {
        const int32_t mid = lo + (hi - lo) / 2;
        if (uint32_t(offset_of(a.cu, mid, a.T)) / g.piece + uint32_t(mid) <= id) lo = mid;
        else hi = mid;
    }
    const int64_t from = offset_of(a.cu, lo, a.T), to = offset_of(a.cu, lo + 1, a.T);
    const uint32_t j0 = uint32_t(from) / g.piece, j = id - uint32_t(lo);
    if (id < uint32_t(lo) || j < j0) return false;
    o.seq = lo;
    o.t0 = max(from, int64_t(j) * g.piece);
    o.t1 = min(to, (int64_t(j) + 1) * g.piece);
    o.last = to <= (int64_t(j) + 1) * g.piece;
    return o.t0 < o.t1;
}

// ------------------------------------------------------- terms and products --

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename E>
struct Scheme {  // BF16
    using V8 = bf16x8;
    static constexpr int kIn = 1, kState = 3, kOut = 2;
    static constexpr bool kScaled = false;
};
template <>
struct Scheme<F16> {
    using V8 = f16x8;
    static constexpr int kIn = 1, kState = 2, kOut = 2;
    static constexpr bool kScaled = true;
};
template <>
struct Scheme<F32> {
    using V8 = bf16x8;
    static constexpr int kIn = 3, kState = 3, kOut = 3;
    static constexpr bool kScaled = false;
};

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// Sums of a_i b_j for T tiles, the small ones first; of three terms each, those
// with i + j <= 2.  The tiles take turns, so that none waits for its own last
// product.
template <int T, int NA, int NB, typename V8>
__device__ __forceinline__ void mma(const V8 (&a)[T][NA], const V8 (&b)[NB], f32x4 (&c)[T]) {
#pragma unroll
    for (int o = NA + NB - 2; o >= 0; --o) {
        if (o > 2) continue;
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (o - i >= 0 && o - i < NB)
#pragma unroll
                for (int t = 0; t < T; ++t) c[t] = mfma(a[t][i], b[o - i], c[t]);
    }
}

// The two 16-bit values nearest to x (float16: toward zero, what is left over is
// whole in float32 either way), and x less those.
__device__ __forceinline__ uint32_t take_term(const bf16x8*, f32x2& x) {
    const uint32_t t = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
    x[0] -= __builtin_bit_cast(float, t << 16);
    x[1] -= __builtin_bit_cast(float, t & 0xffff0000u);
    return t;
}
__device__ __forceinline__ uint32_t take_term(const f16x8*, f32x2& x) {
    const f16x2 t = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x[0], x[1]));
    // x - t in one instruction each, t a half of a register (from a conversion and
    // a difference the compiler does not form it).
    const uint32_t u = __builtin_bit_cast(uint32_t, t);
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(x[0]) : "v"(u), "v"(x[0]));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(x[1]) : "v"(u), "v"(x[1]));
    return u;
}

template <int NT, typename V8>
__device__ __forceinline__ void split8(const float (&v)[8], V8 (&o)[NT]) {
    u32x4 w[NT];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f32x2 x = {v[2 * i], v[2 * i + 1]};
#pragma unroll
        for (int t = 0; t < NT; ++t) w[t][i] = take_term((const V8*)nullptr, x);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t] = __builtin_bit_cast(V8, w[t]);
}

__device__ __forceinline__ float elem_f32(f16x8 v, int i) { return (float)v[i]; }
__device__ __forceinline__ float elem_f32(bf16x8 v, int i) {
    const u32x4 w = __builtin_bit_cast(u32x4, v);
    return __builtin_bit_cast(float, (i & 1) ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
}

// A power of two that takes m > 0 into [2^14, 2^15) (below, where m is under
// 2^-112; any for 0, for infinities and NaN), and its inverse.
__device__ __forceinline__ float scale_for(float m, float& inverse) {
    int e = int((__float_as_uint(m) >> 23) & 0xff) - 127;
    e = min(max(e, -112), 127);
    inverse = __uint_as_float(uint32_t(e - 14 + 127) << 23);
    return __uint_as_float(uint32_t(14 - e + 127) << 23);
}

// The largest of the four lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float max_of_groups(float m) {
    // Both halves of what the swap returns hold, in each lane, one of the pair.
    const uint32_t u = __float_as_uint(m);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// x, which the compiler takes for another value: what is formed from it inside a
// loop is not kept in registers across it (some 40 LDS
// addresses and 40 lane masks otherwise).
__device__ __forceinline__ int fresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// The same of a tile: four registers in a row and not four values.
__device__ __forceinline__ f32x4 fresh(f32x4 x) {
    asm volatile("" : "+v"(x));
    return x;
}

// Eight 16-bit elements, the first `by` dropped and zeros moved in.
__device__ __forceinline__ u32x4 shift_out(u32x4 v, int by) {
    if (by & 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (v[i] >> 16) | (i < 3 ? v[i + 1 < 4 ? i + 1 : 3] << 16 : 0u);
    if (by & 2) v = u32x4{v[1], v[2], v[3], 0};
    if (by & 4) v = u32x4{v[2], v[3], 0, 0};
    return by & 8 ? u32x4{0, 0, 0, 0} : v;
}

// Eight elements of a row as loaded, and as terms.
template <typename E>
struct Raw {
    u32x4 v;
    __device__ __forceinline__ void load(const char* p) {
        typedef u32x4 uv __attribute__((aligned(2)));
        v = *reinterpret_cast<const uv*>(p);
    }
    __device__ __forceinline__ void drop(int by) { v = shift_out(v, by); }
    __device__ __forceinline__ void keep_if(bool keep) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = keep ? v[i] : 0u;
    }
    __device__ __forceinline__ void terms(u32x4 (&o)[1]) const { o[0] = v; }
    __device__ __forceinline__ void put(typename E::T* p) const { *reinterpret_cast<u32x4*>(p) = v; }
};
template <>
struct Raw<F32> {
    float v[8];
    __device__ __forceinline__ void load(const char* p) {
        typedef f32x4 uv __attribute__((aligned(4)));
        const f32x4 a = *reinterpret_cast<const uv*>(p), b = *reinterpret_cast<const uv*>(p + 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = a[i];
            v[i + 4] = b[i];
        }
    }
    __device__ __forceinline__ void drop(int by) {
#pragma unroll
        for (int s = 1; s <= 8; s *= 2)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (by & s) ? (i + s < 8 ? v[(i + s) & 7] : 0.0f) : v[i];
    }
    __device__ __forceinline__ void keep_if(bool keep) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = keep ? v[i] : 0.0f;
    }
    __device__ __forceinline__ void put(float* p) const {
        *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
    }
    __device__ __forceinline__ void terms(u32x4 (&o)[3]) const {
        bf16x8 t[3];
        split8(v, t);
#pragma unroll
        for (int i = 0; i < 3; ++i) o[i] = __builtin_bit_cast(u32x4, t[i]);
    }
};

// A plane of [rows][COLS] 16-bit elements in LDS without padding: the 16-byte
// groups of a row are XORed by a number of the row, chosen so that the reads
// below meet every bank once a phase: of M = COLS / 8 groups (16 at most, 256
// bytes) and k the row in units of 256 bytes, k with its bits rotated left by
// one.  Sixteen rows at one group then take all of them, and so do the group
// pairs of eight rows.  The number has a period of 16 rows.
template <int COLS>
__device__ __forceinline__ int swizzle(int row) {
    constexpr int M = COLS < 128 ? COLS / 8 : 16, L = M == 16 ? 4 : M == 8 ? 3 : 2;
    static_assert(M >= 4, "at least 32 columns");
    const int k = (row / (16 / M)) & (M - 1);
    return ((2 * k) & (M - 1)) | (k >> (L - 1));
}
template <int COLS>
__device__ __forceinline__ int place(int row, int col) {
    return row * COLS + (((col >> 3) ^ swizzle<COLS>(row)) << 3) + (col & 7);
}

// Rows of a chunk on their way to LDS: Q rows of COLS elements over THREADS
// threads, eight at a time.  Every load is whole and inside its row: a vector
// that would pass the row's end starts earlier, if need be before `base`, and is
// moved into place (whole rows hold at least eight elements).  Offsets are 32
// bits from the chunk's first row (the host checks the strides).
// LDS planes have LC columns.
template <typename E, int Q, int COLS, int THREADS, int LC = COLS>
struct Rows {
    static constexpr int kVecs = Q * COLS / 8, kEach = (kVecs + THREADS - 1) / THREADS;
    Raw<E> r[kEach];
    // Offsets in bytes from eight elements before the rows, so that they are never
    // negative and the loads take a scalar base; `at` those of a whole chunk.
    uint32_t at[kEach];
    __device__ __forceinline__ uint32_t offset(int i, int32_t ts, int tokens, int width) const {
        const int v = threadIdx.x + i * THREADS, row = min(v / (COLS / 8), min(tokens, Q) - 1), c = v % (COLS / 8) * 8;
        return uint32_t(row * ts + min(c, width - 8) + 8) * E::kBytes;
    }
    __device__ __forceinline__ void init(int32_t ts, int width) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) at[i] = offset(i, ts, Q, width);
    }
    // Of a whole chunk whose first row lies at `base`, and of one of `tokens` rows.
    __device__ __forceinline__ void load(const typename E::T* base) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) r[i].load(reinterpret_cast<const char*>(base - 8) + at[i]);
    }
    __device__ __forceinline__ void load(const typename E::T* base, int32_t ts, int tokens, int width) {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            r[i].load(reinterpret_cast<const char*>(base - 8) + offset(i, ts, tokens, width));
    }
    __device__ __forceinline__ void trim(int tokens, int width) {
        if (width < COLS) {
            const int v = fresh(threadIdx.x);
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int c = (v + i * THREADS) % (COLS / 8) * 8;
                r[i].drop(min(8, c - min(c, width - 8)));
            }
        }
        if (tokens < Q) {
            const int v = fresh(threadIdx.x);
#pragma unroll
            for (int i = 0; i < kEach; ++i) r[i].keep_if((v + i * THREADS) / (COLS / 8) < tokens);
        }
    }
    // As they are, to [Q][PITCH] of T.
    template <int PITCH>
    __device__ __forceinline__ void store_raw(typename E::T* lds, int tokens, int width) {
        trim(tokens, width);
        const int first = fresh(threadIdx.x);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int v = first + i * THREADS;
            if (kVecs % THREADS == 0 || v < kVecs) r[i].put(lds + v / (COLS / 8) * PITCH + v % (COLS / 8) * 8);
        }
    }
    // To kIn planes; SPLIT: columns c of each 32 in the order of frag_split, c = 16
    // h + 4 g + j at 8 g + 4 h + j.
    template <bool SPLIT = false>
    __device__ __forceinline__ void store(uint16_t* lds, int tokens, int width) {
        trim(tokens, width);
        const int first = fresh(threadIdx.x);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int v = first + i * THREADS;
            if (kVecs % THREADS == 0 || v < kVecs) {
                u32x4 t[Scheme<E>::kIn];
                r[i].terms(t);
#pragma unroll
                for (int k = 0; k < Scheme<E>::kIn; ++k) {
                    const int row = v / (COLS / 8), u = v % (COLS / 8);
                    if constexpr (SPLIT) {
                        const int c = 8 * ((u & ~3) + 2 * (u & 1)) + 4 * ((u >> 1) & 1);
                        *reinterpret_cast<u32x2*>(lds + k * Q * LC + place<LC>(row, c)) = u32x2{t[k][0], t[k][1]};
                        *reinterpret_cast<u32x2*>(lds + k * Q * LC + place<LC>(row, c + 8)) = u32x2{t[k][2], t[k][3]};
                    } else {
                        *reinterpret_cast<u32x4*>(lds + k * Q * LC + place<LC>(row, 8 * u)) = t[k];
                    }
                }
            }
        }
    }
};

// Operand fragments of planes of COLS columns.  r16 is a multiple of 16 rows.
// Lane l: row r16 + l % 16, eight columns from c + 8 (l / 16).
template <typename V8, int COLS>
__device__ __forceinline__ V8 frag_row(const uint16_t* p, int r16, int c, int lane) {
    const int row = lane & 15;
    return *reinterpret_cast<const V8*>(p + r16 * COLS + row * COLS +
                                        (((c >> 3) ^ ((lane >> 4) ^ swizzle<COLS>(row))) << 3));
}
// Lane l: row r16 + l % 16, columns c + 4 (l / 16) .. + 3 and those 16 further on.
template <typename V8, int COLS>
__device__ __forceinline__ V8 frag_split(const uint16_t* p, int r16, int c, int lane) {
    const int row = lane & 15, g = (lane >> 5) ^ swizzle<COLS>(row);
    const uint16_t* q = p + r16 * COLS + row * COLS + 4 * ((lane >> 4) & 1);
    const u32x2 a = *reinterpret_cast<const u32x2*>(q + (((c >> 3) ^ g) << 3));
    const u32x2 b = *reinterpret_cast<const u32x2*>(q + (((c >> 3) ^ 2 ^ g) << 3));
    return __builtin_bit_cast(V8, u32x4{a[0], a[1], b[0], b[1]});
}
// Transposing read: lane 4 j + q of each 16 points at row j, columns 4 q .. + 3;
// lane i receives column i of the four rows.
typedef short i16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2 read_tr(const uint16_t* p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (__attribute__((address_space(3))) i16x4*)(p)));
}
// Lane l: column c + l % 16 (c a multiple of 16), rows r16 + 4 (l / 16) .. + 3.
template <int COLS>
__device__ __forceinline__ u32x2 read_tr(const uint16_t* p, int r16, int c, int lane) {
    const int row = 4 * (lane >> 4) + ((lane >> 2) & 3);
    return read_tr(p + r16 * COLS + row * COLS + (((c >> 3) ^ (((lane >> 1) & 1) ^ swizzle<COLS>(row))) << 3) +
                   4 * (lane & 1));
}
// The same rows and those 16 further on.
template <typename V8, int COLS>
__device__ __forceinline__ V8 frag_tr(const uint16_t* p, int r16, int c, int lane) {
    const u32x2 a = read_tr<COLS>(p, r16, c, lane), b = read_tr<COLS>(p, r16 + 16, c, lane);
    return __builtin_bit_cast(V8, u32x4{a[0], a[1], b[0], b[1]});
}

// ------------------------------------------------------------------- kernel --


template <typename E, int NT, int Q, int WAVES>
struct ChunkShape {
    static constexpr int kPT = 16 * WAVES, kThreads = 64 * WAVES, kIn = Scheme<E>::kIn, kOut = Scheme<E>::kOut;
    static constexpr int kXC = WAVES == 3 ? 64 : kPT;          // columns of x's planes: a power of two
    static constexpr int kZP = kPT + 16 / E::kBytes;
    static constexpr int kTokens = 256;  // whose step sizes are prepared at a time
    // Waves of a SIMD that the registers are held to: three, which hide more of the
    // chain from LDS read to product, where 16-bit types run without a spill then.
    static constexpr int kPerSimd = E::kBytes == 2 && NT <= 128 && (NT < 128 || WAVES > 2) ? 3 : 2;
    struct Lds {
        alignas(16) uint16_t b[kIn * Q * NT], c[kIn * Q * NT], x[kIn * Q * kXC], p[kOut * Q * Q];
        alignas(16) float step[kTokens], hi[kTokens], lo[kTokens], weight[kTokens], fade[kTokens], row[Q];
        float whole[kTokens / Q];
        alignas(16) typename E::T z[Q * kZP];  // the gate's inputs, then the outputs
    };
    struct LdsStates {
        alignas(16) uint16_t b[kIn * Q * NT], x[kIn * Q * kXC];
        alignas(16) float weight[kTokens];
        float whole[kTokens / Q];
    };
    // Blocks of the main kernel that a CU of 160 KB holds.
    static constexpr int kResident = std::min(4 * kPerSimd / WAVES, int(160 * 1024 / sizeof(Lds)));
    static_assert(kResident >= 1, "too much LDS");
};

// MAIN: outputs (and the final states); else the pieces' contributions.
template <typename E, int NT, int Q, int WAVES, bool MAIN>
__global__ __launch_bounds__(64 * WAVES, (ChunkShape<E, NT, Q, WAVES>::kPerSimd)) void chunk_kernel(ChunkArgs g) {
    using T = typename E::T;
    using Sch = Scheme<E>;
    using V8 = typename Sch::V8;
    using Shape = ChunkShape<E, NT, Q, WAVES>;
    constexpr int kThreads = Shape::kThreads, kPT = Shape::kPT, kIn = Sch::kIn, kState = Sch::kState, kOut = Sch::kOut;
    constexpr int kZP = Shape::kZP, kXC = Shape::kXC, kTokens = Shape::kTokens;
    // Tiles of n whose sums take turns; registers hold one of a float16 main kernel.
    constexpr int kTurn = MAIN && Sch::kScaled ? 1 : 2;
    constexpr int kTT = Q / 16, kNN = NT / 16, kKS = Q / 32, kKN = NT / 32;
    __shared__ std::conditional_t<MAIN, typename Shape::Lds, typename Shape::LdsStates> m;
    const ScanArgs& a = g.s;

    if (blockIdx.x >= g.blocks) {
        clear_outside<E>(a, int64_t(blockIdx.x - g.blocks) * kThreads + threadIdx.x, kScanTailBlocks * kThreads);
        return;
    }
    // Blocks go round the eight XCDs in turn; each XCD gets a run of work, whose
    // heads read the same B and C through its L2.
    const uint32_t xcd = blockIdx.x & 7, each = g.blocks >> 3, more = g.blocks & 7;
    const uint32_t job = xcd * each + min(xcd, more) + (blockIdx.x >> 3);
    const uint32_t ph = job / g.ptiles, pt = job - ph * g.ptiles;
    const uint32_t id = ph / uint32_t(a.H), h = ph - id * uint32_t(a.H);
    Piece piece;
    if (!__builtin_amdgcn_readfirstlane(find_piece(g, id, piece))) return;
    // The same for the whole block: kept in scalar registers.
    piece.t0 = __builtin_amdgcn_readfirstlane(int(piece.t0));
    piece.t1 = __builtin_amdgcn_readfirstlane(int(piece.t1));
    piece.seq = __builtin_amdgcn_readfirstlane(piece.seq);
    piece.last = __builtin_amdgcn_readfirstlane(piece.last);
    if (!MAIN && piece.last) return;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 15, lg = lane >> 4;
    const int p0 = int(pt) * kPT, width = min(kPT, a.P - p0);  // columns of x
    const bool active = 16 * wave < width;
    // The wave's turn at the scores: other waves from block to block, since a
    // block's first wave is on the same SIMD in each.
    const int scorer = int((uint32_t(wave) + job) % WAVES);
    const int p = p0 + 16 * wave + lr;
    const int64_t seq = a.cu ? 0 : piece.seq;
    const int group = int(h) / (a.H / a.G);
    const T* bb = static_cast<const T*>(a.B) + seq * a.b_bs + piece.t0 * a.b_ts + group * a.b_gs;
    const T* cb = static_cast<const T*>(a.C) + seq * a.c_bs + piece.t0 * a.c_ts + group * a.c_gs;
    const T* xb = static_cast<const T*>(a.x) + seq * a.x_bs + piece.t0 * a.x_ts + h * a.x_hs + p0;
    const T* zb = static_cast<const T*>(a.z) + seq * a.z_bs + piece.t0 * a.z_ts + h * a.z_hs + p0;
    const float A = a.A[h], bias = a.dt_bias ? a.dt_bias[h] : 0.0f;
    const double A2 = double(A) * 1.4426950408889634;  // exponents are of 2
    const char* dtp = static_cast<const char*>(a.dt) +
                      (seq * a.dt_bs + piece.t0 * a.dt_ts + h * a.dt_hs) * (a.dt_f32 ? 4 : E::kBytes);
    // Token strides: below kScanStrideEnd (the host sees to it).
    const int32_t b_ts = int32_t(a.b_ts), c_ts = int32_t(a.c_ts), x_ts = int32_t(a.x_ts), z_ts = int32_t(a.z_ts);
    const int32_t dt_ts = int32_t(a.dt_ts);
    const int tokens = int(piece.t1 - piece.t0);

    f32x4 S[kNN];  // lane: p = lr; n = 16 i + 4 lg + element
    // Where a lane's part of the piece's state lies in the workspace.
    auto place_of = [&](int ln) __attribute__((always_inline)) {
        return g.ws_state + ((((int64_t(id) * a.H + h) * g.ptiles + pt) * WAVES + wave) * kNN * 64 + ln) * 4;
    };
    const int32_t ys = a.H * a.P;  // token stride of y
    T* yb = static_cast<T*>(a.y) + ((a.cu ? 0 : int64_t(piece.seq) * a.T) + piece.t0) * int64_t(ys) + int64_t(h) * a.P + p0;
    const int64_t state_at = ((int64_t(piece.seq) * a.H + h) * a.P + p) * a.N;
    // Lane ln's part of the state at the piece's start (contributions: 0).
    auto load_state = [&](int ln) __attribute__((always_inline)) {
        const int lg = ln >> 4, p = p0 + 16 * wave + (ln & 15);
        const int64_t state_at = ((int64_t(piece.seq) * a.H + h) * a.P + p) * a.N;
#pragma unroll
        for (int i = 0; i < kNN; ++i) S[i] = f32x4{0, 0, 0, 0};
        if constexpr (MAIN) {
            if (g.ws_state) {
                const float* ws = place_of(ln);
#pragma unroll
                for (int i = 0; i < kNN; ++i)
                    if (16 * i < a.N && active) S[i] = *reinterpret_cast<const f32x4*>(ws + i * 256);
            } else if (a.state_in && p < a.P) {
#pragma unroll
                for (int i = 0; i < kNN; ++i) {
                    const int n = 16 * i + 4 * lg;
                    if (g.state4) {
                        if (n < a.N) S[i] = *reinterpret_cast<const f32x4*>(a.state_in + state_at + n);
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (n + k < a.N) S[i][k] = a.state_in[state_at + n + k];
                    }
                }
            }
        }
    };
    load_state(lane);
    bool have_state = MAIN && (g.ws_state || a.state_in);

    Rows<E, Q, NT, kThreads> rb;
    Rows<E, Q, MAIN ? NT : 32, kThreads> rc;
    Rows<E, Q, kPT, kThreads, kXC> rx;
    Rows<E, Q, kPT, kThreads> rz;
    const bool gated = MAIN && a.z;
    rb.init(b_ts, a.N);
    rx.init(x_ts, a.P - p0);
    if constexpr (MAIN) {
        rc.init(c_ts, a.N);
        rz.init(z_ts, a.P - p0);
    }
    // The next chunk's rows: `left` tokens from where the pointers stand.
    auto fetch = [&](int left) {
        if (left >= Q) {
            rb.load(bb);
            rx.load(xb);
            if constexpr (MAIN) {
                rc.load(cb);
                if (gated) rz.load(zb);
            }
        } else {
            rb.load(bb, b_ts, left, a.N);
            rx.load(xb, x_ts, left, a.P - p0);
            if constexpr (MAIN) {
                rc.load(cb, c_ts, left, a.N);
                if (gated) rz.load(zb, z_ts, left, a.P - p0);
            }
        }
        bb += Q * b_ts;
        xb += Q * x_ts;
        if constexpr (MAIN) {
            cb += Q * c_ts;
            zb += Q * z_ts;
        }
    };
    fetch(tokens);
    // Raw step sizes of the next kTokens, a wave 64 of them at a time.
    constexpr int kParts = kTokens / 64, kOwn = (kParts + WAVES - 1) / WAVES;
    uint32_t raw[kOwn];
    auto fetch_dt = [&](int t) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            raw[i] = dt_bits<E>(a, dtp, step_offset(min(64 * (wave + i * WAVES) + lane, tokens - t - 1), dt_ts));
        dtp += int64_t(kTokens) * dt_ts * (a.dt_f32 ? 4 : E::kBytes);
    };
    fetch_dt(0);
    double sum = 0.0;  // of this piece's exponents
    float wild[MAIN ? 1 : 4] = {};  // NaN once an output (contributions: the state) was not finite
    const float skip = a.D ? a.D[h] : 0.0f;

    for (int t0 = 0; t0 < tokens; t0 += Q) {
        const int left = tokens - t0, at = t0 & (kTokens - 1);
        __syncthreads();
        rb.store(m.b, left, a.N);
        rx.store(m.x, left, a.P - p0);
        if constexpr (MAIN) {
            rc.template store<true>(m.c, left, a.N);
            if (gated) rz.template store_raw<kZP>(m.z, left, a.P - p0);
        }
        if (at == 0) {
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                const int part = wave + i * WAVES, tok = 64 * part + lane;
                if (part < kParts) {
                    const float d = t0 + tok < tokens ? step_size(a, dt_of<E>(a, raw[i]), bias) : 0.0f;
                    // Decays below 2^-4096 are 0 all the same.
                    double e = A2 * double(d);
                    e = e < -4096.0 ? -4096.0 : e;
#pragma unroll
                    for (int o = 1; o < Q; o *= 2) {
                        const double v = __shfl_up(e, o);
                        if ((lane & (Q - 1)) >= o) e += v;
                    }
                    const double all = __shfl(e, lane | (Q - 1));
                    m.weight[tok] = d * __builtin_amdgcn_exp2f(float(all - e));
                    if constexpr (MAIN) {
                        const float hi = float(e);
                        m.step[tok] = d;
                        m.hi[tok] = hi;
                        m.lo[tok] = float(e - double(hi));
                        m.fade[tok] = __builtin_amdgcn_exp2f(hi);
                        if ((lane & (Q - 1)) == 0) m.whole[tok / Q] = __builtin_amdgcn_exp2f(float(all));
                    } else {
                        if ((lane & (Q - 1)) == 0) m.whole[tok / Q] = float(all);
                    }
                }
            }
            if (t0 + kTokens < tokens) fetch_dt(t0 + kTokens);
        }
        if (left > Q) fetch(left - Q);
        __syncthreads();

        // Fragments are read a step ahead of the products that take them; the
        // barriers to the scheduler keep it from moving the reads back (to save
        // registers, it waited for each right after its read: chunks of one
        // block alone took 1.5 times as long).
        int ln = fresh(lane), lr = ln & 15, lg = ln >> 4;
        auto read_c = [&](V8 (&f)[kTT][kIn], int kk) __attribute__((always_inline)) {
#pragma unroll
            for (int tt = 0; tt < kTT; ++tt)
#pragma unroll
                for (int k = 0; k < kIn; ++k) {
                    if constexpr (MAIN) f[tt][k] = frag_row<V8, NT>(m.c + k * Q * NT, 16 * tt, 32 * kk, ln);
                }
        };
        auto read_bt = [&](V8 (&f)[kKS][kTurn][kIn], int i) __attribute__((always_inline)) {
#pragma unroll
            for (int ks = 0; ks < kKS; ++ks)
#pragma unroll
                for (int u = 0; u < kTurn; ++u)
#pragma unroll
                    for (int k = 0; k < kIn; ++k)
                        f[ks][u][k] = frag_tr<V8, NT>(m.b + k * Q * NT, 32 * ks, 16 * (kTurn * i + u), ln);
        };
        // G^T, weighted: P[t][s] = G_ts exp(run_t - run_s) d_s, s <= t, tiles s of
        // 16 up to tile t.
        if constexpr (MAIN) {
            auto scores = [&](auto tiles) __attribute__((always_inline)) {
                constexpr int kS = tiles(), tt = kS - 1;
                const int t = 16 * tt + lr;
                f32x4 w[kS];
#pragma unroll
                for (int s = 0; s < kS; ++s) w[s] = f32x4{0, 0, 0, 0};
                V8 cf[2][kIn], bf[2][kS][kIn];
                auto read = [&](int kk) __attribute__((always_inline)) {
#pragma unroll
                    for (int k = 0; k < kIn; ++k) {
                        cf[kk & 1][k] = frag_row<V8, NT>(m.c + k * Q * NT, 16 * tt, 32 * kk, ln);
#pragma unroll
                        for (int s = 0; s < kS; ++s)
                            bf[kk & 1][s][k] = frag_split<V8, NT>(m.b + k * Q * NT, 16 * s, 32 * kk, ln);
                    }
                };
                read(0);
#pragma unroll
                for (int kk = 0; kk < kKN; ++kk) {
                    if (kk + 1 < kKN) read(kk + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    mma(bf[kk & 1], cf[kk & 1], w);
                }
                const float hi = m.hi[at + t], lo = m.lo[at + t];
                f32x4 e[kS], sd[kS];
#pragma unroll
                for (int s = 0; s < kS; ++s) {
                    const int s0 = 16 * s + 4 * lg;
                    const f32x4 sh = *reinterpret_cast<const f32x4*>(m.hi + at + s0);
                    const f32x4 sl = *reinterpret_cast<const f32x4*>(m.lo + at + s0);
                    sd[s] = *reinterpret_cast<const f32x4*>(m.step + at + s0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) e[s][i] = (hi - sh[i]) + (lo - sl[i]);
                }
                float top = 0.0f;
#pragma unroll
                for (int s = 0; s < kS; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        w[s][i] *= __builtin_amdgcn_exp2f(e[s][i]) * sd[s][i];
                        if (s == tt) w[s][i] = 4 * lg + i <= lr ? w[s][i] : 0.0f;
                        if constexpr (Sch::kScaled) top = fmaxf(top, fabsf(w[s][i]));
                    }
                float factor = 1.0f;
                if constexpr (Sch::kScaled) {
                    float inverse;
                    factor = scale_for(max_of_groups(top), inverse);
                    if (lg == 0) m.row[t] = inverse;
                }
                // In the order of the products over s: s = 16 h + 4 g + j at 8 g + 4 h + j.
#pragma unroll
                for (int s = 0; s < kTT; ++s) {
                    f32x2 u = {0, 0}, v = {0, 0};
                    if (s < kS) {
                        u = f32x2{w[s < kS ? s : 0][0] * factor, w[s < kS ? s : 0][1] * factor};
                        v = f32x2{w[s < kS ? s : 0][2] * factor, w[s < kS ? s : 0][3] * factor};
                    }
#pragma unroll
                    for (int k = 0; k < kOut; ++k)
                        *reinterpret_cast<u32x2*>(m.p + k * Q * Q + place<Q>(t, 8 * lg + 4 * s)) =
                            u32x2{take_term((const V8*)nullptr, u), take_term((const V8*)nullptr, v)};
                }
            };
            static_assert(kTT == 2, "two tiles of tokens");
            if (scorer == 0) scores(std::integral_constant<int, 1>{});
            if (scorer == 1) scores(std::integral_constant<int, 2>{});
        }

        __builtin_amdgcn_sched_barrier(0);
        ln = fresh(ln), lr = ln & 15, lg = ln >> 4;
        // x^T: lane p, s = 32 ks + 4 lg .. + 3 and those 16 further on, the order of
        // all products over s.  In the outputs' layout, x of token tile tt is half of
        // it.
        V8 xf[kKS][kIn];
        f32x4 y[MAIN ? kTT : 1], gate[MAIN ? kTT : 1];
        if constexpr (MAIN) {
#pragma unroll
            for (int tt = 0; tt < kTT; ++tt) y[tt] = f32x4{0, 0, 0, 0};
        }
        if (active) {
            if constexpr (MAIN) {
                // exp(run_t) C S
                if (have_state) {
                    V8 cf[2][kTT][kIn];
                    read_c(cf[0], 0);
                    float factor = 1.0f, inverse = 1.0f;
                    if constexpr (Sch::kScaled) {
                        float top[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int i = 0; i < kNN; ++i)
#pragma unroll
                            for (int k = 0; k < 4; ++k) top[i & 3] = fmaxf(top[i & 3], fabsf(S[i][k]));
                        factor = scale_for(max_of_groups(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]))), inverse);
                    }
#pragma unroll
                    for (int kk = 0; kk < kKN; ++kk) {
                        if (kk + 1 < kKN) read_c(cf[(kk + 1) & 1], kk + 1);
                        __builtin_amdgcn_sched_barrier(0);
                        float v[8];
                        V8 sf[kOut];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            v[i] = S[2 * kk + i / 4][i % 4];
                            if constexpr (Sch::kScaled) v[i] *= factor;
                        }
                        split8(v, sf);
                        mma(cf[kk & 1], sf, y);
                    }
#pragma unroll
                    for (int tt = 0; tt < kTT; ++tt) {
                        const f32x4 f = *reinterpret_cast<const f32x4*>(m.fade + at + 16 * tt + 4 * lg);
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[tt][i] *= Sch::kScaled ? f[i] * inverse : f[i];
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            ln = fresh(ln), lr = ln & 15, lg = ln >> 4;
            // S' = exp(run_Q) S + B^T (w x)
            V8 bf[2][kKS][kTurn][kIn];
#pragma unroll
            for (int ks = 0; ks < kKS; ++ks)
#pragma unroll
                for (int k = 0; k < kIn; ++k)
                    xf[ks][k] = frag_tr<V8, kXC>(m.x + k * Q * kXC, 32 * ks, 16 * wave, ln);
            float whole = m.whole[at / Q];
            read_bt(bf[0], 0);
            if constexpr (!MAIN) {
                sum += double(whole);
                whole = __builtin_amdgcn_exp2f(whole);
            }
            V8 wx[kKS][kState];
            float xv[kKS][8], wv[kKS][8], top = 0.0f, factor = 1.0f, inverse = 1.0f;
#pragma unroll
            for (int ks = 0; ks < kKS; ++ks) {
                const f32x4 w0 = *reinterpret_cast<const f32x4*>(m.weight + at + 32 * ks + 4 * lg);
                const f32x4 w1 = *reinterpret_cast<const f32x4*>(m.weight + at + 32 * ks + 16 + 4 * lg);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float v = elem_f32(xf[ks][0], i);
#pragma unroll
                    for (int k = 1; k < kIn; ++k) v += elem_f32(xf[ks][k], i);
                    xv[ks][i] = v;
                    wv[ks][i] = v * (i < 4 ? w0[i & 3] : w1[i & 3]);
                    if constexpr (Sch::kScaled) top = fmaxf(top, fabsf(wv[ks][i]));
                }
            }
            if constexpr (MAIN) {
                // the skip
#pragma unroll
                for (int tt = 0; tt < kTT; ++tt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[tt][i] = __builtin_fmaf(skip, xv[tt / 2][4 * (tt & 1) + i], y[tt][i]);
            }
            if constexpr (Sch::kScaled) factor = scale_for(max_of_groups(top), inverse);
#pragma unroll
            for (int ks = 0; ks < kKS; ++ks) {
                if constexpr (Sch::kScaled)
#pragma unroll
                    for (int i = 0; i < 8; ++i) wv[ks][i] *= factor;
                split8(wv[ks], wx[ks]);
            }
#pragma unroll
            for (int i = 0; i < kNN / kTurn; ++i) {
                if (i + 1 < kNN / kTurn) read_bt(bf[(i + 1) & 1], i + 1);
                __builtin_amdgcn_sched_barrier(0);
                f32x4 d[kTurn];
#pragma unroll
                for (int u = 0; u < kTurn; ++u)
#pragma unroll
                    for (int k = 0; k < 4; ++k) d[u][k] = Sch::kScaled ? 0.0f : S[kTurn * i + u][k] * whole;
#pragma unroll
                for (int ks = 0; ks < kKS; ++ks) mma(bf[i & 1][ks], wx[ks], d);
#pragma unroll
                for (int u = 0; u < kTurn; ++u)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        S[kTurn * i + u][k] = Sch::kScaled ? __builtin_fmaf(d[u][k], inverse, S[kTurn * i + u][k] * whole) : d[u][k];
            }
            have_state = true;
        }
        if constexpr (MAIN) {
            // The gate's inputs, in the outputs' layout.
            if (active && gated) {
#pragma unroll
                for (int tt = 0; tt < kTT; ++tt) {
                    if constexpr (E::kBytes == 2) {
                        const u32x2 v = read_tr(reinterpret_cast<const uint16_t*>(m.z) +
                                                (16 * tt + 4 * lg + (lr >> 2)) * kZP + 16 * wave + 4 * (lr & 3));
                        const V8 v8 = __builtin_bit_cast(V8, u32x4{v[0], v[1], 0, 0});
#pragma unroll
                        for (int i = 0; i < 4; ++i) gate[tt][i] = silu(elem_f32(v8, i));
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            gate[tt][i] = silu(E::to_f32(m.z[(16 * tt + 4 * lg + i) * kZP + 16 * wave + lr]));
                    }
                }
            }
        }
        if constexpr (MAIN) {
            __syncthreads();
            ln = fresh(ln), lr = ln & 15, lg = ln >> 4;
            if (active) {
                V8 pf[kTT][kOut];
#pragma unroll
                for (int tt = 0; tt < kTT; ++tt)
#pragma unroll
                    for (int k = 0; k < kOut; ++k) pf[tt][k] = frag_row<V8, Q>(m.p + k * Q * Q, 16 * tt, 0, ln);
                f32x4 d[kTT], r[kTT];
#pragma unroll
                for (int tt = 0; tt < kTT; ++tt) {
                    d[tt] = Sch::kScaled ? f32x4{0, 0, 0, 0} : y[tt];
                    if constexpr (Sch::kScaled) r[tt] = *reinterpret_cast<const f32x4*>(m.row + 16 * tt + 4 * lg);
                }
                mma(pf, xf[0], d);
#pragma unroll
                for (int tt = 0; tt < kTT; ++tt) {
                    if constexpr (Sch::kScaled)
#pragma unroll
                        for (int i = 0; i < 4; ++i) d[tt][i] = __builtin_fmaf(d[tt][i], r[tt][i], y[tt][i]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) wild[0] = __builtin_fmaf(d[tt][i], 0.0f, wild[0]);
                    if (gated)
#pragma unroll
                        for (int i = 0; i < 4; ++i) d[tt][i] *= gate[tt][i];
#pragma unroll
                    for (int i = 0; i < 4; ++i) m.z[(16 * tt + 4 * lg + i) * kZP + 16 * wave + lr] = T(d[tt][i]);
                }
                // The wave's columns of y, 16 bytes a lane.
                wave_sync();
                constexpr int kV = 16 / E::kBytes, kL = 16 / kV, kR = 64 / kL;
                const int pc = 16 * wave + kV * (ln % kL), have = width - pc;
                char* yp = reinterpret_cast<char*>(yb);
                const uint32_t yo = uint32_t((ln / kL) * ys + pc) * E::kBytes, yr = uint32_t(kR * ys) * E::kBytes;
#pragma unroll
                for (int i = 0; i < Q / kR; ++i) {
                    const int t = ln / kL + i * kR;
                    const T* from = m.z + t * kZP + pc;
                    if (t < left) {
                        if (have >= kV) {
                            *reinterpret_cast<typename Vec<E, kV>::utype*>(yp + (yo + i * yr)) =
                                *reinterpret_cast<const typename Vec<E, kV>::type*>(from);
                        } else {
#pragma unroll
                            for (int k = 0; k < kV; ++k)
                                if (k < have) reinterpret_cast<T*>(yp + (yo + i * yr))[k] = from[k];
                        }
                    }
                }
            }
            yb += Q * ys;
        }
    }

    if (!active) return;
    // What is not finite has spread (above): the piece again, by the recurrence as
    // rows_kernel has it.  Lanes l ^ 16 and l ^ 32 hold other n of one p.  (What a lane
    // needs for it is formed here: kept through the chunks it spilled registers.)
    if constexpr (!MAIN) {
#pragma unroll
        for (int i = 0; i < kNN; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) wild[k] = __builtin_fmaf(S[i][k], 0.0f, wild[k]);
        wild[0] = (wild[0] + wild[MAIN ? 0 : 1]) + (wild[MAIN ? 0 : 2] + wild[MAIN ? 0 : 3]);
    }
    if (__any(wild[0] != wild[0])) {
        __threadfence();  // outputs are written a second time, by other lanes
        const int ln = fresh(lane), p = p0 + 16 * wave + (ln & 15);
        const int64_t row = min(p, a.P - 1);
        load_state(ln);
#pragma unroll 1
        for (int64_t t = piece.t0; t < piece.t1; ++t) {
            const float d = step_size(a, dt_of<E>(a, dt_bits<E>(a, a.dt, seq * a.dt_bs + t * a.dt_ts + h * a.dt_hs)), bias);
            const float fade = expf(A * d);
            const T* bt = static_cast<const T*>(a.B) + seq * a.b_bs + t * a.b_ts + group * a.b_gs;
            const T* ct = static_cast<const T*>(a.C) + seq * a.c_bs + t * a.c_ts + group * a.c_gs;
            const T x = static_cast<const T*>(a.x)[seq * a.x_bs + t * a.x_ts + h * a.x_hs + row];
            const int n0 = 4 * fresh(ln >> 4);
            // A token's loads at once; a vector that would pass the row's end starts
            // earlier.
            typename Vec<E, 4>::type b[kNN], c[MAIN ? kNN : 1];
#pragma unroll
            for (int i = 0; i < kNN; ++i) {
                const int at = min(16 * i + n0, a.N - 4);
                b[i] = *reinterpret_cast<const typename Vec<E, 4>::utype*>(bt + at);
                if constexpr (MAIN) c[i] = *reinterpret_cast<const typename Vec<E, 4>::utype*>(ct + at);
            }
            __builtin_amdgcn_sched_barrier(0);
            const float xv = p < a.P ? E::to_f32(x) : 0.0f, dx = d * xv;
            float v = 0.0f;
#pragma unroll
            for (int i = 0; i < kNN; ++i) {
                const int n = 16 * i + n0, by = n - min(n, a.N - 4);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    T bk = b[i][k], ck = c[MAIN ? i : 0][k];
#pragma unroll
                    for (int j = k + 1; j < 4; ++j) {
                        bk = by == j - k ? b[i][j] : bk;
                        ck = by == j - k ? c[MAIN ? i : 0][j] : ck;
                    }
                    S[i][k] = n + k < a.N ? __builtin_fmaf(fade, S[i][k], dx * E::to_f32(bk)) : 0.0f;
                    if constexpr (MAIN) v = n + k < a.N ? __builtin_fmaf(E::to_f32(ck), S[i][k], v) : v;
                }
                S[i] = fresh(S[i]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (MAIN) {
                v += __shfl_xor(v, 16);
                v += __shfl_xor(v, 32);
                v = __builtin_fmaf(skip, xv, v);
                if (gated) v *= silu(E::to_f32(static_cast<const T*>(a.z)[seq * a.z_bs + t * a.z_ts + h * a.z_hs + row]));
                if (ln < 16 && p < a.P)
                    static_cast<T*>(a.y)[((a.cu ? 0 : int64_t(piece.seq) * a.T) + t) * ys + int64_t(h) * a.P + p] = T(v);
            }
        }
    }
    if constexpr (!MAIN) {
        float* ws = place_of(lane);
#pragma unroll
        for (int i = 0; i < kNN; ++i)
            if (16 * i < a.N) *reinterpret_cast<f32x4*>(ws + i * 256) = S[i];
        if (pt == 0 && threadIdx.x == 0) {
            // Not 0, but the least above it: an infinite state stays one.
            const float decay = __builtin_amdgcn_exp2f(float(sum));
            g.ws_decay[int64_t(id) * a.H + h] = decay == 0.0f ? 0x1p-149f : decay;
        }
    } else if (piece.last && a.state_out && p < a.P) {
#pragma unroll
        for (int i = 0; i < kNN; ++i) {
            const int n = 16 * i + 4 * lg;
            if (g.state4) {
                if (n < a.N) *reinterpret_cast<f32x4*>(a.state_out + state_at + n) = S[i];
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (n + k < a.N) a.state_out[state_at + n + k] = S[i][k];
            }
        }
    }
}

// The kernels of one element type: launches the pieces' contributions or (main)
// the outputs, or (g null) only tells how many blocks a CU holds.
int chunks_f16(const ChunkArgs* g, int nt, int waves, bool main, hipStream_t stream);
int chunks_bf16(const ChunkArgs* g, int nt, int waves, bool main, hipStream_t stream);
int chunks_f32(const ChunkArgs* g, int nt, int waves, bool main, hipStream_t stream);

template <typename E, int NT, int WAVES>
int chunks(const ChunkArgs* g, bool main, hipStream_t stream) {
    constexpr int Q = 32;
    if (g && main) {
        const uint32_t blocks = g->blocks + (g->s.cu ? kScanTailBlocks : 0);
        chunk_kernel<E, NT, Q, WAVES, true><<<blocks, 64 * WAVES, 0, stream>>>(*g);
    } else if (g) {
        chunk_kernel<E, NT, E::kBytes == 2 && NT <= 128 ? 64 : 32, WAVES, false><<<g->blocks, 64 * WAVES, 0, stream>>>(*g);
    }
    return ChunkShape<E, NT, Q, WAVES>::kResident;
}

template <typename E, int NT>
int chunks(const ChunkArgs* g, int waves, bool main, hipStream_t stream) {
    if constexpr (NT < 256) {
        if (waves == 2) return chunks<E, NT, 2>(g, main, stream);
    }
    if (waves == 3) return chunks<E, NT, 3>(g, main, stream);
    return chunks<E, NT, 4>(g, main, stream);
}

template <typename E>
int chunks(const ChunkArgs* g, int nt, int waves, bool main, hipStream_t stream) {
    switch (nt) {
        case 32: return chunks<E, 32>(g, waves, main, stream);
        case 64: return chunks<E, 64>(g, waves, main, stream);
        case 128: return chunks<E, 128>(g, waves, main, stream);
        default: return chunks<E, 256>(g, waves, main, stream);
    }
}

}  // namespace ssm
}  // namespace pe
