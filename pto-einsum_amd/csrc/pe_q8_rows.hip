// Products of rows in 8 bits for few rows of x: the tokens of a decode step.
//
// Reading the weights bounds these.  A block's waves each take every WAVES-th
// 128 bytes along k of its 16 NT weight rows and 16 MT rows of x, and add up in LDS
// at the end, which for whole numbers is exact in any order.  Until then no wave
// waits for another: each has a ring of DEPTH steps in LDS of its own, filled by
// direct loads of whole lines, eight lanes to a line.  (Loaded straight into the
// registers of the matrix cores, whose lanes 0 to 15 are 16 rows, a load touches 16
// lines with every 16 lanes and the address unit takes four times as long.)
//
// Where x is a few short rows in another type, each block takes them to 8 bits
// itself while its first weights are on their way: that costs it less than a launch
// of its own costs the call.
#include "pe_q8.h"

#include <algorithm>

namespace pe {
namespace q8 {
namespace {

constexpr int kStep = 128;            // bytes of k of a step, two products

// OWN: x is of type E and goes to 8 bits here, 16 rows at most.
constexpr int kOwnChunks = 8;         // of a thread
constexpr int kOwnBytes = 256 * kOwnChunks * rows::kChunk;   // of the rows in 8 bits

template <typename E, int MT, int NT, int WAVES, int DEPTH, bool OWN>
__global__ __launch_bounds__(64 * WAVES) void q8_rows_kernel(Q8Args g) {
    constexpr int STEP = ((OWN ? 0 : MT) + NT) * 16 * kStep, NI = STEP / 1024;
    static_assert((DEPTH - 1) * NI < 64, "loads in flight that vmcnt counts");
    static_assert(DEPTH * STEP >= MT * NT * 1024, "the sums fit the rings");
    static_assert(!OWN || MT == 1, "one tile of rows");
    __shared__ __attribute__((aligned(1024))) int8_t lds[WAVES * DEPTH * STEP];
    __shared__ __attribute__((aligned(16))) int8_t own[OWN ? kOwnBytes : 16];
    __shared__ uint32_t top[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    const int m0 = int(blockIdx.y) * 16 * MT, n0 = int(blockIdx.x) * 16 * NT;
    const int steps = (g.K + kStep - 1) / kStep;
    const uint32_t last = uint32_t(g.K - 1) & ~15u;
    const uint32_t ring = uint32_t(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) int8_t*)lds)) + uint32_t(wave) * DEPTH * STEP;

    // Chunk c of a step is rows 8 c .. 8 c + 7 of w and then of x; the 16-byte group
    // j of row r lies in slot j ^ (r % 8).
    uint32_t off[NI];
#pragma unroll
    for (int c = 0; c < NI; ++c) {
        const int r = 8 * c + lane / 8;
        off[c] = r < 16 * NT ? uint32_t(min(r, g.N - 1 - n0)) * uint32_t(g.w_ns)
                             : uint32_t(min(r - 16 * NT, g.M - 1 - m0)) * uint32_t(g.x_ms);
    }
    const int8_t* wb = g.w + int64_t(n0) * g.w_ns;
    const int8_t* xb = g.x + int64_t(m0) * g.x_ms;
    const uint32_t seg = 16u * ((lane & 7) ^ (lane >> 3));
    // Blocks start at different places along k: rows lie a power of two apart as
    // often as not, and blocks that all read the same k at once would meet in the
    // same few memory channels.
    const int turn = steps > 1 ? int(blockIdx.x % uint32_t(steps)) : 0;
    auto turned = [&](int s) { return s + turn < steps ? s + turn : s + turn - steps; };
    auto issue = [&](int i, int slot) {
        // (past this wave's last step, that one again, which nothing reads)
        const int s = turned(min(wave + waves * i, steps - 1));
        const uint32_t k = min(uint32_t(s) * kStep + seg, last);
#pragma unroll
        for (int c = 0; c < NI; ++c)
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                         : : "v"(off[c] + k), "s"(8 * c < 16 * NT ? wb : xb), "s"(ring + uint32_t(slot) * STEP + uint32_t(c) * 1024u)
                         : "memory", "m0");
    };
    i32x4 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

    const int row = lane & 15;
    const int mine = wave < steps ? (steps - wave + waves - 1) / waves : 0;
    const int pitch = steps * kStep;                     // of the rows in LDS
    if constexpr (OWN) {
        // Chunks of all rows, dealt to the threads; their loads come back before the
        // weights' go out, whose number the compiler's waits do not know of.
        const int threads = 64 * waves, chunks = pitch / rows::kChunk;
        rows::Raw<E> raw[kOwnChunks];
        int at[kOwnChunks], of[kOwnChunks];
#pragma unroll
        for (int j = 0; j < kOwnChunks; ++j) {
            const int c = int(threadIdx.x) + j * threads;
            of[j] = c / chunks;
            at[j] = rows::kChunk * (c - of[j] * chunks);
            if (of[j] < g.M) raw[j].load(g.x, int64_t(of[j]) * g.x_ms + at[j], g.K - at[j]);
        }
        if (threadIdx.x < 16) top[threadIdx.x] = 0;
        uint32_t most[kOwnChunks];
#pragma unroll
        for (int j = 0; j < kOwnChunks; ++j) {
            most[j] = 0;
            if (of[j] < g.M)
#pragma unroll
                for (int e = 0; e < rows::kChunk; ++e) most[j] = max(most[j], rows::magnitude(raw[j][e]));
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (mine > 0)
#pragma unroll
            for (int i = 0; i < DEPTH - 1; ++i) issue(i, i);
#pragma unroll
        for (int j = 0; j < kOwnChunks; ++j)
            if (of[j] < g.M) atomicMax(&top[of[j]], most[j]);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int j = 0; j < kOwnChunks; ++j) {
            if (of[j] >= g.M) continue;
            const rows::Quant qt(top[of[j]]);
            float v[rows::kChunk];
#pragma unroll
            for (int e = 0; e < rows::kChunk; ++e) v[e] = raw[j][e];
            *reinterpret_cast<rows::u32x2*>(own + of[j] * pitch + at[j]) = rows::eight(qt, v);
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    } else if (mine > 0) {
#pragma unroll
        for (int i = 0; i < DEPTH - 1; ++i) issue(i, i);
    }
    if (mine > 0) {
        int slot = 0, free_slot = DEPTH - 1;
        for (int i = 0; i < mine; ++i) {
            // (the last step's fragments have left the slot that is loaded now)
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            issue(i + DEPTH - 1, free_slot);
            free_slot = slot;
            asm volatile("s_waitcnt vmcnt(%0)" : : "n"((DEPTH - 1) * NI) : "memory");
            const int s = turned(wave + waves * i);
            const int left = g.K - s * kStep;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int j16 = 4 * h + (lane >> 4);
                const uint32_t at = ring + uint32_t(slot) * STEP + uint32_t(row * kStep + 16 * (j16 ^ (row & 7)));
                i32x4 a[NT], b[MT];
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    a[t] = *reinterpret_cast<const __attribute__((address_space(3))) i32x4*>(uintptr_t(at + uint32_t(t) * 16 * kStep));
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    b[t] = OWN ? *reinterpret_cast<const i32x4*>(own + min(row, g.M - 1) * pitch + s * kStep + 16 * j16)
                               : *reinterpret_cast<const __attribute__((address_space(3))) i32x4*>(uintptr_t(at + uint32_t(NT + t) * 16 * kStep));
                if (!OWN && left < kStep) {
                    // Zeros for x behind K.
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int bytes = min(max(left - 16 * j16 - 4 * e, 0), 4);
                        const uint32_t keep = bytes == 4 ? 0xffffffffu : (1u << (8 * bytes)) - 1u;
#pragma unroll
                        for (int t = 0; t < MT; ++t) b[t][e] = int32_t(uint32_t(b[t][e]) & keep);
                    }
                }
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int t = 0; t < MT; ++t)
                        acc[u][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u], b[t], acc[u][t], 0, 0, 0);
            }
            slot = slot + 1 == DEPTH ? 0 : slot + 1;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    // The waves' sums, tile by tile.
    i32x4* sums = reinterpret_cast<i32x4*>(lds);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) sums[((wave * NT + i) * MT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    for (int t = wave; t < NT * MT; t += waves) {
        i32x4 sum = {0, 0, 0, 0};
        for (int w = 0; w < waves; ++w) sum += sums[(w * NT * MT + t) * 64 + lane];
        const int m = m0 + 16 * (t % MT) + row, n = n0 + 16 * (t / MT) + 4 * (lane >> 4);
        if (m < g.M) finish<E>(g, column<E>(g, n), OWN ? rows::Quant(top[m]).scale() : g.xs[m], m, n, sum);
    }
}

template <typename E, int MT, int NT, int DEPTH, bool OWN>
int run(const Q8Args& g, hipStream_t stream) {
    constexpr int WAVES = 4;
    const int64_t cols = ceil_div(g.N, 16 * NT), tall = ceil_div(g.M, 16 * MT);
    const int waves = int(std::max<int64_t>(1, std::min<int64_t>(WAVES, ceil_div(g.K, kStep))));
    if (tall > 65535 || cols * tall * 64 * waves >= (int64_t(1) << 32)) return fail(PE_ERR_UNSUPPORTED, "matmul_q8: too many rows");
    q8_rows_kernel<E, MT, NT, WAVES, DEPTH, OWN><<<dim3(uint32_t(cols), uint32_t(tall)), 64 * waves, 0, stream>>>(g);
    return ssm::hip_status_of_launch("matmul_q8");
}

// Weight tiles of a block: what the busiest CU loads for each step, rounds of blocks
// times rows of w and x, is least.  Measured, us with 1 / 2 / 4 tiles: one row of x,
// N x K 4096 x 4096 5.2 / 5.4 / 6.3, 8512 x 2048 6.2 / 6.5 / 5.5; 16 rows 16384 x
// 8192 27.6 / 29.1 / 25.0; 64 rows 4096 x 4096 6.9 / 7.8 / 10.7, 8192 x 4096 13.1 /
// 10.1 / 12.5, 16384 x 4096 25.7 / 20.7 / 18.6.  Four waves and two or three steps
// in the ring, whichever lets more blocks share a CU: eight waves or more steps
// were level or slower.
template <typename E, int MT, bool OWN = false>
int pick(const Q8Args& g, hipStream_t stream) {
    auto cost = [&](int nt) { return ceil_div(ceil_div(g.N, 16 * nt) * ceil_div(g.M, 16 * MT), cu_count()) * (nt + MT); };
    const int64_t one = cost(1), two = cost(2), four = cost(4);
    if (one <= two && one <= four) return run<E, MT, 1, MT == 4 ? 2 : 3, OWN>(g, stream);
    if (two <= four) return run<E, MT, 2, MT == 1 ? 3 : 2, OWN>(g, stream);
    return run<E, MT, 4, 2, OWN>(g, stream);
}

}  // namespace

// Against a launch of their own: 1 x 4096 x 4096 6.7 us against 8.2, 8 rows 8.8 against
// 8.8; but every block takes them again, and with N = 32768 one row takes 32.8 against
// 31.2, with 131072 110 against 98 (8 rows 100 and 100).
bool rows_take_own(int64_t m, int64_t k) {
    const int64_t steps = ceil_div(k, kStep);
    return m <= 16 && m * steps * kStep <= kOwnBytes / 4 * std::min<int64_t>(4, steps);
}

int rows_launch_own(int dtype, const Q8Args& g, hipStream_t stream) {
    return ssm::with_type(dtype, [&](auto e) { return pick<decltype(e), 1, true>(g, stream); });
}

int rows_launch(int y_dtype, const Q8Args& g, hipStream_t stream) {
    return ssm::with_type(y_dtype, [&](auto e) {
        using E = decltype(e);
        return g.M <= 16 ? pick<E, 1>(g, stream) : g.M <= 32 ? pick<E, 2>(g, stream) : pick<E, 4>(g, stream);
    });
}

}  // namespace q8
}  // namespace pe
