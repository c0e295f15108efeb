// Products of rows in 8 bits: tiles through LDS (pe_q8.h).
#include "pe_q8.h"

#include <algorithm>

namespace pe {
namespace q8 {
namespace {

constexpr int kSlab = 64;             // bytes of k of a slab
constexpr int kStages = 4;

// 16-byte group g of row r of a slab lies in slot g ^ swz(r): the 16 rows by four
// groups of one fragment read then fall on different banks.
__device__ __forceinline__ int swz(int r) { return (r >> 1) & 3; }

__device__ __forceinline__ void load_lds(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 : : "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}

template <typename E, int BM, int BN>
__global__ __launch_bounds__(256) void q8_tile_kernel(Q8Args g) {
    constexpr int FM = BM / 32, FN = BN / 32;          // 16-wide blocks of a wave's tile (2 x 2 waves)
    constexpr int STAGE = (BM + BN) * kSlab, NI = (BM + BN) / 64;
    __shared__ __attribute__((aligned(1024))) int8_t lds[kStages * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) int8_t*)lds));
    const int tm = int(blockIdx.x) / g.tiles_n, tn = int(blockIdx.x) - tm * g.tiles_n;
    const int m0 = tm * BM, n0 = tn * BN;
    const int first = int(blockIdx.y) * g.split_slabs;
    const int total = (g.K + kSlab - 1) / kSlab;
    const int count = min(g.split_slabs, total - first);
    const int tail = g.K - (total - 1) * kSlab;          // bytes of the last slab
    const int8_t* xb = g.x + int64_t(m0) * g.x_ms + int64_t(first) * kSlab;
    const int8_t* wb = g.w + int64_t(n0) * g.w_ns + int64_t(first) * kSlab;

    // This lane's place in each of the wave's chunks of 16 rows: rows past the
    // end are the last one again (their sums are not stored).
    uint32_t off[NI];
    int grp[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int r = (i * 4 + wave) * 16 + lane / 4;
        const bool isx = r < BM;
        const int row = isx ? min(r, g.M - 1 - m0) : min(r - BM, g.N - 1 - n0);
        grp[i] = (lane & 3) ^ swz(r);
        off[i] = uint32_t(row) * uint32_t(isx ? g.x_ms : g.w_ns);
    }
    auto issue = [&](int s) {
        const bool last = first + s == total - 1;
        const uint32_t stage = lds0 + uint32_t(s % kStages) * STAGE;
        // The last slab's groups past the row are its last one again; the product
        // reads zeros for x there.
        const int most = last ? (tail - 1) / 16 : 3;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = i * 4 + wave;
            const int8_t* base = (c * 16 < BM ? xb : wb) + int64_t(s) * kSlab;
            load_lds(base, off[i] + uint32_t(16 * min(grp[i], most)), stage + uint32_t(c) * 1024u);
        }
    };

    i32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

    const int ahead = min(kStages - 1, count);
    for (int s = 0; s < ahead; ++s) issue(s);
    const int fr = lane & 15;
    const uint32_t fo = uint32_t(fr * kSlab + 16 * ((lane >> 4) ^ swz(fr)));
    for (int s = 0; s < count; ++s) {
        // Loads come back in their order: all but the later slabs' have to be there.
        if (count - 1 - s >= kStages - 2) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"((kStages - 2) * NI) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        int8_t* st = lds + (s % kStages) * STAGE;
        if (first + s == total - 1 && tail < kSlab) {
            for (int i = tid; i < BM * 4; i += 256) {
                const int r = i >> 2, k = 16 * ((i & 3) ^ swz(r));
                if (k + 16 > tail)
                    for (int b = max(0, tail - k); b < 16; ++b) st[r * kSlab + 16 * (i & 3) + b] = 0;
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        if (s + kStages - 1 < count) issue(s + kStages - 1);
        const uint32_t base = lds0 + uint32_t(s % kStages) * STAGE + fo;
        i32x4 a[FN], b[FM];
        auto read = [&](int row) {
            return *reinterpret_cast<const __attribute__((address_space(3))) i32x4*>(uintptr_t(base + uint32_t(row) * kSlab));
        };
#pragma unroll
        for (int i = 0; i < FN; ++i) a[i] = read(BM + wn * (BN / 2) + 16 * i);
#pragma unroll
        for (int j = 0; j < FM; ++j) b[j] = read(wm * (BM / 2) + 16 * j);
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FM; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i], b[j], acc[i][j], 0, 0, 0);
    }

    // Lane l holds columns 4 (l / 16) .. + 3 of a block, row l % 16.
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int n = n0 + wn * (BN / 2) + 16 * i + 4 * (lane >> 4), m = m0 + wm * (BM / 2) + 16 * j + fr;
            if (m >= g.M || n >= g.N) continue;
            if (g.splits > 1) {
                int32_t* p = g.part + (int64_t(blockIdx.y) * g.M + m) * g.N + n;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n + r < g.N) p[r] = acc[i][j][r];
            } else {
                finish<E>(g, m, n, acc[i][j]);
            }
        }
}

// Sum of the K splits' parts, four columns a lane.
template <typename E>
__global__ __launch_bounds__(256) void q8_join_kernel(Q8Args g) {
    const int cols = (g.N + 3) / 4;
    const int64_t items = int64_t(cols) * g.M;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < items; i += int64_t(gridDim.x) * 256) {
        const int m = int(i / cols), n = 4 * int(i - int64_t(m) * cols);
        i32x4 sum = {0, 0, 0, 0};
        for (int s = 0; s < g.splits; ++s) {
            const int32_t* p = g.part + (int64_t(s) * g.M + m) * g.N + n;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n + r < g.N) sum[r] += p[r];
        }
        finish<E>(g, m, n, sum);
    }
}

template <typename E, int BM, int BN>
int run(Q8Args& g, hipStream_t stream) {
    const int64_t tm = ceil_div(g.M, BM), tn = ceil_div(g.N, BN);
    if (tm * tn > (int64_t(1) << 23)) return fail(PE_ERR_UNSUPPORTED, "matmul_q8: too many tiles");
    g.tiles_m = int32_t(tm);
    g.tiles_n = int32_t(tn);
    g.splits = 1;
    g.split_slabs = int32_t(ceil_div(g.K, kSlab));
    q8_tile_kernel<E, BM, BN><<<dim3(uint32_t(tm * tn), uint32_t(g.splits)), 256, 0, stream>>>(g);
    return ssm::hip_status_of_launch("matmul_q8");
}

template <typename E>
int pick(Q8Args& g, hipStream_t stream) {
    if (ceil_div(g.M, 128) * ceil_div(g.N, 128) >= 2 * cu_count()) return run<E, 128, 128>(g, stream);
    return run<E, 64, 64>(g, stream);
}

}  // namespace

int tile_launch(int y_dtype, Q8Args& g, hipStream_t stream) {
    return ssm::with_type(y_dtype, [&](auto e) { return pick<decltype(e)>(g, stream); });
}

}  // namespace q8
}  // namespace pe
