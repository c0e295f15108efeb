// Products of rows in 8 bits: tiles through LDS (pe_q8.h).
//
// Four waves (2 x 2) share a tile.  K walks in slabs of 64 bytes through a ring of LDS
// stages that direct loads fill; while a slab is multiplied, the next one's fragments
// are read into a second set of registers and the one STAGES - 1 ahead is loaded, one
// read or load at a time between the products.  Of 8192^3 the matrix cores are 58 % busy
// at about 1.8 GHz, 2.4 POPS (the library's int8 product 2.1); a 256 x 256 tile leaves
// one wave a SIMD, with a barrier for each slab, and which wait takes the rest has not
// been measured.  A wave's tile of 128 x 128 reads 16 KB of LDS for 64 products of 16
// cycles, half of what LDS delivers, one of 64 x 64 all of it.  A tile's start and end
// (12 us of a 256 x 256 one, half of it the stores of all CUs at once) bounds products
// of short K.
#include "pe_q8.h"

#include <algorithm>

namespace pe {
namespace q8 {
namespace {

constexpr int kSlab = 64;             // bytes of k of a slab

// 16-byte group g of row r of a slab lies in slot g ^ swz(r): the 16 rows by four
// groups of one fragment read then fall on different banks.
__device__ __forceinline__ int swz(int r) { return (r >> 1) & 3; }

__device__ __forceinline__ void load_lds(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 : : "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}

// Tile of a block of the grid: consecutive tiles of an XCD (blocks go round robin
// to the eight) lie in groups of kGroup tile rows, column by column, so that its L2
// holds the rows of x and w that they share.
constexpr int kGroup = 4;
__device__ __forceinline__ void place(uint32_t b, uint32_t tiles, uint32_t tiles_m, uint32_t tiles_n, int& tm, int& tn) {
    const uint32_t each = tiles / 8, rest = tiles % 8, xcd = b % 8;
    const uint32_t t = xcd * each + min(xcd, rest) + b / 8;
    const uint32_t group = t / (kGroup * tiles_n), in = t - group * kGroup * tiles_n;
    const uint32_t high = min(tiles_m - group * kGroup, uint32_t(kGroup));
    tn = int(in / high);
    tm = int(group * kGroup + in - uint32_t(tn) * high);
}

template <typename E, int BM, int BN, int STAGES, int MINB>
__global__ __launch_bounds__(256, MINB) void q8_tile_kernel(Q8Args g) {
    constexpr int FM = BM / 32, FN = BN / 32;          // 16-wide blocks of a wave's tile (2 x 2 waves)
    constexpr int STAGE = (BM + BN) * kSlab, NI = (BM + BN) / 64;
    constexpr int AHEAD = STAGES - 1;                  // slabs issued before the one multiplied
    __shared__ __attribute__((aligned(1024))) int8_t lds[STAGES * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) int8_t*)lds));
    int tm, tn;
    place(blockIdx.x, gridDim.x, g.tiles_m, g.tiles_n, tm, tn);
    const int m0 = __builtin_amdgcn_readfirstlane(tm) * BM, n0 = __builtin_amdgcn_readfirstlane(tn) * BN;
    const int count = (g.K + kSlab - 1) / kSlab;
    const int tail = g.K - (count - 1) * kSlab;          // bytes of the last slab
    const int tail_at = tail < kSlab ? count - 1 : count;
    const int8_t* xb = g.x + int64_t(m0) * g.x_ms;
    const int8_t* wb = g.w + int64_t(n0) * g.w_ns;

    // This lane's row in each of the wave's chunks of 16 rows (rows past the end are
    // the last one again: their sums are not stored) and its group of 16 bytes.
    uint32_t off[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int r = (i * 4 + wave) * 16 + lane / 4;
        const bool isx = r < BM;
        const int row = isx ? min(r, g.M - 1 - m0) : min(r - BM, g.N - 1 - n0);
        off[i] = uint32_t(row) * uint32_t(isx ? g.x_ms : g.w_ns);
    }
    const uint32_t grp = 16u * ((lane & 3) ^ swz(lane / 4));
    // Load side: slabs go out in order; past the last one it is loaded again, into a
    // stage that nothing reads any more, so that the number in flight stays known
    // and the loop has no branch.
    int ls = 0;
    uint32_t lstage = lds0, koff;
    auto aim = [&] {
        // (the last slab's groups past the row are its last one again; the product
        // finds zeros for x there)
        koff = ls == tail_at ? min(grp, uint32_t((tail - 1) / 16 * 16)) : grp;
    };
    auto load1 = [&](int i) {
        const int c = i * 4 + wave;
        load_lds(c * 16 < BM ? xb : wb, off[i] + koff, lstage + uint32_t(c) * 1024u);
    };
    auto next_load = [&] {
        if (ls + 1 < count) {
            ++ls;
            xb += kSlab;
            wb += kSlab;
        }
        lstage += STAGE;
        if (lstage == lds0 + STAGES * STAGE) lstage = lds0;
        aim();
    };

    i32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

    // Zeros for x behind K in the slab at `stage` if it has a tail.
    auto clear_tail = [&](int slab, uint32_t stage) {
        if (__builtin_expect(slab != tail_at, 1)) return;
        int8_t* st = lds + (stage - lds0);
        for (int i = tid; i < BM * 4; i += 256) {
            const int r = i >> 2, k = 16 * ((i & 3) ^ swz(r));
            for (int b = max(0, tail - k); b < 16; ++b) st[r * kSlab + 16 * (i & 3) + b] = 0;
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };

    const int fr = lane & 15;
    const uint32_t fo = uint32_t(fr * kSlab + 16 * ((lane >> 4) ^ swz(fr)));
    const uint32_t foa = fo + uint32_t(BM + wn * (BN / 2)) * kSlab, fob = fo + uint32_t(wm * (BM / 2)) * kSlab;
    auto read = [&](uint32_t at, int i) {
        return *reinterpret_cast<const __attribute__((address_space(3))) i32x4*>(uintptr_t(at + uint32_t(16 * i) * kSlab));
    };
    // Fragment u in the order in which the products take them.
    auto fragment = [&](i32x4 (&a)[FN], i32x4 (&b)[FM], uint32_t stage, int u) {
        if (u == 0) a[0] = read(stage + foa, 0);
        else if (u <= FM) b[u - 1] = read(stage + fob, u - 1);
        else a[u - FM] = read(stage + foa, u - FM);
    };

    if (count > 0) {
        aim();
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) {
#pragma unroll
            for (int i = 0; i < NI; ++i) load1(i);
            next_load();
        }
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"((AHEAD - 1) * NI) : "memory");
        clear_tail(0, lds0);
        i32x4 xa[FN], xb_[FM], ya[FN], yb[FM];
        uint32_t cstage = lds0;
#pragma unroll
        for (int u = 0; u < FN + FM; ++u) fragment(xa, xb_, cstage, u);
        // Slab s from its fragments, while the next one's are read and the one
        // AHEAD of it is loaded into the stage that slab s - 1 had.
        auto slab = [&](const i32x4 (&ca)[FN], const i32x4 (&cb)[FM], i32x4 (&na)[FN], i32x4 (&nb)[FM], int s) {
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"((AHEAD - 2) * NI) : "memory");
            cstage += STAGE;
            if (cstage == lds0 + STAGES * STAGE) cstage = lds0;
            clear_tail(s + 1, cstage);
            constexpr int T = FM * FN, RD = FM + FN;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < T; ++t) {
                acc[t / FM][t % FM] = __builtin_amdgcn_mfma_i32_16x16x64_i8(ca[t / FM], cb[t % FM], acc[t / FM][t % FM], 0, 0, 0);
                if ((t + 1) * RD / T != t * RD / T) fragment(na, nb, cstage, t * RD / T);
                if ((t + 1) * NI / T != t * NI / T) load1(t * NI / T);
                __builtin_amdgcn_sched_barrier(0);
            }
            next_load();
        };
        // Slabs in pairs, so that each register set keeps its role, behind an odd one.
        int s = count & 1;
        if (s) {
            slab(xa, xb_, ya, yb, 0);
#pragma unroll
            for (int i = 0; i < FN; ++i) xa[i] = ya[i];
#pragma unroll
            for (int j = 0; j < FM; ++j) xb_[j] = yb[j];
        }
        for (; s < count; s += 2) {
            slab(xa, xb_, ya, yb, s);
            slab(ya, yb, xa, xb_, s + 1);
        }
        // (no load may still be on its way to LDS when the block ends)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }

    // (The lane's number anew: the loop above has a register for nothing else.)
    const int lane_out = int(__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u))), row_out = lane_out & 15;
    // Lane l holds columns 4 (l / 16) .. + 3 of a block, row l % 16.
    const int nl = n0 + wn * (BN / 2) + 4 * (lane_out >> 4);
    // The sums lie four columns a lane, which would store 8 bytes of 16 rows at a time
    // (8192 x 8192 in 16 bits took 60 to 100 us that way, for 21 us of writing), so
    // each 16 rows of the wave's tile go through LDS of the wave's own and out in
    // whole 16-byte vectors along the rows, two such places in turn.
    using V = typename ssm::Vec<E, 16 / E::kBytes>;
    constexpr int WN = BN / 2, PITCH = WN * E::kBytes + 16, VPR = WN * E::kBytes / 16;
    static_assert(2 * 4 * 16 * PITCH <= STAGES * STAGE, "the output rows of four waves fit the ring twice");
    asm volatile("s_barrier" ::: "memory");
    Column c[FN];
#pragma unroll
    for (int i = 0; i < FN; ++i) c[i] = column<E>(g, nl + 16 * i);
    float sx[FM];
    bool far = false;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        sx[j] = g.xs[min(m0 + wm * (BM / 2) + 16 * j + row_out, g.M - 1)];
        far = far || large(sx[j]);
    }
    auto out = [&](auto value_of) {
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int m = m0 + wm * (BM / 2) + 16 * j;
            int8_t* mine = lds + (2 * wave + (j & 1)) * 16 * PITCH;
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                typename ssm::Vec<E, 4>::type v;
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = (typename E::T)value_of(c[i], sx[j], r, acc[i][j][r]);
                *reinterpret_cast<typename ssm::Vec<E, 4>::type*>(mine + row_out * PITCH + (16 * i + 4 * (lane_out >> 4)) * E::kBytes) = v;
            }
            ssm::wave_sync();
#pragma unroll
            for (int u = 0; u < 16 * VPR / 64; ++u) {
                const int row = (u * 64 + lane_out) / VPR, at = (u * 64 + lane_out) % VPR;
                const typename V::type v = *reinterpret_cast<const typename V::type*>(mine + row * PITCH + 16 * at);
                const int n = n0 + wn * WN + at * (16 / E::kBytes);
                if (m + row < g.M && n < g.N) {
                    typename E::T* y = static_cast<typename E::T*>(g.y) + int64_t(m + row) * g.N + n;
                    if (n + 16 / E::kBytes <= g.N) {
                        *reinterpret_cast<typename V::utype*>(y) = v;
                    } else {
#pragma unroll
                        for (int e = 0; e < 16 / E::kBytes; ++e)
                            if (n + e < g.N) y[e] = v[e];
                    }
                }
            }
        }
    };
    if (__builtin_expect(__any(far), 0)) out(value_of_large);
    else out(value);
}

constexpr int64_t kMostTiles = (int64_t(1) << 24) - 1;   // blocks of 256 threads in fewer than 2^32

template <typename E, int BM, int BN, int STAGES, int MINB>
int run(const Q8Args& args, hipStream_t stream) {
    Q8Args g = args;
    const int64_t tm = ceil_div(g.M, BM), tn = ceil_div(g.N, BN);
    if (tm * tn > kMostTiles) return fail(PE_ERR_UNSUPPORTED, "matmul_q8: too many tiles");
    g.tiles_m = int32_t(tm);
    g.tiles_n = int32_t(tn);
    q8_tile_kernel<E, BM, BN, STAGES, MINB><<<uint32_t(tm * tn), 256, 0, stream>>>(g);
    return ssm::hip_status_of_launch("matmul_q8");
}

// The tile: rounds of blocks times their start and end, and slabs times what the
// busiest CU takes for each, from fits to 8192 x 8192 x (64 to 8192) and, of the
// small tiles, to few blocks a CU (us).  A CU with fewer blocks than it holds takes a
// slab's latency at least.  Measured, us, in the order below: 8192^3 452 / 526 / 536 /
// 640 / 649 / 880 / 1090; 4096 x 8512 x 2048 100 / 87 / 94 / 93 / 96 / 127 / 152; 512 x
// 8192 x 8192 97 / 82 / 102 / 77 / 58 / 72 / 88; 1000 x 2048 x 2048 12.0 with the last two,
// 17.9 and 13.9 with those of 128 x 128.
struct Tile {
    int bm, bn, blocks;               // blocks that share a CU
    float fixed, latency, slab;
};
constexpr Tile kTiles[kTileKernels] = {
    {256, 256, 1, 12.0f, 0.79f, 0.79f},
    {256, 192, 1, 9.0f, 0.61f, 0.61f},
    {128, 256, 2, 8.0f, 0.65f, 0.49f},
    {128, 128, 3, 5.0f, 0.56f, 0.30f},
    {128, 128, 2, 4.5f, 0.43f, 0.30f},
    {64, 128, 3, 4.0f, 0.27f, 0.27f},
    {64, 64, 5, 3.5f, 0.24f, 0.17f},
};

template <typename E>
int pick(const Q8Args& g, int kernel, hipStream_t stream) {
    int best = 0;
    float least = 0.0f;
    for (int i = 0; i < kTileKernels; ++i) {
        const Tile& t = kTiles[i];
        const int64_t tiles = ceil_div(g.M, t.bm) * ceil_div(g.N, t.bn);
        const int64_t each = ceil_div(tiles, cu_count()), rounds = ceil_div(each, t.blocks);
        const float us = float(rounds) * t.fixed + float(ceil_div(g.K, kSlab)) * std::max(float(rounds) * t.latency, float(each) * t.slab);
        if (i == 0 || (us < least && tiles <= kMostTiles)) {
            best = i;
            least = us;
        }
    }
    switch (kernel ? kernel - 2 : best) {
        case 0: return run<E, 256, 256, 4, 1>(g, stream);
        case 1: return run<E, 256, 192, 4, 1>(g, stream);
        case 2: return run<E, 128, 256, 3, 2>(g, stream);
        case 3: return run<E, 128, 128, 3, 3>(g, stream);
        case 4: return run<E, 128, 128, 4, 2>(g, stream);
        case 5: return run<E, 64, 128, 4, 2>(g, stream);
        default: return run<E, 64, 64, 4, 2>(g, stream);
    }
}

}  // namespace

int tile_launch(int y_dtype, const Q8Args& g, int kernel, hipStream_t stream) {
    return ssm::with_type(y_dtype, [&](auto e) { return pick<decltype(e)>(g, kernel, stream); });
}

}  // namespace q8
}  // namespace pe
