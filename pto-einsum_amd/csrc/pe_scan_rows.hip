// Selective scan token by token: the recurrence itself, for single tokens
// (state in the cache's slots) and for prompts of up to 16 tokens (and any whose
// rows or strides the chunks do not take).
//
//   S[p, n] = exp(A d) S[p, n] + d x[p] B[n],    y[p] = sum_n C[n] S[p, n] + D x[p]
//
// A single token reads and writes its states and little else, 8 bytes for 5
// flops: HBM bounds it.  A row p of the state lies across LPR lanes, 4 n (16
// bytes) each; a wave holds R x 64 / LPR rows, so a lane has R loads in flight
// and B, C serve R rows.  The R sums over n are reduced together: log2 R halving
// exchanges, each lane keeping half the rows it held, then butterflies.
//
// One token of 128 sequences, 64 heads of 64 x 128: 537 MB of states read and
// written in 106 us, 5.1 TB/s (a large copy moves 5.1 to 6.5 here).  Of one
// sequence, 32 heads: 6.6 to 7 us, of a call of 13.
#include "pe_scan.h"

namespace pe {
namespace ssm {
namespace {

constexpr int kThreads = 256;
constexpr int kTailBlocks = 64;

// N4: rows of N = 4 k elements, 16-byte accesses; else element by element.  NT:
// streaming loads and stores of the states (launch()).
template <typename E, int LPR, int R, bool N4, bool NT>
__global__ __launch_bounds__(kThreads) void rows_kernel(ScanArgs g, uint32_t tiles, uint32_t main_blocks) {
    using T = typename E::T;
    constexpr int G = 64 / LPR, TR = G * R;
    if (blockIdx.x >= main_blocks) {
        clear_outside<E>(g, int64_t(blockIdx.x - main_blocks) * kThreads + threadIdx.x, kTailBlocks * kThreads);
        return;
    }
    const int lane = threadIdx.x & 63, l = lane % LPR, grp = lane / LPR;
    const uint32_t wave = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t sh = wave / tiles;
    const int s = int(sh / uint32_t(g.H)), h = int(sh - uint32_t(s) * uint32_t(g.H));
    if (s >= g.nseq) return;
    const int p0 = int(wave - sh * tiles) * TR;
    const int group = h / (g.H / g.G);

    int64_t slot = s, t0 = 0, t1 = g.T;
    if (g.slots) {
        slot = g.slots[s];
        t1 = 1;
    } else if (g.cu) {
        t0 = offset_of(g.cu, s, g.T);
        t1 = offset_of(g.cu, s + 1, g.T);
    }
    const int64_t seq = g.cu ? 0 : s;
    T* y = static_cast<T*>(g.y) + (g.cu ? 0 : int64_t(s) * g.T * g.H * g.P) + int64_t(h) * g.P;
    // The row whose sum a lane ends up with, and whether it stores it.
    int r_of = 0;
    bool keeper = true;
    {
        int cnt = R;
#pragma unroll
        for (int m = LPR / 2; m >= 1; m /= 2) {
            if (cnt > 1) {
                if (l & m) r_of += cnt / 2;
                cnt /= 2;
            } else if (l & m) keeper = false;
        }
    }
    const int p_of = p0 + r_of * G + grp;
    if (slot < 0 || slot >= g.nslots) {  // a row without a sequence
        if (keeper && p_of < g.P) y[p_of] = T(0.0f);
        return;
    }

    const int n0 = l * 4;
    const int64_t state_at = (slot * g.H + h) * g.P * int64_t(g.N);
    float st[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int p = p0 + r * G + grp;
#pragma unroll
        for (int i = 0; i < 4; ++i) st[r][i] = 0.0f;
        if (g.state_in && p < g.P && n0 < g.N) {
            const float* sp = g.state_in + state_at + int64_t(p) * g.N + n0;
            if (N4) {
                const f32x4* q = reinterpret_cast<const f32x4*>(sp);
                const f32x4 v = NT ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
                for (int i = 0; i < 4; ++i) st[r][i] = v[i];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n0 + i < g.N) st[r][i] = sp[i];
            }
        }
    }
    // Lanes past N keep a state of 0: an infinite x times their B of 0 would be NaN.
    const bool mine = n0 < g.N;
    const float A = g.A[h], bias = g.dt_bias ? g.dt_bias[h] : 0.0f, skip = g.D ? g.D[h] : 0.0f;
    for (int64_t t = t0; t < t1; ++t) {
        const float step = step_size(g, dt_of<E>(g, dt_bits<E>(g, g.dt, seq * g.dt_bs + t * g.dt_ts + h * g.dt_hs)), bias);
        const float d = mine ? step : 0.0f, a = mine ? expf(A * step) : 0.0f;
        float b[4], c[4];
        const int left = g.N - n0;
        load_f32<E, 4>(static_cast<const T*>(g.B) + seq * g.b_bs + t * g.b_ts + group * g.b_gs + n0, left, b);
        load_f32<E, 4>(static_cast<const T*>(g.C) + seq * g.c_bs + t * g.c_ts + group * g.c_gs + n0, left, c);
        const T* x = static_cast<const T*>(g.x) + seq * g.x_bs + t * g.x_ts + h * g.x_hs;
        float sum[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int p = p0 + r * G + grp;
            const float dx = d * (p < g.P && mine ? E::to_f32(x[p]) : 0.0f);
            float v = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                st[r][i] = N4 || i < left ? __builtin_fmaf(a, st[r][i], dx * b[i]) : 0.0f;
                v = __builtin_fmaf(c[i], st[r][i], v);
            }
            sum[r] = v;
        }
        int cnt = R;
#pragma unroll
        for (int m = LPR / 2; m >= 1; m /= 2) {
            if (cnt > 1) {
                cnt /= 2;
#pragma unroll
                for (int i = 0; i < R / 2; ++i)
                    if (i < cnt) {
                        const float keep = (l & m) ? sum[i + cnt] : sum[i], give = (l & m) ? sum[i] : sum[i + cnt];
                        sum[i] = keep + __shfl_xor(give, m);
                    }
            } else {
                sum[0] += __shfl_xor(sum[0], m);
            }
        }
        if (keeper && p_of < g.P) {
            float v = __builtin_fmaf(skip, E::to_f32(x[p_of]), sum[0]);
            if (g.z)
                v *= silu(E::to_f32(static_cast<const T*>(g.z)[seq * g.z_bs + t * g.z_ts + h * g.z_hs + p_of]));
            y[t * g.H * g.P + p_of] = T(v);
        }
    }
    if (!g.state_out) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int p = p0 + r * G + grp;
        if (p < g.P && n0 < g.N) {
            float* sp = g.state_out + state_at + int64_t(p) * g.N + n0;
            if (N4) {
                f32x4 v;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = st[r][i];
                if constexpr (NT) store_nt(reinterpret_cast<f32x4*>(sp), v);
                else *reinterpret_cast<f32x4*>(sp) = v;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n0 + i < g.N) sp[i] = st[r][i];
            }
        }
    }
}

template <typename E, int LPR, int R>
int launch(const ScanArgs& g, hipStream_t stream) {
    constexpr int TR = 64 / LPR * R;
    const uint32_t tiles = uint32_t(ceil_div(g.P, TR));
    const __int128 waves = __int128(g.nseq) * g.H * tiles;
    // Fewer than 2^32 threads.
    if (waves >= (1 << 26) - 4 * kTailBlocks) return fail(PE_ERR_UNSUPPORTED, "selective_scan: too many rows");
    const uint32_t blocks = uint32_t(ceil_div(int64_t(waves), kThreads / 64));
    const uint32_t all = blocks + (g.cu ? kTailBlocks : 0);
    // States of 32 MB and more pass the caches by: with states of several calls in
    // turn, us ordinary / streaming: 34 MB 16.6 / 15.3, 67 MB 33 / 30, 134 MB 68 / 60,
    // 268 MB 124 / 110 (4.9 TB/s), 537 MB 231 / 213.
    const bool nt = 4 * int64_t(g.nseq) * g.H * g.P * g.N >= PE_NT_MIN_BYTES;
    if (!(g.N % 4 == 0 && aligned(g.state_in, 16) && aligned(g.state_out, 16)))
        rows_kernel<E, LPR, R, false, false><<<all, kThreads, 0, stream>>>(g, tiles, blocks);
    else if (nt)
        rows_kernel<E, LPR, R, true, true><<<all, kThreads, 0, stream>>>(g, tiles, blocks);
    else
        rows_kernel<E, LPR, R, true, false><<<all, kThreads, 0, stream>>>(g, tiles, blocks);
    return hip_status_of_launch("selective_scan");
}

}  // namespace

int launch_rows(int dtype, const ScanArgs& g, hipStream_t stream) {
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        if (g.N <= 16) return launch<E, 4, 4>(g, stream);
        if (g.N <= 32) return launch<E, 8, 8>(g, stream);
        if (g.N <= 64) return launch<E, 16, 8>(g, stream);
        if (g.N <= 128) return launch<E, 32, 8>(g, stream);
        return launch<E, 64, 8>(g, stream);
    });
}

}  // namespace ssm
}  // namespace pe
