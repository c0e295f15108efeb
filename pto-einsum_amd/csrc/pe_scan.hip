// Entry points of the selective scan: checks, the choice of kernel, and the
// states at the starts of a sequence's pieces.
#include "pe_scan_chunk.h"

#include <algorithm>
#include <cmath>

namespace pe {
namespace ssm {
namespace {

int check(const pe_scan_desc* d, bool step, bool packed, const void* z) {
    if (!d) return fail(PE_ERR_INVALID, "selective_scan: null descriptor");
    if (!dtype_ok(d->dtype)) return fail(PE_ERR_UNSUPPORTED, "selective_scan: dtype must be PE_F32, PE_F16 or PE_BF16");
    if (d->dt_dtype != d->dtype && d->dt_dtype != PE_F32)
        return fail(PE_ERR_UNSUPPORTED, "selective_scan: dt must be of x's dtype or PE_F32");
    if (d->reserved != 0) return fail(PE_ERR_INVALID, "selective_scan: reserved field must be 0");
    if (d->nseq < 0 || d->H < 0 || d->P < 0 || d->N < 0 || (!step && d->T < 0) || (step && d->nslots < 0))
        return fail(PE_ERR_INVALID, "selective_scan: negative extent");
    if (d->G < 1 || d->H % d->G != 0) return fail(PE_ERR_INVALID, "selective_scan: H is no multiple of G");
    if (d->N > PE_SCAN_MAX_N)
        return fail(PE_ERR_UNSUPPORTED, "selective_scan: N above " + std::to_string(PE_SCAN_MAX_N));
    const int64_t big = int64_t(1) << 31;
    if (d->nseq >= big || d->H >= big || d->P >= big || (!step && d->T >= big))
        return fail(PE_ERR_UNSUPPORTED, "selective_scan: an extent of 2^31 or more");
    const int64_t T = step ? 1 : d->T, seqs = packed ? 1 : d->nseq;
    auto in = [&](int64_t bs, int64_t ts, int64_t hs, int64_t heads, int64_t inner, int64_t numel) {
        return within({{seqs, bs}, {T, ts}, {heads, hs}, {inner, 1}}, numel);
    };
    if (!in(d->x_bs, d->x_ts, d->x_hs, d->H, d->P, d->x_numel) ||
        (z && !in(d->z_bs, d->z_ts, d->z_hs, d->H, d->P, d->z_numel)) ||
        !in(d->dt_bs, d->dt_ts, d->dt_hs, d->H, 1, d->dt_numel) ||
        !in(d->b_bs, d->b_ts, d->b_gs, d->G, d->N, d->b_numel) ||
        !in(d->c_bs, d->c_ts, d->c_gs, d->G, d->N, d->c_numel))
        return fail(PE_ERR_BOUNDS, "selective_scan: strides address past an operand");
    return PE_OK;
}

ScanArgs arguments(const pe_scan_desc& d, const void* x, const void* dt, const float* A, const void* B, const void* C,
                   const float* D, const void* z, const float* dt_bias) {
    ScanArgs g{};
    g.x = x; g.dt = dt; g.A = A; g.B = B; g.C = C; g.D = D; g.z = z; g.dt_bias = dt_bias;
    g.x_bs = d.x_bs; g.x_ts = d.x_ts; g.x_hs = d.x_hs;
    g.z_bs = d.z_bs; g.z_ts = d.z_ts; g.z_hs = d.z_hs;
    g.dt_bs = d.dt_bs; g.dt_ts = d.dt_ts; g.dt_hs = d.dt_hs;
    g.b_bs = d.b_bs; g.b_ts = d.b_ts; g.b_gs = d.b_gs;
    g.c_bs = d.c_bs; g.c_ts = d.c_ts; g.c_gs = d.c_gs;
    g.nseq = int32_t(d.nseq); g.H = int32_t(d.H); g.P = int32_t(d.P); g.G = int32_t(d.G); g.N = int32_t(d.N);
    g.dt_f32 = d.dt_dtype == PE_F32;
    g.softplus = d.softplus;
    return g;
}

// How a prompt is run: token by token (rows), or in chunks.
struct Plan {
    bool chunks = false;
    int nt = 0, waves = 0;
    int64_t ptiles = 0, piece = 0, per_seq = 0, pieces = 0;
    int64_t state_floats = 0, decay_floats = 0;   // workspace
};

// Blocks of carry_kernel for a sequence and head.
constexpr int kCarryThreads = 256, kAhead = 8;
int64_t carry_blocks(const Plan& p) { return ceil_div(p.ptiles * p.waves * (p.nt / 16) * 64, kCarryThreads); }

auto chunks_of(int dtype) { return dtype == PE_F16 ? chunks_f16 : dtype == PE_BF16 ? chunks_bf16 : chunks_f32; }

Plan plan_of(const pe_scan_desc& d, bool packed) {
    Plan p;
    // Up to 16 tokens the recurrence is as quick; rows of less than eight
    // elements cannot be loaded as whole vectors.
    if (d.T <= 16 || d.N < 8 || d.P < 8) return p;
    // Offsets of rows within a chunk are 32 bits.
    for (const int64_t ts : {d.x_ts, d.z_ts, d.dt_ts, d.b_ts, d.c_ts, d.H * d.P})
        if (ts >= kScanStrideEnd) return p;
    p.chunks = true;
    p.nt = d.N <= 32 ? 32 : d.N <= 64 ? 64 : d.N <= 128 ? 128 : 256;
    // Tiles of up to 64 rows p, as even as waves of 16 allow.
    p.ptiles = ceil_div(d.P, 64);
    p.waves = int(std::max<int64_t>(p.nt == 256 ? 3 : 2, ceil_div(ceil_div(d.P, 16), p.ptiles)));
    // Pieces of a sequence (packed: of the whole buffer), of 64 tokens at least.
    // What a choice costs, in chunks of 32 tokens that a block walks: those of a
    // piece and one for its start, in as many rounds as the blocks need; with
    // several pieces half of that again for their contributions, 6 for the states
    // of 1000 blocks of 64 x 128, and 2 for two launches more.  Measured, us for 1, 2,
    // 4, 8, 16 pieces (chosen: *): 1 x 128 tokens, 32 heads 17* 20 20; 2 x 256, 16
    // heads 28 27 22* 25; 1 x 1024, 32 heads 105 76 47 39 38*; 2 x 4096, 64 heads 404
    // 270 182 179 184, 161 for 6*; 1 x 16384, 24 heads 1400 920 468 243 162, 121 for
    // 32* (64 x 128 a head, 16-bit types; float32 and other heads take the same
    // constants, of which only the hand-over's is scaled to their size).
    const int64_t seqs = packed ? 1 : d.nseq, across = d.H * p.ptiles, chunks = ceil_div(d.T, 32);
    const double slots = double(cu_count()) * chunks_of(d.dtype)(nullptr, p.nt, p.waves, true, nullptr);
    double best = 0.0;
    for (int64_t k = 1; k <= std::max<int64_t>(1, std::min<int64_t>(chunks / 2, 96)); ++k) {
        const int64_t piece = ceil_div(chunks, k);
        if (k > 1 && ceil_div(chunks, k - 1) == piece) continue;
        const double blocks = double(seqs) * double(across) * double(ceil_div(chunks, piece));
        double cost = std::ceil(blocks / slots) * double(piece + 1);
        if (k > 1) cost = 2.0 + 1.5 * cost + 0.006 * blocks * (p.waves * p.nt / 512.0);
        if (k == 1 || cost < best) {
            best = cost;
            p.piece = 32 * piece;
        }
    }
    p.per_seq = ceil_div(d.T, p.piece);
    p.pieces = packed ? p.per_seq + d.nseq : p.per_seq * d.nseq;
    // What passes a launch's threads goes token by token: so many sequences and
    // heads fill the card that way too.
    const __int128 most = (int64_t(1) << 32) - 1;
    const bool several = packed || p.per_seq > 1;
    if ((__int128(p.pieces) * across + kScanTailBlocks) * 64 * p.waves > most ||
        (several && __int128(d.nseq) * d.H * carry_blocks(p) * kCarryThreads > most))
        return Plan{};
    if (several) {
        p.decay_floats = ceil_div(p.pieces * d.H, 4) * 4;
        p.state_floats = p.pieces * d.H * p.ptiles * p.waves * (p.nt / 16) * 256;
    }
    return p;
}

// From the pieces' contributions to the states at their starts, in place, and
// the final states.  A thread follows four n of a row p through its sequence;
// the next kAhead contributions are on their way.
__global__ __launch_bounds__(kCarryThreads) void carry_kernel(ChunkArgs g, uint32_t vecs, uint32_t frags, uint32_t wave_rows,
                                                              uint32_t head_blocks) {
    const ScanArgs& a = g.s;
    const uint32_t sh = blockIdx.x / head_blocks, per_head = g.ptiles * vecs;
    const uint32_t at = (blockIdx.x - sh * head_blocks) * kCarryThreads + threadIdx.x;
    if (at >= per_head) return;
    const int s = int(sh / uint32_t(a.H)), h = int(sh - uint32_t(s) * uint32_t(a.H));
    const uint32_t pt = at / vecs, v = at - pt * vecs, lane = v & 63, frag = v >> 6;
    const uint32_t wave = frag / frags, i = frag - wave * frags;
    const int64_t p = int64_t(pt) * 16 * wave_rows + 16 * wave + (lane & 15), n = 16 * i + 4 * (lane >> 4);
    if (p - (lane & 15) >= a.P || int(16 * i) >= a.N) return;  // beside the state
    int64_t id, count;
    if (a.cu) {
        const int64_t from = offset_of(a.cu, s, a.T), to = offset_of(a.cu, s + 1, a.T);
        id = from / g.piece + s;
        count = to > from ? (to - 1) / g.piece + s - id + 1 : 0;
    } else {
        id = int64_t(s) * g.per_seq;
        count = g.per_seq;
    }
    const int64_t state_at = ((int64_t(s) * a.H + h) * a.P + p) * a.N + n;
    f32x4 S = {0, 0, 0, 0};
    if (a.state_in && p < a.P) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (n + k < a.N) S[k] = a.state_in[state_at + k];
    }
    const int64_t stride = int64_t(a.H) * per_head;
    f32x4* ws = reinterpret_cast<f32x4*>(g.ws_state) + (id * a.H + h) * per_head + at;
    const float* decay = g.ws_decay + id * a.H + h;
    // The last piece's contribution is its own block's.
    for (int64_t j = 0; j < count; j += kAhead) {
        f32x4 add[kAhead];
        float f[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int64_t u = min(j + k, max(count - 2, int64_t(0)));
            add[k] = ws[u * stride];
            f[k] = decay[u * a.H];
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (j + k < count) ws[(j + k) * stride] = S;
#pragma unroll
            for (int e = 0; e < 4; ++e) S[e] = __builtin_fmaf(f[k], S[e], add[k][e]);
        }
    }
    if (count == 0 && a.state_out && p < a.P) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (n + k < a.N) a.state_out[state_at + k] = S[k];
    }
}

int launch_plan(const pe_scan_desc& d, const Plan& p, const ScanArgs& a, void* ws, hipStream_t stream) {
    ChunkArgs g{};
    g.s = a;
    g.piece = uint32_t(p.piece); g.pieces = uint32_t(p.pieces); g.per_seq = uint32_t(p.per_seq);
    g.ptiles = uint32_t(p.ptiles); g.blocks = uint32_t(p.pieces * d.H * p.ptiles);
    g.state4 = a.N % 4 == 0 && aligned(a.state_in, 16) && aligned(a.state_out, 16);
    if (p.state_floats) {
        g.ws_decay = static_cast<float*>(ws);
        g.ws_state = g.ws_decay + p.decay_floats;
    }
    const auto run = chunks_of(d.dtype);
    if (p.state_floats) {
        run(&g, p.nt, p.waves, false, stream);
        const uint32_t frags = uint32_t(p.nt / 16), vecs = uint32_t(p.waves) * frags * 64;
        const uint32_t head_blocks = uint32_t(carry_blocks(p));
        carry_kernel<<<uint32_t(d.nseq * d.H) * head_blocks, kCarryThreads, 0, stream>>>(g, vecs, frags,
                                                                                         uint32_t(p.waves), head_blocks);
    }
    run(&g, p.nt, p.waves, true, stream);
    return hip_status_of_launch("selective_scan");
}

}  // namespace
}  // namespace ssm
}  // namespace pe

using namespace pe;
using namespace pe::ssm;

extern "C" int64_t pe_selective_scan_workspace_bytes(const pe_scan_desc* d, int packed) {
    if (check(d, false, packed != 0, nullptr) != PE_OK || d->nseq == 0 || d->H == 0 || d->P == 0) return 0;
    const Plan p = plan_of(*d, packed != 0);
    return 4 * (p.state_floats + p.decay_floats);
}

extern "C" int pe_selective_scan(const pe_scan_desc* d, const void* x, const void* dt, const float* A, const void* B,
                                 const void* C, const float* D, const void* z, const float* dt_bias,
                                 const float* state_in, const int32_t* cu, void* y, float* state_out, void* ws,
                                 int64_t ws_bytes, void* stream) {
    if (int rc = check(d, false, cu != nullptr, z)) return rc;
    if (cu && d->nseq < 1) return fail(PE_ERR_INVALID, "selective_scan: packed tokens without a sequence");
    if (d->nseq == 0 || d->H == 0 || d->P == 0) return PE_OK;
    if (!A || (d->T > 0 && (!x || !dt || !y || (d->N > 0 && (!B || !C)))))
        return fail(PE_ERR_INVALID, "selective_scan: null pointer");
    const Plan p = plan_of(*d, cu != nullptr);
    const int64_t need = 4 * (p.state_floats + p.decay_floats);
    if (need && (!ws || ws_bytes < need || !aligned(ws, 16)))
        return fail(PE_ERR_WORKSPACE, "selective_scan: workspace missing, misaligned or too small");
    ScanArgs g = arguments(*d, x, dt, A, B, C, D, z, dt_bias);
    g.cu = cu; g.T = d->T; g.y = y; g.state_in = state_in; g.state_out = state_out;
    g.nslots = d->nseq;
    auto s = static_cast<hipStream_t>(stream);
    return p.chunks ? launch_plan(*d, p, g, ws, s) : launch_rows(d->dtype, g, s);
}

extern "C" int pe_selective_scan_step(const pe_scan_desc* d, const void* x, const void* dt, const float* A,
                                      const void* B, const void* C, const float* D, const void* z,
                                      const float* dt_bias, float* state, const int32_t* slots, void* y,
                                      void* stream) {
    if (int rc = check(d, true, false, z)) return rc;
    if (d->nseq == 0 || d->H == 0 || d->P == 0) return PE_OK;
    if (!A || !x || !dt || !y || (d->N > 0 && (!B || !C || !state)))
        return fail(PE_ERR_INVALID, "selective_scan_step: null pointer");
    if (!slots && d->nslots < d->nseq) return fail(PE_ERR_BOUNDS, "selective_scan_step: fewer states than rows");
    ScanArgs g = arguments(*d, x, dt, A, B, C, D, z, dt_bias);
    g.T = 1; g.y = y; g.state_in = state; g.state_out = state; g.slots = slots;
    g.nslots = d->nslots;
    return launch_rows(d->dtype, g, static_cast<hipStream_t>(stream));
}
