// Short causal convolution of each channel (depthwise, width 2 to 8) with bias
// and activation, for prompts and for single tokens.
//
//   y[t, d] = act(bias[d] + sum_{j < W} w[d, j] x[t - W + 1 + j, d])
//
// Reading x and writing y bound it: 2 W flops for two elements moved.  A thread
// owns V channels (16 bytes) and walks a run of consecutive tokens with the
// last W - 1 inputs in registers, so x is read once but for W - 1 tokens at the
// run's start.  A group of tokens is loaded while the one before is worked on.
// Sums are float32 in the order of j after the bias; the output is rounded once.
//
// Four prompts of 4096 x 4352 float16: 65 us a call, 4.4 TB/s (without the loads
// ahead and with the library's exp and divide 142); 3993 x 1283 bfloat16 in packed
// prompts 13 us; one token of 64 x 4352 4 us of a call of 10.5.  Stores that pass
// the caches by made the large call 62 us back to back but 82 instead of 76 alone.
#include "pe_ssm.h"

#include <algorithm>

namespace pe {
namespace ssm {
namespace {

constexpr int kThreads = 256;

struct ConvArgs {
    const void *x, *w, *bias, *state_in;
    const int32_t* cu;
    void *y, *state_out;
    int64_t x_bs, x_ts;
    int64_t nseq, T, D;
    int64_t nslots;
    const int32_t* slots;
    uint32_t runs;       // runs of `run` tokens a sequence (dense) or in all (packed)
    uint32_t run;
    uint32_t vecs;       // ceil(D / V)
    uint32_t rows;       // rows of `vecs` threads
    int silu;
};

template <typename E, int W, int V>
struct Taps {
    float w[W][V], b[V];
    __device__ __forceinline__ void load(const ConvArgs& g, int64_t d, int n) {
        using T = typename E::T;
        const T* wp = static_cast<const T*>(g.w) + d * W;
        if (n >= V) {
            T all[W * V];
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const typename Vec<E, V>::utype v = *reinterpret_cast<const typename Vec<E, V>::utype*>(wp + j * V);
#pragma unroll
                for (int i = 0; i < V; ++i) all[j * V + i] = v[i];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                b[i] = 0.0f;
#pragma unroll
                for (int j = 0; j < W; ++j) w[j][i] = E::to_f32(all[i * W + j]);
            }
            if (g.bias) load_f32<E, V>(static_cast<const T*>(g.bias) + d, n, b);
            return;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][i] = i < n ? E::to_f32(wp[i * W + j]) : 0.0f;
            b[i] = g.bias && i < n ? E::to_f32(static_cast<const typename E::T*>(g.bias)[d + i]) : 0.0f;
        }
    }
    // The output for inputs h (oldest first) and x.
    __device__ __forceinline__ void apply(const float (&h)[W - 1][V], const float (&x)[V], int act,
                                          float (&o)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float s = b[i];
#pragma unroll
            for (int j = 0; j < W - 1; ++j) s = __builtin_fmaf(w[j][i], h[j][i], s);
            s = __builtin_fmaf(w[W - 1][i], x[i], s);
            o[i] = act ? silu(s) : s;
        }
    }
};

template <int W, int V>
__device__ __forceinline__ void push(float (&h)[W - 1][V], const float (&x)[V]) {
#pragma unroll
    for (int j = 0; j + 1 < W - 1; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) h[j][i] = h[j + 1][i];
#pragma unroll
    for (int i = 0; i < V; ++i) h[W - 2][i] = x[i];
}

// The W - 1 inputs before token t of sequence s, whose first token lies at xs.
template <typename E, int W, int V>
__device__ __forceinline__ void history(const ConvArgs& g, const typename E::T* xs, int64_t s, int64_t t, int64_t d,
                                        int n, float (&h)[W - 1][V]) {
    using T = typename E::T;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
        const int64_t at = t - (W - 1) + j;
        if (at >= 0) load_f32<E, V>(xs + at * g.x_ts, n, h[j]);
        else if (g.state_in)
            load_f32<E, V>(static_cast<const T*>(g.state_in) + (s * (W - 1) + (W - 1) + at) * g.D + d, n, h[j]);
        else
#pragma unroll
            for (int i = 0; i < V; ++i) h[j][i] = 0.0f;
    }
}

template <typename E, int W, int V>
__device__ __forceinline__ void write_state(const ConvArgs& g, int64_t s, int64_t d, int n,
                                            const float (&h)[W - 1][V]) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
        store_f32<E, V>(static_cast<typename E::T*>(g.state_out) + (s * (W - 1) + j) * g.D + d, n, h[j]);
}

// A row of D / V threads walks a run of tokens (dense: runs of each sequence in
// turn); nseq rows more carry the states of empty sequences over.
template <typename E, int W, int V, int U>
__global__ __launch_bounds__(kThreads) void conv_kernel(ConvArgs g) {
    using T = typename E::T;
    const uint32_t at = blockIdx.x * kThreads + threadIdx.x;
    const uint32_t row = at / g.vecs, vec = at - row * g.vecs;
    if (row >= g.rows) return;
    // The last channels' thread takes V of them all the same, some of which its
    // neighbour computes too (and both write the same).
    const int64_t d = g.D < V ? 0 : min(int64_t(vec) * V, g.D - V);
    const int n = int(g.D - d < V ? g.D - d : V);
    const T* x = static_cast<const T*>(g.x) + d;
    T* y = static_cast<T*>(g.y) + d;
    float h[W - 1][V];

    const uint32_t token_rows = g.cu ? g.runs : g.runs * uint32_t(g.nseq);
    if (row >= token_rows) {  // an empty sequence keeps its state
        const int64_t s = row - token_rows;
        if (!g.state_out) return;
        if (g.cu ? offset_of(g.cu, s + 1, g.T) > offset_of(g.cu, s, g.T) : g.T > 0) return;
        history<E, W, V>(g, x, s, 0, d, n, h);
        write_state<E, W, V>(g, s, d, n, h);
        return;
    }

    Taps<E, W, V> taps;
    taps.load(g, d, n);
    int64_t s, first, t, end, last;  // sequence, its first token, this run's tokens, the sequence's end
    if (!g.cu) {
        s = row / g.runs;
        first = 0;
        last = g.T;
        t = int64_t(row - uint32_t(s) * g.runs) * g.run;
        x += s * g.x_bs;
        y += s * g.T * g.D;
        end = t + g.run < g.T ? t + g.run : g.T;
    } else {
        t = int64_t(row) * g.run;
        end = t + g.run < g.T ? t + g.run : g.T;
        // the last sequence that starts at or before t
        int64_t lo = 0, hi = g.nseq;
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) / 2;
            if (offset_of(g.cu, mid, g.T) <= t) lo = mid;
            else hi = mid;
        }
        s = lo;
        first = offset_of(g.cu, s, g.T);
        last = offset_of(g.cu, s + 1, g.T);
    }

    while (t < end) {
        if (g.cu) {
            while (t >= last && s + 1 < g.nseq) {
                ++s;
                first = offset_of(g.cu, s, g.T);
                last = offset_of(g.cu, s + 1, g.T);
            }
            if (t < first || t >= last) {  // no sequence's token
                const int64_t stop = t < first && first < end ? first : end;
                const float zero[V] = {};
                for (; t < stop; ++t) store_f32<E, V>(y + t * g.D, n, zero);
                continue;
            }
        }
        const T* xs = x + first * g.x_ts;
        history<E, W, V>(g, xs, s, t - first, d, n, h);
        const int64_t stop = last < end ? last : end;
        if (n >= V) {
            typename Vec<E, V>::type even[U], odd[U];
            auto load = [&](typename Vec<E, V>::type (&v)[U], int64_t at) __attribute__((always_inline)) {
                if (at + U <= stop)
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        v[u] = *reinterpret_cast<const typename Vec<E, V>::utype*>(x + (at + u) * g.x_ts);
            };
            auto work = [&](const typename Vec<E, V>::type (&r)[U]) __attribute__((always_inline)) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float v[V], o[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] = E::to_f32(r[u][i]);
                    taps.apply(h, v, g.silu, o);
                    push<W, V>(h, v);
                    store_f32<E, V>(y + (t + u) * g.D, V, o);
                }
                t += U;
            };
            load(even, t);
            while (t + U <= stop) {
                load(odd, t + U);
                work(even);
                if (t + U > stop) break;
                load(even, t + U);
                work(odd);
            }
        }
        for (; t < stop; ++t) {
            float v[V], o[V];
            load_f32<E, V>(x + t * g.x_ts, n, v);
            taps.apply(h, v, g.silu, o);
            push<W, V>(h, v);
            store_f32<E, V>(y + t * g.D, n, o);
        }
        if (t == last && g.state_out) write_state<E, W, V>(g, s, d, n, h);
    }
}

template <typename E, int W, int V>
__global__ __launch_bounds__(kThreads) void conv_step_kernel(ConvArgs g) {
    using T = typename E::T;
    const uint32_t at = blockIdx.x * kThreads + threadIdx.x;
    const int64_t row = at / g.vecs;
    if (row >= g.nseq) return;
    const int64_t d = int64_t(at - uint32_t(row) * g.vecs) * V;
    const int n = int(g.D - d < V ? g.D - d : V);
    const int64_t slot = g.slots ? int64_t(g.slots[row]) : row;
    T* y = static_cast<T*>(g.y) + row * g.D + d;
    float h[W - 1][V], v[V], o[V];
    if (slot < 0 || slot >= g.nslots) {
        const float zero[V] = {};
        store_f32<E, V>(y, n, zero);
        return;
    }
    T* st = static_cast<T*>(g.state_out) + slot * (W - 1) * g.D + d;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) load_f32<E, V>(st + j * g.D, n, h[j]);
    load_f32<E, V>(static_cast<const T*>(g.x) + row * g.x_bs + d, n, v);
    Taps<E, W, V> taps;
    taps.load(g, d, n);
    taps.apply(h, v, g.silu, o);
    store_f32<E, V>(y, n, o);
    push<W, V>(h, v);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_f32<E, V>(st + j * g.D, n, h[j]);
}

template <typename F>
int with_width(int w, F f) {
    switch (w) {
        case 2: return f(std::integral_constant<int, 2>{});
        case 3: return f(std::integral_constant<int, 3>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 5: return f(std::integral_constant<int, 5>{});
        case 6: return f(std::integral_constant<int, 6>{});
        case 7: return f(std::integral_constant<int, 7>{});
        default: return f(std::integral_constant<int, 8>{});
    }
}

int check(const pe_conv_desc* d, bool step) {
    if (!d) return fail(PE_ERR_INVALID, "causal_conv: null descriptor");
    if (!dtype_ok(d->dtype)) return fail(PE_ERR_UNSUPPORTED, "causal_conv: dtype must be PE_F32, PE_F16 or PE_BF16");
    if (d->width < 2 || d->width > PE_CONV_MAX_WIDTH)
        return fail(PE_ERR_UNSUPPORTED, "causal_conv: width outside 2.." + std::to_string(PE_CONV_MAX_WIDTH));
    if (d->reserved != 0) return fail(PE_ERR_INVALID, "causal_conv: reserved field must be 0");
    if (d->nseq < 0 || d->D < 0 || (!step && d->T < 0) || (step && d->nslots < 0))
        return fail(PE_ERR_INVALID, "causal_conv: negative extent");
    if (d->nseq >= (int64_t(1) << 31) || d->T >= (int64_t(1) << 31) || d->D >= (int64_t(1) << 31))
        return fail(PE_ERR_UNSUPPORTED, "causal_conv: an extent of 2^31 or more");
    return PE_OK;
}

}  // namespace
}  // namespace ssm
}  // namespace pe

using namespace pe;
using namespace pe::ssm;

extern "C" int pe_causal_conv(const pe_conv_desc* d, const void* x, const void* weight, const void* bias,
                              const void* state_in, const int32_t* cu, void* y, void* state_out, void* stream) {
    if (int rc = check(d, false)) return rc;
    const bool in = cu ? within({{d->T, d->x_ts}, {d->D, 1}}, d->x_numel)
                       : within({{d->nseq, d->x_bs}, {d->T, d->x_ts}, {d->D, 1}}, d->x_numel);
    if (!in) return fail(PE_ERR_BOUNDS, "causal_conv: strides address past x");
    if (cu && d->nseq < 1) return fail(PE_ERR_INVALID, "causal_conv: packed tokens without a sequence");
    if (d->D == 0 || d->nseq == 0) return PE_OK;
    const bool tokens = d->T > 0;
    if (!weight || (tokens && (!x || !y))) return fail(PE_ERR_INVALID, "causal_conv: null pointer");
    ConvArgs g{};
    g.x = x; g.w = weight; g.bias = bias; g.state_in = state_in; g.cu = cu; g.y = y; g.state_out = state_out;
    g.x_bs = d->x_bs; g.x_ts = d->x_ts; g.nseq = d->nseq; g.T = d->T; g.D = d->D; g.silu = d->silu;
    return with_type(d->dtype, [&](auto e) {
        using E = decltype(e);
        return with_width(d->width, [&](auto w) {
            constexpr int W = w(), V = 16 / E::kBytes, U = 4;
            g.vecs = uint32_t(ceil_div(d->D, V));
            // Tokens a thread walks: of longer runs fewer inputs are read twice,
            // shorter ones make more threads (some four waves for each SIMD).
            g.run = 32;
            while (g.run > 8 && __int128(ceil_div(d->T, g.run)) * (cu ? 1 : d->nseq) * g.vecs < 1 << 18) g.run /= 2;
            g.runs = uint32_t(ceil_div(d->T, g.run));
            const int64_t rows = (cu ? int64_t(g.runs) : int64_t(g.runs) * d->nseq) +
                                 (cu || d->T == 0 ? d->nseq : 0);
            const __int128 blocks = (__int128(rows) * g.vecs + kThreads - 1) / kThreads;
            if (blocks >= (1 << 24)) return fail(PE_ERR_UNSUPPORTED, "causal_conv: too many tokens");
            g.rows = uint32_t(rows);
            conv_kernel<E, W, V, U><<<uint32_t(blocks), kThreads, 0, static_cast<hipStream_t>(stream)>>>(g);
            return hip_status_of_launch("causal_conv");
        });
    });
}

extern "C" int pe_causal_conv_step(const pe_conv_desc* d, const void* x, const void* weight, const void* bias,
                                   void* state, const int32_t* slots, void* y, void* stream) {
    if (int rc = check(d, true)) return rc;
    if (!within({{d->nseq, d->x_bs}, {d->D, 1}}, d->x_numel))
        return fail(PE_ERR_BOUNDS, "causal_conv_step: strides address past x");
    if (d->D == 0 || d->nseq == 0) return PE_OK;
    if (!x || !weight || !state || !y) return fail(PE_ERR_INVALID, "causal_conv_step: null pointer");
    if (!slots && d->nslots < d->nseq) return fail(PE_ERR_BOUNDS, "causal_conv_step: fewer states than rows");
    ConvArgs g{};
    g.x = x; g.w = weight; g.bias = bias; g.y = y; g.state_out = state; g.slots = slots;
    g.x_bs = d->x_bs; g.nseq = d->nseq; g.D = d->D; g.nslots = d->nslots; g.silu = d->silu;
    return with_type(d->dtype, [&](auto e) {
        using E = decltype(e);
        return with_width(d->width, [&](auto w) {
            constexpr int W = w(), V = 8 / E::kBytes;
            g.vecs = uint32_t(ceil_div(d->D, V));
            const int64_t blocks = ceil_div(int64_t(g.vecs) * d->nseq, kThreads);
            if (blocks >= (int64_t(1) << 24)) return fail(PE_ERR_UNSUPPORTED, "causal_conv_step: too many rows");
            conv_step_kernel<E, W, V><<<uint32_t(blocks), kThreads, 0, static_cast<hipStream_t>(stream)>>>(g);
            return hip_status_of_launch("causal_conv_step");
        });
    });
}
