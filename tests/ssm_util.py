"""64-bit definitions of the state-space operators and of the 4-bit product,
token by token on the CPU, and the error bounds that follow from them."""
import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
ALL = [torch.float16, torch.bfloat16, torch.float32]
IDS = ["f16", "bf16", "f32"]


def silu(v):
    return v / (1 + torch.exp(-v))


def conv(x, weight, bias, act, state):
    """One sequence: y [T, D], the state after it, and sum |w x| + |bias|."""
    w = weight.double()
    width = w.shape[1]
    line = torch.cat([state.double(), x.double()])
    T = x.shape[0]
    y = torch.zeros(T, x.shape[1], dtype=torch.float64)
    size = torch.zeros_like(y)
    for j in range(width):
        y += line[j:j + T] * w[:, j]
        size += (line[j:j + T] * w[:, j]).abs()
    if bias is not None:
        y += bias.double()
        size += bias.double().abs()
    return (silu(y) if act else y), line[line.shape[0] - (width - 1):], size


def conv_bound(ref, size, dtype):
    """Each of the width + 1 additions and the activation's four operations (exp
    good to 2 units, slope at most 1.1) rounds to float32; then one rounding
    to dtype."""
    return HALF[dtype] * ref.abs() + 16 * 2.0 ** -24 * (size + ref.abs()) + TINY[dtype]


def scan(x, dt, A, B, C, D, z, dt_bias, softplus, state):
    """One sequence: y [T, H, P], the state after it [H, P, N], and the same
    with every term's absolute value (what rounding errors scale with)."""
    x, dt, B, C = (t.double() for t in (x, dt, B, C))
    T, H, P = x.shape
    rep = H // B.shape[1]
    B, C = B.repeat_interleave(rep, 1), C.repeat_interleave(rep, 1)
    d = dt if dt_bias is None else dt + dt_bias.double()
    if softplus:
        d = torch.clamp(d, min=0) + torch.log1p(torch.exp(-d.abs()))
    fade = torch.exp(d * A.double())
    S, Sa = state.double().clone(), state.double().abs()
    y, ya = torch.zeros(T, H, P, dtype=torch.float64), torch.zeros(T, H, P, dtype=torch.float64)
    for t in range(T):
        add = (d[t, :, None] * x[t])[:, :, None] * B[t][:, None, :]
        S = fade[t, :, None, None] * S + add
        Sa = fade[t, :, None, None] * Sa + add.abs()
        y[t] = (S * C[t][:, None, :]).sum(-1)
        ya[t] = (Sa * C[t].abs()[:, None, :]).sum(-1)
        if D is not None:
            y[t] += D.double()[:, None] * x[t]
            ya[t] += (D.double()[:, None] * x[t]).abs()
    if z is not None:
        g = silu(z.double())
        y, ya = y * g, ya * g.abs()
    return y, S, ya, Sa


def scan_bound(T, N, d_max, a_max):
    """Relative to the sums of absolute values: a term passes through at most T
    decays, each good to (2 + |A d|) roundings of which what matters survives
    |A d| summed to 20, and as many additions; step size, product with x and B
    and the sum over N round some 8 + log2 N + T / 16 times more."""
    return 2.0 ** -24 * (4 * T + 40 + N)


def q4(x, packed, scales, zeros, group, K):
    q = torch.empty(packed.shape[0], 2 * packed.shape[1], dtype=torch.float64)
    q[:, 0::2] = (packed & 15).double()
    q[:, 1::2] = (packed >> 4).double()
    zero = 8.0 if zeros is None else zeros.double().repeat_interleave(group, 1)[:, :K]
    s = scales.double().repeat_interleave(group, 1)[:, :K]
    w = (q[:, :K] - zero) * s
    # what the roundings of q x and z x, added up apart, scale with
    big = (q[:, :K] + (8.0 if zeros is None else zero.abs())) * s.abs()
    return x.double() @ w.t(), x.double().abs() @ big.t()


def q4_bound(ref, size, K, dtype):
    """Float32 sums of K products in some order, K / group fused multiply-adds and
    eight parts; then one rounding to dtype."""
    return HALF[dtype] * ref.abs() + 2.0 ** -24 * (K + 16) * size + TINY[dtype]
