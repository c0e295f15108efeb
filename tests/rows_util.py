"""64-bit definitions of rows in 8 bits, their products and the norms between
blocks, and the error bounds that follow from them."""
import torch

from ssm_util import ALL, HALF, IDS, TINY, silu  # noqa: F401

U = 2.0 ** -24


def quantize(x):
    """(q as float64, scale as float64) of rows of x.  In 64 bits 127 x is exact
    and the quotient of float32 values lies a relative 2^-32 or more away from
    every half it is not equal to, so its rounding is the exact one."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True) if x.shape[-1] else x.new_zeros((*x.shape[:-1], 1))
    q = torch.where(top > 0, torch.round(127 * x / torch.where(top > 0, top, 1.0)), 0.0)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    return torch.where(bad, 0.0, q), torch.where(bad, float("nan"), top / 127)[..., 0]


def product(q, scales, w, ws, bias):
    """y, and the size that the float32 roundings behind the exact sums scale with."""
    y = (q.double() @ w.double().t()) * scales.double()[..., None] * ws.double()
    size = y.abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def product_bound(ref, size, dtype):
    """The sum's conversion, the scale of a row given as float32 where it is formed
    in the call, two products and a sum; then one rounding to dtype."""
    return HALF[dtype] * ref.abs() + 6 * U * size + TINY[dtype]


def norm(u, eps, groups=1):
    """u over its root mean square in each group, and that factor."""
    v = u.unflatten(-1, (groups, -1))
    inv = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    return (v * inv).flatten(-2), inv.expand(v.shape).flatten(-2)


def gated(x, weight, z, eps, groups, norm_first):
    """y, and its relative error in float32 in units of U: a sum of D / groups
    squares over at least 64 lanes, each a chain, halved by the root; the gate's
    exponent, where it counts, is off by its own size times U."""
    x = x.double()
    gate = 1.0 if z is None else silu(z.double())
    gerr = 0.0 if z is None else z.double().abs() + 8
    y, _ = norm(x if norm_first else x * gate, eps, groups)
    if weight is not None:
        y = y * weight.double()
    if norm_first:
        y = y * gate
    chain = 16 + x.shape[-1] / groups / 64
    most = 0.0 if z is None else float(gerr.amax()) if gerr.numel() else 0.0
    return y, chain + 12 + gerr + most


def gated_bound(ref, units, dtype):
    return HALF[dtype] * ref.abs() + U * units * ref.abs() + TINY[dtype]


def residual(x, res, weight, post_weight, gate, scale, eps):
    """(y, r) and the absolute errors of each in float32 (before their last
    rounding): r's terms each pass a handful of roundings, y's factor the sum of
    squares, whose own error is that of the r's."""
    x = x.double()
    u = x
    chain = 16 + x.shape[-1] / 64
    if post_weight is not None:
        u = norm(u, eps)[0] * post_weight.double()
    if gate is not None:
        u = u * gate.double()
    r = res.double() + scale * u
    r_err = U * ((chain + 8) * (scale * u).abs() + r.abs())
    _, inv = norm(r, eps)
    w = 1.0 if weight is None else weight.double()
    y = r * inv * w
    # the root mean square is off by at most that of the errors
    rms = torch.sqrt((r_err * r_err).mean(-1, keepdim=True)) * inv
    y_err = (r_err * inv * abs(w)) + y.abs() * (rms + U * (chain + 8))
    return y, r, y_err, r_err


def bound(ref, err, dtype):
    return HALF[dtype] * ref.abs() + (1 + HALF[dtype]) * err + TINY[dtype]


def rows_bound(ref, err, scales):
    """What rows in 8 bits stand for differs from ref by half a step, by its own
    error, and by that of the row's largest value, which the step follows."""
    return 0.5 * scales.double()[..., None] * (1 + 8 * U) + err + err.amax(-1, keepdim=True) + TINY[torch.float32]


def assert_within(got, ref, limit, what=""):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)} for {tuple(ref.shape)}"
    off = (got - ref).abs() - limit
    bad = ~(off <= 0)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, the worst by {float(off.max()):.3e} beyond its "
                           f"bound, first at {bad.nonzero()[0].tolist()}")
