"""Norms between the blocks of a layer on the GPU.

``gated_norm`` is the norm behind a scan, fused with its gate; ``residual_norm``
ends one block and starts the next: a norm and a gate of the block's output, the
residual sum with its scale, and the norm of that sum.  Both read each value once
and answer either in the operands' type or, with ``quantize=True``, with rows in
8 bits and their scales: the operands of ``matmul_q8``.

Types, streams, captures and refusals are those of the state-space operators:
float16, bfloat16 or float32, sums and norms in float32, every output rounded
once, no gradients.
"""
from __future__ import annotations

import ctypes
import operator

import torch

from . import abi, runtime
from .ssm import DTYPES, _plans, _ptr, check, dense, extent, inner, layout, lib, on, ready, remember


def row_bytes(k: int) -> int:
    """Bytes of a row in 8 bits, in the groups of 16 that the product reads."""
    return -(-k // 16) * 16


def row_pitch(k: int) -> int:
    """Bytes from one row in 8 bits to the next: long rows start on whole lines."""
    return row_bytes(k) if k < 1024 else -(-k // 128) * 128


def _stride(axes):
    """The one stride of some (size, stride) axes, or None."""
    axes = [a for a in axes if a[0] != 1]
    if any(n == 0 for n, _ in axes):
        return 0
    for (_, s), (n, t) in zip(axes, axes[1:]):
        if s != n * t:
            return None
    return axes[-1][1] if axes else 0


def places(lead, tensors):
    """The leading axes ``lead`` as two, and every tensor's strides along them
    (None: that tensor has no such strides; None in its place: not given): the
    split that suits most tensors."""
    best = None
    for p in range(len(lead) + 1):
        found = []
        for t in tensors:
            if t is None or not t.numel():
                # (of no elements nothing is addressed; torch calls them contiguous in any order)
                found.append((0, 0))
                continue
            axes = list(zip(lead, t.stride()))
            pair = _stride(axes[:p]), _stride(axes[p:len(lead)])
            found.append(None if None in pair else pair)
        if best is None or found.count(None) < best[1].count(None):
            best = p, found
    p, found = best
    rows0, rows1 = torch.Size(lead[:p]).numel(), torch.Size(lead[p:]).numel()
    return rows0, rows1, found


def _operands(what, x, **others):
    if x.dtype not in DTYPES:
        raise TypeError(f"{what}: unsupported dtype {x.dtype} for x")
    if x.dim() < 1:
        raise ValueError(f"{what}: x must have an axis")
    for name, t in others.items():
        check(what, name, t, (x.shape[-1],), x.dtype)


def number(what, name, v, kind=float):
    """A number; a tensor's value is not known here."""
    if type(v) is kind:
        return v
    if isinstance(v, torch.Tensor):
        raise TypeError(f"{what}: {name} must be a number, got a tensor")
    return float(v) if kind is float else operator.index(v)


def _held(what, name, v):
    """v, which float32 holds: neither as infinity nor, where it is not 0, as 0."""
    if not abs(v) <= torch.finfo(torch.float32).max or 0.0 < abs(v) < 2.0 ** -149:
        raise ValueError(f"{what}: {name} must be finite and in float32's range, got {v}")
    return v


def _eps(what, eps):
    if not eps >= 0.0:
        raise ValueError(f"{what}: eps must be finite and 0 or more, got {eps}")
    return _held(what, "eps", eps)


# eps and scale may change from call to call, and calls on several threads have their
# own: a plan keeps a descriptor for each of the last numbers, not one plan for each.
MOST_NUMBERS = 64


def numbered(what, base, made, eps, scale):
    """A plan's descriptor with these numbers, kept with those already made."""
    d = abi.RowsDesc.from_buffer_copy(base)
    d.eps, d.scale = _eps(what, eps), _held(what, "scale", scale)
    if len(made) >= MOST_NUMBERS:
        made.clear()
    made[eps, scale] = d
    return d


def fresh(shape, dtype):
    """How a contiguous result is allocated: shape, strides and dtype, kept with the
    plan (``empty_strided`` takes 1.5 us where ``new_empty`` takes 2 to 3)."""
    strides, n = [], 1
    for size in reversed(shape):
        strides.append(n)
        n *= max(size, 1)
    return tuple(shape), tuple(reversed(strides)), dtype


def alloc(how, device):
    return torch.empty_strided(how[0], how[1], dtype=how[2], device=device)


def fresh8(shape):
    """The same of rows in 8 bits for values of that shape: the rows with what pads
    them, their length (None: nothing does), the scales."""
    k = shape[-1]
    pitch = row_pitch(k)
    return fresh((*shape[:-1], pitch), torch.int8), None if k == pitch else k, fresh(shape[:-1], torch.float32)


def alloc8(how, device):
    """(values, scales) of such rows."""
    q = alloc(how[0], device)
    return (q if how[1] is None else q[..., :how[1]]), alloc(how[2], device)


def quantize_q8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of x in 8 bits: (q int8 of x's shape, scales float32 [...]) with

        scales = max_k |x| / 127,   q = x / scales rounded to the nearest whole number

    ties to even, as the exact quotient 127 x / max decides.  A row of zeros gets
    scale 0; one that holds an infinity or NaN gets scale NaN and values 0, so
    that whatever is formed with it is NaN.  x [..., K] float16, bfloat16 or
    float32.  q's rows start every 16 bytes (K rounded up to 16, from 1024 on to
    128, the rest 0), which is how ``matmul_q8`` reads rows of x and of weights."""
    what = "quantize_q8"
    key = (what, layout(x))
    plan = _plans.get(key)
    if plan is None:
        _operands(what, x)
        ready(what, x)
        laid = inner(x)
        rows0, rows1, (pair,) = places(x.shape[:-1], (laid,))
        if pair is None or laid is not x:
            return quantize_q8(laid.contiguous())
        d = abi.RowsDesc(dtype=DTYPES[x.dtype], rows0=rows0, rows1=rows1, D=x.shape[-1], groups=1, x_s0=pair[0],
                         x_s1=pair[1], q_ms=row_pitch(x.shape[-1]), x_numel=extent(x))
        plan = remember(key, (d, fresh8(x.shape)))
    d, rows = plan
    dev = ready(what, x)
    with on(dev):
        q, scales = alloc8(rows, x.device)
        rc = lib().pe_quantize_q8(ctypes.byref(d), x.data_ptr(), q.data_ptr(), scales.data_ptr(),
                                  runtime.raw_stream(dev))
    runtime.check(rc, "pe_quantize_q8")
    return q, scales


def gated_norm(x: torch.Tensor, weight: torch.Tensor | None = None, z: torch.Tensor | None = None, *,
               eps: float = 1e-5, groups: int = 1, norm_first: bool = False, quantize: bool = False):
    """Root-mean-square norm with a gate, over each of ``groups`` equal parts of
    the last axis:

        u = x * silu(z),  y = u / sqrt(mean(u^2) + eps) * weight                (z given)
        y = x / sqrt(mean(x^2) + eps) * weight * silu(z)                        (and norm_first)

    with silu(z) = z / (1 + exp(-z)); without z the plain norm.  x and z [..., D]
    (any strides but along the last axis), weight [D], all of x's dtype.  Returns
    y of x's shape and dtype, or with ``quantize`` what ``quantize_q8`` gives for
    the float32 y: (q, scales), one scale for a row of D (at most 8192 groups)."""
    what = "gated_norm"
    eps, groups = number(what, "eps", eps), number(what, "groups", groups, int)
    key = (what, layout(x), layout(weight), layout(z), groups, bool(norm_first), bool(quantize))
    plan = _plans.get(key)
    if plan is None:
        _operands(what, x, weight=weight)
        check(what, "z", z, x.shape, x.dtype)
        D = x.shape[-1]
        if groups < 1 or D % groups:
            raise ValueError(f"{what}: {D} elements are no {groups} equal groups")
        if quantize and groups > 8192:
            raise ValueError(f"{what}: at most 8192 groups with quantize, got {groups}")
        _eps(what, eps)
        ready(what, x, weight, z)
        given = (x, weight, z)
        laid = [inner(x), dense(weight), None if z is None else inner(z)]
        rows0, rows1, pairs = places(x.shape[:-1], (laid[0], laid[2]))
        for i, pair in zip((0, 2), pairs):
            if pair is None:
                laid[i] = laid[i].contiguous()
        if any(g is not t for g, t in zip(given, laid)):
            return gated_norm(*laid, eps=eps, groups=groups, norm_first=norm_first, quantize=quantize)
        d = abi.RowsDesc(dtype=DTYPES[x.dtype], norm_first=bool(norm_first), rows0=rows0, rows1=rows1, D=D,
                         groups=groups, x_s0=pairs[0][0], x_s1=pairs[0][1], g_s0=pairs[1][0], g_s1=pairs[1][1],
                         q_ms=row_pitch(D), x_numel=extent(x), g_numel=0 if z is None else extent(z))
        plan = remember(key, (d, {}, fresh8(x.shape) if quantize else fresh(x.shape, x.dtype)))
    base, made, result = plan
    d = made.get((eps, 1.0)) or numbered(what, base, made, eps, 1.0)
    dev = ready(what, x, weight, z)
    with on(dev):
        y, scales = alloc8(result, x.device) if quantize else (alloc(result, x.device), None)
        out = (None, y.data_ptr(), scales.data_ptr()) if quantize else (y.data_ptr(), None, None)
        rc = lib().pe_gated_norm(ctypes.byref(d), x.data_ptr(), _ptr(weight), _ptr(z), *out, runtime.raw_stream(dev))
    runtime.check(rc, "pe_gated_norm")
    return (y, scales) if quantize else y


def residual_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None, *,
                  post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float = 1.0,
                  eps: float = 1e-5, quantize: bool = False):
    """The end of one block, x, and the start of the next:

        u = x / sqrt(mean(x^2) + eps) * post_weight     (post_weight given, else u = x)
        r = residual + scale * gate * u                 (gate given, else 1)
        y = r / sqrt(mean(r^2) + eps) * weight

    x [..., D]; residual of x's shape and dtype, or float32; weight and
    post_weight [D] and gate of x's dtype; gate of any shape that broadcasts to
    x's (a gate for each channel, sequence, token or value).  Any strides but
    along the last axis.  scale and eps are numbers, finite and in float32's
    range.  Returns (y, r): y of x's dtype, formed from r before r
    is rounded to the residual's dtype, or with ``quantize`` ((q, scales), r) as
    ``quantize_q8`` gives them for the float32 y."""
    what = "residual_norm"
    scale, eps = number(what, "scale", scale), number(what, "eps", eps)
    key = (what, layout(x), layout(residual), layout(weight), layout(post_weight), layout(gate), bool(quantize))
    plan = _plans.get(key)
    if plan is None:
        _operands(what, x, weight=weight, post_weight=post_weight)
        check(what, "residual", residual, x.shape, x.dtype if residual.dtype is x.dtype else torch.float32)
        D, lead = x.shape[-1], x.shape[:-1]
        _eps(what, eps), _held(what, "scale", scale)
        wide = gate
        if gate is not None:
            check(what, "gate", gate, gate.shape, x.dtype)
            try:
                wide = gate.expand((*lead, 1 if gate.shape[-1:] in ((), (1,)) else D))
            except RuntimeError:
                raise ValueError(f"{what}: gate of shape {tuple(gate.shape)} does not broadcast to {tuple(x.shape)}") from None
        ready(what, x, residual, weight, post_weight, gate)
        given = [x, residual, weight, post_weight, gate]
        laid = [inner(x), inner(residual), dense(weight), dense(post_weight),
                gate if gate is None or wide.stride(-1) == 1 or wide.shape[-1] == 1 else gate.clone(
                    memory_format=torch.contiguous_format)]
        if laid[4] is gate:
            rows0, rows1, pairs = places(lead, (laid[0], laid[1], wide))
            for i, t, pair in zip((0, 1, 4), (laid[0], laid[1], wide), pairs):
                if pair is None:
                    laid[i] = t.contiguous()
        if any(g is not t for g, t in zip(given, laid)):
            return residual_norm(*laid[:3], post_weight=laid[3], gate=laid[4], scale=scale, eps=eps, quantize=quantize)
        (xs, rs, gs) = pairs
        d = abi.RowsDesc(dtype=DTYPES[x.dtype], res_dtype=DTYPES[residual.dtype],
                         gate_row=gate is not None and wide.shape[-1] == 1, rows0=rows0, rows1=rows1, D=D, groups=1,
                         x_s0=xs[0], x_s1=xs[1], g_s0=gs[0], g_s1=gs[1], r_s0=rs[0], r_s1=rs[1], q_ms=row_pitch(D),
                         x_numel=extent(x), g_numel=0 if gate is None else extent(gate), r_numel=extent(residual))
        plan = remember(key, (d, {}, fresh8(x.shape) if quantize else fresh(x.shape, x.dtype),
                              fresh(x.shape, residual.dtype)))
    base, made, result, total = plan
    d = made.get((eps, scale)) or numbered(what, base, made, eps, scale)
    dev = ready(what, x, residual, weight, post_weight, gate)
    with on(dev):
        y, scales = alloc8(result, x.device) if quantize else (alloc(result, x.device), None)
        r = alloc(total, x.device)
        out = (None, r.data_ptr(), y.data_ptr(), scales.data_ptr()) if quantize else (y.data_ptr(), r.data_ptr(), None,
                                                                                     None)
        rc = lib().pe_residual_norm(ctypes.byref(d), x.data_ptr(), residual.data_ptr(), _ptr(weight),
                                    _ptr(post_weight), _ptr(gate), *out, runtime.raw_stream(dev))
    runtime.check(rc, "pe_residual_norm")
    return ((y, scales) if quantize else y), r
