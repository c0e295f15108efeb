"""Products with 4-bit weights on the GPU.

``matvec_q4(x, packed, scales, zeros)`` is ``einsum("mk,nk->mn", x, W)`` for a
weight W kept as 4-bit whole numbers with a scale, and optionally a zero point,
for every group of 32, 64 or 128 along k.  It is meant for the few rows of x of
a decode step: reading W bounds it, at half a byte a weight.  The whole numbers
enter the matrix cores exactly and scales are applied to float32 group sums,
so nothing is rounded but the float32 sums and the result.
"""
from __future__ import annotations

import ctypes

import torch

from . import abi, runtime
from .ssm import DTYPES, _plans, _ptr, check, dense, extent, inner, layout, lib, on, ready, remember


def matvec_q4(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
              group: int = 128) -> torch.Tensor:
    """y[..., n] = sum_k x[..., k] * scales[n, k // group] * (q[n, k] - zeros[n, k // group]).

    x [..., K] float16, bfloat16 or float32; packed uint8 [N, ceil(K / 2)] with
    q[n, k] in the low half of byte k // 2 for even k, in the high half for odd
    k; scales and zeros (none: 8) [N, ceil(K / group)] of x's dtype.  Sums are
    float32; y has x's dtype.  The weights are read once for every 64 rows of x."""
    what = "matvec_q4"
    key = (what, layout(x), layout(packed), layout(scales), layout(zeros), group)
    plan = _plans.get(key)
    if plan is None:
        if x.dtype not in DTYPES:
            raise TypeError(f"{what}: unsupported dtype {x.dtype} for x")
        if x.dim() < 1:
            raise ValueError(f"{what}: x must have an axis")
        if group not in (32, 64, 128):
            raise ValueError(f"{what}: group must be 32, 64 or 128, got {group}")
        K = x.shape[-1]
        if packed.dtype is not torch.uint8 or packed.dim() != 2:
            raise TypeError(f"{what}: packed must be a 2-D uint8 tensor, got {packed.dtype} of shape "
                            f"{tuple(packed.shape)}")
        N = packed.shape[0]
        if packed.shape[1] != (K + 1) // 2:
            raise ValueError(f"{what}: packed must have shape {(N, (K + 1) // 2)}, got {tuple(packed.shape)}")
        groups = (N, -(-K // group))
        check(what, "scales", scales, groups, x.dtype)
        check(what, "zeros", zeros, groups, x.dtype)
        ready(what, x, packed, scales, zeros)
        if x.dim() != 2:
            rows = x.reshape(-1, K) if K else x.reshape(x.shape[:-1].numel(), 0)
            return matvec_q4(rows, packed, scales, zeros, group=group).reshape(*x.shape[:-1], N)
        given, laid = (x, packed, scales, zeros), (inner(x), dense(packed), dense(scales), dense(zeros))
        if any(g is not t for g, t in zip(given, laid)):
            return matvec_q4(*laid, group=group)
        d = abi.Q4Desc(DTYPES[x.dtype], group, x.shape[0], N, K, x.stride(0), extent(x))
        plan = remember(key, (d, (x.shape[0], N)))
    d, shape = plan
    dev = ready(what, x, packed, scales, zeros)
    with on(dev):
        y = x.new_empty(shape)
        rc = lib().pe_matvec_q4(ctypes.byref(d), x.data_ptr(), packed.data_ptr(), scales.data_ptr(), _ptr(zeros),
                                y.data_ptr(), runtime.raw_stream(dev))
    runtime.check(rc, "pe_matvec_q4")
    return y
