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
from .ssm import DTYPES, _ptr, extent, inner, lib, no_grad, of_shape, of_type, same_gpu


def matvec_q4(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
              group: int = 128) -> torch.Tensor:
    """y[..., n] = sum_k x[..., k] * scales[n, k // group] * (q[n, k] - zeros[n, k // group]).

    x [..., K] float16, bfloat16 or float32; packed uint8 [N, ceil(K / 2)] with
    q[n, k] in the low half of byte k // 2 for even k, in the high half for odd
    k; scales and zeros (none: 8) [N, ceil(K / group)] of x's dtype.  Sums are
    float32; y has x's dtype.  The weights are read once for every 64 rows of x."""
    what = "matvec_q4"
    if x.dtype not in DTYPES:
        raise TypeError(f"{what}: unsupported dtype {x.dtype} for x")
    if x.dim() < 1:
        raise ValueError(f"{what}: x must have an axis")
    if group not in (32, 64, 128):
        raise ValueError(f"{what}: group must be 32, 64 or 128, got {group}")
    K = x.shape[-1]
    if packed.dtype != torch.uint8 or packed.dim() != 2:
        raise TypeError(f"{what}: packed must be a 2-D uint8 tensor, got {packed.dtype} of shape {tuple(packed.shape)}")
    N = packed.shape[0]
    of_type(what, x.dtype, scales=scales, zeros=zeros)
    of_shape(what, packed=(packed, (N, (K + 1) // 2)), scales=(scales, (N, -(-K // group))),
             zeros=(zeros, (N, -(-K // group))))
    no_grad(what, x, scales, zeros)
    dev = same_gpu(what, x, packed=packed, scales=scales, zeros=zeros)
    rows = inner(x if x.dim() == 2 else x.reshape(-1, K) if K else x.reshape(x.shape[:-1].numel(), 0))
    packed, scales = packed.contiguous(), scales.contiguous()
    zeros = None if zeros is None else zeros.contiguous()
    d = abi.Q4Desc(dtype=DTYPES[x.dtype], group=group, M=rows.shape[0], N=N, K=K, x_ms=rows.stride(0),
                   x_numel=extent(rows))
    with torch.cuda.device(dev):
        y = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=dev)
        rc = lib().pe_matvec_q4(ctypes.byref(d), _ptr(rows), _ptr(packed), _ptr(scales), _ptr(zeros), _ptr(y),
                                runtime.raw_stream(dev.index))
    runtime.check(rc, "pe_matvec_q4")
    return y
