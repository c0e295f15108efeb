"""Products with weights of 4 or 8 bits on the GPU.

``matvec_q4(x, packed, scales, zeros)`` is ``einsum("mk,nk->mn", x, W)`` for a
weight W kept as 4-bit whole numbers with a scale, and optionally a zero point,
for every group of 32, 64 or 128 along k.  It is meant for the few rows of x of
a decode step: reading W bounds it, at half a byte a weight.  The whole numbers
enter the matrix cores exactly and scales are applied to float32 group sums,
so nothing is rounded but the float32 sums and the result.

``matmul_q8(x, weight, weight_scales)`` multiplies rows in 8 bits, x's tokens with
a weight's channels, in whole numbers on the matrix cores: for prompts twice the
rate of 16-bit products, for single tokens half their bytes.
"""
from __future__ import annotations

import ctypes

import torch

from . import abi, launch, runtime
from .norm import _stride, alloc, fresh, row_bytes, row_pitch
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


MAX_K8 = 131071    # sums of 32 bits hold 128 * 128 * K


def _apart(t: torch.Tensor):
    """The one stride of t's rows, all axes but the last taken as one, or None.  (Of no
    elements, which torch calls contiguous in any order: 0.)"""
    return 0 if not t.numel() else _stride(list(zip(t.shape[:-1], t.stride())))


def _apart8(t: torch.Tensor) -> int:
    """The same of rows in 8 bits; of one row, or none, as if there were more."""
    return _apart(t) if t.numel() and t.shape[:-1].numel() > 1 else row_bytes(t.shape[-1])


def _laid8(t: torch.Tensor) -> bool:
    """Whether t's rows in 8 bits lie as the product reads them: whole 16-byte
    groups from 16-byte addresses.  (Where K is no multiple of 16 the last group
    ends behind the row, which the storage has to hold.)"""
    k = t.shape[-1]
    if t.data_ptr() % 16:
        return False
    return k % 16 == 0 or not t.numel() or extent(t) + row_bytes(k) - k <= t.untyped_storage().nbytes() - t.storage_offset()


def _lay8(t: torch.Tensor) -> torch.Tensor:
    """t in rows that start every 16 bytes."""
    k = t.shape[-1]
    out = t.new_zeros((*t.shape[:-1], row_pitch(k)))[..., :k]
    out.copy_(t)
    return out


def _rows_ok(t: torch.Tensor) -> bool:
    """Whether t's strides are those of rows in 8 bits."""
    k, apart = t.shape[-1], _apart(t)
    if t.numel() == 0:
        return True
    if apart is None or (t.stride(-1) != 1 and k != 1):
        return False
    apart = _apart8(t)
    return apart % 16 == 0 and row_bytes(k) <= apart <= 1 << 23


def matmul_q8(x: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, *,
              scales: torch.Tensor | None = None, bias: torch.Tensor | None = None,
              dtype: torch.dtype | None = None) -> torch.Tensor:
    """y[..., n] = scales[...] * weight_scales[n] * sum_k x[..., k] * weight[n, k] + bias[n]

    in 8-bit whole numbers, with a scale for each row of x (a token) and each row
    of the weight (an output channel).  weight int8 [N, K] with K <= 131071,
    weight_scales float32 [N]: what ``quantize_q8`` gives for a weight.  x is
    either int8 [..., K] with ``scales`` float32 [...], from ``quantize_q8`` or a
    norm with ``quantize``, or float16, bfloat16 or float32, whose rows the call
    takes to 8 bits first.  Sums of products are exact; scales and bias (float32
    or of the result's dtype) are applied in float32 and the result is rounded
    once to ``dtype`` (none: x's, float32 for int8 x).

    Rows that do not start every 16 bytes (a contiguous weight whose K is no
    multiple of 16) are copied first, in every call: keep weights as
    ``quantize_q8`` lays them out."""
    what = "matmul_q8"
    key = (what, layout(x), layout(weight), layout(weight_scales), layout(scales), layout(bias), dtype)
    plan = _plans.get(key)
    if plan is None:
        whole = x.dtype is torch.int8
        if not whole and x.dtype not in DTYPES:
            raise TypeError(f"{what}: unsupported dtype {x.dtype} for x")
        if x.dim() < 1:
            raise ValueError(f"{what}: x must have an axis")
        if weight.dtype is not torch.int8 or weight.dim() != 2:
            raise TypeError(f"{what}: weight must be a 2-D int8 tensor, got {weight.dtype} of shape "
                            f"{tuple(weight.shape)}")
        (N, K), lead = weight.shape, x.shape[:-1]
        if x.shape[-1] != K:
            raise ValueError(f"{what}: x must be [..., {K}] for a weight of shape {(N, K)}, got {tuple(x.shape)}")
        if K > MAX_K8:
            raise ValueError(f"{what}: K must be at most {MAX_K8} for sums of 32 bits, got {K}")
        if whole == (scales is None):
            raise ValueError(f"{what}: " + ("int8 x needs its scales" if whole else
                                            f"scales belong to int8 x, got {x.dtype}"))
        out = dtype if dtype is not None else torch.float32 if whole else x.dtype
        if out not in DTYPES:
            raise TypeError(f"{what}: unsupported dtype {out} for the result")
        check(what, "weight_scales", weight_scales, (N,), torch.float32)
        check(what, "scales", scales, lead, torch.float32)
        check(what, "bias", bias, (N,), out if bias is None or bias.dtype is out else torch.float32)
        ready(what, x, weight, weight_scales, scales, bias)
        given = (x, weight, weight_scales, scales, bias)
        laid = (_lay8(x) if whole and not _rows_ok(x) else x if whole or _apart(x) is not None and inner(x) is x
                else x.contiguous(), weight if _rows_ok(weight) else _lay8(weight), dense(weight_scales),
                dense(scales), dense(bias))
        if any(g is not t for g, t in zip(given, laid)):
            return matmul_q8(*laid[:3], scales=laid[3], bias=laid[4], dtype=dtype)
        M, kp = lead.numel(), row_bytes(K)
        d = abi.Q8Desc(launch.DT_I8 if whole else DTYPES[x.dtype], DTYPES[out],
                       launch.DT_F32 if bias is None else DTYPES[bias.dtype], 0, M, N, K,
                       _apart8(x) if whole else _apart(x), _apart8(weight),
                       extent(x) + (kp - K if whole else 0), extent(weight) + kp - K)
        plan = remember(key, (d, fresh((*lead, N), out), whole, lib().pe_matmul_q8_workspace_bytes(ctypes.byref(d))))
    d, result, whole, ws_bytes = plan
    dev = ready(what, x, weight, weight_scales, scales, bias)
    rows_lie, weight_lies = not whole or _laid8(x), _laid8(weight)
    if not (rows_lie and weight_lies):
        return matmul_q8(x if rows_lie else _lay8(x), weight if weight_lies else _lay8(weight), weight_scales,
                         scales=scales, bias=bias, dtype=dtype)
    with on(dev):
        y = alloc(result, x.device)
        ws = weight.new_empty(ws_bytes) if ws_bytes else None
        rc = lib().pe_matmul_q8(ctypes.byref(d), x.data_ptr(), _ptr(scales), weight.data_ptr(),
                                weight_scales.data_ptr(), _ptr(bias), y.data_ptr(), _ptr(ws), ws_bytes,
                                runtime.raw_stream(dev))
    runtime.check(rc, "pe_matmul_q8")
    return y
