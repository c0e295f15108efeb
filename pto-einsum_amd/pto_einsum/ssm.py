"""The serving operators of a state-space layer on the GPU.

A layer convolves each channel with a short causal filter, scans the result
through a state of P x N values per head whose decay and input depend on the
token, and projects.  ``causal_conv`` and ``selective_scan`` run prompts
(dense batches or packed sequences, from a carried state to a new one),
``causal_conv_step`` and ``selective_scan_step`` one token of each sequence
against caches of states that they update in place.

Operands are float16, bfloat16 or float32 and share a dtype, which the output
has too: it is the next operator's operand, unlike a contraction's float32
result.  Sums and scan states are float32.  Calls enqueue on the current
stream, allocate through torch only and neither synchronise nor clear memory
with a memset, so they can be captured in a ``StageGraph``.  ``cu_seqlens`` and
``slots`` are read on the GPU; offsets outside the buffer are clamped to it and
slots outside the cache mark rows without a sequence.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import abi, launch, runtime

DTYPES = {torch.float32: launch.DT_F32, torch.float16: launch.DT_F16, torch.bfloat16: launch.DT_BF16}
MAX_WIDTH = 8      # PE_CONV_MAX_WIDTH
MAX_N = 256        # PE_SCAN_MAX_N


@functools.lru_cache(maxsize=None)
def lib():
    """The core library with its argument types set."""
    return abi.bind()


def extent(t: torch.Tensor) -> int:
    """Elements addressable from t's first element to the end of its storage."""
    return t.untyped_storage().nbytes() // t.element_size() - t.storage_offset()


def inner(t: torch.Tensor) -> torch.Tensor:
    """t with its last axis contiguous and no negative or overlapping inner
    layout: t itself where that holds (other axes keep their strides)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def same_gpu(what: str, x: torch.Tensor, **others) -> torch.device:
    if x.device.type != "cuda":
        raise ValueError(f"{what}: operands must live on a GPU, got {x.device}")
    for name, t in others.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{what}: operands must all live on one GPU, {name} is on {t.device}, not {x.device}")
    return x.device


def no_grad(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or on detached operands")


def of_type(what: str, dtype, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.dtype != dtype:
            raise TypeError(f"{what}: {name} must be {dtype}, got {t.dtype}")


def of_shape(what: str, **tensors) -> None:
    """``name=(tensor, shape)``: each tensor that is given has that shape."""
    for name, (t, shape) in tensors.items():
        if t is not None and tuple(t.shape) != tuple(shape):
            raise ValueError(f"{what}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _index(what: str, name: str, t, length: int | None):
    """An int32 index vector, contiguous."""
    if t is None:
        return None
    if t.dtype != torch.int32 or t.dim() != 1:
        raise TypeError(f"{what}: {name} must be a 1-D int32 tensor, got {t.dtype} of shape {tuple(t.shape)}")
    if length is not None and t.shape[0] != length:
        raise ValueError(f"{what}: {name} must have {length} entries, got {t.shape[0]}")
    return t.contiguous()


def _sequences(what: str, x, cu_seqlens, dims: int):
    """(number of sequences, tokens) of x, dense [nseq, T, ...] with ``dims``
    axes or packed [T, ...] with one less."""
    cu = _index(what, "cu_seqlens", cu_seqlens, None)
    if cu is None:
        if x.dim() != dims:
            raise ValueError(f"{what}: x must have {dims} axes (sequences first), got shape {tuple(x.shape)}")
        return x.shape[0], x.shape[1], None
    if x.dim() != dims - 1:
        raise ValueError(f"{what}: packed x must have {dims - 1} axes (tokens first), got shape {tuple(x.shape)}")
    if cu.shape[0] < 2:
        raise ValueError(f"{what}: cu_seqlens needs the offsets of at least one sequence")
    return cu.shape[0] - 1, x.shape[0], cu


def _lead(t, packed: bool):
    """(sequence stride, token stride) of a prompt's tensor."""
    return (0, t.stride(0)) if packed else (t.stride(0), t.stride(1))


# --------------------------------------------------------------- convolution --

def _conv_operands(what, x, weight, bias, activation):
    if x.dtype not in DTYPES:
        raise TypeError(f"{what}: unsupported dtype {x.dtype} for x")
    if activation not in (None, "silu"):
        raise ValueError(f"{what}: activation must be None or 'silu', got {activation!r}")
    if weight.dim() != 2 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"{what}: weight must be [{x.shape[-1]}, width], got shape {tuple(weight.shape)}")
    width = weight.shape[1]
    if not 2 <= width <= MAX_WIDTH:
        raise ValueError(f"{what}: width must be 2 to {MAX_WIDTH}, got {width}")
    of_type(what, x.dtype, weight=weight, bias=bias)
    of_shape(what, bias=(bias, (x.shape[-1],)))
    return width, weight.contiguous(), None if bias is None else bias.contiguous()


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                activation: str | None = None, initial_state: torch.Tensor | None = None,
                cu_seqlens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Causal convolution of each channel along the tokens of prompts:

        y[t, d] = act(bias[d] + sum_j weight[d, j] * x[t - width + 1 + j, d])

    x [nseq, T, D], or packed [T, D] with ``cu_seqlens`` (int32 offsets on the
    GPU, nseq + 1 of them, from 0 up; tokens past the last get y = 0); weight
    [D, width] with 2 <= width <= 8; ``activation`` None or "silu".
    ``initial_state`` [nseq, width - 1, D] holds the inputs before each
    sequence's first token, oldest first (none: zeros).  Returns y of x's
    shape and the state after each sequence, both of x's dtype."""
    what = "causal_conv"
    nseq, T, cu = _sequences(what, x, cu_seqlens, 3)
    D = x.shape[-1]
    width, weight, bias = _conv_operands(what, x, weight, bias, activation)
    of_type(what, x.dtype, initial_state=initial_state)
    of_shape(what, initial_state=(initial_state, (nseq, width - 1, D)))
    no_grad(what, x, weight, bias, initial_state)
    dev = same_gpu(what, x, weight=weight, bias=bias, initial_state=initial_state, cu_seqlens=cu)
    x = inner(x)
    first = None if initial_state is None else initial_state.contiguous()
    d = abi.ConvDesc(dtype=DTYPES[x.dtype], width=width, silu=activation is not None, nseq=nseq, T=T, D=D,
                     x_numel=extent(x))
    d.x_bs, d.x_ts = _lead(x, cu is not None)
    with torch.cuda.device(dev):
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        state = torch.empty((nseq, width - 1, D), dtype=x.dtype, device=dev)
        rc = lib().pe_causal_conv(ctypes.byref(d), _ptr(x), _ptr(weight), _ptr(bias), _ptr(first), _ptr(cu), _ptr(y),
                                  _ptr(state), runtime.raw_stream(dev.index))
    runtime.check(rc, "pe_causal_conv")
    return y, state


def causal_conv_step(x: torch.Tensor, weight: torch.Tensor, state: torch.Tensor, bias: torch.Tensor | None = None, *,
                     activation: str | None = None, slots: torch.Tensor | None = None) -> torch.Tensor:
    """``causal_conv`` of one further token of each of B sequences: x [B, D],
    ``state`` [S, width - 1, D], contiguous, the cache of their last inputs,
    updated in place.  Row b uses state ``slots[b]`` (int32 [B] on the GPU, no
    two rows the same; none: state b); a slot outside [0, S) marks a row
    without a sequence, whose output is zero.  Returns y [B, D]."""
    what = "causal_conv_step"
    if x.dim() != 2:
        raise ValueError(f"{what}: x must be [B, D], got shape {tuple(x.shape)}")
    B, D = x.shape
    width, weight, bias = _conv_operands(what, x, weight, bias, activation)
    of_type(what, x.dtype, state=state)
    S = _cache(what, state, (width - 1, D), B, slots)
    slots = _index(what, "slots", slots, B)
    no_grad(what, x, weight, bias, state)
    dev = same_gpu(what, x, weight=weight, bias=bias, state=state, slots=slots)
    x = inner(x)
    d = abi.ConvDesc(dtype=DTYPES[x.dtype], width=width, silu=activation is not None, nseq=B, D=D, x_bs=x.stride(0),
                     nslots=S, x_numel=extent(x))
    with torch.cuda.device(dev):
        y = torch.empty((B, D), dtype=x.dtype, device=dev)
        rc = lib().pe_causal_conv_step(ctypes.byref(d), _ptr(x), _ptr(weight), _ptr(bias), _ptr(state), _ptr(slots),
                                       _ptr(y), runtime.raw_stream(dev.index))
    runtime.check(rc, "pe_causal_conv_step")
    return y


def _cache(what, state, shape, B, slots) -> int:
    """The rows of a cache of states [S, *shape]."""
    if state.dim() != 1 + len(shape) or tuple(state.shape[1:]) != tuple(shape) or not state.is_contiguous():
        raise ValueError(f"{what}: state must be contiguous [S, {', '.join(map(str, shape))}], got shape "
                         f"{tuple(state.shape)}, strides {state.stride()}")
    if slots is None and state.shape[0] < B:
        raise ValueError(f"{what}: {state.shape[0]} states for {B} rows")
    return state.shape[0]


# --------------------------------------------------------------------- scan --

def _scan_desc(what, lead, x, dt, A, B, C, D, z, dt_bias, dt_softplus):
    """Checks the operands of a scan whose tensors start with the axes ``lead``;
    its descriptor (extents without nseq and T), and the operands laid out."""
    if x.dtype not in DTYPES:
        raise TypeError(f"{what}: unsupported dtype {x.dtype} for x")
    H, P = x.shape[-2:]
    if B.dim() != len(lead) + 2 or tuple(B.shape[:-2]) != lead:
        raise ValueError(f"{what}: B must be {list(lead)} + [groups, N], got shape {tuple(B.shape)}")
    G, N = B.shape[-2:]
    if G < 1 or H % G:
        raise ValueError(f"{what}: {H} heads do not share {G} groups of B and C evenly")
    if N > MAX_N:
        raise ValueError(f"{what}: N must be at most {MAX_N}, got {N}")
    of_shape(what, C=(C, B.shape), dt=(dt, (*lead, H)), z=(z, x.shape), A=(A, (H,)), D=(D, (H,)),
             dt_bias=(dt_bias, (H,)))
    of_type(what, x.dtype, B=B, C=C, z=z)
    of_type(what, torch.float32, A=A, D=D, dt_bias=dt_bias)
    if dt.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"{what}: dt must be {x.dtype} or float32, got {dt.dtype}")
    no_grad(what, x, dt, A, B, C, D, z, dt_bias)
    x, B, C = inner(x), inner(B), inner(C)
    z = None if z is None else inner(z)
    A, D, dt_bias = (None if t is None else t.contiguous() for t in (A, D, dt_bias))
    d = abi.ScanDesc(dtype=DTYPES[x.dtype], dt_dtype=DTYPES[dt.dtype], softplus=bool(dt_softplus), H=H, P=P, G=G, N=N,
                     x_hs=x.stride(-2), dt_hs=dt.stride(-1), b_gs=B.stride(-2), c_gs=C.stride(-2),
                     x_numel=extent(x), dt_numel=extent(dt), b_numel=extent(B), c_numel=extent(C))
    if z is not None:
        d.z_hs, d.z_numel = z.stride(-2), extent(z)
    return d, x, dt, A, B, C, D, z, dt_bias


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, *,
                   D: torch.Tensor | None = None, z: torch.Tensor | None = None, dt_bias: torch.Tensor | None = None,
                   dt_softplus: bool = False, initial_state: torch.Tensor | None = None,
                   cu_seqlens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Selective state-space scan of prompts: per sequence and head h, with
    group g = h // (H // G) of B and C,

        d_t = dt_t + dt_bias (through log(1 + exp(.)) if ``dt_softplus``)
        S_t = exp(A d_t) S_{t-1} + d_t x_t B_t^T            [P, N]
        y_t = (S_t C_t + D x_t) * (z_t / (1 + exp(-z_t)) if z is given)

    x, z [nseq, T, H, P], dt [nseq, T, H] (x's dtype or float32), B, C [nseq,
    T, G, N] with N <= 256, any strides but along the last axis; or packed,
    without the first axis, with ``cu_seqlens`` (int32 offsets on the GPU, nseq +
    1 of them, from 0 up; tokens past the last get y = 0).  A, D, dt_bias are
    float32 [H]; ``initial_state`` float32 [nseq, H, P, N] (none: zeros).
    Returns y (x's shape and dtype) and the float32 states after each
    sequence."""
    what = "selective_scan"
    nseq, T, cu = _sequences(what, x, cu_seqlens, 4)
    packed = cu is not None
    lead = (T,) if packed else (nseq, T)
    d, x, dt, A, B, C, D, z, dt_bias = _scan_desc(what, lead, x, dt, A, B, C, D, z, dt_bias, dt_softplus)
    of_type(what, torch.float32, initial_state=initial_state)
    of_shape(what, initial_state=(initial_state, (nseq, d.H, d.P, d.N)))
    no_grad(what, initial_state)
    dev = same_gpu(what, x, dt=dt, A=A, B=B, C=C, D=D, z=z, dt_bias=dt_bias, initial_state=initial_state,
                   cu_seqlens=cu)
    first = None if initial_state is None else initial_state.contiguous()
    d.nseq, d.T = nseq, T
    d.x_bs, d.x_ts = _lead(x, packed)
    d.dt_bs, d.dt_ts = _lead(dt, packed)
    d.b_bs, d.b_ts = _lead(B, packed)
    d.c_bs, d.c_ts = _lead(C, packed)
    if z is not None:
        d.z_bs, d.z_ts = _lead(z, packed)
    core = lib()
    with torch.cuda.device(dev):
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        state = torch.empty((nseq, d.H, d.P, d.N), dtype=torch.float32, device=dev)
        ws_bytes = core.pe_selective_scan_workspace_bytes(ctypes.byref(d), packed)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
        rc = core.pe_selective_scan(ctypes.byref(d), _ptr(x), _ptr(dt), _ptr(A), _ptr(B), _ptr(C), _ptr(D), _ptr(z),
                                    _ptr(dt_bias), _ptr(first), _ptr(cu), _ptr(y), _ptr(state), _ptr(ws), ws_bytes,
                                    runtime.raw_stream(dev.index))
    runtime.check(rc, "pe_selective_scan")
    return y, state


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                        state: torch.Tensor, *, D: torch.Tensor | None = None, z: torch.Tensor | None = None,
                        dt_bias: torch.Tensor | None = None, dt_softplus: bool = False,
                        slots: torch.Tensor | None = None) -> torch.Tensor:
    """``selective_scan`` of one further token of each of n sequences: x, z [n,
    H, P], dt [n, H], B, C [n, G, N], ``state`` float32 [S, H, P, N],
    contiguous, the cache of their states, updated in place.  Row i uses state
    ``slots[i]`` (int32 [n] on the GPU, no two rows the same; none: state i); a
    slot outside [0, S) marks a row without a sequence, whose output is zero.
    Returns y [n, H, P] of x's dtype."""
    what = "selective_scan_step"
    if x.dim() != 3:
        raise ValueError(f"{what}: x must be [n, H, P], got shape {tuple(x.shape)}")
    n = x.shape[0]
    d, x, dt, A, B, C, D, z, dt_bias = _scan_desc(what, (n,), x, dt, A, B, C, D, z, dt_bias, dt_softplus)
    of_type(what, torch.float32, state=state)
    d.nslots = _cache(what, state, (d.H, d.P, d.N), n, slots)
    slots = _index(what, "slots", slots, n)
    no_grad(what, state)
    dev = same_gpu(what, x, dt=dt, A=A, B=B, C=C, D=D, z=z, dt_bias=dt_bias, state=state, slots=slots)
    d.nseq = n
    d.x_bs, d.dt_bs, d.b_bs, d.c_bs = x.stride(0), dt.stride(0), B.stride(0), C.stride(0)
    if z is not None:
        d.z_bs = z.stride(0)
    with torch.cuda.device(dev):
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        rc = lib().pe_selective_scan_step(ctypes.byref(d), _ptr(x), _ptr(dt), _ptr(A), _ptr(B), _ptr(C), _ptr(D),
                                          _ptr(z), _ptr(dt_bias), _ptr(state), _ptr(slots), _ptr(y),
                                          runtime.raw_stream(dev.index))
    runtime.check(rc, "pe_selective_scan_step")
    return y
