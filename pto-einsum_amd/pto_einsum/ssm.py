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
``slots`` are read on the GPU; offsets outside the buffer are clamped to it (where
they fall, the outputs and new states mean nothing), and slots outside the cache
mark rows without a sequence.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools

import torch
from torch.autograd import forward_ad

from . import abi, launch, runtime

DTYPES = {torch.float32: launch.DT_F32, torch.float16: launch.DT_F16, torch.bfloat16: launch.DT_BF16}
MAX_WIDTH = 8      # PE_CONV_MAX_WIDTH
MAX_N = 256        # PE_SCAN_MAX_N


@functools.lru_cache(maxsize=None)
def lib():
    """The core library with its argument types set."""
    return abi.bind()


# A call of single tokens lasts a few microseconds on the GPU, and checking ten
# operands and filling a descriptor takes longer than that.  So the descriptor of
# operands that passed is kept by their layouts -- shapes, strides, dtypes and
# flags, nothing of the tensors themselves -- and a later call of the same layouts
# only looks at devices and gradients.
_plans: dict = {}


def remember(key, plan):
    """Keeps a plan; all are dropped when there are many (prompts of ever new
    lengths)."""
    if len(_plans) >= 4096:
        _plans.clear()
    _plans[key] = plan
    return plan


def layout(t):
    return None if t is None else (t.shape, t.stride(), t.dtype)


def extent(t: torch.Tensor) -> int:
    """Elements from t's first to its last, which torch keeps inside its storage."""
    return 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else 0


def inner(t: torch.Tensor) -> torch.Tensor:
    """t with its last axis contiguous and no negative or overlapping inner
    layout: t itself where that holds (other axes keep their strides)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def dense(t):
    return None if t is None else t.contiguous()


def check(what: str, name: str, t, shape, dtype) -> None:
    """t, where it is given, has that shape and dtype."""
    if t is not None:
        if t.shape != shape:
            raise ValueError(f"{what}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
        if t.dtype is not dtype:
            raise TypeError(f"{what}: {name} must be {dtype}, got {t.dtype}")


def ready(what: str, x, *others) -> int:
    """The index of the GPU that x and all others (None: not given) live on; no
    gradient is asked of them, and none carries a forward-mode tangent."""
    index = x.get_device()
    grad = torch.is_grad_enabled()
    # (Without a dual level open there are no tangents, and asking every operand
    # for its own costs 0.4 us each.)
    if forward_ad._current_level >= 0:
        for t in (x, *others):
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} has no forward-mode gradient: call it on detached operands")
    if grad and x.requires_grad:
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or on detached operands")
    alike = True
    for t in others:
        if t is not None:
            if grad and t.requires_grad:
                raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or on detached operands")
            alike = alike and t.get_device() == index
    if index < 0 or not x.is_cuda:
        raise ValueError(f"{what}: operands must live on a GPU, got {x.device}")
    if not alike:
        where = sorted({str(t.device) for t in others if t is not None} | {str(x.device)})
        raise ValueError(f"{what}: operands must all live on one GPU, got {', '.join(where)}")
    return index


_HERE = contextlib.nullcontext()


def on(index: int):
    """A context in which GPU ``index`` is the current device."""
    return _HERE if torch.cuda.current_device() == index else torch.cuda.device(index)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _index(what: str, name: str, t, length: int | None):
    """An int32 index vector, contiguous."""
    if t is None:
        return None
    if t.dtype is not torch.int32 or t.dim() != 1:
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
    if activation is not None and activation != "silu":
        raise ValueError(f"{what}: activation must be None or 'silu', got {activation!r}")
    D = x.shape[-1]
    if weight.dim() != 2 or weight.shape[0] != D:
        raise ValueError(f"{what}: weight must be [{D}, width], got shape {tuple(weight.shape)}")
    width = weight.shape[1]
    if not 2 <= width <= MAX_WIDTH:
        raise ValueError(f"{what}: width must be 2 to {MAX_WIDTH}, got {width}")
    if weight.dtype is not x.dtype:
        raise TypeError(f"{what}: weight must be {x.dtype}, got {weight.dtype}")
    check(what, "bias", bias, (D,), x.dtype)
    return width, weight.contiguous(), dense(bias)


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                activation: str | None = None, initial_state: torch.Tensor | None = None,
                cu_seqlens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Causal convolution of each channel along the tokens of prompts:

        y[t, d] = act(bias[d] + sum_j weight[d, j] * x[t - width + 1 + j, d])

    x [nseq, T, D], or packed [T, D] with ``cu_seqlens`` (int32 offsets on the
    GPU, nseq + 1 of them that do not fall; tokens before the first and from the
    last on get y = 0); weight [D, width] with 2 <= width <= 8; ``activation`` None or "silu".
    ``initial_state`` [nseq, width - 1, D] holds the inputs before each
    sequence's first token, oldest first (none: zeros).  Returns y of x's
    shape and the state after each sequence, both of x's dtype."""
    what = "causal_conv"
    key = (what, layout(x), layout(weight), layout(bias), activation, layout(initial_state), layout(cu_seqlens))
    plan = _plans.get(key)
    if plan is None:
        nseq, T, cu = _sequences(what, x, cu_seqlens, 3)
        D = x.shape[-1]
        width, w, b = _conv_operands(what, x, weight, bias, activation)
        check(what, "initial_state", initial_state, (nseq, width - 1, D), x.dtype)
        ready(what, x, weight, bias, initial_state, cu)
        given, laid = (x, weight, bias, initial_state, cu_seqlens), (inner(x), w, b, dense(initial_state), cu)
        if any(g is not t for g, t in zip(given, laid)):
            return causal_conv(*laid[:3], activation=activation, initial_state=laid[3], cu_seqlens=cu)
        x_bs, x_ts = _lead(x, cu is not None)
        plan = remember(key, (abi.ConvDesc(DTYPES[x.dtype], width, activation is not None, 0, nseq, T, D, x_bs, x_ts, 0,
                                           extent(x)), (nseq, width - 1, D)))
    d, state_shape = plan
    dev = ready(what, x, weight, bias, initial_state, cu_seqlens)
    with on(dev):
        y = x.new_empty(x.shape)
        state = x.new_empty(state_shape)
        rc = lib().pe_causal_conv(ctypes.byref(d), x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(initial_state),
                                  _ptr(cu_seqlens), y.data_ptr(), state.data_ptr(), runtime.raw_stream(dev))
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
    key = (what, layout(x), layout(weight), layout(state), layout(bias), activation, layout(slots))
    d = _plans.get(key)
    if d is None:
        if x.dim() != 2:
            raise ValueError(f"{what}: x must be [B, D], got shape {tuple(x.shape)}")
        B, D = x.shape
        width, w, b = _conv_operands(what, x, weight, bias, activation)
        S = _cache(what, state, (width - 1, D), x.dtype, B, slots)
        at = _index(what, "slots", slots, B)
        ready(what, x, weight, bias, state, slots)
        given, laid = (x, weight, bias, slots), (inner(x), w, b, at)
        if any(g is not t for g, t in zip(given, laid)):
            return causal_conv_step(laid[0], w, state, b, activation=activation, slots=at)
        d = remember(key, abi.ConvDesc(DTYPES[x.dtype], width, activation is not None, 0, B, 0, D, x.stride(0), 0, S,
                                       extent(x)))
    dev = ready(what, x, weight, bias, state, slots)
    with on(dev):
        y = x.new_empty(x.shape)
        rc = lib().pe_causal_conv_step(ctypes.byref(d), x.data_ptr(), weight.data_ptr(), _ptr(bias), state.data_ptr(),
                                       _ptr(slots), y.data_ptr(), runtime.raw_stream(dev))
    runtime.check(rc, "pe_causal_conv_step")
    return y


def _cache(what, state, shape, dtype, B, slots) -> int:
    """The rows of a cache of states [S, *shape]."""
    if state.dtype is not dtype:
        raise TypeError(f"{what}: state must be {dtype}, got {state.dtype}")
    if state.dim() != 1 + len(shape) or state.shape[1:] != shape or not state.is_contiguous():
        raise ValueError(f"{what}: state must be contiguous [S, {', '.join(map(str, shape))}], got shape "
                         f"{tuple(state.shape)}, strides {state.stride()}")
    if slots is None and state.shape[0] < B:
        raise ValueError(f"{what}: {state.shape[0]} states for {B} rows")
    return state.shape[0]


# --------------------------------------------------------------------- scan --

def _scan_operands(what, lead, x, dt, A, B, C, D, z, dt_bias):
    """Checks the operands of a scan whose tensors start with the axes ``lead``;
    (H, P, G, N) and the operands laid out."""
    dtype = x.dtype
    if dtype not in DTYPES:
        raise TypeError(f"{what}: unsupported dtype {dtype} for x")
    H, P = x.shape[-2:]
    if B.dim() != len(lead) + 2 or B.shape[:-2] != lead:
        raise ValueError(f"{what}: B must be {list(lead)} + [groups, N], got shape {tuple(B.shape)}")
    G, N = B.shape[-2:]
    if G < 1 or H % G:
        raise ValueError(f"{what}: {H} heads do not share {G} groups of B and C evenly")
    if N > MAX_N:
        raise ValueError(f"{what}: N must be at most {MAX_N}, got {N}")
    if B.dtype is not dtype:
        raise TypeError(f"{what}: B must be {dtype}, got {B.dtype}")
    check(what, "C", C, B.shape, dtype)
    check(what, "dt", dt, (*lead, H), dtype if dt.dtype is dtype else torch.float32)
    check(what, "z", z, x.shape, dtype)
    heads, f32 = (H,), torch.float32
    check(what, "A", A, heads, f32)
    check(what, "D", D, heads, f32)
    check(what, "dt_bias", dt_bias, heads, f32)
    return (H, P, G, N), (inner(x), dt, A.contiguous(), inner(B), inner(C), dense(D), None if z is None else inner(z),
                          dense(dt_bias))


def _scan_desc(x, dt, B, C, z, softplus, nseq, T, H, P, G, N, slots, lead):
    """The descriptor; ``lead`` gives a tensor's (sequence stride, token stride)."""
    xs, dts, bs, cs = lead(x), lead(dt), lead(B), lead(C)
    zs = (0, 0) if z is None else lead(z)
    z_hs, z_numel = (0, 0) if z is None else (z.stride(-2), extent(z))
    return abi.ScanDesc(DTYPES[x.dtype], DTYPES[dt.dtype], softplus, 0, nseq, T, H, P, G, N, *xs, x.stride(-2), *zs,
                        z_hs, *dts, dt.stride(-1), *bs, B.stride(-2), *cs, C.stride(-2), slots, extent(x), z_numel,
                        extent(dt), extent(B), extent(C))


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
    1 of them that do not fall; tokens before the first and from the last on get
    y = 0).  A, D, dt_bias are float32 [H]; ``initial_state`` float32 [nseq, H, P, N] (none: zeros).
    Returns y (x's shape and dtype) and the float32 states after each
    sequence."""
    what = "selective_scan"
    key = (what, layout(x), layout(dt), layout(A), layout(B), layout(C), layout(D), layout(z), layout(dt_bias),
           bool(dt_softplus), layout(initial_state), layout(cu_seqlens))
    plan = _plans.get(key)
    if plan is None:
        nseq, T, cu = _sequences(what, x, cu_seqlens, 4)
        packed = cu is not None
        given = (x, dt, A, B, C, D, z, dt_bias)
        (H, P, G, N), laid = _scan_operands(what, (T,) if packed else (nseq, T), *given)
        check(what, "initial_state", initial_state, (nseq, H, P, N), torch.float32)
        ready(what, *given, initial_state, cu)
        first = dense(initial_state)
        if any(g is not t for g, t in zip((*given, initial_state, cu_seqlens), (*laid, first, cu))):
            x, dt, A, B, C, D, z, dt_bias = laid
            return selective_scan(x, dt, A, B, C, D=D, z=z, dt_bias=dt_bias, dt_softplus=dt_softplus,
                                  initial_state=first, cu_seqlens=cu)
        d = _scan_desc(x, dt, B, C, z, bool(dt_softplus), nseq, T, H, P, G, N, 0,
                       (lambda t: (0, t.stride(0))) if packed else (lambda t: t.stride()[:2]))
        plan = remember(key, (d, (nseq, H, P, N), lib().pe_selective_scan_workspace_bytes(ctypes.byref(d), packed)))
    d, state_shape, ws_bytes = plan
    dev = ready(what, x, dt, A, B, C, D, z, dt_bias, initial_state, cu_seqlens)
    with on(dev):
        y = x.new_empty(x.shape)
        state = A.new_empty(state_shape)
        ws = A.new_empty(ws_bytes // 4) if ws_bytes else None
        rc = lib().pe_selective_scan(ctypes.byref(d), x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(),
                                     C.data_ptr(), _ptr(D), _ptr(z), _ptr(dt_bias), _ptr(initial_state),
                                     _ptr(cu_seqlens), y.data_ptr(), state.data_ptr(), _ptr(ws), ws_bytes,
                                     runtime.raw_stream(dev))
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
    key = (what, layout(x), layout(dt), layout(A), layout(B), layout(C), layout(state), layout(D), layout(z),
           layout(dt_bias), bool(dt_softplus), layout(slots))
    d = _plans.get(key)
    if d is None:
        if x.dim() != 3:
            raise ValueError(f"{what}: x must be [n, H, P], got shape {tuple(x.shape)}")
        n = x.shape[0]
        given = (x, dt, A, B, C, D, z, dt_bias)
        (H, P, G, N), laid = _scan_operands(what, (n,), *given)
        S = _cache(what, state, (H, P, N), torch.float32, n, slots)
        at = _index(what, "slots", slots, n)
        ready(what, *given, state, slots)
        if any(g is not t for g, t in zip((*given, slots), (*laid, at))):
            x, dt, A, B, C, D, z, dt_bias = laid
            return selective_scan_step(x, dt, A, B, C, state, D=D, z=z, dt_bias=dt_bias, dt_softplus=dt_softplus,
                                       slots=at)
        d = remember(key, _scan_desc(x, dt, B, C, z, bool(dt_softplus), n, 0, H, P, G, N, S,
                                     lambda t: (t.stride(0), 0)))
    dev = ready(what, x, dt, A, B, C, D, z, dt_bias, state, slots)
    with on(dev):
        y = x.new_empty(x.shape)
        rc = lib().pe_selective_scan_step(ctypes.byref(d), x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(),
                                          C.data_ptr(), _ptr(D), _ptr(z), _ptr(dt_bias), state.data_ptr(), _ptr(slots),
                                          y.data_ptr(), runtime.raw_stream(dev))
    runtime.check(rc, "pe_selective_scan_step")
    return y
