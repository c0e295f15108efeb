"""What the norms, the row quantiser and the 8-bit product refuse, on the CPU: all
checks come before the GPU is touched."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from pto_einsum import abi, gated_norm, matmul_q8, quantize_q8, residual_norm, runtime

f16, bf16, f32, i8 = torch.float16, torch.bfloat16, torch.float32, torch.int8
z = torch.zeros


@pytest.mark.parametrize("x,err,text", [
    (z(3, 4), ValueError, "GPU"),
    (z(3, 4, dtype=torch.float64), TypeError, "dtype"),
    (z(3, 4, dtype=i8), TypeError, "dtype"),
    (z(()), ValueError, "axis"),
    (z(3, 4, requires_grad=True), RuntimeError, "gradient"),
])
def test_quantize(x, err, text):
    with pytest.raises(err, match=text):
        quantize_q8(x)


def gated_args(**kw):
    return {**dict(x=z(2, 12, dtype=f16), weight=z(12, dtype=f16), z=z(2, 12, dtype=f16)), **kw}


@pytest.mark.parametrize("kw,err,text", [
    (dict(), ValueError, "GPU"),
    (dict(x=z(2, 12, dtype=torch.int32)), TypeError, "dtype"),
    (dict(weight=z(11, dtype=f16)), ValueError, "weight"),
    (dict(weight=z(12)), TypeError, "weight"),
    (dict(z=z(12, dtype=f16)), ValueError, "z must"),
    (dict(z=z(2, 12)), TypeError, "z must"),
    (dict(groups=5), ValueError, "groups"),
    (dict(groups=0), ValueError, "groups"),
    (dict(x=z(1, 16386, dtype=f16), weight=None, z=None, groups=8193, quantize=True), ValueError, "8192"),
    (dict(eps=-1e-5), ValueError, "eps"),
    (dict(eps=float("nan")), ValueError, "eps"),
    (dict(eps=float("inf")), ValueError, "eps"),
    (dict(eps=1e39), ValueError, "eps"),
    (dict(eps=torch.tensor(1e-5)), TypeError, "eps"),
    (dict(groups=torch.tensor(2)), TypeError, "groups"),
    (dict(groups=2.0), TypeError, "integer"),
    (dict(z=z(2, 12, dtype=f16, requires_grad=True)), RuntimeError, "gradient"),
    (dict(weight=z(12, dtype=f16, requires_grad=True)), RuntimeError, "gradient"),
])
def test_gated(kw, err, text):
    with pytest.raises(err, match=text):
        gated_norm(**gated_args(**kw))


def residual_args(**kw):
    return {**dict(x=z(2, 3, 12, dtype=f16), residual=z(2, 3, 12, dtype=f16), weight=z(12, dtype=f16),
                   post_weight=z(12, dtype=f16), gate=z(12, dtype=f16)), **kw}


@pytest.mark.parametrize("kw,err,text", [
    (dict(), ValueError, "GPU"),
    (dict(residual=z(2, 3, 12)), ValueError, "GPU"),
    (dict(gate=z(2, 1, 1, dtype=f16)), ValueError, "GPU"),
    (dict(residual=z(2, 3, 12, dtype=bf16)), TypeError, "residual"),
    (dict(residual=z(3, 12, dtype=f16)), ValueError, "residual"),
    (dict(weight=z(1, dtype=f16)), ValueError, "weight"),
    (dict(post_weight=z(12)), TypeError, "post_weight"),
    (dict(gate=z(2, dtype=f16)), ValueError, "gate"),
    (dict(gate=z(3, 3, 12, dtype=f16)), ValueError, "gate"),
    (dict(gate=z(1, 2, 3, 12, dtype=f16)), ValueError, "gate"),
    (dict(gate=z(12)), TypeError, "gate"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(scale=torch.tensor(0.5)), TypeError, "scale"),
    (dict(gate=z(12, dtype=f16, requires_grad=True)), RuntimeError, "gradient"),
    (dict(residual=z(2, 3, 12, dtype=f16, requires_grad=True)), RuntimeError, "gradient"),
])
def test_residual(kw, err, text):
    with pytest.raises(err, match=text):
        residual_norm(**residual_args(**kw))


def product_args(**kw):
    return {**dict(x=z(2, 3, 32, dtype=f16), weight=z(5, 32, dtype=i8), weight_scales=z(5), bias=z(5)), **kw}


@pytest.mark.parametrize("kw,err,text", [
    (dict(), ValueError, "GPU"),
    (dict(x=z(2, 32, dtype=i8), scales=z(2)), ValueError, "GPU"),
    (dict(bias=z(5, dtype=f16)), ValueError, "GPU"),
    (dict(dtype=bf16, bias=z(5, dtype=bf16)), ValueError, "GPU"),
    (dict(x=z(2, 32, dtype=torch.int16)), TypeError, "dtype"),
    (dict(x=z(())), ValueError, "axis"),
    (dict(x=z(2, 31, dtype=f16)), ValueError, "x must"),
    (dict(weight=z(5, 32, dtype=torch.uint8)), TypeError, "weight"),
    (dict(weight=z(32, dtype=i8)), TypeError, "weight"),
    (dict(weight_scales=z(4)), ValueError, "weight_scales"),
    (dict(weight_scales=z(5, dtype=f16)), TypeError, "weight_scales"),
    (dict(x=z(2, 32, dtype=i8)), ValueError, "scales"),
    (dict(scales=z(2, 3)), ValueError, "scales"),
    (dict(x=z(2, 32, dtype=i8), scales=z(2, 1)), ValueError, "scales"),
    (dict(x=z(2, 32, dtype=i8), scales=z(2, dtype=f16)), TypeError, "scales"),
    (dict(bias=z(4)), ValueError, "bias"),
    (dict(bias=z(5, dtype=bf16)), TypeError, "bias"),
    (dict(dtype=torch.float64), TypeError, "dtype"),
    (dict(dtype=i8), TypeError, "dtype"),
    (dict(x=z(1, 131072, dtype=f16), weight=z(5, 131072, dtype=i8)), ValueError, "131071"),
    (dict(x=z(2, 3, 32, dtype=f16, requires_grad=True)), RuntimeError, "gradient"),
    (dict(weight_scales=z(5, requires_grad=True)), RuntimeError, "gradient"),
])
def test_product(kw, err, text):
    with pytest.raises(err, match=text):
        matmul_q8(**product_args(**kw))


CALLS = [(quantize_q8, dict(x=z(3, 4)), ("x",)),
         (gated_norm, gated_args(), ("x", "weight", "z")),
         (residual_norm, residual_args(), ("x", "residual", "weight", "post_weight", "gate")),
         (matmul_q8, product_args(), ("x", "weight_scales", "bias"))]


@pytest.mark.parametrize("f,args,name", [(f, a, n) for f, a, names in CALLS for n in names],
                         ids=[f"{f.__name__}-{n}" for f, _, names in CALLS for n in names])
def test_tangents_are_refused(f, args, name):
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(**{**args, name: dual})


# ------------------------------------------------------------------ C entries --

def status(name, d, pointers, *more):
    """The status of a call whose operands lie at an address that nothing may read."""
    lib = abi.bind()
    rc = getattr(lib, name)(ctypes.byref(d) if d is not None else None, *pointers, *more)
    return rc, runtime.last_error()


def rows_desc(**kw):
    return abi.RowsDesc(**{**dict(rows0=2, rows1=3, D=20, groups=1, x_s0=60, x_s1=20, g_s0=60, g_s1=20, r_s0=60, r_s1=20,
                                  q_ms=32, x_numel=120, g_numel=120, r_numel=120, eps=1e-5, scale=1.0), **kw})


INVALID, BOUNDS, UNSUPPORTED, WORKSPACE = -1, -2, -3, -4


@pytest.mark.parametrize("kw,want", [
    (dict(dtype=3), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED), (dict(rows0=-1), INVALID), (dict(D=-4), INVALID),
    (dict(groups=0), INVALID), (dict(groups=3), INVALID), (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID),
    (dict(x_numel=119), BOUNDS), (dict(x_s0=-60), BOUNDS), (dict(x_s1=1 << 62, rows1=1 << 20), BOUNDS),
    (dict(rows0=1 << 40, rows1=1 << 40), UNSUPPORTED), (dict(rows0=1 << 31, rows1=1, x_s0=0), UNSUPPORTED),
    (dict(D=1 << 32), UNSUPPORTED), (dict(q_ms=16), INVALID), (dict(q_ms=144), INVALID), (dict(q_ms=20), INVALID),
])
def test_rows_descriptor(kw, want):
    assert status("pe_quantize_q8", rows_desc(**kw), (64, 64, 64, None))[0] == want


def test_norm_descriptors():
    at = 64
    assert status("pe_gated_norm", None, (at, at, at, at, None, None, None))[0] == INVALID
    assert status("pe_gated_norm", rows_desc(g_numel=119), (at, at, at, at, None, None, None))[0] == BOUNDS
    assert status("pe_gated_norm", rows_desc(gate_row=1), (at, at, at, at, None, None, None))[0] == INVALID
    assert status("pe_gated_norm", rows_desc(), (None, at, at, at, None, None, None))[0] == INVALID
    assert status("pe_gated_norm", rows_desc(), (at, at, at, None, None, None, None))[0] == INVALID
    assert status("pe_gated_norm", rows_desc(), (at, at, at, None, None, at, None))[0] == INVALID
    assert status("pe_gated_norm", rows_desc(D=16384, groups=16384, rows0=0, q_ms=16384),
                  (at, at, at, None, at, at, None))[0] == UNSUPPORTED
    args = (at, at, at, at, at, at, at, None, None, None)
    assert status("pe_residual_norm", rows_desc(groups=2), args)[0] == INVALID
    assert status("pe_residual_norm", rows_desc(res_dtype=2), args)[0] == UNSUPPORTED
    assert status("pe_residual_norm", rows_desc(dtype=1, res_dtype=2), args)[0] == UNSUPPORTED
    assert status("pe_residual_norm", rows_desc(r_numel=1), args)[0] == BOUNDS
    assert status("pe_residual_norm", rows_desc(gate_row=1, g_numel=80), args)[0] == BOUNDS
    for i in (0, 1, 5, 6):
        assert status("pe_residual_norm", rows_desc(), args[:i] + (None,) + args[i + 1:])[0] == INVALID


def q8_desc(**kw):
    return abi.Q8Desc(**{**dict(x_dtype=3, y_dtype=0, bias_dtype=0, M=4, N=5, K=100, x_ms=112, w_ns=112, x_numel=448,
                                w_numel=560), **kw})


@pytest.mark.parametrize("kw,want", [
    (dict(x_dtype=4), UNSUPPORTED), (dict(y_dtype=3), UNSUPPORTED), (dict(bias_dtype=1), UNSUPPORTED),
    (dict(kernel=-1), INVALID), (dict(kernel=9), INVALID), (dict(M=-1), INVALID), (dict(K=131072, x_ms=131072, w_ns=131072), UNSUPPORTED), (dict(M=1 << 31), UNSUPPORTED),
    (dict(x_ms=100), UNSUPPORTED), (dict(x_ms=96), UNSUPPORTED), (dict(w_ns=104), UNSUPPORTED), (dict(w_ns=96), UNSUPPORTED),
    (dict(w_ns=(1 << 23) + 16), UNSUPPORTED), (dict(x_ms=-112), UNSUPPORTED),
    (dict(x_numel=447), BOUNDS), (dict(w_numel=559), BOUNDS), (dict(x_dtype=1, x_ms=100, x_numel=399), BOUNDS),
    (dict(x_dtype=1, x_ms=100, x_numel=400), WORKSPACE),
])
def test_product_descriptor(kw, want):
    at = 64
    assert status("pe_matmul_q8", q8_desc(**kw), (at, at, at, at, None, at, None), 0, None)[0] == want


def test_product_pointers():
    at = 64
    args = (at, at, at, at, None, at, None)
    for i in (0, 1, 2, 3, 5):
        assert status("pe_matmul_q8", q8_desc(), args[:i] + (None,) + args[i + 1:], 0, None)[0] == INVALID
    for i in (0, 2):
        assert status("pe_matmul_q8", q8_desc(), args[:i] + (at + 8,) + args[i + 1:], 0, None)[0] == UNSUPPORTED
    d = q8_desc(x_dtype=1, x_ms=100, x_numel=400)
    need = abi.bind().pe_matmul_q8_workspace_bytes(ctypes.byref(d))
    assert need >= 4 * 112 + 16
    assert status("pe_matmul_q8", d, args[:6] + (at,), need - 1, None)[0] == WORKSPACE
    assert status("pe_matmul_q8", d, args[:6] + (at + 4,), need, None)[0] == WORKSPACE
    assert abi.bind().pe_matmul_q8_workspace_bytes(ctypes.byref(q8_desc(M=-1))) == 0
