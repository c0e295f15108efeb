"""What the state-space operators and the 4-bit product refuse, on the CPU: all
checks come before the GPU is touched."""
import ctypes

import pytest
import torch

from pto_einsum import (abi, causal_conv, causal_conv_step, matvec_q4, runtime, selective_scan, selective_scan_step)

f16, f32 = torch.float16, torch.float32


def conv_args(**kw):
    a = dict(x=torch.zeros(2, 5, 8, dtype=f16), weight=torch.zeros(8, 4, dtype=f16), bias=torch.zeros(8, dtype=f16))
    return {**a, **kw}


@pytest.mark.parametrize("kw,err,text", [
    (dict(), ValueError, "GPU"),
    (dict(x=torch.zeros(2, 5, 8, dtype=torch.float64)), TypeError, "dtype"),
    (dict(x=torch.zeros(5, 8, dtype=f16)), ValueError, "3 axes"),
    (dict(weight=torch.zeros(8, 1, dtype=f16)), ValueError, "width"),
    (dict(weight=torch.zeros(8, 9, dtype=f16)), ValueError, "width"),
    (dict(weight=torch.zeros(7, 4, dtype=f16)), ValueError, "weight"),
    (dict(weight=torch.zeros(8, 4)), TypeError, "weight"),
    (dict(bias=torch.zeros(7, dtype=f16)), ValueError, "bias"),
    (dict(bias=torch.zeros(8)), TypeError, "bias"),
    (dict(activation="gelu"), ValueError, "activation"),
    (dict(initial_state=torch.zeros(2, 4, 8, dtype=f16)), ValueError, "initial_state"),
    (dict(initial_state=torch.zeros(2, 3, 8)), TypeError, "initial_state"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), ValueError, "2 axes"),
    (dict(x=torch.zeros(5, 8, dtype=f16), cu_seqlens=torch.zeros(3, dtype=torch.int64)), TypeError, "int32"),
    (dict(x=torch.zeros(5, 8, dtype=f16), cu_seqlens=torch.zeros(1, dtype=torch.int32)), ValueError, "one sequence"),
    (dict(weight=torch.zeros(8, 4, dtype=f16, requires_grad=True)), RuntimeError, "gradient"),
])
def test_causal_conv(kw, err, text):
    with pytest.raises(err, match=text):
        causal_conv(**conv_args(**kw))


@pytest.mark.parametrize("kw,err,text", [
    (dict(), ValueError, "GPU"),
    (dict(x=torch.zeros(2, 5, 8, dtype=f16)), ValueError, "x must be"),
    (dict(state=torch.zeros(2, 4, 8, dtype=f16)), ValueError, "state"),
    (dict(state=torch.zeros(2, 3, 16, dtype=f16)[..., ::2]), ValueError, "contiguous"),
    (dict(state=torch.zeros(2, 3, 8)), TypeError, "state"),
    (dict(state=torch.zeros(1, 3, 8, dtype=f16)), ValueError, "1 states"),
    (dict(slots=torch.zeros(3, dtype=torch.int32)), ValueError, "slots"),
    (dict(slots=torch.zeros(2, dtype=torch.int64)), TypeError, "slots"),
])
def test_causal_conv_step(kw, err, text):
    a = conv_args(x=torch.zeros(2, 8, dtype=f16), state=torch.zeros(2, 3, 8, dtype=f16))
    with pytest.raises(err, match=text):
        causal_conv_step(**{**a, **kw})


def scan_args(lead=(2, 5), **kw):
    a = dict(x=torch.zeros(*lead, 4, 8, dtype=f16), dt=torch.zeros(*lead, 4, dtype=f16), A=torch.zeros(4),
             B=torch.zeros(*lead, 2, 16, dtype=f16), C=torch.zeros(*lead, 2, 16, dtype=f16))
    return {**a, **kw}


SCAN = [
    (dict(), ValueError, "GPU"),
    (dict(dt=torch.zeros(2, 5, 3, dtype=f16)), ValueError, "dt"),
    (dict(dt=torch.zeros(2, 5, 4, dtype=torch.bfloat16)), TypeError, "dt"),
    (dict(A=torch.zeros(3)), ValueError, "A"),
    (dict(A=torch.zeros(4, dtype=f16)), TypeError, "A"),
    (dict(B=torch.zeros(2, 5, 3, 16, dtype=f16)), ValueError, "groups"),
    (dict(B=torch.zeros(2, 5, 0, 16, dtype=f16)), ValueError, "groups"),
    (dict(B=torch.zeros(2, 5, 2, 257, dtype=f16)), ValueError, "N must"),
    (dict(B=torch.zeros(2, 4, 2, 16, dtype=f16)), ValueError, "B must"),
    (dict(C=torch.zeros(2, 5, 2, 15, dtype=f16)), ValueError, "C"),
    (dict(C=torch.zeros(2, 5, 2, 16)), TypeError, "C"),
    (dict(D=torch.zeros(4, dtype=f16)), TypeError, "D"),
    (dict(z=torch.zeros(2, 5, 4, 7, dtype=f16)), ValueError, "z"),
    (dict(dt_bias=torch.zeros(5)), ValueError, "dt_bias"),
    (dict(x=torch.zeros(2, 5, 4, 8, dtype=torch.float64)), TypeError, "dtype"),
    (dict(A=torch.zeros(4, requires_grad=True)), RuntimeError, "gradient"),
]


@pytest.mark.parametrize("kw,err,text", SCAN + [
    (dict(initial_state=torch.zeros(2, 4, 8, 15)), ValueError, "initial_state"),
    (dict(initial_state=torch.zeros(2, 4, 8, 16, dtype=f16)), TypeError, "initial_state"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), ValueError, "3 axes"),
])
def test_selective_scan(kw, err, text):
    with pytest.raises(err, match=text):
        selective_scan(**scan_args(**kw))


@pytest.mark.parametrize("kw,err,text", [
    (dict(), ValueError, "GPU"),
    (dict(x=torch.zeros(2, 5, 4, 8, dtype=f16)), ValueError, "x must be"),
    (dict(state=torch.zeros(2, 4, 8, 15)), ValueError, "state"),
    (dict(state=torch.zeros(2, 4, 8, 16, dtype=f16)), TypeError, "state"),
    (dict(state=torch.zeros(1, 4, 8, 16)), ValueError, "1 states"),
    (dict(slots=torch.zeros(1, dtype=torch.int32)), ValueError, "slots"),
])
def test_selective_scan_step(kw, err, text):
    a = scan_args(lead=(2,), state=torch.zeros(2, 4, 8, 16))
    with pytest.raises(err, match=text):
        selective_scan_step(**{**a, **kw})


@pytest.mark.parametrize("kw,err,text", [
    (dict(), ValueError, "GPU"),
    (dict(group=16), ValueError, "group"),
    (dict(packed=torch.zeros(3, 25, dtype=torch.int32)), TypeError, "uint8"),
    (dict(packed=torch.zeros(3, 24, dtype=torch.uint8)), ValueError, "packed"),
    (dict(scales=torch.zeros(3, 3, dtype=f16)), ValueError, "scales"),
    (dict(scales=torch.zeros(3, 2)), TypeError, "scales"),
    (dict(zeros=torch.zeros(2, 2, dtype=f16)), ValueError, "zeros"),
    (dict(x=torch.zeros((), dtype=f16)), ValueError, "axis"),
    (dict(x=torch.zeros(2, 50, dtype=torch.int8)), TypeError, "dtype"),
    (dict(x=torch.zeros(2, 50, dtype=f16, requires_grad=True)), RuntimeError, "gradient"),
])
def test_matvec_q4(kw, err, text):
    a = dict(x=torch.zeros(2, 50, dtype=f16), packed=torch.zeros(3, 25, dtype=torch.uint8),
             scales=torch.zeros(3, 2, dtype=f16), group=32)
    with pytest.raises(err, match=text):
        matvec_q4(**{**a, **kw})


# ------------------------------------------------ the C entry points' checks --

def _status(name, d, nargs, ptrs=None):
    """The entry point's status for a descriptor, all pointers null but ``ptrs``;
    no case below reaches a launch."""
    args = [None] * nargs
    for i, v in (ptrs or {}).items():
        args[i] = v
    rc = getattr(abi.bind(), name)(ctypes.byref(d), *args)
    return rc, runtime.last_error()


def _conv(**kw):
    return abi.ConvDesc(**{**dict(dtype=1, width=4, nseq=2, T=5, D=8, x_bs=40, x_ts=8, nslots=2, x_numel=80), **kw})


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=3), -3), (dict(width=1), -3), (dict(width=9), -3), (dict(reserved=1), -1), (dict(T=-1), -1),
    (dict(x_numel=79), -2), (dict(x_bs=-1), -2), (dict(D=1 << 31), -3), (dict(), -1)])
def test_conv_descriptor(kw, status):
    assert _status("pe_causal_conv", _conv(**kw), 8)[0] == status


def test_conv_descriptor_packed_and_step():
    assert _status("pe_causal_conv", _conv(nseq=0), 8, {4: 16})[0] == -1     # offsets, no sequence
    assert _status("pe_causal_conv", _conv(nseq=0), 8)[0] == 0               # nothing to do
    assert _status("pe_causal_conv_step", _conv(x_numel=47), 7)[0] == -2
    assert _status("pe_causal_conv_step", _conv(nslots=1), 7, {0: 16, 1: 16, 3: 16, 5: 16})[0] == -2
    assert _status("pe_causal_conv_step", _conv(nslots=-1), 7)[0] == -1


def _scan(**kw):
    a = dict(dtype=2, dt_dtype=0, nseq=2, T=5, H=4, P=8, G=2, N=16, x_bs=160, x_ts=32, x_hs=8, z_bs=160, z_ts=32,
             z_hs=8, dt_bs=20, dt_ts=4, dt_hs=1, b_bs=160, b_ts=32, b_gs=16, c_bs=160, c_ts=32, c_gs=16, nslots=2,
             x_numel=320, z_numel=320, dt_numel=40, b_numel=320, c_numel=320)
    return abi.ScanDesc(**{**a, **kw})


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=5), -3), (dict(dt_dtype=1), -3), (dict(N=257), -3), (dict(H=5), -1), (dict(G=0), -1),
    (dict(P=-1), -1), (dict(x_numel=319), -2), (dict(dt_numel=39), -2), (dict(b_numel=319), -2),
    (dict(c_gs=-1), -2), (dict(reserved=2), -1), (dict(), -1)])
def test_scan_descriptor(kw, status):
    assert _status("pe_selective_scan", _scan(**kw), 15, {13: 0})[0] == status


def test_scan_descriptor_gate_packed_and_step():
    assert _status("pe_selective_scan", _scan(z_numel=319), 15, {6: 16, 13: 0})[0] == -2
    assert _status("pe_selective_scan", _scan(nseq=0), 15, {9: 16, 13: 0})[0] == -1
    assert _status("pe_selective_scan", _scan(nseq=0), 15, {13: 0})[0] == 0
    everything = {i: 16 for i in (0, 1, 2, 3, 4, 8, 10)}
    assert _status("pe_selective_scan_step", _scan(nslots=1), 12, everything)[0] == -2
    assert _status("pe_selective_scan_step", _scan(), 12)[0] == -1


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=-1), -3), (dict(group=16), -3), (dict(M=-1), -1), (dict(x_numel=99), -2), (dict(N=1 << 31), -3),
    (dict(M=0), 0), (dict(), -1)])
def test_q4_descriptor(kw, status):
    d = abi.Q4Desc(**{**dict(dtype=0, group=32, M=2, N=3, K=50, x_ms=50, x_numel=100), **kw})
    assert _status("pe_matvec_q4", d, 6)[0] == status


STRUCTS = [("pe_conv_desc", abi.ConvDesc), ("pe_scan_desc", abi.ScanDesc), ("pe_q4_desc", abi.Q4Desc)]


def test_struct_layout_matches_c(tmp_path):
    import os
    import subprocess

    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    lines = []
    for c, py in STRUCTS:
        lines.append(f'printf("{c} %zu\\n", sizeof({c}));')
        lines += [f'printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    (tmp_path / "p.cpp").write_text('#include <cstdio>\n#include <cstddef>\n#include "pto_einsum_hip.h"\nint main() {'
                                    + "".join(lines) + "}")
    subprocess.run(["g++", "-std=c++17", "-I", header, str(tmp_path / "p.cpp"), "-o", str(tmp_path / "p")], check=True)
    out = subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout
    vals = dict(line.rsplit(" ", 1) for line in out.splitlines())
    for c, py in STRUCTS:
        assert int(vals[c]) == ctypes.sizeof(py)
        for f, _ in py._fields_:
            assert int(vals[f"{c}.{f}"]) == getattr(py, f).offset, (c, f)
