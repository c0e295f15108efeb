"""How a prompt's scan is cut, as far as its workspace shows it, and the
workspace's refusals; on the CPU."""
import ctypes

import pytest

from pto_einsum import abi, runtime

DENSE = dict(dtype=1, dt_dtype=1, nseq=2, T=4096, H=64, P=64, G=1, N=128)


def _desc(**kw):
    a = {**DENSE, **kw}
    h, p, g, n, t = a["H"], a["P"], a["G"], a["N"], a["T"]
    a.update(x_bs=t * h * p, x_ts=h * p, x_hs=p, dt_bs=t * h, dt_ts=h, dt_hs=1, b_bs=t * g * n, b_ts=g * n, b_gs=n,
             c_bs=t * g * n, c_ts=g * n, c_gs=n, x_numel=1 << 40, dt_numel=1 << 40, b_numel=1 << 40, c_numel=1 << 40)
    return abi.ScanDesc(**a)


def _bytes(packed=0, **kw):
    return abi.bind().pe_selective_scan_workspace_bytes(ctypes.byref(_desc(**kw)), packed)


def test_workspace_bytes():
    # a state of 64 x 128 for each head and piece, and its decay
    state = 64 * 64 * 128 * 4
    assert _bytes() > 2 * 2 * state and _bytes() % 16 == 0
    assert _bytes() < 2 * 4096 // 64 * (state + 64 * 4) + 64
    assert _bytes(T=16) == 0                      # token by token
    assert _bytes(N=7) == 0 and _bytes(P=7) == 0
    assert _bytes(nseq=4096, T=128) == 0          # enough sequences: one piece each
    assert _bytes(T=0) == 0 and _bytes(nseq=0) == 0
    assert _bytes(dtype=9) == 0                   # refused by the call itself
    assert _bytes(packed=1, T=200, nseq=3) > 0    # how long sequences are shows on the GPU


@pytest.mark.parametrize("ws,size", [(None, 1 << 40), (16, 1024), (8, 1 << 40)], ids=["none", "small", "misaligned"])
def test_workspace_refusals(ws, size):
    d = _desc()
    args = [16] * 5 + [None, None, None, None, None, 16, 16, ws, size, None]
    assert abi.bind().pe_selective_scan(ctypes.byref(d), *args) == -4
    assert "workspace" in runtime.last_error()
