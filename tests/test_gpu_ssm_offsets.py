"""Packed prompts whose offsets start past the buffer's first token, and offsets
that make no sense: outputs of tokens that no sequence has are zero whatever
memory held, and nothing beside the outputs is written."""
import ctypes

import pytest
import torch

import ssm_util as u
from pto_einsum import abi, runtime
from pto_einsum.ssm import DTYPES
from test_gpu_ssm import _check_conv, _check_scan, _conv_case, _cuda, _scan_case

pytestmark = pytest.mark.gpu


def _stale(n, dtype):
    """NaN in the memory that the allocator gives out next for n elements."""
    t = torch.full((n,), float("nan"), dtype=dtype, device="cuda")
    torch.cuda.synchronize()
    del t


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("cu", [[5, 20, 60, 90], [40, 40, 90, 100], [100, 100, 100, 100], [3, 4, 4, 9]],
                         ids=["late", "empty", "none", "few"])
def test_tokens_before_the_first_sequence(dtype, cu):
    from pto_einsum import causal_conv, selective_scan

    T, H, P, N = (100 if cu[0] != 3 else 12), 2, 32, 64
    c = _scan_case(dtype, [T], H, P, 1, N, seed=cu[0])
    t = {k: _cuda(v) for k, v in c.items()}
    first = torch.randn(3, H, P, N, generator=torch.Generator().manual_seed(0))
    offsets = torch.tensor(cu, dtype=torch.int32).cuda()
    first_gpu = first.cuda()
    print(f"selective_scan {dtype} offsets {cu}", flush=True)
    _stale(T * H * P, dtype)
    y, st = selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], D=t["D"], z=t["z"], dt_bias=t["dt_bias"],
                           dt_softplus=True, initial_state=first_gpu, cu_seqlens=offsets)
    assert bool((y[:cu[0]] == 0).all()) and bool((y[cu[3]:] == 0).all())
    lens = [b - a for a, b in zip(cu, cu[1:])]
    cut = {k: (v[cu[0]:cu[3]] if k in ("x", "dt", "B", "C", "z") else v) for k, v in c.items()}
    _check_scan(y[cu[0]:cu[3]], st, {**cut, "st": first}, lens, dtype)
    x, w, b, cs = _conv_case(dtype, [T, 0, 0], 24, 4)
    _stale(T * 24, dtype)
    y, state = causal_conv(x.cuda(), w.cuda(), b.cuda(), initial_state=cs.cuda(), cu_seqlens=offsets)
    assert bool((y[:cu[0]] == 0).all()) and bool((y[cu[3]:] == 0).all())
    _check_conv(y[cu[0]:cu[3]], state, x[cu[0]:cu[3]], w, b, False, cs, lens, dtype)


class Guarded:
    """A tensor between two stretches of a value that nothing computes."""

    def __init__(self, shape, dtype, pad=4096):
        n = torch.Size(shape).numel()
        self.whole = torch.full((n + 2 * pad,), 12345.0, dtype=dtype, device="cuda")
        self.part, self.pad = self.whole[pad:pad + n].view(shape), pad

    def intact(self):
        return bool((self.whole[:self.pad] == 12345.0).all()) and bool((self.whole[-self.pad:] == 12345.0).all())


@pytest.mark.parametrize("T", [200, 12], ids=["chunks", "rows"])
@pytest.mark.parametrize("cu", [[0, 150, 20, 200], [-5, 90, 1 << 30, 7], [200, 200, 0, 0], [7, 3, 5, 1]])
def test_falling_offsets_write_their_outputs_only(cu, T):
    """The C entry points with guards around what they write."""
    dtype, H, P, N, D, W = torch.float16, 2, 32, 64, 50, 4
    c = _scan_case(dtype, [T], H, P, 1, N, seed=4, gate=False)
    t = {k: _cuda(v) for k, v in c.items()}
    before = {k: v.clone() for k, v in t.items() if v is not None}
    offsets = torch.tensor(cu, dtype=torch.int32).cuda()
    lib, stream = abi.bind(), runtime.raw_stream(0)
    d = abi.ScanDesc(DTYPES[dtype], DTYPES[dtype], 1, 0, 3, T, H, P, 1, N, 0, H * P, P, 0, 0, 0, 0, H, 1, 0, N, N, 0, N, N, 0,
                     T * H * P, 0, T * H, T * N, T * N)
    size = lib.pe_selective_scan_workspace_bytes(ctypes.byref(d), 1)
    y, st, ws = Guarded((T, H, P), dtype), Guarded((3, H, P, N), torch.float32), Guarded((size // 4,), torch.float32)
    print(f"offsets {cu} of {T} tokens", flush=True)
    rc = lib.pe_selective_scan(ctypes.byref(d), t["x"].data_ptr(), t["dt"].data_ptr(), t["A"].data_ptr(),
                               t["B"].data_ptr(), t["C"].data_ptr(), t["D"].data_ptr(), None, t["dt_bias"].data_ptr(),
                               None, offsets.data_ptr(), y.part.data_ptr(), st.part.data_ptr(), ws.part.data_ptr(),
                               size, stream)
    assert rc == 0, runtime.last_error()
    x = torch.randn(T, D, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    w = torch.ones(D, W, dtype=dtype, device="cuda")
    cy, cs = Guarded((T, D), dtype), Guarded((3, W - 1, D), dtype)
    cd = abi.ConvDesc(DTYPES[dtype], W, 1, 0, 3, T, D, 0, D, 0, T * D)
    rc = lib.pe_causal_conv(ctypes.byref(cd), x.data_ptr(), w.data_ptr(), None, None, offsets.data_ptr(),
                            cy.part.data_ptr(), cs.part.data_ptr(), stream)
    assert rc == 0, runtime.last_error()
    torch.cuda.synchronize()
    assert y.intact() and st.intact() and ws.intact() and cy.intact() and cs.intact()
    assert all(torch.equal(t[k], v) for k, v in before.items())
    assert offsets.tolist() == cu
