"""Scans whose step sizes lie far apart: a time-major buffer shared by many
channels, of which a call takes a few."""
import pytest
import torch

import ssm_util as u
from pto_einsum.ssm import DTYPES
from test_gpu_ssm import _cuda, _scan_case
from test_gpu_ssm_pieces import _check_scan
from test_ssm_plan import _bytes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,P,ts", [(torch.float16, 16, 9000001), (torch.bfloat16, 48, 5700001),
                                        (torch.float32, 64, 8500001)], ids=["two", "three", "four"])
def test_steps_far_apart(dtype, P, ts):
    """Pieces of 400 tokens, whose 255th step size (with three waves a block the
    383rd) lies past 2^31 elements from the first."""
    from pto_einsum import selective_scan

    T, H, nseq, N, G = 400, 64, 24, 16, 1
    assert _bytes(nseq=nseq, T=T, H=H, P=P, N=N, dtype=DTYPES[dtype], dt_dtype=DTYPES[dtype]) == 0   # one piece each
    one = _scan_case(dtype, [T], H, P, G, N, seed=P)
    t = {k: _cuda(v) for k, v in one.items()}
    far = torch.empty(T * ts, dtype=dtype, device="cuda").as_strided((nseq, T, H), (H, ts, 1))
    far.copy_(t["dt"][None].expand(nseq, -1, -1))
    print(f"selective_scan {dtype} P {P} steps {ts} apart", flush=True)

    def wide(v):
        return v[None].expand(nseq, *v.shape)

    y, st = selective_scan(wide(t["x"]), far, t["A"], wide(t["B"]), wide(t["C"]), D=t["D"], z=wide(t["z"]),
                           dt_bias=t["dt_bias"], dt_softplus=True, initial_state=t["st"].expand(nseq, -1, -1, -1))
    _check_scan(y[0], st[:1], one, [T], dtype)
    for i in range(1, nseq):
        assert torch.equal(y[i], y[0]) and torch.equal(st[i], st[0])
