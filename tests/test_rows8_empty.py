"""Operands without elements, their leading axes in any order."""
import pytest
import torch

from pto_einsum.norm import places
from pto_einsum.quant import _apart

EMPTY = [torch.zeros(4, 3, 2, 0).permute(2, 1, 0, 3), torch.zeros(2, 3, 0).transpose(0, 1), torch.zeros(5, 4, 0, 8).transpose(0, 1),
         torch.zeros(3, 4, 5, 0)[::2, 1:3].permute(1, 2, 0, 3), torch.zeros(6, 0)[::3], torch.zeros(0)]


@pytest.mark.parametrize("t", EMPTY, ids=[str(tuple(t.shape)) for t in EMPTY])
def test_strides(t):
    rows0, rows1, (pair, none) = places(t.shape[:-1], (t, None))
    assert rows0 * rows1 == t.shape[:-1].numel() and pair is not None and none == (0, 0)
    assert _apart(t) is not None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("t", EMPTY, ids=[str(tuple(t.shape)) for t in EMPTY])
def test_calls(t, dtype):
    from pto_einsum import gated_norm, matmul_q8, quantize_q8, residual_norm

    x = torch.empty_strided(t.shape, t.stride(), dtype=dtype, device="cuda")
    q, s = quantize_q8(x)
    assert q.shape == x.shape and s.shape == x.shape[:-1] and not s.any()
    y = gated_norm(x, None, x)
    assert y.shape == x.shape
    q, s = gated_norm(x, quantize=True)
    assert q.shape == x.shape and s.shape == x.shape[:-1] and not s.any()
    for gate in (None, x, x.new_ones(()), x.new_ones(1)):
        y, r = residual_norm(x, x, gate=gate)
        assert y.shape == x.shape and r.shape == x.shape
        (q, s), r = residual_norm(x, x.float(), gate=gate, quantize=True)
        assert q.shape == x.shape and s.shape == x.shape[:-1] and not s.any()
    w, ws = torch.zeros(7, x.shape[-1], dtype=torch.int8, device="cuda"), torch.ones(7, device="cuda")
    assert matmul_q8(x, w, ws).shape == (*x.shape[:-1], 7)
    y = matmul_q8(torch.empty_strided(t.shape, t.stride(), dtype=torch.int8, device="cuda"), w, ws,
                  scales=torch.ones(x.shape[:-1], device="cuda"), bias=ws)
    assert torch.equal(y, torch.ones(*x.shape[:-1], 7, device="cuda"))
