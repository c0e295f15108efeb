"""Which products of few rows take x to 8 bits in their own blocks, as the workspace
that a call needs tells, up to the most channels that an operand may have."""
import ctypes

import pytest

from pto_einsum import abi


@pytest.mark.parametrize("m", [1, 3, 16])
@pytest.mark.parametrize("n,own", [(100, True), (1 << 20, True), ((1 << 30) - 64, True), ((1 << 30) - 63, False),
                                   ((1 << 30) + 200, False), ((1 << 31) - 4096, False)])
def test_workspace(m, n, own):
    k = 16
    d = abi.Q8Desc(x_dtype=1, y_dtype=1, bias_dtype=0, M=m, N=n, K=k, x_ms=k, w_ns=k, x_numel=m * k, w_numel=n * k)
    need = abi.bind().pe_matmul_q8_workspace_bytes(ctypes.byref(d))
    assert (need == 0) == own and (own or need >= m * (k + 4))
