"""Groups of rows without elements."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("groups", [1, 2, 7, 8192])
@pytest.mark.parametrize("shape", [(3, 0), (2, 5, 0), (0,), (0, 0), (70000, 0)])
def test_rows_in_8_bits(shape, groups, dtype):
    from pto_einsum import gated_norm

    x = torch.zeros(shape, dtype=dtype, device="cuda")
    for norm_first in (False, True):
        for z in (None, x):
            q, s = gated_norm(x, None, z, groups=groups, norm_first=norm_first, eps=0.0, quantize=True)
            assert q.shape == shape and s.shape == shape[:-1] and torch.equal(s, torch.zeros(shape[:-1], device="cuda"))
            assert gated_norm(x, None, z, groups=groups, norm_first=norm_first).shape == shape
