"""Products of few rows with more channels than the kernel for few rows has a launch for."""
import pytest
import torch

import rows_util as ru

pytestmark = pytest.mark.gpu


def test_more_than_2_to_the_30_channels():
    from pto_einsum import matmul_q8, quantize_q8

    n, k = (1 << 30) + 200, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    ws = torch.rand(n, generator=g, device="cuda")
    at = torch.tensor([0, 1, n // 2, n - 201, n - 2, n - 1], device="cuda")
    x = torch.randn(3, k, generator=g, device="cuda").half()
    q, s = quantize_q8(x)
    for m in (1, 3):
        ref, size = ru.product(q[:m].cpu(), s[:m].cpu(), w[at].cpu(), ws[at].cpu(), None)
        y = matmul_q8(x[:m], w, ws)
        ru.assert_within(y[:, at], ref, ru.product_bound(ref, size, torch.float16))
        y2 = matmul_q8(q[:m], w, ws, scales=s[:m], dtype=torch.float16)
        assert torch.equal(y, y2)
        del y, y2
    del w, ws
    torch.cuda.empty_cache()
