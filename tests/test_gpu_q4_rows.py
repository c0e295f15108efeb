"""4-bit products of more rows of x than one launch holds."""
import pytest
import torch

import ssm_util as u

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_rows_past_a_launch(dtype):
    """65535 tiles of 64 rows, and 100 rows more."""
    from pto_einsum import matvec_q4

    M, N, K, group = 65535 * 64 + 100, 5, 33, 32
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    packed = torch.randint(0, 256, (N, (K + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand(N, 2, generator=g, device="cuda") * 0.02 + 0.01).to(dtype)
    print(f"matvec_q4 {dtype} {M} rows", flush=True)
    y = matvec_q4(x, packed, scales, group=group)
    some = torch.cat([torch.arange(0, 70), torch.arange(65535 * 64 - 70, M)]).cuda()
    ref, size = u.q4(x[some].cpu(), packed.cpu(), scales.cpu(), None, group, K)
    assert bool(((y[some].double().cpu() - ref).abs() <= u.q4_bound(ref, size, K, dtype)).all())
    # the rest: the same rows in a call of their own
    part = matvec_q4(x[1000000:1000064], packed, scales, group=group)
    assert torch.equal(y[1000000:1000064], part)
