"""Products with 4-bit weights of infinite, NaN and very large x: what the
definition gives, output by output."""
import pytest
import torch

import ssm_util as u
from test_gpu_q4 import _case, _run

pytestmark = pytest.mark.gpu


def _definition(x, packed, scales, zeros, group):
    K = x.shape[-1]
    q = torch.stack([packed & 15, packed >> 4], -1).flatten(1)[:, :K].double()
    zero = 8.0 if zeros is None else zeros.double().repeat_interleave(group, 1)[:, :K]
    w = (q - zero) * scales.double().repeat_interleave(group, 1)[:, :K]
    return (x.double()[:, None] * w).sum(-1), w


@pytest.mark.parametrize("dtype", u.ALL, ids=u.IDS)
@pytest.mark.parametrize("zeros", [False, True], ids=["sym", "zeros"])
@pytest.mark.parametrize("M,N,K,group", [(3, 40, 96, 32), (5, 33, 1001, 64), (20, 50, 4700, 128)])
def test_infinite_x(dtype, zeros, M, N, K, group):
    """An infinity gives +-inf where its weight is not 0 and NaN where it is, two of
    opposite signs as the weights' signs have it, a NaN its row; other rows stay."""
    x, packed, scales, z = _case(dtype, M, N, K, group, zeros, seed=K + M)
    if zeros:
        z = z.round()          # some weights are 0
    x[0, 5] = float("inf")
    x[1, K - 1], x[1, 3] = float("-inf"), float("inf")
    x[2, 17] = float("nan")
    print(f"matvec_q4 {dtype} M {M} N {N} K {K} infinities", flush=True)
    y = _run(x, packed, scales, z, group).double().cpu()
    ref, w = _definition(x, packed, scales, z, group)
    assert bool((w[:, 5] == 0).any()) and bool(torch.isinf(ref[0]).any())
    assert torch.equal(torch.isnan(y[:3]), torch.isnan(ref[:3]))
    there = ~torch.isnan(ref[:3])
    assert torch.equal(y[:3][there], ref[:3][there])
    if M > 3:
        good, size = u.q4(x[3:], packed, scales, z, group, K)
        assert bool(((y[3:] - good).abs() <= u.q4_bound(good, size, K, dtype)).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("zeros", [False, True], ids=["sym", "zeros"])
@pytest.mark.parametrize("K", [32, 333])
def test_x_near_the_largest(dtype, zeros, K):
    """Sums of q x pass float32's range, the outputs do not: each product rounds
    twice, each addition once, and the result to dtype."""
    x, packed, scales, z = _case(dtype, 4, 35, K, 32, zeros, seed=K)
    top = torch.finfo(dtype).max
    x[0] = (x[0].float().sign() * top).to(dtype)
    x[1] = (x[1].float() * 2.0 ** 123).to(dtype)
    scales = (scales.float() / 64).to(dtype)
    x[2, 9] = top
    y = _run(x, packed, scales, z, 32).double().cpu()
    ref, w = _definition(x, packed, scales, z, 32)
    size = (x.double().abs()[:, None] * w.abs()).sum(-1)
    assert bool((size < 3e38).all())
    assert bool(((y[:3] - ref[:3]).abs() <= u.HALF[dtype] * ref[:3].abs() + 2.0 ** -24 * (K + 3) * size[:3]).all())


@pytest.mark.parametrize("e", [-100, -112, -124, -130, -140])
def test_small_float32_x(e):
    """x down to float32's subnormals."""
    x, packed, scales, z = _case(torch.float32, 2, 40, 300, 32, True, seed=1)
    x = (x.double() * 2.0 ** e).float()
    y = _run(x, packed, scales, z, 32).double().cpu()
    ref, size = u.q4(x, packed, scales, z, 32, 300)
    assert bool(((y - ref).abs() <= u.q4_bound(ref, size, 300, torch.float32)).all())
